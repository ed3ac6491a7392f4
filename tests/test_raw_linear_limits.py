"""The longest K of a raw linear: a tile's rows are addressed by 31 bits of bytes."""

from __future__ import annotations

import pytest
import torch

from selas_amd import _lib
from selas_amd.linear import raw_linear

from .test_operator_checks import problem, query


def rows(m, n, k, **kw):
    return problem(L=m, N=n, K=k, x_sl=k, ldw=k, y_sl=n, **kw)


@pytest.mark.parametrize("m,n,k", [(256, 256, 4194241), (40, 256, 1 << 23), (300, 70, (1 << 22) + 1), (33, 65, 16519041),
                                   (4608, 3000, (1 << 30) - 1)])
def test_a_longer_k_is_refused(m, n, k):
    for p in (rows(m, n, k), rows(m, n, 64) + rows(m, n, k)):
        with pytest.raises(_lib.Unsupported, match="2\\^31 bytes"):
            query(*[p[i:i + _lib.RAW_LINEAR_PROBLEM.size] for i in range(0, len(p), _lib.RAW_LINEAR_PROBLEM.size)])
        with pytest.raises(_lib.Unsupported, match="2\\^31 bytes"):
            _lib.call("selas_raw_linear", p, len(p) // _lib.RAW_LINEAR_PROBLEM.size, _lib.BF16, None, 0, None)


@pytest.mark.parametrize("m,n,k", [(256, 256, 4194240), (40, 100, 1 << 23), (33, 65, 16519040), (32, 300, 1 << 26),
                                   (300, 64, 1 << 26), (0, 300, 1 << 26)])
def test_others_are_not(m, n, k):
    assert query(rows(m, n, k)) >= 0


@pytest.mark.gpu
def test_the_longest_k_of_65_columns(dev):
    # Both operands copied (an odd K), rows of 33 MB, the tile's last one 2.11 GB behind its first. Few columns hold
    # anything: the sums are whole numbers.
    m, n, k = 33, 65, 16500003
    x, w = (torch.zeros(r, k, dtype=torch.bfloat16, device=dev) for r in (m, n))
    at = torch.tensor([0, 1, 63, 64, 8250001, 16499967, 16499968, k - 2, k - 1], device=dev)
    xs = (torch.arange(m * len(at), device=dev).view(m, -1) * 7 % 11 - 5).to(torch.bfloat16)
    ws = (torch.arange(n * len(at), device=dev).view(n, -1) * 5 % 13 - 6).to(torch.bfloat16)
    x[:, at], w[:, at] = xs, ws
    y = raw_linear(x, w, out_dtype=torch.float32)
    assert torch.equal(y.cpu().double(), xs.cpu().double() @ ws.cpu().double().t())
