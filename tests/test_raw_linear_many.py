"""More raw linears than one launch takes: refused as a whole, ahead of the first launch."""

from __future__ import annotations

import pytest
import torch

from selas_amd import _lib
from selas_amd.linear import RawLinear, raw_linear_batched

BF = torch.bfloat16


def problems(dev):
    return [RawLinear(torch.ones(4, 16, dtype=BF, device=dev), torch.ones(8, 16, dtype=BF, device=dev),
                      out=torch.full((4, 8), 7.0, dtype=BF, device=dev)) for _ in range(6)]


@pytest.mark.parametrize("i,j", [(0, 5), (5, 0), (1, 4), (4, 3)])
@pytest.mark.parametrize("what", ["x", "weight", "bias", "gate", "residual", "out"])
def test_overlaps_between_launches_are_refused(i, j, what):
    ps = problems("cpu")
    buf = torch.zeros(128, dtype=BF)
    shape = {"x": (4, 16), "weight": (8, 16), "bias": (8,), "gate": (8,), "residual": (4, 8), "out": (4, 8)}[what]
    n = torch.Size(shape).numel()
    ps[i] = ps[i]._replace(out=buf[:32].view(4, 8))
    ps[j] = ps[j]._replace(**{what: buf[128 - n:].view(shape) if n == 128 else buf[31:31 + n].view(shape)})
    with pytest.raises(ValueError, match=f"out of problem {i if what != 'out' else min(i, j)} overlaps a tensor of problem"):
        raw_linear_batched(ps)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["act", "bias", "out", "k"])
def test_a_bad_problem_of_a_later_launch_leaves_all_as_it_was(dev, bad):
    ps = problems(dev)
    error = ValueError
    if bad == "act":
        ps[5] = ps[5]._replace(act="relu")
    elif bad == "bias":
        ps[5] = ps[5]._replace(bias=torch.zeros(9, dtype=BF, device=dev))
    elif bad == "out":
        ps[5] = ps[5]._replace(out=torch.zeros(8, 4, dtype=BF, device=dev).t())
    else:  # refused by the library, not in Python: never read
        row, error = torch.empty(1, 1 << 31, dtype=BF, device=dev), _lib.Unsupported
        ps[5] = RawLinear(row, row)
    with pytest.raises(error):
        raw_linear_batched(ps)
    torch.cuda.synchronize()
    assert all(bool((p.out == 7.0).all()) for p in ps[:5])
    ps[5] = problems(dev)[5]
    assert all(bool((y == 16.0).all()) for y in raw_linear_batched(ps))
