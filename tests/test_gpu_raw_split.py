"""Raw linears whose K is split over workgroups, on whole numbers: few rows of x or of w, and several problems in one tiled
launch, some with fewer steps of K than there are ranges and some with operands that are copied first. The sums stay
below 2^24, so every order of additions gives the one right answer."""

from __future__ import annotations

import ctypes

import pytest
import torch

from selas_amd import _lib
from selas_amd.linear import RawLinear, raw_linear, raw_linear_batched

from .conftest import seeded
from .test_operator_checks import problem, query

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(shape, seed, lo=-3, hi=4, dtype=BF):
    return torch.randint(lo, hi, shape, generator=seeded(seed)).to(dtype)


def shape_of(m, n, k, off=0, b=1):
    # Rows of k elements from an element `off` past 16 bytes on: no vector of 8 with off 1 or an odd k.
    return problem(x=4096 + 2 * off, B=b, L=m // b, N=n, K=k, x_sb=m // b * k, x_sl=k, ldw=k, y_sb=m // b * n, y_sl=n)


# (rows, columns, K, images): x few, then w few; those with an odd K or offset run raw_few_kernel, the others raw_stream_kernel.
FEW = [(1, 96, 12288, 1), (28, 1000, 3072, 2), (17, 41, 2048, 1), (32, 300, 4096, 4), (28, 999, 3001, 1), (1, 97, 12289, 1),
       (9, 99, 3001, 3), (1024, 64, 3072, 4), (300, 33, 4096, 3), (300, 17, 4096, 1), (2000, 16, 2048, 2), (40, 1, 8192, 2),
       (300, 33, 4099, 3), (70, 64, 12289, 2), (41, 49, 3079, 1)]


@pytest.mark.parametrize("m,n,k,b", FEW)
@pytest.mark.parametrize("off", [0, 1])
def test_these_few_rows_are_split(m, n, k, b, off):
    need = query(shape_of(m, n, k, off, b))
    ranges = need // (4 * m * n)
    assert ranges > 1 and need == -(-4 * ranges * m * n // 16) * 16  # partial sums and nothing else


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,b", FEW)
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype,out", [(BF, F32), (FP, FP)])
def test_few_rows(dev, m, n, k, b, off, dtype, out):
    buf = ints((m * k + 8,), 1, dtype=dtype).to(dev)
    x, w = buf[off:off + m * k].view(b, m // b, k), ints((n, k), 2, dtype=dtype).to(dev)
    bias, gate = ints((n,), 3, dtype=dtype).to(dev), ints((b, 1, n), 4, dtype=F32).to(dev)
    res = ints((b, m // b, n), 5, -50, 50, dtype=out).to(dev)
    z = x.double() @ w.double().t() + bias.double()
    want = (res.double() + gate.double() * z).to(out)
    assert torch.equal(raw_linear(x, w, bias, gate=gate, residual=res), want)
    assert torch.equal(raw_linear(x, w, bias, out_dtype=F32).double(), z)
    wide = torch.full((b, m // b, n + 3), 7.0, dtype=out, device=dev)
    raw_linear(x, w, bias, gate=gate, residual=res, out=wide[..., 1:n + 1])
    assert torch.equal(wide[..., 1:n + 1], want) and bool((wide[..., n + 1:] == 7.0).all()) and bool((wide[..., 0] == 7.0).all())
    assert raw_linear(x, w, bias, gate=gate, residual=res, out=res) is res and torch.equal(res, want)


def ranges_of(shapes):
    out = [ctypes.c_int64() for _ in range(3)]
    ps = [problem(L=m, N=n, K=k, x_sl=k, ldw=k, y_sl=n) for m, n, k in shapes]
    _lib.call("selas_raw_linear_tile", b"".join(ps), len(ps), _lib.BF16, *map(ctypes.byref, out))
    return out[2].value


# Long beside short K (most ranges of the short one are empty), copied operands beside others, few rows among them.
BATCHES = [[(130, 600, 8200), (70, 300, 64), (100, 129, 67), (40, 96, 4096)],
           [(130, 600, 8200), (70, 300, 64), (200, 129, 72), (40, 97, 4099)],
           [(512, 640, 4096), (28, 1000, 3072), (60, 70, 1)],
           [(65, 300, 12288), (65, 300, 0), (33, 65, 129)]]


@pytest.mark.parametrize("shapes", BATCHES)
def test_these_batches_are_split(shapes):
    assert ranges_of(shapes) > 1


@pytest.mark.parametrize("shapes", BATCHES)
def test_their_workspace(shapes):
    # Partial sums of every problem, of a tiled one in the launch's ranges, and copies (rows of K rounded up to 64) of the
    # operands whose rows are not whole vectors of 8.
    want = 0
    for m, n, k in shapes:
        few = m <= 32 or n <= 64
        parts = query(shape_of(m, n, k)) // (4 * m * n) if few else ranges_of(shapes)
        want += -(-4 * parts * m * n // 16) * 16 if parts > 1 else 0
        want += 0 if few or k % 8 == 0 else (m + n) * -(-k // 64) * 128
    assert query(*[shape_of(*s) for s in shapes]) == want


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", BATCHES)
@pytest.mark.parametrize("dtype,out", [(BF, F32), (FP, FP)])
def test_batches(dev, shapes, dtype, out):
    ps, want = [], []
    for i, (m, n, k) in enumerate(shapes):
        x, w = ints((m, k), 10 + i, dtype=dtype).to(dev), ints((n, k), 20 + i, dtype=dtype).to(dev)
        bias, gate = ints((n,), 30 + i, dtype=dtype).to(dev), ints((n,), 40 + i, dtype=F32).to(dev)
        res = ints((m, n), 50 + i, dtype=out).to(dev)
        ps.append(RawLinear(x, w, bias, gate=gate, residual=res))
        want.append((res.double() + gate.double() * (x.double() @ w.double().t() + bias.double())).to(out))
    for p, y, r in zip(ps, raw_linear_batched(ps), want):
        assert torch.equal(y, r) and torch.equal(raw_linear(p.x, p.weight, p.bias, gate=p.gate, residual=p.residual), r)
    ps = [p._replace(out=p.residual) for p in ps]
    assert all(torch.equal(y, r) for y, r in zip(raw_linear_batched(ps), want))
