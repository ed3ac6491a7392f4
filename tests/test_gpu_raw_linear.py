"""Linears with unquantized weights and their epilogue (raw_linear) against the formula in 64 bits.

Two kinds of checks. Whole-number inputs whose sums stay below 2^24 have one right answer, so the result has to be
equal to it. Random inputs: with S = |x| |w|^T, each of the K fp32 additions is off by at most 2^-23 of a partial
sum (products of 16-bit values are exact in fp32), so the sum by (K + 2) 2^-23 S. An activation has slope at most 1.13; its
own evaluation multiplies by 1 / (1 + 2^u) where u has 3 roundings and the exponential, the sum and the
reciprocal one each: (|u| + 4) 2^-22 of its value. The gate and the residual add a rounding each, and storing
half a step of the output's type."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from selas_amd import _lib
from selas_amd.linear import RawLinear, raw_linear, raw_linear_batched

from .conftest import seeded

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(shape, seed, lo=-3, hi=4, dtype=BF):
    return torch.randint(lo, hi, shape, generator=seeded(seed)).to(dtype)


def normal(shape, seed, std=1.0, dtype=BF):
    return (torch.randn(shape, generator=seeded(seed)) * std).to(dtype)


def reference(x, w, bias=None, act=None, gate=None, residual=None):
    """(value, bound of the error ahead of the last rounding) in 64 bits on the CPU."""
    x, w = x.detach().cpu().double(), w.detach().cpu().double()
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z = z + bias.cpu().double()
    err = (x.shape[-1] + 2) * 2.0 ** -23 * s + 2.0 ** -23 * z.abs()
    a = z
    if act is not None:
        u = z if act == "silu" else math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)
        a = z * torch.sigmoid(u)
        err = 1.13 * err + a.abs() * (u.abs() * 1.4427 + 4) * 2.0 ** -22
    if gate is not None:
        g = gate.cpu().double()
        if g.dim() == 2 and a.dim() == 3:
            g = g.unsqueeze(1)
        a = g * a
        err = g.abs() * err + 2.0 ** -23 * a.abs()
    if residual is not None:
        a = residual.cpu().double() + a
        err = err + 2.0 ** -23 * a.abs()
    return a, err


def check(y, ref_err):
    ref, err = ref_err
    fi = torch.finfo(y.dtype)
    # Half a step of the type (of the computed value, which may be err larger), or of its smallest steps.
    tol = err + (ref.abs() + err) * fi.eps / 2 + fi.smallest_normal * fi.eps
    d = (y.detach().cpu().double() - ref).abs()
    assert y.shape == ref.shape
    assert bool((d <= tol).all()), f"worst {(d / tol).max().item()} of the bound at {(d / tol).argmax().item()}"


SHAPES = [(1, 1, 1, 1), (1, 1, 64, 64), (1, 7, 33, 65), (2, 33, 70, 40), (1, 16, 200, 1032), (3, 100, 129, 72),
          (1, 257, 300, 520), (2, 130, 1431, 667), (1, 300, 64, 3), (1, 31, 1000, 256), (5, 13, 96, 2048),
          (1, 515, 520, 1160), (1, 1024, 768, 320)]


@pytest.mark.parametrize("b,l,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_whole_numbers_are_exact(dev, b, l, n, k, dtype):
    x, w = ints((b, l, k), 1, dtype=dtype), ints((n, k), 2, dtype=dtype)
    bias, gate = ints((n,), 3, dtype=dtype), ints((b, 1, n), 4, dtype=F32)
    residual = ints((b, l, n), 5, -50, 50, dtype=F32)
    z = x.double() @ w.double().t() + bias.double()
    y = raw_linear(x.to(dev), w.to(dev), bias.to(dev), out_dtype=F32)
    assert y.dtype == F32 and torch.equal(y.cpu().double(), z)
    y = raw_linear(x.to(dev), w.to(dev), bias.to(dev), gate=gate.to(dev), residual=residual.to(dev))
    assert y.dtype == F32 and torch.equal(y.cpu().double(), residual.double() + gate.double() * z)
    y = raw_linear(x.to(dev), w.to(dev))
    assert y.dtype == dtype and torch.equal(y.cpu(), (x.double() @ w.double().t()).to(dtype))


@pytest.mark.parametrize("b,l,n,k", SHAPES)
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (FP, FP)])
def test_against_the_formula(dev, b, l, n, k, act, dtype, out):
    x, w = normal((b, l, k), 11, dtype=dtype), normal((n, k), 12, 2 * k ** -0.5, dtype=dtype)
    bias, gate, residual = normal((n,), 13, dtype=dtype), normal((b, n), 14, dtype=F32), normal((b, l, n), 15, dtype=out)
    y = raw_linear(x.to(dev), w.to(dev), bias.to(dev), act=act, gate=gate.to(dev), residual=residual.to(dev))
    assert y.dtype == out
    check(y, reference(x, w, bias, act, gate, residual))
    check(raw_linear(x.to(dev), w.to(dev), bias.to(dev), act=act, out_dtype=out), reference(x, w, bias, act))


@pytest.mark.parametrize("which", ["gate", "residual", "bias", "none"])
def test_each_part_of_the_epilogue_alone(dev, which):
    x, w = normal((2, 50, 128), 21), normal((96, 128), 22, 0.1)
    kw = {"gate": normal((2, 1, 96), 23, dtype=BF), "residual": normal((2, 50, 96), 24, dtype=BF),
          "bias": normal((96,), 25, dtype=F32)}
    kw = {which: kw[which]} if which in kw else {}
    y = raw_linear(x.to(dev), w.to(dev), **{n: t.to(dev) for n, t in kw.items()})
    assert y.dtype == BF
    check(y, reference(x, w, **kw))


def tile(m, n, k):
    out = [ctypes.c_int64() for _ in range(3)]
    p = _lib.RAW_LINEAR_PROBLEM.pack(4096, 0, k, 4096, k, 0, 0, 0, 0, 0, 0, 4096, 0, n, 1, m, n, k, 0, 0, 0, 2, 0, 0)
    _lib.call("selas_raw_linear_tile", p, 1, _lib.BF16, *map(ctypes.byref, out))
    return tuple(o.value for o in out)


# Every tile and both kinds of K (whole steps of 64 or not), whole and split, with sizes that fill no tile.
@pytest.mark.parametrize("m,n,k,want", [(1030, 12280, 320, (256, 256, 1)), (700, 12279, 1352, (256, 256, 1)),
                                        (130, 6008, 8200, (256, 256, 8)), (300, 12280, 640, (256, 128, 1)),
                                        (300, 12279, 1352, (256, 128, 1)), (130, 6008, 6152, (256, 128, 4)),
                                        (300, 500, 640, (128, 128, 1)), (130, 3064, 1352, (128, 128, 1)),
                                        (70, 300, 1352, (128, 128, 6))])
def test_every_tile_on_whole_numbers(dev, m, n, k, want):
    if torch.cuda.get_device_properties(dev).multi_processor_count == 256:  # the choice goes by the CU count
        assert tile(m, n, k) == want
    x, w = ints((m, k), 1).to(dev), ints((n, k), 2).to(dev)
    bias, gate, res = ints((n,), 3, dtype=F32).to(dev), ints((n,), 4, dtype=F32).to(dev), ints((m, n), 5, dtype=F32).to(dev)
    z = x.double() @ w.double().t() + bias.double()
    assert torch.equal(raw_linear(x, w, bias, gate=gate, residual=res).double(), res.double() + gate.double() * z)
    assert torch.equal(raw_linear(x, w, bias), z.to(BF))


# Few rows against weights of one to seven blocks of 16 rows per CU of 256, the last block and round not full.
@pytest.mark.parametrize("n", [4000, 5000, 9208, 12283, 16376, 18424, 21499, 24568, 29000])
@pytest.mark.parametrize("m,k", [(1, 72), (16, 640), (28, 1352), (32, 64)])
def test_few_rows_on_whole_numbers(dev, m, n, k):
    x, w = ints((m, k), 1).to(dev), ints((n, k), 2).to(dev)
    bias, gate, res = ints((n,), 3, dtype=F32).to(dev), ints((n,), 4, dtype=F32).to(dev), ints((m, n), 5, dtype=F32).to(dev)
    z = x.double() @ w.double().t() + bias.double()
    assert torch.equal(raw_linear(x, w, bias, gate=gate, residual=res).double(), res.double() + gate.double() * z)
    assert torch.equal(raw_linear(x, w, bias), z.to(BF))


# Outputs off every alignment (odd N; a residual and a result that start at an odd element), tiles across images.
@pytest.mark.parametrize("b,l,n,k", [(3, 100, 129, 72), (4, 33, 1431, 667), (2, 350, 12279, 200), (2, 150, 12279, 1352)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gates,gate_t,res_t", [("image", "w", F32), ("image", F32, "w"), ("one", "w", "w"), ("one", F32, F32),
                                                ("none", F32, "w")])
def test_epilogues_off_alignment(dev, b, l, n, k, dtype, gates, gate_t, res_t):
    gate_t, res_t = dtype if gate_t == "w" else gate_t, dtype if res_t == "w" else res_t
    x, w, bias = ints((b, l, k), 31, dtype=dtype).to(dev), ints((n, k), 32, dtype=dtype).to(dev), ints((n,), 33, dtype=dtype).to(dev)
    gate = {"image": ints((b, 1, n), 34, dtype=gate_t).to(dev), "one": ints((n,), 34, dtype=gate_t).to(dev), "none": None}[gates]
    buf = ints((b * l * n + 2 * n,), 35, dtype=res_t).to(dev)
    res = buf[1:1 + b * l * n].view(b, l, n)
    z = x.double() @ w.double().t() + bias.double()
    want = (res.double() + (z if gate is None else gate.double() * z)).to(res_t)
    ends = buf[0].clone(), buf[1 + b * l * n:].clone()
    assert torch.equal(raw_linear(x, w, bias, gate=gate, residual=res), want)
    assert torch.equal(raw_linear(x, w, bias, gate=gate, residual=res, out=res), want)
    assert torch.equal(res, want) and torch.equal(buf[0], ends[0]) and torch.equal(buf[1 + b * l * n:], ends[1])


def test_gate_shapes(dev):
    x, w, g = normal((3, 9, 64), 31), normal((40, 64), 32), normal((3, 40), 33, dtype=F32)
    a = raw_linear(x.to(dev), w.to(dev), gate=g.to(dev))
    b = raw_linear(x.to(dev), w.to(dev), gate=g[:, None].to(dev))
    wide = normal((3, 1, 120), 34, dtype=F32).to(dev)
    wide[..., 80:] = g[:, None].to(dev)
    assert torch.equal(a, b) and torch.equal(a, raw_linear(x.to(dev), w.to(dev), gate=wide[..., 80:]))
    for shape in ((40,), (1, 40), (1, 1, 40)):
        one = raw_linear(x.to(dev), w.to(dev), gate=g[0].view(shape).to(dev))
        check(one, reference(x, w, gate=g[0]))


@pytest.mark.parametrize("m", [1, 5, 20, 40, 300])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_views_with_strides_of_their_own(dev, m, offset):
    # x: columns of a wider buffer behind rows of another stream; weight: rows and columns of a wider one; out: columns.
    n, k = 136, 192
    wide = ints((2, m + 6, k + 24), 41).to(dev)
    x = wide[:, 6:, offset:offset + k]
    w = ints((n + 8, k + 16), 42).to(dev)[8:, offset:offset + k]
    res = ints((2, m + 2, n + 12), 43, -9, 9, F32).to(dev)[:, 2:, 4 + offset:4 + offset + n]
    buf = torch.full((2, m + 1, n + 32), 7.0, device=dev)
    out = buf[:, 1:, 16 + offset:16 + offset + n]
    y = raw_linear(x, w, residual=res, out=out)
    assert y is out
    assert torch.equal(out.cpu().double(), res.cpu().double() + x.cpu().double() @ w.cpu().double().t())
    buf[:, 1:, 16 + offset:16 + offset + n] = 7.0
    assert bool((buf == 7.0).all()), "the launch wrote outside out"


@pytest.mark.parametrize("b,l,n,k", [(2, 21, 64, 64), (1, 300, 520, 256), (1, 3, 2048, 512), (2, 640, 512, 4096)])
def test_residual_in_place_and_inputs_untouched(dev, b, l, n, k):
    x, w, r = ints((b, l, k), 51).to(dev), ints((n, k), 52).to(dev), ints((b, l, n), 53, dtype=F32).to(dev)
    x0, w0, ref = x.clone(), w.clone(), r.cpu().double() + x.cpu().double() @ w.cpu().double().t()
    assert raw_linear(x, w, residual=r, out=r) is r
    assert torch.equal(r.cpu().double(), ref) and torch.equal(x, x0) and torch.equal(w, w0)


def test_rows_that_are_not_finite_stay_alone(dev):
    for m, n, k in ((9, 64, 64), (200, 136, 128)):
        x, w = ints((m, k), 61).to(dev), ints((n, k), 62).to(dev)
        ref = raw_linear(x, w, out_dtype=F32)
        x[3, 5], x[7, k - 1] = float("nan"), float("inf")
        w[11, 0] = float("inf")
        y = raw_linear(x, w, out_dtype=F32)
        rows = [i for i in range(m) if i not in (3, 7)]
        cols = [j for j in range(n) if j != 11]
        assert bool(y[3].isnan().all()) and torch.equal(y[rows][:, cols], ref[rows][:, cols])
        want = x[7].double().cpu() @ w.double().cpu().t()
        assert torch.equal(y[7].isnan().cpu(), want.isnan()) and torch.equal(y[7].isinf().cpu(), want.isinf())


def test_large_magnitudes_of_the_activations(dev):
    # +-large pre-activations: gelu and silu go to x or to zero without NaN.
    w = torch.eye(64, dtype=BF)
    x = torch.tensor([-1e30, -3e4, -100.0, -20.0, -0.0, 0.0, 1e-30, 20.0, 100.0, 3e4, 1e30]).to(BF)
    x = x[:, None].expand(-1, 64).contiguous()
    for act in ("gelu", "silu"):
        y = raw_linear(x.to(dev), w.to(dev), act=act, out_dtype=F32).cpu().double()
        z = x.double()
        u = z if act == "silu" else math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)
        ref = z * torch.sigmoid(u)
        # Values below fp32's normal range may come out as zero (hardware exponential).
        assert bool(((y - ref).abs() <= ref.abs() * 2.0 ** -15 + 1e-36).all()), (act, y[:, 0], ref[:, 0])


def test_overflow_of_fp16_is_infinite(dev):
    x, w = torch.full((3, 64), 100.0, dtype=FP), torch.full((8, 64), 100.0, dtype=FP)
    assert bool(raw_linear(x.to(dev), w.to(dev)).isinf().all())
    assert bool((raw_linear(x.to(dev), w.to(dev), out_dtype=F32) == 640000.0).all())


def test_empty_sizes(dev):
    w, b = ints((24, 16), 71).to(dev), ints((24,), 72).to(dev)
    assert raw_linear(torch.zeros(0, 16, dtype=BF, device=dev), w, b).shape == (0, 24)
    assert raw_linear(torch.zeros(2, 0, 16, dtype=BF, device=dev), w, b).shape == (2, 0, 24)
    assert raw_linear(torch.zeros(5, 16, dtype=BF, device=dev), w[:0]).shape == (5, 0)
    y = raw_linear(torch.zeros(5, 0, dtype=BF, device=dev), w[:, :0], b)
    assert torch.equal(y, b.expand(5, -1))
    assert raw_linear(torch.ones(16, dtype=BF, device=dev), w, b).shape == (24,)
    assert raw_linear_batched([]) == []


@pytest.mark.parametrize("lead", [(2, 3, 0), (2, 0, 4), (0, 3, 4), (2, 0, 0, 5)])
def test_empty_higher_dims(dev, lead):
    x, w = torch.zeros(*lead, 16, dtype=BF, device=dev), ints((24, 16), 73).to(dev)
    r = torch.zeros(*lead, 24, dtype=BF, device=dev)
    assert raw_linear(x, w, residual=r).shape == (*lead, 24)
    assert raw_linear(x, w, residual=r, out=r).shape == (*lead, 24)


def test_higher_dims(dev):
    x, w = ints((2, 3, 4, 64), 81).to(dev), ints((40, 64), 82).to(dev)
    ref = (x.cpu().double() @ w.cpu().double().t()).to(BF)
    assert torch.equal(raw_linear(x, w).cpu(), ref)
    out = torch.empty(2, 3, 4, 40, dtype=BF, device=dev)
    assert raw_linear(x, w, out=out) is out and torch.equal(out.cpu(), ref)
    assert torch.equal(raw_linear(x[0, 0, 0], w).cpu(), ref[0, 0, 0])


def test_batched_equals_single(dev):
    probs = []
    for i, (b, l, n, k) in enumerate([(1, 512, 264, 192), (1, 77, 264, 192), (2, 3, 96, 72), (1, 130, 41, 33),
                                      (1, 40, 512, 64), (1, 1, 9, 9)]):
        probs.append(RawLinear(normal((b, l, k), i).to(dev), normal((n, k), 50 + i, 0.1).to(dev),
                               act=(None, "gelu", "silu")[i % 3], residual=normal((b, l, n), 99 + i, dtype=F32).to(dev)))
    outs = raw_linear_batched(probs)
    for p, y in zip(probs, outs):
        check(y, reference(p.x, p.weight, p.bias, p.act, p.gate, p.residual))
        again = raw_linear(*p[:3], act=p.act, residual=p.residual)
        check(again, reference(p.x, p.weight, p.bias, p.act, p.gate, p.residual))


def test_equal_calls_give_equal_bits(dev):
    for m, n, k in ((1, 3072, 768), (28, 1000, 3072), (512, 640, 4096), (1030, 264, 200)):
        x, w = normal((m, k), 91).to(dev), normal((n, k), 92, 0.05).to(dev)
        first = raw_linear(x, w, act="gelu", out_dtype=F32)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = [raw_linear(x, w, act="gelu", out_dtype=F32) for _ in range(3)]
        s.synchronize()
        assert all(torch.equal(first, o) for o in other)


def test_two_streams_at_once(dev):
    xs = [normal((m, 1024), m).to(dev) for m in (300, 40)]
    ws = [normal((640, 1024), 7 + i, 0.05).to(dev) for i in range(2)]
    ref = [raw_linear(x, w, out_dtype=F32) for x, w in zip(xs, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(raw_linear(xs[i], ws[i], out_dtype=F32))
    torch.cuda.synchronize()
    assert all(torch.equal(ref[i], y) for i in range(2) for y in got[i])


@pytest.mark.parametrize("m,n,k", [(1, 512, 768), (512, 640, 4096), (300, 264, 200)])
def test_captured_and_replayed(dev, m, n, k):
    x, w, r = normal((m, k), 1).to(dev), normal((n, k), 2, 0.05).to(dev), normal((m, n), 3, dtype=F32).to(dev)
    eager = raw_linear(x, w, act="silu", residual=r)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = raw_linear(x, w, act="silu", residual=r)
    for i in range(4):
        x.copy_(normal((m, k), 10 + i).to(dev))
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        eager = raw_linear(x, w, act="silu", residual=r)
        assert torch.equal(y, eager), i


def test_refusals(dev):
    x, w = torch.zeros(4, 16, dtype=BF, device=dev), torch.zeros(8, 16, dtype=BF, device=dev)
    with pytest.raises(_lib.Unsupported, match="bf16 or fp16"):
        raw_linear(x.float(), w.float())
    for kw, match in (({"act": "relu"}, "act"), ({"bias": torch.zeros(7, dtype=BF, device=dev)}, "bias"),
                      ({"residual": torch.zeros(4, 9, dtype=BF, device=dev)}, "residual"),
                      ({"gate": torch.zeros(2, 8, dtype=BF, device=dev)}, "gate"),
                      ({"gate": torch.zeros(8, dtype=FP, device=dev)}, "gate"),
                      ({"out_dtype": FP}, "out"), ({"out": torch.zeros(4, 9, dtype=BF, device=dev)}, "out"),
                      ({"out": torch.zeros(1, 8, dtype=BF, device=dev).expand(4, 8)}, "own address"),
                      ({"out": torch.zeros(8, 4, dtype=BF, device=dev).t()}, "unit column")):
        with pytest.raises(ValueError, match=match):
            raw_linear(x, w, **kw)
    with pytest.raises(ValueError, match="weight"):
        raw_linear(x, w[:, :8])
    with pytest.raises(ValueError, match="must be"):
        raw_linear(x, w.to(FP))
    sq = torch.zeros(16, 16, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        raw_linear(sq, sq, out=sq)
    big = torch.zeros(5, 8, dtype=BF, device=dev)
    with pytest.raises(ValueError, match="overlaps"):
        raw_linear(x, w, residual=big[:4], out=big[1:])
    with pytest.raises(ValueError, match="problem"):
        raw_linear_batched([RawLinear(x, w, out=big[:4]), RawLinear(x, w, out=big[1:])])
    with pytest.raises(ValueError, match="GPU"):
        raw_linear(x.cpu(), w)
