"""The fp16 guard of raw linears: act(..) clamped to +-65504 ahead of the gate and the residual.

Whole numbers have one right answer below 2^24, infinite sums too; NaN (0 times an infinite input) passes through. The
blocks are compared with the oracle's guarded ones at the tolerance of the raw blocks: relative L2 <= 4e-3 of the
update, over the rows that overflow and over the others."""

from __future__ import annotations

import pytest
import torch

from oracle import flux as OF
from oracle import segments as S
from selas_amd import flux as F
from selas_amd.linear import RawLinear, raw_linear, raw_linear_batched

from .conftest import seeded

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
MAX = 65504.0


def ints(shape, seed, lo=-3, hi=4, dtype=FP):
    return torch.randint(lo, hi, shape, generator=seeded(seed)).to(dtype)


def same(y, want):
    want = want.to(y.dtype)
    return torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(7.0, 9e4, -9e4), want.nan_to_num(7.0, 9e4, -9e4))


# Every route: few rows of x and of w, with aligned rows and others, whole and split; the three tiles, whole and split, with
# outputs on alignment and off.
@pytest.mark.parametrize("b,l,n,k", [(1, 28, 1000, 640), (1, 28, 1000, 4096), (1, 9, 130, 67), (2, 9, 99, 3001), (2, 150, 64, 128),
                                     (1, 300, 64, 4096), (1, 300, 33, 65), (1, 300, 520, 640), (2, 65, 129, 72),
                                     (1, 70, 300, 1352), (2, 35, 299, 4099), (1, 1030, 12280, 72), (1, 300, 12279, 640)])
@pytest.mark.parametrize("res_t", [F32, FP])
def test_every_route_clamps(dev, b, l, n, k, res_t):
    x, w = ints((b, l, k), 1).to(dev), ints((n, k), 2).to(dev)
    x[0, 1], x[b - 1, l - 1, 0], x[0, 2, k - 1] = 300.0, float("inf"), float("-inf")
    bias, gate, res = ints((n,), 3).to(dev), ints((b, 1, n), 4, dtype=F32).to(dev), ints((b, l, n), 5, dtype=res_t).to(dev)
    z = x.double() @ w.double().t() + bias.double()
    assert bool(z.isinf().any()) and bool(z.isnan().any())
    c = z.clamp(-MAX, MAX)
    assert same(raw_linear(x, w, bias, gate=gate, residual=res, guard=True), res.double() + gate.double() * c)
    assert same(raw_linear(x, w, bias, guard=True, out_dtype=F32), c)
    assert same(raw_linear(x, w, bias, out_dtype=F32), z)  # off unless asked for


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,n", [(4, 64), (200, 136), (200, 137)])
def test_after_the_activation(dev, act, m, n):
    x = torch.full((m, 128), 1000.0, dtype=BF, device=dev)
    x[1::2] = -1000.0
    y = raw_linear(x, torch.ones(n, 128, dtype=BF, device=dev), act=act, guard=True, out_dtype=F32)
    assert bool((y[0::2] == MAX).all()) and bool((y[1::2] == 0).all())


def test_each_problem_of_a_launch_has_its_own(dev):
    x, w = torch.full((200, 64), 100.0, dtype=FP, device=dev), torch.full((136, 64), 100.0, dtype=FP, device=dev)
    a, b = raw_linear_batched([RawLinear(x, w, out_dtype=F32, guard=True), RawLinear(x, w, out_dtype=F32)])
    assert bool((a == MAX).all()) and bool((b == 640000.0).all())


KW = dict(hidden=256, heads=2, mlp_hidden=1024, depth_double=1, depth_single=1, in_channels=64, context_dim=128,
          vec_dim=64, axes_dim=(16, 56, 56))
CFG, OCFG = F.FluxConfig(**KW), OF.FluxConfig(**KW)


def overflow(unit, prefix, row):
    """One output of a linear above fp16's range for the tokens where its sum is positive, far from the border."""
    unit.get(prefix + ".weight")[row] *= 4000.0
    unit.get(prefix + ".bias")[row] = MAX


def oracle_unit(view):
    enc = {n: (e.codec, e.shape, e.meta, {k: v.cpu() for k, v in e.parts.items()}) for n, e in view.tensors.items()}
    return OF.OracleUnit.from_encoded(enc, FP, FP)


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def close(got, ref, before):
    # Rows with +-65504 times a gate in them; the others reach 64000 times a weight of 0.08 and a gate.
    far = (ref - before).abs().amax(-1) > 15000.0
    assert bool(far.any()) and not bool(far.all()) and bool(ref.isfinite().all())
    got = got.cpu()
    assert bool(got.isfinite().all())
    for rows in (far, ~far):
        assert rel((got - before)[rows], (ref - before)[rows]) < 4e-3


def test_blocks_whose_hidden_values_overflow_stay_finite(dev):
    m = F.RandomFlux(CFG, "cuda", FP, seed=4, quant="raw", with_mods=False)
    d, s = m.doubles[0], m.singles[0]
    for unit, prefix, row in ((d, "img_mlp.0", 5), (d, "txt_mlp.0", 700), (s, "linear1", 3 * CFG.hidden + 9)):
        overflow(unit, prefix, row)
    g = seeded(8)
    img, txt = torch.randn(2, 35, CFG.hidden, generator=g), torch.randn(2, 20, CFG.hidden, generator=g)
    x = torch.cat((txt, img), dim=1)
    ids = torch.cat((torch.zeros(20, 3), F.image_ids(5, 7)))
    cos, sin = S.rope_tables(ids, CFG.axes_dim, CFG.theta)
    dmod = (torch.randn(2, 12 * CFG.hidden, generator=g) * 0.3).to(FP)
    smod = (torch.randn(2, 3 * CFG.hidden, generator=g) * 0.3).to(FP)
    ri, rt = OF.double_block(oracle_unit(d), img, txt, dmod, cos, sin, OCFG, FP, True)
    rx = OF.single_block(oracle_unit(s), x, smod, cos, sin, OCFG, FP, True)
    args = (cos.cuda(), sin.cuda(), CFG, FP)
    gi, gt = F.double_block(d, img.cuda(), txt.cuda(), dmod.cuda(), *args, True)
    gx = F.single_block(s, x.cuda(), smod.cuda(), *args, True)
    close(gi, ri, img), close(gt, rt, txt), close(gx, rx, x)
    gi, gt = F.double_block(d, img.cuda(), txt.cuda(), dmod.cuda(), *args, False)
    gx = F.single_block(s, x.cuda(), smod.cuda(), *args, False)
    assert not any(bool(t.isfinite().all()) for t in (gi, gt, gx))
