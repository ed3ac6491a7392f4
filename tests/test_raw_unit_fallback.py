"""Units with fused_raw set that raw_linear does not take run as units without it, bit for bit."""

from __future__ import annotations

import pytest
import torch

from oracle import segments as S
from selas_amd import flux as F
from selas_amd.codecs import encode_nf4, encode_raw
from selas_amd.kernels import FUSED
from selas_amd.linear import UnitView

from .conftest import seeded

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
CFG = F.FluxConfig(hidden=256, heads=2, mlp_hidden=512, depth_double=1, depth_single=1, in_channels=64, context_dim=128,
                   vec_dim=64, axes_dim=(16, 56, 56))


def test_what_raw_linear_takes():
    w, b = torch.randn(64, 64), torch.randn(64)
    raw = {"a.weight": encode_raw("a.weight", w, BF), "a.bias": encode_raw("a.bias", b, F32)}
    for dt, want in ((BF, True), (FP, True), (F32, False)):
        assert UnitView(raw, dt).takes_raw_linear() is want
    coded = encode_raw("b.weight", w, BF)._replace(codec="nf4")
    assert not UnitView({**raw, "b.weight": coded}, BF).takes_raw_linear()


class Segments:
    """The segments of a runner of another package."""

    def __getattr__(self, name):
        return getattr(FUSED, name)


def blocks(m, dt, fused, k=FUSED):
    for u in (m.globals, *m.doubles, *m.singles, *m.mods):
        u.fused_raw = fused
    g = seeded(2)
    img, txt = torch.randn(1, 12, 256, generator=g).cuda(), torch.randn(1, 7, 256, generator=g).cuda()
    cos, sin = (t.cuda() for t in S.rope_tables(torch.cat((torch.zeros(7, 3), F.image_ids(3, 4))), CFG.axes_dim, CFG.theta))
    dmod, smod = torch.randn(1, 12 * 256, generator=g).to(dt).cuda(), torch.randn(1, 3 * 256, generator=g).to(dt).cuda()
    a, b = F.double_block(m.doubles[0], img, txt, dmod, cos, sin, CFG, dt, dt == FP, k)
    c = F.single_block(m.singles[0], torch.cat((b, a), 1), smod, cos, sin, CFG, dt, dt == FP, k)
    return [a, b, c, F.final_layer(m.globals, a, smod[:, :512], dt, k), F.mlp_embed(m.globals, "vector_in", img[:, 0, :64].to(dt), k)]


def steps(m, fused, k=FUSED):
    for u in (m.globals, *m.doubles, *m.singles, *m.mods):
        u.fused_raw = fused
    runner, g = F.FluxRunner(m, k), seeded(3)
    pooled, txt, lat = torch.randn(1, 64, generator=g), torch.randn(1, 7, 128, generator=g), torch.randn(1, 12, 64, generator=g)
    cond = runner.prepare([1.0, 0.5], 3.5, pooled, txt, F.image_ids(3, 4), F.text_ids(7))
    return [runner.step(0, lat.cuda(), cond)[0], cond.txt, cond.final_mod, *cond.mods.values()]


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_fp32_units(dev):
    m = F.RandomFlux(CFG, dev, F32, seed=5, quant="raw")
    assert equal(blocks(m, F32, True), blocks(m, F32, False)) and equal(steps(m, True), steps(m, False))


@pytest.mark.gpu
@pytest.mark.parametrize("names", [("img_mlp.0", "linear1"), ("txt_attn.proj", "linear2")])
def test_units_with_a_quantized_matrix(dev, names):
    m = F.RandomFlux(CFG, dev, BF, seed=6, quant="raw")
    for u, name in ((m.doubles[0], names[0]), (m.singles[0], names[1]), (m.mods[0], "img_mod.lin"), (m.globals, "vector_in.in_layer")):
        w = u.get(name + ".weight")
        u._views.clear()
        u.tensors[name + ".weight"] = encode_nf4(name + ".weight", w)
    assert equal(blocks(m, BF, True), blocks(m, BF, False)) and equal(steps(m, True), steps(m, False))


@pytest.mark.gpu
def test_a_runner_with_other_segments(dev):
    m = F.RandomFlux(CFG, dev, BF, seed=7, quant="raw")
    assert equal(blocks(m, BF, True, Segments()), blocks(m, BF, False, Segments()))
    assert equal(steps(m, True, Segments()), steps(m, False, Segments()))
