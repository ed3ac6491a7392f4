"""FLUX blocks and steps with raw (unquantized) weights on raw_linear, and images at positions of their own on rope_qk,
against the oracle on the CPU.

Tolerance: the residual update (out - in) and the velocity at relative L2 <= 4e-3, as for the quantized blocks. The
oracle rounds the outputs of mlp.0 (linear1) and of the linears ahead of a residual to 16 bits, which these blocks do
not: two more roundings, each 2^-8 / sqrt(12) = 1.1e-3 of the branch in the L2 norm at bf16, beside the ones both have."""

from __future__ import annotations

import pytest
import torch

from oracle import flux as OF
from oracle import segments as S
from selas_amd import flux as F

from .conftest import seeded

pytestmark = pytest.mark.gpu

KW = dict(hidden=256, heads=2, mlp_hidden=1024, depth_double=2, depth_single=2, in_channels=64, context_dim=128,
          vec_dim=64, axes_dim=(16, 56, 56))
CFG, OCFG = F.FluxConfig(**KW), OF.FluxConfig(**KW)
BF, FP = torch.bfloat16, torch.float16
L2 = 4e-3


def oracle_unit(view, dt=BF):
    enc = {n: (e.codec, e.shape, e.meta, {k: v.cpu() for k, v in e.parts.items()}) for n, e in view.tensors.items()}
    return OF.OracleUnit.from_encoded(enc, dt, dt)


def rel(a, b):
    return ((a.double().cpu() - b.double()).norm() / b.double().norm()).item()


@pytest.fixture(scope="module")
def models():
    return {dt: F.RandomFlux(CFG, "cuda", dt, seed=3, quant="raw") for dt in (BF, FP)}


def inputs(b, lt, h, w):
    g = seeded(21)
    img, txt = torch.randn(b, h * w, CFG.hidden, generator=g), torch.randn(b, lt, CFG.hidden, generator=g)
    return img, txt, torch.cat((torch.zeros(lt, 3), F.image_ids(h, w)), dim=0)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("b,lt,h,w", [(2, 64, 8, 8), (1, 60, 7, 7), (3, 5, 2, 3)])
def test_blocks(models, dt, b, lt, h, w):
    m = models[dt]
    assert m.doubles[0].codec("img_mlp.0.weight") == "raw" and m.doubles[0].fused_raw
    img, txt, ids = inputs(b, lt, h, w)
    cos, sin = S.rope_tables(ids, CFG.axes_dim, CFG.theta)
    dmod = (torch.randn(b, 12 * CFG.hidden, generator=seeded(22)) * 0.3).to(dt)
    smod = (torch.randn(b, 3 * CFG.hidden, generator=seeded(23)) * 0.3).to(dt)
    x = torch.cat((txt, img), dim=1)
    cu = lambda t: t.cuda()  # noqa: E731
    ri, rt = OF.double_block(oracle_unit(m.doubles[0], dt), img, txt, dmod, cos, sin, OCFG, dt, dt == FP)
    rx = OF.single_block(oracle_unit(m.singles[0], dt), x, smod, cos, sin, OCFG, dt, dt == FP)
    every = ids.expand(b, -1, -1)
    for args in ((cu(cos), cu(sin)), (None, None)):
        kw = {} if args[0] is not None else {"ids": cu(every)}
        gi, gt = F.double_block(m.doubles[0], cu(img), cu(txt), cu(dmod), *args, CFG, dt, dt == FP, **kw)
        assert rel(gi - img.cuda(), ri - img) < L2 and rel(gt - txt.cuda(), rt - txt) < L2
        gx = F.single_block(m.singles[0], cu(x), cu(smod), *args, CFG, dt, dt == FP, **kw)
        assert rel(gx - x.cuda(), rx - x) < L2


def test_next_blocks_input_equals_its_own_mod_in(models):
    m = models[BF]
    img, txt, ids = inputs(2, 16, 4, 8)
    cos, sin = (t.cuda() for t in S.rope_tables(ids, CFG.axes_dim, CFG.theta))
    img, txt, x = img.cuda(), txt.cuda(), torch.cat((txt, img), dim=1).cuda()
    dmod, dnext = (torch.randn(2, 12 * CFG.hidden, generator=seeded(s)).cuda() * 0.3 for s in (1, 2))
    smod, snext = (torch.randn(2, 3 * CFG.hidden, generator=seeded(s)).cuda() * 0.3 for s in (3, 4))
    i1, t1 = F.double_block(m.doubles[1], img, txt, dmod, cos, sin, CFG, BF, False)
    i2, t2, (hi, ht) = F.double_block(m.doubles[1], img, txt, dmod, cos, sin, CFG, BF, False, next_mod=dnext)
    n = dnext.unsqueeze(1).chunk(12, dim=-1)
    assert torch.equal(i1, i2) and torch.equal(t1, t2)
    assert torch.equal(hi, F.FUSED.mod_in(i1, n[0], n[1], BF)) and torch.equal(ht, F.FUSED.mod_in(t1, n[6], n[7], BF))
    x1 = F.single_block(m.singles[1], x, smod, cos, sin, CFG, BF, False)
    x2, h = F.single_block(m.singles[1], x, smod, cos, sin, CFG, BF, False, next_mod=snext)
    n = snext.unsqueeze(1).chunk(3, dim=-1)
    assert torch.equal(x1, x2) and torch.equal(h, F.FUSED.mod_in(x1, n[0], n[1], BF))


def test_a_run_with_positions_of_each_image(models):
    # Prologue, two steps and their Euler updates, two images of one token count and other shapes and offsets, against
    # the oracle run on each image alone.
    m = models[BF]
    runner = F.FluxRunner(m)
    g = seeded(5)
    sigmas = F.get_schedule(2, 24)
    pooled, txt = torch.randn(2, CFG.vec_dim, generator=g), torch.randn(2, 10, CFG.context_dim, generator=g)
    lat = torch.randn(2, 24, 64, generator=g)
    own = torch.stack((F.image_ids(4, 6), F.image_ids(6, 4) + torch.tensor([0.0, 3.0, 5.0])))
    cond = runner.prepare(sigmas, 3.5, pooled, txt, own, F.text_ids(10))
    assert cond.cos is None and cond.ids.shape == (2, 34, 3)
    out = runner.denoise(lat.cuda(), cond)
    gu, du, su = oracle_unit(m.globals), [oracle_unit(u) for u in m.doubles], [oracle_unit(u) for u in m.singles]
    mu = [oracle_unit(u) for u in m.mods]
    for i in range(2):
        sv = OF.svec(gu, OCFG, sigmas, 3.5, pooled[i:i + 1], BF)
        mods = OF.modulations(mu, [sv], 2)[0]
        c = OF.prepare(gu, OCFG, sigmas, 3.5, pooled[i:i + 1], txt[i:i + 1], own[i], F.text_ids(10), mods, BF)
        x = lat[i:i + 1]
        for s in range(2):
            x = OF.euler(x, sigmas, s, OF.step(gu, du, su, OCFG, s, x, c, BF))
        # The velocity of two steps through svec (three more 16-bit linears) and four blocks.
        assert rel(out[i:i + 1].cpu() - lat[i:i + 1], x - lat[i:i + 1]) < 2 * L2
    # Chunks of one image give every image the bits of the whole batch's tiles or its own sums' order: close, not equal.
    chunked = F.FluxRunner(m, micro_batch=1).denoise(lat.cuda(), cond)
    assert rel(chunked - lat.cuda(), out.cpu() - lat) < L2


def test_shared_positions_give_the_tables_result(models):
    m = models[BF]
    runner = F.FluxRunner(m)
    g = seeded(6)
    sigmas = [1.0, 0.5]
    pooled, txt = torch.randn(2, CFG.vec_dim, generator=g), torch.randn(2, 7, CFG.context_dim, generator=g)
    lat = torch.randn(2, 20, 64, generator=g).cuda()
    ids = F.image_ids(4, 5)
    a = runner.step(0, lat, runner.prepare(sigmas, 3.5, pooled, txt, ids, F.text_ids(7)))[0]
    b = runner.step(0, lat, runner.prepare(sigmas, 3.5, pooled, txt, ids[None], F.text_ids(7)))[0]
    assert rel(a, b.cpu()) < L2
    with pytest.raises(ValueError, match="img_ids"):
        runner.prepare(sigmas, 3.5, pooled, txt, ids[None].expand(3, -1, -1), F.text_ids(7))


def test_quantized_blocks_at_positions_of_their_own():
    m = F.RandomFlux(CFG, "cuda", BF, seed=8, n_double=1, n_single=1)
    img, txt, ids = inputs(2, 64, 8, 8)
    every = torch.stack((ids, ids + 2.0))
    dmod = (torch.randn(2, 12 * CFG.hidden, generator=seeded(22)) * 0.3).to(BF)
    smod = (torch.randn(2, 3 * CFG.hidden, generator=seeded(23)) * 0.3).to(BF)
    x = torch.cat((txt, img), dim=1)
    gi, gt = F.double_block(m.doubles[0], img.cuda(), txt.cuda(), dmod.cuda(), None, None, CFG, BF, False, ids=every.cuda())
    gx = F.single_block(m.singles[0], x.cuda(), smod.cuda(), None, None, CFG, BF, False, ids=every.cuda())
    for i in range(2):
        cos, sin = S.rope_tables(every[i], CFG.axes_dim, CFG.theta)
        s = slice(i, i + 1)
        ri, rt = OF.double_block(oracle_unit(m.doubles[0]), img[s], txt[s], dmod[s], cos, sin, OCFG, BF, False)
        rx = OF.single_block(oracle_unit(m.singles[0]), x[s], smod[s], cos, sin, OCFG, BF, False)
        assert rel(gi[s].cpu() - img[s], ri - img[s]) < L2 and rel(gt[s].cpu() - txt[s], rt - txt[s]) < L2
        assert rel(gx[s].cpu() - x[s], rx - x[s]) < L2


def test_the_default_of_a_raw_unit_is_unchanged():
    # Without fused_raw a raw unit's blocks run the library linear and the separate kernels, bit for bit as before.
    m = F.RandomFlux(CFG, "cuda", BF, seed=9, n_double=0, n_single=1, with_mods=False, quant="raw")
    u = m.singles[0]
    u.fused_raw = False
    x = torch.randn(1, 40, CFG.hidden, generator=seeded(1)).cuda()
    smod = torch.randn(1, 3 * CFG.hidden, generator=seeded(2)).cuda() * 0.3
    cos, sin = (t.cuda() for t in S.rope_tables(torch.zeros(40, 3), CFG.axes_dim, CFG.theta))
    got = F.single_block(u, x, smod, cos, sin, CFG, BF, False)
    k, (sh, sc, g) = F.FUSED, smod.unsqueeze(1).chunk(3, dim=-1)
    y = torch.nn.functional.linear(k.mod_in(x, sh, sc, BF), u.get("linear1.weight"), u.get("linear1.bias"))
    qkv, mlp = y.split([3 * CFG.hidden, CFG.mlp_hidden], dim=-1)
    q, kk, v = k.qkv_single(qkv, u.get("norm.query_norm.scale", torch.float32), u.get("norm.key_norm.scale", torch.float32),
                            cos, sin, CFG.heads, BF)
    z = torch.nn.functional.linear(k.attn_mlp(F.attention(q, kk, v), mlp), u.get("linear2.weight"), u.get("linear2.bias"))
    assert torch.equal(got, k.gated_add(x, g, z, False))
