"""Rotary positions with several axes (rope_qk) against the formula in 64 bits.

Bound: sin and cos come from a remainder that is rounded to fp32 (off by at most 2^-24 of at most pi/4) and sums of
6 or 7 terms, within 2^-22; each product and the sum add 2^-24: (|z0| + |z1|) 2^-21 for a turned pair. The RMS
norm sums Dh squares in a tree of at most 16 + 6 additions and takes a root, a quotient and two products: 2^-19 of
a value. Then half a step of the type. The 64-bit reference's own angle is off by 2^-53 of pos, below 2^-29 here."""

from __future__ import annotations

import pytest
import torch

from selas_amd import _lib
from selas_amd.attention import attention
from selas_amd.linear import raw_linear
from selas_amd.rope import rope_qk

from .conftest import seeded

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(shape, seed, std=1.0, dtype=F32, mean=0.0):
    return (torch.randn(shape, generator=seeded(seed)) * std + mean).to(dtype)


def grid(b, l, axes, seed, hi=200, dtype=F32):
    return torch.randint(0, hi, (b, l, axes), generator=seeded(seed)).to(dtype)


def reference(x, scale, ids, axes, theta, pairs, inverse):
    """(value, bound ahead of the last rounding) in 64 bits."""
    z = x.detach().cpu().double()
    err = torch.zeros_like(z)
    if scale is not None:
        z = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * scale.cpu().double()
        err = 2.0 ** -19 * z.abs()
    pos = ids.cpu().double()
    pos = pos[None] if pos.dim() == 2 else pos
    ang = torch.cat([pos[..., i:i + 1] * float(theta) ** (-torch.arange(0, d, 2).double() / d)
                     for i, d in enumerate(axes)], -1)[:, None]
    c, s = ang.cos(), ang.sin() * (-1 if inverse else 1)
    n = ang.shape[-1]
    i0, i1 = (torch.arange(0, 2 * n, 2), torch.arange(1, 2 * n, 2)) if pairs == "interleaved" else (torch.arange(n),
                                                                                                torch.arange(n, 2 * n))
    out = z.clone()
    a, b, e = z[..., i0], z[..., i1], err[..., i0] + err[..., i1] + (z[..., i0].abs() + z[..., i1].abs()) * 2.0 ** -21
    out[..., i0], out[..., i1] = a * c - b * s, a * s + b * c
    err[..., i0], err[..., i1] = e, e
    return out, err


def check(y, ref_err):
    ref, err = ref_err
    fi = torch.finfo(y.dtype)
    tol = err + (ref.abs() + err) * fi.eps / 2 + fi.smallest_normal * fi.eps
    d = (y.detach().cpu().double() - ref).abs()
    assert y.shape == ref.shape and bool((d <= tol).all()), f"worst {(d / tol).max().item()} of the bound"


# (b, l, heads, k heads, dh, axes): vectors of 8 and 4 channels and single ones, whole and partly turned heads.
SHAPES = [(1, 1, 1, 1, 2, (2,)), (1, 1, 24, 24, 128, (16, 56, 56)), (2, 37, 3, 1, 64, (16, 24, 24)), (1, 5, 2, 2, 80, (20, 20, 40)),
          (2, 129, 4, 2, 96, (16, 28, 28)), (1, 33, 5, 1, 128, (32, 32)), (3, 7, 2, 1, 72, (12, 12, 12)),
          (1, 50, 3, 3, 20, (6, 6)), (1, 9, 2, 2, 21, (2, 4, 6, 8)), (2, 64, 2, 2, 256, (64, 96, 96)),
          (1, 1000, 12, 4, 128, (44, 42, 42)), (1, 6, 1, 2, 10, (0, 6))]


@pytest.mark.parametrize("b,l,h,hk,dh,axes", SHAPES)
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("norm", [False, True])
def test_against_the_formula(dev, b, l, h, hk, dh, axes, pairs, dtype, norm):
    q, k, v = normal((b, h, l, dh), 1, 2, dtype), normal((b, hk, l, dh), 2, 1, dtype), normal((b, hk, l, dh), 3, 1, dtype)
    ids = grid(b, l, len(axes), 4)
    qs, ks = (normal((dh,), 5, 0.2, mean=1.0), normal((dh,), 6, 0.2, mean=1.0)) if norm else (None, None)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = rope_qk(to(q), to(k), to(ids), axes, v=to(v), q_scale=to(qs), k_scale=to(ks), pairs=pairs)
    assert len(y) == 3 and all(t.is_contiguous() and t.dtype == dtype for t in y) and torch.equal(y[2].cpu(), v)
    check(y[0], reference(q, qs, ids, axes, 10000.0, pairs, False))
    check(y[1], reference(k, ks, ids, axes, 10000.0, pairs, False))
    if not norm:
        y = rope_qk(to(q), to(k), to(ids), axes, 500.0, pairs=pairs, inverse=True)
        assert len(y) == 2
        check(y[0], reference(q, None, ids, axes, 500.0, pairs, True))
        check(y[1], reference(k, None, ids, axes, 500.0, pairs, True))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, F32])
def test_positions_far_out_negative_and_fractional(dev, dtype):
    q, k = normal((2, 2, 40, 64), 1), normal((2, 1, 40, 64), 2)
    ids = torch.randint(-(1 << 24), 1 << 24, (2, 40, 2), generator=seeded(3))
    ids[0, :5], ids[1, 7] = 0, (1 << 24) - 1
    ids = ids.to(dtype) if dtype != F32 else ids.float() / 1024 + 0.25
    y = rope_qk(q.to(dev), k.to(dev), ids.to(dev), (32, 32))
    check(y[0], reference(q, None, ids, (32, 32), 10000.0, "interleaved", False))
    check(y[1], reference(k, None, ids, (32, 32), 10000.0, "interleaved", False))
    if dtype != F32:  # (the fp32 positions are a quarter off whole numbers)
        assert torch.equal(y[0][0, :, :5].cpu(), q[0, :, :5])  # position 0 turns nothing


def test_positions_that_are_not_finite_stay_in_their_row(dev):
    q = normal((1, 2, 8, 64), 1).to(dev)
    ids = grid(1, 8, 2, 2).to(dev)
    ref = rope_qk(q, q, ids, (32, 32))[0]
    ids[0, 3, 0], ids[0, 5, 1] = float("nan"), float("inf")
    y = rope_qk(q, q, ids, (32, 32))[0]
    rows = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[:, :, rows], ref[:, :, rows])
    assert bool(y[:, :, 3, :32].isnan().all()) and torch.equal(y[:, :, 3, 32:], ref[:, :, 3, 32:])
    assert bool(y[:, :, 5, 32:].isnan().all()) and torch.equal(y[:, :, 5, :32], ref[:, :, 5, :32])


def test_shared_and_broadcast_positions(dev):
    q, k = normal((3, 2, 17, 64), 1, dtype=BF).to(dev), normal((3, 2, 17, 64), 2, dtype=BF).to(dev)
    ids = grid(1, 17, 3, 3).to(dev)
    axes = (16, 24, 24)
    a = rope_qk(q, k, ids[0], axes)
    for other in (ids, ids.expand(3, -1, -1), ids.repeat(3, 1, 1), torch.cat([ids, ids], -1)[..., :3],
                  ids.transpose(1, 2).contiguous().transpose(1, 2)):
        assert all(torch.equal(s, t) for s, t in zip(a, rope_qk(q, k, other, axes)))


@pytest.mark.parametrize("dtype,dh,axes", [(BF, 128, (16, 56, 56)), (FP, 96, (16, 28, 28)), (F32, 20, (6, 6)),
                                           (BF, 36, (6, 6, 6))])
def test_views_of_one_linear_output_and_in_place(dev, dtype, dh, axes):
    b, l, h = 2, 45, 3
    qkv = normal((b, l, 3 * h * dh + 3), 1, dtype=dtype).to(dev)
    for off in (0, 3):  # off 3: rows off every vector
        view = qkv[..., off:off + 3 * h * dh]
        q, k, v = view.unflatten(-1, (3, h, dh)).permute(2, 0, 3, 1, 4)
        ids = grid(b, l, len(axes), 2).to(dev)
        ref = rope_qk(q.contiguous(), k.contiguous(), ids, axes, v=v.contiguous())
        got = rope_qk(q, k, ids, axes, v=v)
        assert all(torch.allclose(s.float(), t.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-6)
                   for s, t in zip(ref, got))
        # In place over q and k, v untouched; the rest of the buffer too.
        buf = qkv.clone()
        bq, bk, bv = buf[..., off:off + 3 * h * dh].unflatten(-1, (3, h, dh)).permute(2, 0, 3, 1, 4)
        out = rope_qk(bq, bk, ids, axes, out=(bq, bk))
        assert out[0] is bq and torch.equal(bq, got[0]) and torch.equal(bk, got[1]) and torch.equal(bv, v)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[..., off:off + 2 * h * dh] = False
        assert torch.equal(buf[mask], qkv[mask])


def test_destinations_inside_a_joint_buffer(dev):
    # Text and image tokens written into one [B, H, Lt + Li, Dh] buffer, as a double block's attention reads them.
    b, h, lt, li, dh, axes = 2, 3, 11, 30, 64, (16, 24, 24)
    ids = grid(b, lt + li, 3, 1).to(dev)
    x = [normal((b, h, n, dh), i, dtype=BF).to(dev) for i, n in enumerate((lt, li, lt, li))]
    q, k = torch.full((b, h, lt + li, dh), 9.0, dtype=BF, device=dev), torch.empty(b, h, lt + li, dh, dtype=BF, device=dev)
    rope_qk(x[0], x[2], ids[:, :lt], axes, out=(q[:, :, :lt], k[:, :, :lt]))
    assert bool((q[:, :, lt:] == 9.0).all())
    rope_qk(x[1], x[3], ids[:, lt:], axes, out=(q[:, :, lt:], k[:, :, lt:]))
    ref = rope_qk(torch.cat((x[0], x[1]), 2), torch.cat((x[2], x[3]), 2), ids, axes)
    assert torch.equal(q, ref[0]) and torch.equal(k, ref[1])


def test_empty(dev):
    z = torch.zeros(2, 3, 0, 64, dtype=BF, device=dev)
    assert rope_qk(z, z, torch.zeros(0, 1, device=dev), (64,))[0].shape == (2, 3, 0, 64)
    one = torch.ones(1, 2, 4, 64, dtype=BF, device=dev)
    y = rope_qk(one, one[:, :0], torch.ones(4, 1, device=dev), (64,))
    assert y[1].shape == (1, 0, 4, 64) and not torch.equal(y[0], one)


def test_inverse_is_the_gradient(dev):
    # f = <w, rope(q)> has the gradient rope_inverse(w); differences of f are exact for a linear f up to rounding.
    for pairs in ("interleaved", "halves"):
        q, w = normal((1, 2, 6, 40), 1), normal((1, 2, 6, 40), 2)
        ids, axes = grid(1, 6, 2, 3).to(dev), (12, 20)
        f = lambda t: (rope_qk(t, t, ids, axes, pairs=pairs)[0].double() * w.to(dev).double()).sum().item()  # noqa: E731
        grad = rope_qk(w.to(dev), w.to(dev), ids, axes, pairs=pairs, inverse=True)[0]
        base = torch.zeros(1, 2, 6, 40)
        for at in ((0, 0, 0, 0), (0, 1, 3, 13), (0, 0, 5, 31), (0, 1, 2, 39)):
            step = base.clone()
            step[at] = 1.0
            # f is a sum of at most two products of values within 2^-22 of theirs.
            assert abs(f(step.to(dev)) - grad[at].item()) <= 2.0 ** -20 * w.abs().max().item()
        back = rope_qk(*rope_qk(q.to(dev), q.to(dev), ids, axes, pairs=pairs), ids, axes, pairs=pairs, inverse=True)[0]
        assert bool(((back.cpu() - q).abs() <= 2.0 ** -19 * q.abs().max()).all())


def test_streams_and_a_captured_graph(dev):
    q, k = normal((2, 4, 100, 128), 1, dtype=BF).to(dev), normal((2, 4, 100, 128), 2, dtype=BF).to(dev)
    ids, axes = grid(2, 100, 3, 3).to(dev), (16, 56, 56)
    ref = rope_qk(q, k, ids, axes)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = rope_qk(q, k, ids, axes)
    s.synchronize()
    assert torch.equal(ref[0], other[0]) and torch.equal(ref[1], other[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rope_qk(q, k, ids, axes)
    for i in range(3):
        q.copy_(normal((2, 4, 100, 128), 10 + i, dtype=BF).to(dev))
        ids.add_(1)
        g.replay()
        torch.cuda.synchronize()
        want = rope_qk(q, k, ids, axes)
        assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])


def test_a_destination_over_the_positions_or_a_scale_is_refused(dev):
    x, buf = torch.ones(1, 2, 8, 64, device=dev), torch.ones(2048, device=dev)
    over, free = buf[:1024].view(1, 2, 8, 64), torch.empty(1, 2, 8, 64, device=dev)
    for kw in ({"ids": buf[1000:1008].view(8, 1)}, {"ids": buf[2000:2008].view(8, 1), "q_scale": buf[960:1024]},
               {"ids": buf[2000:2008].view(8, 1), "k_scale": buf[:64]}):
        with pytest.raises(ValueError, match="overlaps"):
            rope_qk(x, x, axes_dim=(64,), out=(free, over), **kw)
    rope_qk(x, x, buf[2000:2008].view(8, 1), (64,), q_scale=buf[1024:1088], out=(free, over))
    assert bool(buf[1024:].eq(1).all())


def test_refusals(dev):
    q = torch.zeros(2, 3, 5, 64, dtype=BF, device=dev)
    ids = torch.zeros(5, 2, device=dev)
    axes = (32, 32)
    for args, kw, match in (((q[0], q, ids, axes), {}, "B, heads"), ((q, q[:1], ids, axes), {}, "does not go"),
                            ((q, q.float(), ids, axes), {}, "does not go"), ((q, q, ids[:4], axes), {}, "positions"),
                            ((q, q, ids, (32, 16, 16)), {}, "positions"), ((q, q, ids.double(), axes), {}, "positions"),
                            ((q, q, ids, (33, 31)), {}, "even"), ((q, q, ids, (64, 2)), {}, "heads 64"),
                            ((q, q, ids, ()), {}, "axes"), ((q, q, ids, axes, -1.0), {}, "theta"),
                            ((q, q, ids, axes, float("nan")), {}, "theta"), ((q, q, ids, axes), {"pairs": "x"}, "pairs"),
                            ((q, q, ids, axes), {"q_scale": torch.ones(3, device=dev)}, "q_scale"),
                            ((q, q, ids, axes), {"inverse": True, "k_scale": torch.ones(64, device=dev)}, "inverse"),
                            ((q, q, ids, axes), {"out": (q,)}, "out"), ((q, q, ids, axes), {"out": (q, q)}, "overlaps"),
                            ((q.cpu(), q, ids, axes), {}, "GPU")):
        with pytest.raises(ValueError, match=match):
            rope_qk(*args, **kw)
    with pytest.raises(_lib.Unsupported, match="dtype"):
        rope_qk(q.double(), q.double(), ids, axes)
    wide = torch.zeros(1, 1, 2, 320, dtype=BF, device=dev)
    with pytest.raises(_lib.Unsupported, match="head_dim"):
        rope_qk(wide, wide, torch.zeros(2, 1, device=dev), (320,))
    odd = torch.zeros(1, 1, 2, 162, dtype=BF, device=dev)
    with pytest.raises(_lib.Unsupported, match="alignment"):
        rope_qk(odd, odd, torch.zeros(2, 1, device=dev), (162,))


def test_qkv_linear_rope_attention_and_gated_projection(dev):
    # The attention half of a block with raw weights, as it is used: two images at positions of their own.
    b, l, h, dh = 2, 150, 2, 128
    d = h * dh
    x = normal((b, l, d), 1, dtype=BF)
    wqkv, wo = normal((3 * d, d), 2, d ** -0.5, BF), normal((d, d), 3, d ** -0.5, BF)
    bqkv, gate, res = normal((3 * d,), 4, 0.1, BF), normal((b, 1, d), 5, 0.5), normal((b, l, d), 6)
    qs, ks = normal((dh,), 7, 0.1, mean=1.0), normal((dh,), 8, 0.1, mean=1.0)
    ids, axes = grid(b, l, 3, 9, hi=64), (16, 56, 56)
    qkv = raw_linear(x.to(dev), wqkv.to(dev), bqkv.to(dev))
    q, k, v = qkv.unflatten(-1, (3, h, dh)).permute(2, 0, 3, 1, 4)
    q, k, v = rope_qk(q, k, ids.to(dev), axes, v=v, q_scale=qs.to(dev), k_scale=ks.to(dev))
    y = raw_linear(attention(q, k, v), wo.to(dev), gate=gate.to(dev), residual=res.to(dev))
    # 64 bits throughout; each 16-bit intermediate rounding (qkv, q, k, v, probabilities, attention) is 2^-8 at most, so the
    # gated branch is compared at 6 of them in the L2 norm.
    z = (x.double() @ wqkv.double().t() + bqkv.double()).unflatten(-1, (3, h, dh)).permute(2, 0, 3, 1, 4)
    rq = reference(z[0], qs, ids, axes, 10000.0, "interleaved", False)[0]
    rk = reference(z[1], ks, ids, axes, 10000.0, "interleaved", False)[0]
    a = torch.softmax(rq @ rk.transpose(-1, -2) / dh ** 0.5, -1) @ z[2]
    branch = gate.double() * (a.transpose(1, 2).reshape(b, l, d) @ wo.double().t())
    diff = y.cpu().double() - res.double() - branch
    assert diff.norm() <= 6 * 2.0 ** -8 * branch.norm()
