"""The gradients of cross_attention and text_attention against the formula's in 64 bits (bounds:
text_attention_reference.py) and against differences of the forward pass."""

from __future__ import annotations

import pytest
import torch

from selas_amd.text_attention import (cross_attention, cross_attention_backward, text_attention, text_attention_backward)

from .conftest import seeded
from .test_gpu_text_attention import BF, F32, FP, heads, inputs, table_of
from .text_attention_reference import Reference, within

pytestmark = pytest.mark.gpu


def grad_of(q, seed=11, std=1.0):
    b, h, l, dh = q.shape
    return (torch.randn(b, l, h * dh, generator=seeded(seed)) * std).to(q.dtype).cuda()


def check(q, k, v, *args, grad=None, **kw):
    grad = grad_of(q) if grad is None else grad
    if args or "causal" in kw or "q_start" in kw:
        out, lse = text_attention(q, k, v, *args, return_lse=True, **kw)
        run = lambda: text_attention_backward(grad, q, k, v, out, lse, *args, **kw)  # noqa: E731
    else:
        out, lse = cross_attention(q, k, v, return_lse=True, **kw)
        run = lambda: (*cross_attention_backward(grad, q, k, v, out, lse, **kw), None)  # noqa: E731
    got, ref = run(), Reference(q, k, v, *args, **kw).backward(grad)
    for name, y, want in zip(("dq", "dk", "dv", "dtable"), got, ref):
        assert (y is None) == (want is None), name
        if y is not None:
            print(name, flush=True)
            within(y, *want)
    again = run()
    assert all(torch.equal(x, y) for x, y in zip(got, again) if x is not None)
    return got


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 200), (200, 1), (33, 65), (64, 64), (128, 128), (130, 77), (77, 300), (300, 450)])
@pytest.mark.parametrize("dh", [40, 64, 128])
def test_gradients(lq, lk, dh, dtype):
    check(*inputs(2, 2, 2, lq, lk, dh, seed=lq + lk, dtype=dtype))


@pytest.mark.parametrize("h,hk", [(4, 2), (8, 1), (6, 2)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_shared_key_heads(h, hk, dtype):
    check(*inputs(2, h, hk, 100, 150, 72, seed=h, dtype=dtype))


@pytest.mark.parametrize("lq,lk", [(3000, 70), (40, 3000), (2049, 2049)])
def test_long_axes_are_split(lq, lk):
    check(*inputs(1, 2, 1, lq, lk, 64, seed=lq))
    check(*inputs(1, 1, 1, lq, lk, 128, seed=lk))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq", [1, 40, 150])
def test_lengths_and_masks(lq, dtype):
    q, k, v = inputs(5, 4, 2, lq, 200, 64, seed=lq, dtype=dtype)
    lengths = torch.tensor([0, 1, 64, 130, 200], dtype=torch.int32).cuda()
    mask = torch.rand(5, 200, generator=seeded(3)) < 0.6
    mask[3, :128] = False
    mask = mask.cuda()
    dq, dk, dv, _ = check(q, k, v, lengths=lengths)
    assert not dq[0].any() and not dk[1, :, 1:].any() and not dv[0].any()
    check(q, k, v, mask=mask)
    want = check(q, k, v, mask=mask, lengths=lengths)
    hidden = (~mask | (torch.arange(200, device="cuda") >= lengths[:, None]))[:, None, :, None]
    k, v = k.masked_fill(hidden, float("nan")), v.masked_fill(hidden, float("inf"))
    out, lse = cross_attention(q, k, v, mask=mask, lengths=lengths, return_lse=True)
    got = cross_attention_backward(grad_of(q), q, k, v, out, lse, mask=mask, lengths=lengths)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("l", [1, 31, 77, 128, 200, 600])
@pytest.mark.parametrize("buckets,distance,both", [(32, 128, True), (32, 128, False), (4, 3, True), (24, 200, False),
                                                   (256, 512, True)])
def test_bias(l, buckets, distance, both, dtype):
    q, k, v = inputs(2, 4, 2, l, l, 64, seed=l, dtype=dtype, std=0.125)
    kw = dict(max_distance=distance, bidirectional=both, scale=1.0)
    check(q, k, v, table_of(buckets, 4, dtype=dtype), **kw)
    check(q, k, v, table_of(buckets, 4, dtype=F32), causal=True, **kw)


@pytest.mark.parametrize("dh", [72, 128])
def test_bias_of_wide_heads(dh):
    q, k, v = inputs(2, 4, 4, 300, 450, dh, seed=dh)
    for kw in (dict(), dict(causal=True), dict(q_start=150), dict(q_start=-100, causal=True), dict(bidirectional=False, q_start=2000),
               dict(max_distance=512, lengths=torch.tensor([450, 77]).cuda()),
               dict(mask=(torch.rand(2, 450, generator=seeded(5)) < 0.5).cuda(), causal=True, q_start=torch.tensor([150, 3]).cuda())):
        check(q, k, v, table_of(32, 4), **kw)


@pytest.mark.parametrize("l", [1, 63, 77, 129, 300])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_causal(l, dtype):
    q, k, v = inputs(3, 4, 4, l, l, 64, seed=l, dtype=dtype)
    check(q, k, v, causal=True)
    check(q, k, v, causal=True, lengths=torch.tensor([l, l // 2, 0], dtype=torch.int32).cuda())
    mask = torch.rand(3, l, generator=seeded(3)) < 0.5
    mask[0, 0] = False
    check(q, k, v, causal=True, mask=mask.cuda())


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 1e3])
def test_fp16_gradients_of_any_size(size):
    # dS is held with a power of two of its own: small gradients keep their digits, large ones do not overflow inside.
    q, k, v = inputs(2, 4, 2, 150, 333, 64, seed=5, dtype=FP)
    check(q, k, v, grad=grad_of(q, std=size))
    check(q, k, v * 50, grad=grad_of(q, std=size))


def test_differences_of_the_forward_pass():
    # Along a direction: (f(x + t d) - f(x - t d)) / 2t of f = sum(out * grad). The outputs are off by their bounds, which
    # the sum collects at random (sqrt(n) of the mean square; 6 of them), and the third derivative adds t^2.
    q, k, v = inputs(2, 4, 2, 65, 77, 64, seed=3, dtype=FP)
    table, grad = table_of(32, 4, dtype=F32), grad_of(q)
    out, lse = text_attention(q, k, v, table, return_lse=True)
    got = text_attention_backward(grad, q, k, v, out, lse, table)
    xs, t = [q, k, v, table], 2.0 ** -5
    for i, d in enumerate(got):
        way = torch.randint(0, 2, xs[i].shape, generator=seeded(i)).mul(2).sub(1).to(xs[i].dtype).cuda()
        ends, noise = [], 0.0
        for sign in (1, -1):
            moved = [x + sign * t * way if j == i else x for j, x in enumerate(xs)]
            step = (moved[i].double() - xs[i].double()).abs().mean().item()
            ref = Reference(*moved)
            ends.append((text_attention(*moved).double() * grad.double()).sum().item())
            noise += ((ref.out_bound * grad.cpu().double()) ** 2).sum().item()
        slope = (ends[0] - ends[1]) / (2 * step)
        # x + t d is rounded to x's type: half a step of each element, with a random sign.
        exact = (d.double() * (xs[i] + t * way - (xs[i] - t * way)).double()).sum().item() / (2 * step)
        curve = step ** 2 * (d.double().abs().sum().item())
        assert abs(slope - exact) <= 6 * noise ** 0.5 / (2 * step) + curve, (i, slope, exact)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [40, 64, 128])
def test_rows_of_one_key_have_no_gradient_of_their_scores(dh, dtype):
    # The weight is 1 whatever the score, out is that key's value and dP - D is 0 exactly.
    q, k, v = inputs(2, 4, 2, 100, 1, dh, seed=dh, dtype=dtype)
    dq, dk, _, dtable = check(q, k, v, table_of(32, 4))
    assert not dq.any() and not dk.any() and not dtable.any()
    q, k, v = inputs(2, 4, 4, 70, 70, dh, seed=dh, dtype=dtype)
    dq, _, _, _ = check(q, k, v, causal=True)
    assert not dq[:, :, 0].any() and dq[:, :, 1].any()
    dq, dk, _, _ = check(q, k, v, lengths=torch.tensor([1, 1]).cuda())
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize("dtype,half", [(BF, 2.0 ** -8), (FP, 2.0 ** -11)])
@pytest.mark.parametrize("l", [2, 16, 77, 256])
def test_gradients_lose_no_more_than_two_roundings(l, dtype, half):
    # dS and the result are rounded once each; errors of one rounding are spread evenly over +-half a step of values of
    # every mantissa: 0.42 of `half` in the mean square (sqrt of the mean of 1 / (3 m^2) over m in 1 .. 2, weighted by 1 / m).
    # Two of them are 0.6; D's own share, where few keys carry a row, would make it 0.73. A tenth is left for chance.
    q, k, v = inputs(2, 8, 8, l, l, 64, seed=l, dtype=dtype)
    grad, table = grad_of(q), table_of(32, 8, dtype=dtype)
    kw = dict(causal=True, bidirectional=False)
    out, lse = text_attention(q, k, v, table, return_lse=True, **kw)
    got = text_attention_backward(grad, q, k, v, out, lse, table, **kw)
    for y, (ref, _) in zip(got, Reference(q, k, v, table, **kw).backward(grad)):
        assert (y.cpu().double() - ref).norm() <= 1.1 * 0.6 * half * ref.norm()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [8, 32, 48, 56, 80, 88, 96, 104, 120])
def test_head_dims(dh, dtype):
    q, k, v = inputs(2, 4, 2, 150, 210, dh, seed=dh, dtype=dtype)
    check(q, k, v)
    check(q, k, v, table_of(32, 4), causal=True, q_start=5)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_the_widest_tables(dtype):
    # As much LDS as a call can take: 128 channels and the largest distances.
    q, k, v = inputs(1, 4, 2, 150, 1300, 128, seed=1, dtype=dtype)
    check(q, k, v, table_of(256, 4), max_distance=512, q_start=600)
    check(q, k, v, table_of(128, 4), max_distance=512, bidirectional=False, causal=True, q_start=1100)
