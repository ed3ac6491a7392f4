"""cross_attention and text_attention against the definition in 64 bits (bounds: text_attention_reference.py)."""

from __future__ import annotations

import pytest
import torch

from selas_amd.text_attention import cross_attention, text_attention

from .conftest import seeded
from .text_attention_reference import Reference, within

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def heads(b, h, l, dh, seed, dtype=BF, std=1.0):
    """[b, h, l, dh] as a view of a linear's output."""
    return (torch.randn(b, l, h, dh, generator=seeded(seed)) * std).to(dtype).cuda().transpose(1, 2)


def inputs(b, h, hk, lq, lk, dh, seed=0, dtype=BF, std=1.0):
    return heads(b, h, lq, dh, seed, dtype, std), heads(b, hk, lk, dh, seed + 1, dtype), heads(b, hk, lk, dh, seed + 2, dtype)


def table_of(buckets, h, seed=7, dtype=BF, std=1.0):
    return (torch.randn(buckets, h, generator=seeded(seed)) * std).to(dtype).cuda()


def check(fn, q, k, v, *args, **kw):
    out, lse = fn(q, k, v, *args, return_lse=True, **kw)
    ref = Reference(q, k, v, *args, **kw)
    within(out, ref.out, ref.out_bound)
    within(lse, ref.lse, ref.lse_bound)
    assert torch.equal(fn(q, k, v, *args, **kw).view(torch.int16), out.view(torch.int16))
    return out


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq", [1, 2, 3, 7, 8])
@pytest.mark.parametrize("lk,dh", [(1, 64), (2, 128), (63, 8), (64, 64), (65, 72), (517, 128), (1000, 40)])
def test_few_queries(lq, lk, dh, dtype):
    check(cross_attention, *inputs(2, 3, 3, lq, lk, dh, seed=lq + lk, dtype=dtype))


@pytest.mark.parametrize("lq,h,hk", [(1, 4, 2), (1, 8, 1), (2, 8, 2), (3, 4, 2), (1, 6, 2)])
def test_few_queries_of_shared_key_heads(lq, h, hk):
    check(cross_attention, *inputs(2, h, hk, lq, 333, 96, seed=lq))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lq", [9, 32, 33, 64, 65, 128, 131, 300])
@pytest.mark.parametrize("lk,dh", [(1, 64), (64, 128), (65, 72), (77, 40), (200, 128), (449, 64)])
def test_many_queries(lq, lk, dh, dtype):
    check(cross_attention, *inputs(2, 4, 2, lq, lk, dh, seed=lq + lk, dtype=dtype))


@pytest.mark.parametrize("lq", [1, 5, 33, 130])
@pytest.mark.parametrize("dh", [64, 128])
def test_a_long_axis_is_split(lq, dh):
    # One image and few heads: the keys are dealt to several workgroups and joined.
    q, k, v = inputs(1, 2, 1, lq, 9001, dh, seed=lq)
    check(cross_attention, q, k, v)
    check(cross_attention, q, k, v, lengths=torch.tensor([4100], dtype=torch.int32).cuda())
    check(text_attention, q, k, v, table_of(32, 2), causal=True, q_start=8000)


@pytest.mark.parametrize("lq", [1, 4, 40, 150])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_lengths(lq, itype):
    q, k, v = inputs(6, 4, 2, lq, 200, 64, seed=lq)
    lengths = torch.tensor([0, 1, 64, 65, 199, 200], dtype=itype).cuda()
    out = check(cross_attention, q, k, v, lengths=lengths)
    assert not out[0].any()
    for i, n in enumerate((0, 1, 64, 65, 199)):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    assert torch.equal(cross_attention(q, k, v, lengths=lengths), out)
    # Past either end: as the nearer end.
    assert torch.equal(cross_attention(q, k, v, lengths=torch.tensor([-5, 1, 64, 65, 199, 1 << 30], dtype=itype).cuda()), out)


@pytest.mark.parametrize("lq,dtype", [(1, BF), (4, FP), (40, BF), (150, FP)])
def test_masks(lq, dtype):
    q, k, v = inputs(4, 4, 2, lq, 333, 96, seed=lq, dtype=dtype)
    mask = torch.rand(4, 333, generator=seeded(3)) < 0.6
    mask[0], mask[1, :128], mask[2, 70:] = False, False, False
    mask = mask.cuda()
    out = check(cross_attention, q, k, v, mask=mask)
    assert not out[0].any()
    hidden = ~mask[:, None, :, None]
    k2, v2 = k.masked_fill(hidden, float("nan")), v.masked_fill(hidden, float("inf"))
    assert torch.equal(cross_attention(q, k2, v2, mask=mask), out)
    check(cross_attention, q, k, v, mask=mask, lengths=torch.tensor([333, 200, 64, 129], dtype=torch.int32).cuda())
    check(cross_attention, q, k, v, mask=mask[3:4])
    check(cross_attention, q, k, v, mask=mask.t().contiguous().t())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("l", [1, 31, 77, 128, 200, 600])
@pytest.mark.parametrize("buckets,distance,both", [(32, 128, True), (32, 128, False), (4, 3, True), (2, 2, False), (24, 200, False),
                                                   (256, 512, True)])
def test_bias(l, buckets, distance, both, dtype):
    q, k, v = inputs(2, 4, 2, l, l, 64, seed=l, dtype=dtype, std=0.125)
    kw = dict(max_distance=distance, bidirectional=both, scale=1.0)
    for t in (BF, F32):
        check(text_attention, q, k, v, table_of(buckets, 4, dtype=t), **kw)
    check(text_attention, q, k, v, table_of(buckets, 4, std=5.0), causal=True, **kw)


@pytest.mark.parametrize("dh", [72, 128])
def test_bias_of_wide_heads(dh):
    q, k, v = inputs(2, 4, 4, 300, 450, dh, seed=dh)
    for kw in (dict(), dict(causal=True), dict(q_start=150), dict(q_start=-100, causal=True), dict(bidirectional=False, q_start=2000)):
        check(text_attention, q, k, v, table_of(32, 4), **kw)


@pytest.mark.parametrize("l", [1, 32, 63, 77, 129, 300])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_causal(l, dtype):
    q, k, v = inputs(3, 4, 4, l, l, 64, seed=l, dtype=dtype)
    check(text_attention, q, k, v, causal=True)
    lengths = torch.tensor([l, l // 2, 0], dtype=torch.int32).cuda()
    check(text_attention, q, k, v, causal=True, lengths=lengths)
    mask = torch.rand(3, l, generator=seeded(3)) < 0.5
    mask[0, 0] = False  # a first row that sees nothing
    out = check(text_attention, q, k, v, causal=True, mask=mask.cuda())
    assert not out[0, 0].any()


@pytest.mark.parametrize("lq", [1, 3, 20, 70])
def test_later_tokens_over_a_cache_equal_the_whole_texts_rows(lq):
    b, h, hk, l = 3, 8, 4, 500
    q, k, v = inputs(b, h, hk, l, l, 64, seed=1, std=0.125)
    table, lengths = table_of(32, h), torch.tensor([500, 317, 71], dtype=torch.int32).cuda()
    kw = dict(bidirectional=False, causal=True, scale=1.0)
    start = lengths - lq
    last = torch.stack([q[i, :, n - lq:n] for i, n in enumerate((500, 317, 71))])
    check(text_attention, last, k, v, table, q_start=start, lengths=lengths, **kw)
    whole = Reference(q, k, v, table, lengths=lengths, **kw)
    out = text_attention(last, k, v, table, q_start=start, lengths=lengths, **kw)
    for i, n in enumerate((500, 317, 71)):
        within(out[i], whole.out[i, n - lq:n], whole.out_bound[i, n - lq:n])
    # int64 positions and lengths say the same
    assert torch.equal(out, text_attention(last, k, v, table, q_start=start.long(), lengths=lengths.long(), **kw))
    same = text_attention(last, k, v, table, q_start=300, **kw)
    assert torch.equal(same, text_attention(last, k, v, table, q_start=torch.full((b,), 300).cuda(), **kw))


@pytest.mark.parametrize("dh", [8, 32, 48, 56, 80, 88, 96, 104, 120])
@pytest.mark.parametrize("lq", [3, 70, 200])
def test_head_dims(dh, lq):
    q, k, v = inputs(2, 4, 2, lq, 210, dh, seed=dh + lq)
    check(cross_attention, q, k, v)
    check(text_attention, q, k, v, table_of(32, 4), causal=True, q_start=5)


@pytest.mark.parametrize("lq,h,hk", [(1, 8, 1), (150, 4, 2)])
def test_the_widest_tables(lq, h, hk):
    # As much LDS as a call can take: 128 channels and the largest distances.
    q, k, v = inputs(1, h, hk, lq, 1300, 128, seed=lq)
    check(text_attention, q, k, v, table_of(256, h), max_distance=512, q_start=600)
    check(text_attention, q, k, v, table_of(128, h), max_distance=512, bidirectional=False, causal=True, q_start=1100)
