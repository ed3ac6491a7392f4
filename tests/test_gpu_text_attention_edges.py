"""cross_attention and text_attention at the edges of what they take: axes of no and of one element, strides that say
nothing, weight on few of many keys, extreme entries of the bias table."""

from __future__ import annotations

import pytest
import torch

from selas_amd.text_attention import (cross_attention, cross_attention_backward, text_attention, text_attention_backward)

from .test_gpu_text_attention import BF, F32, FP, inputs, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [64, 96, 128])
@pytest.mark.parametrize("lk", [1, 77, 3000])
def test_without_queries_the_gradients_are_zeros(dtype, dh, lk):
    q, k, v = inputs(2, 4, 2, 0, lk, dh, dtype=dtype)
    mask = torch.ones(2, lk, dtype=torch.bool).cuda()
    out, lse = cross_attention(q, k, v, return_lse=True)
    assert out.shape == (2, 0, 4 * dh) and lse.shape == (2, 4, 0)
    for kw in (dict(), dict(mask=mask), dict(lengths=torch.tensor([lk, 1]).cuda())):
        stale = [torch.full_like(t, float("nan")) for t in (k, v)]
        del stale  # what the allocator hands out next holds no zeros
        dq, dk, dv = cross_attention_backward(out, q, k, v, out, lse, **kw)
        assert (dq.shape, dk.shape, dv.shape) == (q.shape, k.shape, v.shape) and not dk.any() and not dv.any()
    for t in (dtype, F32):
        table = table_of(32, 4, dtype=t)
        out, lse = text_attention(q, k, v, table, causal=True, return_lse=True)
        dq, dk, dv, dtable = text_attention_backward(out, q, k, v, out, lse, table, causal=True)
        assert not dk.any() and not dv.any() and dtable.shape == table.shape and dtable.dtype == t and not dtable.any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("dh", [64, 72, 128])
@pytest.mark.parametrize("lk", [1, 40, 200, 2000])  # up to 2000: one range of keys, and several
@pytest.mark.parametrize("stride", [0, 8, 4096])
def test_the_row_stride_of_one_row_says_nothing(dtype, dh, lk, stride):
    # 16 query heads of one key head: the kernel of 32 rows, of which one exists.
    q, k, v = inputs(2, 16, 1, 1, lk, dh, seed=lk, dtype=dtype)
    want = cross_attention(q, k, v)
    n = 16 * dh
    for b in (1, 2):
        given = torch.full((2 * n + 8,), 7.0, dtype=dtype, device="cuda")
        out = given[4:].as_strided((b, 1, n), (n, stride, 1))
        assert torch.equal(cross_attention(q[:b], k[:b], v[:b], out=out), want[:b])
        assert bool((given[:4] == 7).all()) and bool((given[4 + b * n:] == 7).all())


@pytest.mark.parametrize("lq", [1, 3])
def test_strides_of_axes_of_one_element_are_not_looked_at(lq):
    q, k, v = inputs(1, 16, 1, lq, 100, 64, seed=lq)
    want, n = cross_attention(q, k, v), 16 * 64
    for sb, sl in ((0, n), (3, n), (1 << 40, n), (n, n if lq > 1 else 1), (n, n if lq > 1 else 1 << 30)):
        out = torch.empty(lq * n, dtype=BF, device="cuda").as_strided((1, lq, n), (sb, sl, 1))
        assert torch.equal(cross_attention(q, k, v, out=out), want)
        assert out.stride() == (sb, sl, 1)
    with pytest.raises(ValueError, match="out must be"):
        cross_attention(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1),
                        out=torch.empty(2 * lq * n + 3, dtype=BF, device="cuda").as_strided((2, lq, n), (lq * n + 3, n, 1)))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_gradients_of_one_query_and_one_key_at_any_stride(dtype):
    q, k, v = inputs(2, 16, 2, 1, 1, 64, dtype=dtype)
    q2, k2, v2 = inputs(2, 16, 2, 1, 90, 64, dtype=dtype)
    grad = torch.ones(2, 1, 1024, dtype=dtype, device="cuda")

    def folded(t, stride):  # the same elements, the row stride of the one row replaced
        t = t.contiguous()
        return t.as_strided(t.shape, (*t.stride()[:-2], stride, 1))

    for args in ((q, k, v), (q2, k2, v2)):
        out, lse = cross_attention(*args, return_lse=True)
        want = (out, lse, *cross_attention_backward(grad, *args, out, lse))
        for stride in (0, 8, 1 << 30):
            x = [folded(t, stride) if t.shape[2] == 1 else t for t in args]
            out, lse = cross_attention(*x, return_lse=True)
            got = (out, lse, *cross_attention_backward(folded(grad, stride), *x, folded(out, stride), lse))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
