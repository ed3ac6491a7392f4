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
