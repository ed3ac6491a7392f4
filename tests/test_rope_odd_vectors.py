"""Rotated channels that are an odd number of vectors of 4 (sum(axes_dim) a multiple of 4 but not of 8): adjacent pairs run
in vectors, at heads above 128 channels too. Bounds as in test_gpu_rope.py."""

from __future__ import annotations

import pytest
import torch

from selas_amd import _lib
from selas_amd.rope import rope_qk

from .test_gpu_rope import BF, F32, FP, check, grid, normal, reference
from .test_operator_checks import rope


@pytest.mark.parametrize("dh,dims,halves", [(256, (130,), 0), (256, (4, 64, 64), 1), (256, (2, 2), 1), (132, (66, 66), 1),
                                            (130, (128,), 0), (130, (128,), 1)])
def test_wide_heads_off_vectors_are_refused(dh, dims, halves):
    with pytest.raises(_lib.Unsupported, match="alignment"):
        rope(Dh=dh, ids_sl=len(dims), dims=dims, halves=halves)


@pytest.mark.gpu
@pytest.mark.parametrize("dh,axes", [(256, (4, 64, 64)), (256, (132,)), (256, (2, 2)), (256, (252,)), (132, (2, 6, 4)),
                                     (136, (66, 66)), (128, (6, 4, 2)), (128, (124,)), (72, (12, 12, 12)), (20, (6, 6)),
                                     (12, (12,)), (4, (4,)), (8, (2, 2)), (64, (0, 28, 0))])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("norm", [False, True])
def test_adjacent_pairs(dev, dh, axes, dtype, norm):
    b, l, h, hk = 2, 37, 3, 1
    q, k, v = normal((b, h, l, dh), 1, 2, dtype), normal((b, hk, l, dh), 2, 1, dtype), normal((b, hk, l, dh), 3, 1, dtype)
    ids = grid(b, l, len(axes), 4)
    qs, ks = (normal((dh,), 5, 0.2, mean=1.0), normal((dh,), 6, 0.2, mean=1.0)) if norm else (None, None)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = rope_qk(to(q), to(k), to(ids), axes, v=to(v), q_scale=to(qs), k_scale=to(ks))
    assert torch.equal(y[2].cpu(), v)
    check(y[0], reference(q, qs, ids, axes, 10000.0, "interleaved", False))
    check(y[1], reference(k, ks, ids, axes, 10000.0, "interleaved", False))
    # In place, in a buffer whose other elements stay: vectors and single elements (an odd start) give one result.
    if norm:
        return
    for at in (8, 1):
        if dh > 128 and at == 1:
            with pytest.raises(_lib.Unsupported, match="alignment"):
                buf = torch.zeros(b * h * l * dh + 16, dtype=dtype, device=dev)
                rope_qk(buf[at:at + q.numel()].view(q.shape), to(k), to(ids), axes)
            continue
        buf = torch.full((q.numel() + 16,), 5.0, dtype=dtype, device=dev)
        x = buf[at:at + q.numel()].view(q.shape)
        x.copy_(q)
        kk = to(k)
        rope_qk(x, kk, to(ids), axes, out=(x, kk))
        assert torch.equal(x, y[0]) and torch.equal(kk, y[1])
        assert bool((buf[:at] == 5.0).all()) and bool((buf[at + q.numel():] == 5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_channels_that_are_not_turned_keep_what_is_not_finite(dev, dtype):
    # 12 of 20 channels turned: the third vector's unit also holds the first vector that is not.
    q = normal((1, 2, 9, 20), 1, 1, dtype)
    q[..., 12], q[..., 14], q[..., 19] = float("inf"), float("nan"), float("-inf")
    y = rope_qk(q.to(dev), q.to(dev), grid(1, 9, 1, 2).to(dev), (12,))[0].cpu()
    assert bool(y[..., :12].isfinite().all())
    for c in (13, 15, 16, 17, 18):
        assert torch.equal(y[..., c], q[..., c])
    assert torch.equal(y[..., 12], q[..., 12]) and torch.equal(y[..., 19], q[..., 19]) and bool(y[..., 14].isnan().all())
