"""Rotary positions with several axes (time, row, column) as a gfx950 kernel.

The segments ``Kernels.qkv_single`` and ``qkv_double`` take cos/sin tables that all images of a batch share
(selas/models/flux.py:106-121, 179-191). ``rope_qk`` takes the positions themselves, [L, axes] or one set per
image, [B, L, axes]: grids of other shapes or offsets in one batch, clips with a time axis, heads that are only
partly rotated, k with fewer heads than q, and pairs of adjacent channels or of the two halves. The norm of the
heads that precedes the rotation (flux.py:124-126) and the layout of v run in the same pass.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from ._layout import distinct, may_meet, same_elements

PAIRS = ("interleaved", "halves")
_ID_CODES = {torch.float32: _lib.F32, torch.int32: _lib.I32, torch.int64: _lib.I64}


def _check_heads(name: str, t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if t.dim() != 4:
        raise ValueError(f"rope_qk: {name} must be [B, heads, L, Dh], got shape {tuple(t.shape)}")
    if t.shape[0] != like.shape[0] or t.shape[2:] != like.shape[2:] or t.dtype != like.dtype:
        raise ValueError(f"rope_qk: {name} {tuple(t.shape)} {t.dtype} does not go with q {tuple(like.shape)} "
                         f"{like.dtype}")
    return t if t.shape[3] == 1 or t.stride(3) == 1 else t.contiguous()


def _check_scale(name: str, s: torch.Tensor | None, dh: int) -> torch.Tensor | None:
    if s is None:
        return None
    if s.numel() != dh:
        raise ValueError(f"rope_qk: {name} has {s.numel()} values, head_dim is {dh}")
    if s.dtype != torch.float32 or not s.is_contiguous():
        s = s.float().contiguous()
    return s


def rope_qk(q: torch.Tensor, k: torch.Tensor, ids: torch.Tensor, axes_dim, theta: float = 10000.0, *,
            v: torch.Tensor | None = None, q_scale: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
            pairs: str = "interleaved", inverse: bool = False, out=None) -> tuple[torch.Tensor, ...]:
    """(q, k) or (q, k, v), turned by the positions: [B, heads, L, Dh], contiguous unless ``out`` is given.

    q [B, H, L, Dh] and k, v [B, Hk, L, Dh] (bf16, fp16 or fp32) may have any strides, such as views of one
    linear's output. ``ids``: [L, axes] or [B, L, axes] (B or 1), fp32, int32 or int64. Axis a owns
    axes_dim[a] channels (even); its pair j turns by ``ids[..., a] * theta ** (-2 j / axes_dim[a])``. The pairs of
    the axes follow each other: pair i is channels (2 i, 2 i + 1), or (i, i + sum(axes_dim) / 2) with
    ``pairs="halves"``; channels past sum(axes_dim) are not turned. ``q_scale``, ``k_scale`` [Dh]: RMS norm
    (eps 1e-6) of each head and its scale ahead of the rotation. v is only laid out. ``inverse`` turns by the
    negative angles, which is the gradient of a rotation (without norms). Angles are formed in fp64, the
    arithmetic is fp32 with one rounding.

    ``out``: destinations (q_out, k_out[, v_out]) of the same shapes with unit channel stride; a tensor may be its
    own destination, any other overlap is refused. Heads above 256 channels raise ``Unsupported``, and so
    do those above 128 that are not read in vectors of 4 elements: addresses, strides, Dh and sum(axes_dim) (half of it with
    ``pairs="halves"``) are multiples of 4 elements there."""
    if q.dim() != 4:
        raise ValueError(f"rope_qk: q must be [B, heads, L, Dh], got shape {tuple(q.shape)}")
    if pairs not in PAIRS:
        raise ValueError(f"rope_qk: pairs must be one of {PAIRS}, got {pairs!r}")
    b, _, l, dh = q.shape
    axes = tuple(axes_dim)
    if not 1 <= len(axes) <= _lib.ROPE_MAX_AXES:
        raise ValueError(f"rope_qk: takes 1 to {_lib.ROPE_MAX_AXES} axes, got {len(axes)}")
    dtype = _lib.DTYPE_CODES.get(q.dtype)
    if dtype is None:
        raise _lib.Unsupported(f"rope_qk: dtype {q.dtype}")
    dev = _lib.require_gpu(q, k, v, ids, q_scale, k_scale)
    xs = [_check_heads("q", q, q), _check_heads("k", k, q)]
    if v is not None:
        xs.append(_check_heads("v", v, q))
    lead = ids.shape[:-2]
    if (ids.dim() not in (2, 3) or ids.shape[-1] != len(axes) or ids.shape[-2] != l
            or (len(lead) == 1 and lead[0] not in (1, b))):
        raise ValueError(f"rope_qk: positions {tuple(ids.shape)} are not [{l}, {len(axes)}] or [{b}, {l}, {len(axes)}]")
    id_code = _ID_CODES.get(ids.dtype)
    if id_code is None:
        raise ValueError(f"rope_qk: positions are float32, int32 or int64, got {ids.dtype}")
    if ids.stride(-1) != 1 and len(axes) > 1:
        ids = ids.contiguous()
    ids_sb = ids.stride(0) if lead and lead[0] > 1 else 0
    scales = (_check_scale("q_scale", q_scale, dh), _check_scale("k_scale", k_scale, dh), None)
    if out is None:
        ys = [t.new_empty(t.shape) for t in xs]
    else:
        ys = list(out)
        _check_out(xs, ys, dev, [t for t in (ids, *scales) if t is not None])
    parts = b"".join([_lib.ROPE_PART.pack(x.data_ptr(), *x.stride()[:3], y.data_ptr(), *y.stride()[:3],
                                          0 if scale is None else scale.data_ptr(), x.shape[1], i < 2)
                      for i, (x, y, scale) in enumerate(zip(xs, ys, scales))])
    with _lib.on(dev):
        _lib.call("selas_rope", parts, len(xs), b, l, dh, ids.data_ptr(), id_code, ids_sb, ids.stride(-2), len(axes),
                  struct.pack(f"@{len(axes)}q", *axes), float(theta), pairs == "halves", bool(inverse), dtype,
                  _lib.stream(dev))
    return tuple(ys)


def _check_out(xs, ys, dev, read) -> None:
    if len(ys) != len(xs):
        raise ValueError(f"rope_qk: out has {len(ys)} tensors for {len(xs)}")
    for i, (x, y) in enumerate(zip(xs, ys)):
        if y.shape != x.shape or y.dtype != x.dtype or y.device != dev or (y.shape[3] > 1 and y.stride(3) != 1):
            raise ValueError(f"rope_qk: out[{i}] must be {tuple(x.shape)} {x.dtype} on {dev} with unit channel stride, "
                             f"got {tuple(y.shape)} {y.dtype} strides {y.stride()}")
        if not distinct(y):
            raise ValueError(f"rope_qk: out[{i}] has elements at one address (strides {y.stride()})")
        others = [t for j, t in enumerate(xs) if j != i or not same_elements(x, y)]
        others += [t for j, t in enumerate(ys) if j != i] + read
        if any(may_meet(y, t) for t in others):
            raise ValueError(f"rope_qk: out[{i}] overlaps another tensor of the call")
