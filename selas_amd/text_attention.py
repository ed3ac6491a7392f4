"""Attention of the text side as gfx950 kernels: what the text encoders run, and what reads their states.

``attention.attention`` is the FLUX blocks' own: q, k and v of one length, no mask. The two here take keys of another
length than the queries, key heads that several query heads share, images or texts whose keys end early (``lengths``) or
are masked (``mask``), head dims of whole 8 up to 128, bf16 and fp16:

``cross_attention``  queries of one stream (image tokens, learned queries) over an encoder's states.
``text_attention``   a text encoder's or decoder's own attention: a learned bias for each head by buckets of the distance
                     between key and query (selas/models/t5.py:66 has one), a causal mask (selas/models/clip.py:34), and
                     ``q_start`` for single tokens over the keys so far.

Each has its gradient as a function of its own, ``cross_attention_backward`` and ``text_attention_backward``; the forward
pass hands it ``lse`` (``return_lse=True``).
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from ._layout import distinct, may_meet

# selas_text_attention_problem (include/selas_amd.h).
_PROBLEM = struct.Struct("@P3qP3qP3qP2qPPPqPqPq8qd4i")
_SIZES = ctypes.c_int64


def _heads(t: torch.Tensor) -> torch.Tensor:
    """t [B, heads, L, Dh] as the kernels read it: unit channel stride, rows of whole 16 bytes at aligned addresses."""
    sb, sh, sl, sc = t.stride()
    if sc != 1 or (sb | sh | sl) & 7 or sl > 1 << 23 or t.data_ptr() & 15:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _no_graph(what: str, *ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} records no graph: call it under torch.no_grad() and take the gradients from "
                                 f"{what}_backward")


def _per_image(what: str, name: str, t: torch.Tensor, b: int, hi: int) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64) or t.shape != (b,):
        raise ValueError(f"{what}: {name} must be int32 or int64 [{b}], got {t.dtype} {tuple(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(-hi, hi).to(torch.int32)
    return t if b <= 1 or t.stride(0) == 1 else t.contiguous()


class _Call:
    """The checked arguments of a call: `problem` fills the C structure with given outputs."""

    def __init__(self, what, q, k, v, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale):
        if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
            raise ValueError(f"{what}: q, k and v are [B, heads, L, Dh], got {tuple(q.shape)}, {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
        b, h, lq, dh = q.shape
        hk, lk = k.shape[1], k.shape[2]
        if k.shape != v.shape or k.shape[0] != b or k.shape[3] != dh or (h % hk if hk else h):
            raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} do not go with q {tuple(q.shape)}")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError(f"{what}: q {q.dtype}, k {k.dtype} and v {v.dtype} must have one type")
        dev = self.dev = q.device
        if not q.is_cuda or k.device != dev or v.device != dev or table is not None or lengths is not None or mask is not None:
            _lib.require_gpu(q, k, v, table, lengths, mask)
        dtype = _lib.DTYPE_CODES.get(q.dtype)
        if dtype is None or dtype == _lib.F32:
            raise _lib.Unsupported(f"{what}: takes bf16 or fp16, got {q.dtype}")
        if dh % 8 or dh > 128:
            raise _lib.Unsupported(f"{what}: takes head dims of whole 8 up to 128, got {dh}")
        self.dtype, self.shape = dtype, (b, h, hk, lq, lk, dh)
        self.q, self.k, self.v = _heads(q), _heads(k), _heads(v)
        self.lengths = None if lengths is None else _per_image(what, "lengths", lengths, b, lk)
        if mask is not None:
            if mask.dtype != torch.bool or mask.dim() != 2 or mask.shape[1] != lk or mask.shape[0] not in (1, b):
                raise ValueError(f"{what}: mask must be bool [{b}, {lk}] (True: the key is seen), got {mask.dtype} "
                                 f"{tuple(mask.shape)}")
            if lk > 1 and mask.stride(1) != 1:
                mask = mask.contiguous()
        self.mask = mask
        self.start, start0 = None, 0
        if isinstance(q_start, torch.Tensor):
            _lib.require_gpu(q, q_start)
            self.start = _per_image(what, "q_start", q_start, b, 1 << 29)
        else:
            start0 = int(q_start)
            if abs(start0) > 1 << 29:
                raise ValueError(f"{what}: q_start {start0} is outside +-2^29")
        self.table, table_row, table_type, buckets = None, 0, 0, 0
        if table is not None:
            if table.dim() != 2 or table.shape[1] != h:
                raise ValueError(f"{what}: the table must be [buckets, {h}], got {tuple(table.shape)}")
            table_type, buckets = _lib.dtype_code(table.dtype), table.shape[0]
            if not buckets:
                raise ValueError(f"{what}: the table has no buckets")
            if h > 1 and table.stride(1) != 1:
                table = table.contiguous()
            self.table, table_row = table, table.stride(0)
        q, k, v, (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _) = (self.q, self.k, self.v, self.q.stride(), self.k.stride(),
                                                                     self.v.stride())
        self._head = (q.data_ptr(), q0, q1, q2, k.data_ptr(), k0, k1, k2, v.data_ptr(), v0, v1, v2)
        self._tail = (0 if lengths is None else self.lengths.data_ptr(), 0 if mask is None else mask.data_ptr(),
                      0 if mask is None or mask.shape[0] == 1 else mask.stride(0),
                      0 if self.start is None else self.start.data_ptr(), start0, 0 if table is None else table.data_ptr(),
                      table_row, b, h, hk, lq, lk, dh, buckets, int(max_distance),
                      dh ** -0.5 if scale is None else float(scale), table_type, bool(bidirectional), bool(causal), 0)

    def problem(self, out, lse) -> bytes:
        o0, o1, _ = out.stride()
        return _PROBLEM.pack(*self._head, out.data_ptr(), o0, o1, 0 if lse is None else lse.data_ptr(), *self._tail)

    def reads(self):
        return [t for t in (self.q, self.k, self.v, self.lengths, self.mask, self.start, self.table) if t is not None]


def _forward(what, q, k, v, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale, out, return_lse):
    _no_graph(what, q, k, v, table)
    call = _Call(what, q, k, v, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale)
    b, h, _, lq, _, dh = call.shape
    if out is None:
        out = torch.empty(b, lq, h * dh, dtype=q.dtype, device=call.dev)
    else:
        if (out.shape != (b, lq, h * dh) or out.dtype != q.dtype or out.device != call.dev
                or (h * dh > 1 and out.stride(2) != 1) or (b > 1 and out.stride(0) & 3) or (lq > 1 and out.stride(1) & 3)
                or out.data_ptr() & 7):
            raise ValueError(f"{what}: out must be [{b}, {lq}, {h * dh}] {q.dtype} on {call.dev} with unit column stride and "
                             f"rows of whole 8 bytes, got {tuple(out.shape)} {out.dtype} strides {out.stride()}")
        if not distinct(out):
            raise ValueError(f"{what}: out has elements at one address (strides {out.stride()})")
        if any(may_meet(out, t) for t in call.reads()):
            raise ValueError(f"{what}: out overlaps another tensor of the call")
    lse = torch.empty(b, h, lq, dtype=torch.float32, device=call.dev) if return_lse else None
    problem, size = call.problem(out, lse), _SIZES()
    with _lib.on(call.dev):
        _lib.call("selas_text_attention_workspace_bytes", problem, call.dtype, ctypes.byref(size))
        n = size.value
        ws = torch.empty(n, dtype=torch.uint8, device=call.dev) if n else None
        _lib.call("selas_text_attention", problem, call.dtype, _lib.ptr(ws), n, _lib.stream(call.dev))
    return (out, lse) if return_lse else out


def _backward(what, grad, q, k, v, out, lse, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale):
    call = _Call(what, q, k, v, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale)
    b, h, hk, lq, lk, dh = call.shape
    _lib.require_gpu(q, grad, out, lse)
    for name, t in (("grad", grad), ("out", out)):
        if t.shape != (b, lq, h * dh) or t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} must be [{b}, {lq}, {h * dh}] {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if lse.shape != (b, h, lq) or lse.dtype != torch.float32:
        raise ValueError(f"{what}: lse must be float32 [{b}, {h}, {lq}], got {lse.dtype} {tuple(lse.shape)}")
    s = grad.stride()
    if s[2] != 1 or (s[0] | s[1]) & 7 or s[1] > 1 << 23 or grad.data_ptr() & 15:
        grad = grad.clone(memory_format=torch.contiguous_format)
    s = out.stride()
    if s[2] != 1 or (s[0] | s[1]) & 3 or out.data_ptr() & 7:
        out = out.clone(memory_format=torch.contiguous_format)
    lse = lse.contiguous()
    dq = torch.empty(b, h, lq, dh, dtype=q.dtype, device=call.dev)
    dk, dv = (torch.empty(b, hk, lk, dh, dtype=q.dtype, device=call.dev) for _ in range(2))
    dtable = None if table is None else torch.empty(table.shape, dtype=table.dtype, device=call.dev)
    problem, size = call.problem(out, lse), _SIZES()
    with _lib.on(call.dev):
        _lib.call("selas_text_attention_backward_workspace_bytes", problem, call.dtype, ctypes.byref(size))
        n = size.value
        ws = torch.empty(n, dtype=torch.uint8, device=call.dev) if n else None
        _lib.call("selas_text_attention_backward", problem, grad.data_ptr(), grad.stride(0), grad.stride(1), dq.data_ptr(),
                  dk.data_ptr(), dv.data_ptr(), _lib.ptr(dtable), call.dtype, _lib.ptr(ws), n, _lib.stream(call.dev))
    return dq, dk, dv, dtable


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, lengths: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                    return_lse: bool = False):
    """softmax(scale q k^T) v for q [B, H, Lq, Dh] over k, v [B, Hk, Lk, Dh] -> [B, Lq, H * Dh], and with ``return_lse``
    the fp32 logarithms of the rows' sums [B, H, Lq].

    H is a multiple of Hk: query head h reads key head h // (H // Hk). Any strides (views of linears' outputs); what the
    kernels cannot read in 16-byte chunks is copied first. ``lengths`` [B] (int32, int64): image b has its first lengths[b]
    keys. ``mask`` [B, Lk] or [1, Lk] (bool): True where the key is seen. What keys that no query sees hold does not
    matter, NaN included; a query that sees none gets zeros and an lse of -inf. ``scale``: 1 / sqrt(Dh) unless given.
    ``out``: optional destination with unit column stride and rows of whole 8 bytes, overlapping nothing the call reads.

    bf16 or fp16, Dh of whole 8 up to 128, otherwise ``Unsupported``. Scores, maxima and sums are fp32
    (scores are to stay below 10^7 in magnitude, where fp32 holds little more than whole numbers), the probabilities are
    rounded to the type for the product with v. No graph is recorded: tensors that require grad are refused outside
    torch.no_grad(), and ``cross_attention_backward`` gives the gradients."""
    return _forward("cross_attention", q, k, v, None, 0, True, False, 0, lengths, mask, scale, out, return_lse)


def text_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor | None = None, *,
                   max_distance: int = 128, bidirectional: bool = True, causal: bool = False,
                   q_start: int | torch.Tensor = 0, lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """``cross_attention`` with positions: key j is at j, query i of image b at q_start (one for all, or [B]) + i.

    ``table`` [buckets, H] (bf16, fp16 or fp32): a learned bias, table[bucket(j - position), h], is added to the scaled
    score. With n buckets a direction (half of them each with ``bidirectional``; otherwise all of them for the keys before
    the query, and bucket 0 for those after it) distance a has bucket a below n // 2, and above it
    n // 2 + floor((n - n // 2) log(a / (n // 2)) / log(max_distance / (n // 2))), at most n - 1; keys after the query
    have the second half. Distances are compared in exact arithmetic. 2 to 128 buckets a direction, max_distance up to 512.
    An entry of -inf leaves its keys no weight; finite ones beyond +-2^17 count as +-2^17, which leaves a key no weight
    beside others, and weights by their products to keys that all have it.
    ``causal``: a query sees the keys up to its own position (a NaN in the value of a key that later queries see reaches
    the earlier ones too, as in a product with weights of 0). For one more token over a cache give q [B, H, 1, Dh],
    ``lengths`` and ``q_start = lengths - 1`` (int32: no conversion)."""
    return _forward("text_attention", q, k, v, table, max_distance, bidirectional, causal, q_start, lengths, mask, scale, out,
                    return_lse)


def cross_attention_backward(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, *, lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                             scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv), contiguous and in the type of q, for ``grad`` [B, Lq, H * Dh], the gradient of ``cross_attention``'s
    output; ``out`` and ``lse`` are what that call returned, the other arguments what it was given.

    Each is the gradient of the tensor as given: dk and dv are summed over the query heads that share a key head; a
    broadcast input (an expanded batch) still has its own sum to take. Keys that are not seen and queries that see none
    (by ``lengths``, ``mask`` or a causal mask) have zeros, and what they and their rows of ``grad`` hold does not matter.
    Sums are fp32 in one order: equal calls give equal bits."""
    return _backward("cross_attention_backward", grad, q, k, v, out, lse, None, 0, True, False, 0, lengths, mask, scale)[:3]


def text_attention_backward(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                            lse: torch.Tensor, table: torch.Tensor | None = None, *, max_distance: int = 128,
                            bidirectional: bool = True, causal: bool = False, q_start: int | torch.Tensor = 0,
                            lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                            scale: float | None = None):
    """(dq, dk, dv, dtable) of ``text_attention``, as in ``cross_attention_backward``. dtable [buckets, H] is in the table's
    type, summed in fp32 over images, queries and keys; None without a table."""
    return _backward("text_attention_backward", grad, q, k, v, out, lse, table, max_distance, bidirectional, causal, q_start,
                     lengths, mask, scale)
