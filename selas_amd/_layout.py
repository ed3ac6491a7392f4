"""Whether tensors given as destinations may be written while a launch reads or writes others."""

from __future__ import annotations

import torch


def distinct(t: torch.Tensor) -> bool:
    """Whether the elements of a tensor are at addresses of their own (no broadcast or folded dimension)."""
    span = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda d: d[1]):
        if size > 1:
            if stride < span:
                return False
            span += (size - 1) * stride
    return True


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """A tensor of at most four dims as [B, heads, L, C]."""
    if t.dim() == 3:
        return t.unsqueeze(1)
    while t.dim() < 4:
        t = t.unsqueeze(0)
    return t


def may_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors (non-negative strides) may share an element. False for address ranges apart, and for two
    [..., L, C] or [B, heads, L, C] tensors at different columns of one matrix of rows: the q, k and v of one linear's
    output, the two halves of a linear's input."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size = a.element_size()
    ends = [t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            for t in (a, b)]
    if ends[0] <= b.data_ptr() or ends[1] <= a.data_ptr():
        return False
    gap = b.data_ptr() - a.data_ptr()
    if a.dim() > 4 or b.dim() > 4 or b.element_size() != size or gap % size:
        return True
    a, b = _as_rows(a), _as_rows(b)
    row = a.stride(2)
    if row <= 0 or row != b.stride(2) or any(t.shape[0] > 1 and t.stride(0) % row for t in (a, b)):
        return True
    # Each tensor keeps to columns [at, at + width) of every row, counted from a's first.
    width = [(t.shape[1] - 1) * t.stride(1) + (t.shape[3] - 1) * t.stride(3) + 1 for t in (a, b)]
    at = gap // size % row
    return not (width[0] <= at and at + width[1] <= row)


def same_elements(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors are the same view: element for element at the same address."""
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
