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


def may_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors (non-negative strides) may share an element. False for address ranges apart, and for two
    [B, heads, L, Dh] tensors at different columns of one matrix of rows: the q, k and v of one linear's output."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size = a.element_size()
    ends = [t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            for t in (a, b)]
    if ends[0] <= b.data_ptr() or ends[1] <= a.data_ptr():
        return False
    if a.dim() != 4 or b.dim() != 4 or b.element_size() != size:
        return True
    row, gap = a.stride(2), b.data_ptr() - a.data_ptr()
    if (row <= 0 or row != b.stride(2) or a.stride(0) != b.stride(0) or gap % size
            or (a.shape[0] > 1 or b.shape[0] > 1) and a.stride(0) % row):
        return True
    # Each tensor keeps to columns [at, at + width) of every row, counted from a's first.
    width = [(t.shape[1] - 1) * t.stride(1) + (t.shape[3] - 1) * t.stride(3) + 1 for t in (a, b)]
    at = gap // size % row
    return not (width[0] <= at and at + width[1] <= row)


def same_elements(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors are the same view: element for element at the same address."""
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype
