"""Whether tensors share memory: the assertions behind the native front ends, which decide the same way (csrc/memory_regions.h)."""
from __future__ import annotations

import torch


def apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors that are not empty are shown to share no byte: they lie in ranges of memory apart from each other, or, modulo one of
    their strides, in ranges apart (slices of the columns of one wide buffer).  Interleaved in another way they count as overlapping."""

    def dims(t):
        return [(n, s * t.element_size()) for n, s in zip(t.shape, t.stride()) if n > 1]

    def span(t, modulus=0):
        return t.element_size() + sum((n - 1) * s for n, s in dims(t) if modulus == 0 or s % modulus != 0)

    x, y = a.data_ptr(), b.data_ptr()
    if x + span(a) <= y or y + span(b) <= x:
        return True
    for _, m in dims(a) + dims(b):
        if m > 0 and span(a, m) <= (y - x) % m <= m - span(b, m):
            return True
    return False


def rows_apart(t: torch.Tensor) -> bool:
    """Whether no two elements of [tokens, heads] or [tokens, heads, row], the last of unit stride, share memory: one of the two outer strides
    spans the other dimension's rows."""
    row = t.shape[2] if t.dim() == 3 else 1
    (n0, n1), (s0, s1) = t.shape[:2], t.stride()[:2]
    return (n1 == 1 or s1 >= row) and (n0 == 1 or s0 >= row) and (n0 == 1 or n1 == 1 or s0 >= (n1 - 1) * s1 + row or s1 >= (n0 - 1) * s0 + row)
