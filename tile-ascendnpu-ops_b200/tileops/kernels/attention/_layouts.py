"""What the rotary and paged-cache kernels know of their arguments' layouts.

A layout (shapes, strides, types and devices) decides which arguments have to be copied, the strides
that go to the entry point and the shapes of outputs: it is worked out once and kept (the host
spends 0.1 to 0.3 us on each attribute of a tensor that it looks at).
"""

from __future__ import annotations

from typing import Sequence

import torch

__all__ = ["Apart", "Layouts", "NO_PLAN", "channels_last", "layout_of", "overlaps", "plan_of", "row_of"]


def layout_of(*tensors):
    """What of the tensors decides how they are handled; None where one is no (strided) tensor."""
    try:
        return tuple([None if t is None else
                      (t.shape, t.is_contiguous() or t.stride(), t.dtype, t.get_device())
                      for t in tensors])
    except (AttributeError, TypeError, RuntimeError):
        return None


class Layouts(dict):
    """What was worked out for the last layouts."""

    def keep(self, layout, found):
        if layout is not None:
            if len(self) >= 256:
                self.clear()
            self[layout] = found
        return found


NO_PLAN = ()


def plan_of(kernel, *args):
    """What a kernel works out once for a layout; NO_PLAN where the class whose ``forward`` it has (an
    op's override) makes none, since that forward takes the op's arguments only."""
    for cls in type(kernel).__mro__:
        if "forward" in vars(cls):
            return kernel.plan(*args) if "plan" in vars(cls) else NO_PLAN
    return NO_PLAN


def overlaps(shape: Sequence[int], strides: Sequence[int]) -> bool:
    """Whether two indices of a tensor can share an element (never wrongly no)."""
    reach = 0
    for stride, size in sorted((st, n) for st, n in zip(strides, shape) if n > 1):
        if stride <= reach:
            return True
        reach += stride * (size - 1)
    return False


class Apart:
    """Whether two tensors of these layouts share no element, by where they begin; distances that were
    found good are remembered."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor):
        # Element index of a less that of b: a sum of i stride, low <= i <= high, over the strides.
        terms: dict = {}
        for t, sign in ((a, 1), (b, -1)):
            for n, stride in zip(t.shape, t.stride()):
                low, high = terms.get(stride, (0, 0))
                reach = sign * (n - 1)
                terms[stride] = low + min(reach, 0), high + max(reach, 0)
        self.terms = sorted(((s, *r) for s, r in terms.items() if s and any(r)), reverse=True)
        self.ends = [(0, 0)]  # of the sums over the last terms
        for stride, low, high in reversed(self.terms):
            self.ends.insert(0, (self.ends[0][0] + low * stride, self.ends[0][1] + high * stride))
        self.size = a.element_size()
        self.empty = a.numel() == 0 or b.numel() == 0
        self.good: set = set()

    def __call__(self, a_at: int, b_at: int) -> bool:
        distance = b_at - a_at
        if distance in self.good or self.empty:
            return True
        elements, part = divmod(distance, self.size)
        if self._meet(elements, 0) or part and self._meet(elements + 1, 0):
            return False
        if len(self.good) >= 256:
            self.good.clear()
        self.good.add(distance)
        return True

    def _meet(self, distance: int, n: int) -> bool:
        """Whether the terms from the n-th on have this sum.  A stride above the reach of those behind it,
        as in tensors without elements in common, leaves two or three multiples to look at."""
        if n == len(self.terms):
            return distance == 0
        stride, low, high = self.terms[n]
        rest_low, rest_high = self.ends[n + 1]
        first, last = -((rest_high - distance) // stride), (distance - rest_low) // stride
        return any(self._meet(distance - i * stride, n + 1)
                   for i in range(max(first, low), min(last, high) + 1))


def channels_last(t: torch.Tensor) -> bool:
    """Whether a tensor's channels are contiguous."""
    return t.stride(-1) == 1 or t.shape[-1] <= 1


def row_of(t: torch.Tensor) -> torch.Tensor:
    """One element in the shape of ``t``: ``empty_like`` of it is dense, and costs the host half of
    what ``empty`` does."""
    return torch.empty(1, dtype=t.dtype, device=t.device).expand(t.shape)
