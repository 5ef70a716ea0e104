"""What the rotary and paged-cache kernels know of their arguments' layouts.

A layout (shapes, strides, types and devices) decides which arguments have to be copied, the strides
that go to the entry point and the shapes of outputs: it is worked out once and kept (the host
spends 0.1 to 0.3 us on each attribute of a tensor that it looks at).
"""

from __future__ import annotations

from typing import Sequence

import torch

__all__ = ["Layouts", "NO_PLAN", "channels_last", "layout_of", "overlaps", "plan_of", "row_of"]


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


def channels_last(t: torch.Tensor) -> bool:
    """Whether a tensor's channels are contiguous."""
    return t.stride(-1) == 1 or t.shape[-1] <= 1


def row_of(t: torch.Tensor) -> torch.Tensor:
    """One element in the shape of ``t``: ``empty_like`` of it is dense, and costs the host half of
    what ``empty`` does."""
    return torch.empty(1, dtype=t.dtype, device=t.device).expand(t.shape)
