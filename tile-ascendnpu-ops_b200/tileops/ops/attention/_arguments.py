"""Argument checks of the rotary and paged-cache ops."""

from __future__ import annotations

import torch

from tileops.device import get_device_backend

__all__ = ["check_tensor"]


def check_tensor(device: torch.device, name: str, t: torch.Tensor, shape: tuple,
                 dtype: torch.dtype) -> None:
    """Raise unless ``t`` is a device tensor on ``device`` of this shape and type."""
    backend = get_device_backend()
    if not backend.is_device_tensor(t):
        raise ValueError(f"{name} must be a {backend.name} tensor, "
                         f"got {getattr(t, 'device', type(t).__name__)}")
    if t.device != device:
        raise ValueError(f"Expected {name} on {device}, got {t.device}")
    if t.shape != shape:
        raise ValueError(f"Expected {name}.shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"Expected {name}.dtype {dtype}, got {t.dtype}")
