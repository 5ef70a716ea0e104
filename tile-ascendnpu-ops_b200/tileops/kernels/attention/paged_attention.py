"""Paged-cache kernels: appending keys and values, attention of one new token.

Shims over ``tileops_paged_kv_append`` (``csrc/rotary.cu``) and
``tileops_paged_decode_fwd`` (``csrc/paged_attention.cu``).  A cache is
``(pages, page_size, heads_kv, dim)`` with contiguous channels and any other
strides: a head-major one, ``(pages, heads_kv, page_size, dim)``, is its
transposed view.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from tileops import _native
from tileops.kernels.attention.rotary_embedding import (
    channels_last,
    check_rotation,
    dense_like,
    overlaps,
    turns_array,
)
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["PagedAttentionDecodeKernel", "PagedKVAppendKernel"]

_KEPT = 64  # layouts an op keeps the stride arrays of


def _keep(kept: dict, key, made):
    if len(kept) >= _KEPT:
        kept.clear()
    kept[key] = made
    return made


class PagedKVAppendKernel(Kernel):
    """New tokens into a paged cache, keys (and queries) rotated on the way.

    Args:
        heads_kv, dim, page_size: the cache's.
        heads: query heads that are rotated beside (0: none).
        rotary_dim, interleaved, frequencies, amplitude: as in the rotary kernels.
        dtype: float32, float16 or bfloat16.
        config: Optional config dict (no tunables).
    """

    SUPPORTED_DTYPES = (torch.float32, torch.float16, torch.bfloat16)

    def __init__(self, heads_kv: int, dim: int, page_size: int, heads: int, rotary_dim: int,
                 interleaved: bool, frequencies: Sequence[float], amplitude: float = 1.0,
                 dtype: torch.dtype = torch.bfloat16, config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if (not 1 <= heads_kv <= 4096 or not 0 <= heads <= 4096 or not 1 <= dim <= 4096
                or not 1 <= page_size < 2**31):
            raise ValueError(f"{type(self).__name__} supports heads_kv 1..4096, heads 0..4096, dim "
                             f"1..4096 and page_size 1..2^31 - 1, got ({heads_kv}, {heads}, {dim}, "
                             f"{page_size})")
        check_rotation(type(self).__name__, dim, rotary_dim, frequencies, amplitude)
        self.heads, self.heads_kv, self.dim, self.page_size = heads, heads_kv, dim, page_size
        self.rotary_dim, self.interleaved = rotary_dim, bool(interleaved)
        self.amplitude = float(amplitude)
        self.dtype = dtype
        self._code = _native.dtype_code(dtype)
        self._turns = turns_array(frequencies)
        self._strides: dict = {}
        self.init_config(config)

    def _layout(self, k_cache, v_cache):
        """The caches' strides; refuses caches whose slots share memory."""
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if c.stride(-1) != 1 and c.shape[-1] > 1:
                raise ValueError(f"{name} must have contiguous channels, got strides {c.stride()}")
            if overlaps(c.shape, c.stride()):
                raise ValueError(f"{name} has slots that share memory: shape {tuple(c.shape)}, "
                                 f"strides {c.stride()}")
        return k_cache.stride()[:3] + v_cache.stride()[:3]

    def forward(self, k, v, k_cache, v_cache, page_table, seq_lens, q=None, cu_seqlens=None):
        """Write the caches; return the rotated queries (None without ``q``)."""
        k, v = channels_last(k), channels_last(v)
        q = None if q is None else channels_last(q)
        if page_table.stride(-1) != 1:
            page_table = page_table.contiguous()
        if seq_lens.stride(0) != 1:
            seq_lens = seq_lens.contiguous()
        if cu_seqlens is not None and cu_seqlens.stride(0) != 1:
            cu_seqlens = cu_seqlens.contiguous()
        q_out = None if q is None else dense_like(q)
        key = (k.stride(), v.stride(), k_cache.stride(), v_cache.stride(), k_cache.shape[0],
               None if q is None else q.stride(), cu_seqlens is None)
        strides = self._strides.get(key)
        if strides is None:
            values = []
            for t in (q, k, v, q_out):
                s = (0, 0, 0) if t is None else t.stride()[:-1]
                if len(s) == 2:  # rows of packed sequences, or one token each
                    s = (s[0], 0, s[1]) if cu_seqlens is None else (0, s[0], s[1])
                values += s
            values += self._layout(k_cache, v_cache)
            strides = _keep(self._strides, key, (ctypes.c_int64 * 18)(*values))
        tokens = k.shape[0] if k.dim() == 3 else k.shape[0] * k.shape[1]
        _native.launch(
            "tileops_paged_kv_append", k.device, _native.data_ptr(q), k.data_ptr(), v.data_ptr(),
            _native.data_ptr(q_out), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
            seq_lens.data_ptr(), _native.data_ptr(cu_seqlens), self._turns, seq_lens.shape[0],
            tokens, 0 if q is None else self.heads, self.heads_kv, self.dim, self.rotary_dim,
            k_cache.shape[0], self.page_size, page_table.shape[1], page_table.stride(0), strides,
            self.interleaved, self.amplitude, self._code)
        return q_out


class PagedAttentionDecodeKernel(Kernel):
    """Attention of one new token of every sequence over a paged cache.

    Args:
        heads, heads_kv, dim, page_size: problem shape.
        scale: factor on the scores.
        window: tokens a query sees, the last ones (0: all).
        dtype: float16 or bfloat16.
        config: Optional config dict (no tunables).
    """

    SUPPORTED_DTYPES = (torch.float16, torch.bfloat16)

    def __init__(self, heads: int, heads_kv: int, dim: int, page_size: int, scale: float,
                 window: int = 0, dtype: torch.dtype = torch.bfloat16,
                 config: Optional[dict] = None):
        super().__init__()
        check_dtype(self, dtype, self.SUPPORTED_DTYPES)
        if (not 1 <= heads <= 4096 or heads_kv < 1 or heads % heads_kv or not 8 <= dim <= 256
                or dim % 8 or not 1 <= page_size < 2**31 - 64):
            raise ValueError(f"{type(self).__name__} supports up to 4096 heads in groups of "
                             f"heads / heads_kv, dim a multiple of 8 up to 256 and page_size 1..2^31 "
                             f"- 65, got ({heads}, {heads_kv}, {dim}, {page_size})")
        if not abs(scale) <= 2.0**100:
            raise ValueError(f"scale must be finite and at most 2^100, got {scale}")
        if not 0 <= window < 2**31:
            raise ValueError(f"window must be at least 1 token and below 2^31, got {window}")
        self.heads, self.heads_kv, self.dim, self.page_size = heads, heads_kv, dim, page_size
        self.scale, self.window = float(scale), int(window)
        self.dtype = dtype
        self._code = _native.dtype_code(dtype)
        self._ws_bytes: Optional[int] = None
        self._strides: dict = {}
        self.init_config(config)

    def _layout(self, q, k_cache, v_cache):
        """Strides of q and the caches, multiples of 16 bytes (copies are never made of a cache)."""
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if c.stride(-1) != 1 or any(s % 8 for s, n in zip(c.stride()[:3], c.shape) if n > 1):
                raise ValueError(f"{name} must have contiguous channels and strides that are "
                                 f"multiples of 8, got {c.stride()}")
        strides = [*q.stride()[:2]]
        for c in (k_cache, v_cache):  # what a single page, slot or head is apart has no say
            strides += [s if n > 1 else 0 for s, n in zip(c.stride()[:3], c.shape)]
        return (ctypes.c_int64 * 8)(*strides)

    def forward(self, q, k_cache, v_cache, page_table, seq_lens):
        """Return ``(o, lse)``."""
        dev = q.device
        if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
        if page_table.stride(-1) != 1:
            page_table = page_table.contiguous()
        if seq_lens.stride(0) != 1:
            seq_lens = seq_lens.contiguous()
        key = (q.stride(), k_cache.stride(), v_cache.stride(), k_cache.shape[0])
        strides = self._strides.get(key)
        if strides is None:
            strides = _keep(self._strides, key, self._layout(q, k_cache, v_cache))
        if self._ws_bytes is None:
            self._ws_bytes = _native.lib().tileops_paged_decode_workspace_bytes(
                self.heads, self.heads_kv, self.dim)
        o = dense_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
        ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=dev)
        _native.launch(
            "tileops_paged_decode_fwd", dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            page_table.data_ptr(), seq_lens.data_ptr(), o.data_ptr(), lse.data_ptr(), ws.data_ptr(),
            q.shape[0], self.heads, self.heads_kv, self.dim, k_cache.shape[0], self.page_size,
            page_table.shape[1], page_table.stride(0), strides, self.window, self.scale, self._code)
        return o, lse
