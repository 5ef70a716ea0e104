"""Paged-cache ops: appending keys and values, attention of one new token.

A cache is (num_pages, page_size, heads_kv, dim) of ``dtype`` with contiguous channels and any
other strides (a head-major one, (num_pages, heads_kv, page_size, dim), is passed as its
``transpose(1, 2)``; one without pages, (batch, length, heads_kv, dim), as pages of ``length``
with the table ``arange(batch)[:, None]``).  Token p of sequence b lies in slot p % page_size of
page ``page_table[b, p // page_size]``; table entries behind a sequence's end are not read.
page_table (batch, columns) and seq_lens (batch,) are int32 and stay on the device.

    PagedKVAppendOp(heads_kv, dim, page_size, heads=0, rotary_dim=0, interleaved=False,
                    frequencies=None, amplitude=1.0, dtype=torch.bfloat16, kernel_map=None)
    forward(k, v, k_cache, v_cache, page_table, seq_lens, q=None, cu_seqlens=None) -> q_out or None

Writes each sequence's new tokens, its last ones (``seq_lens``: lengths after the call), into the
caches, keys rotated by their positions as by RotaryEmbeddingFwdOp, and returns the queries
rotated likewise.  k, v (and q): (batch, heads, dim), one token a sequence; (batch, tokens, heads,
dim); or packed (tokens, heads, dim) with ``cu_seqlens``, batch + 1 int32 offsets 0, ..., at most
tokens.  Token i of n has position seq_lens[b] - n + i; one of a negative position is padding, as
are packed rows behind the last sequence: zeros in q_out, nothing in the caches.  No two rows may
have the same slot.

    PagedAttentionDecodeOp(heads, heads_kv, dim, page_size, scale=None, window=None,
                           dtype=torch.bfloat16, kernel_map=None)
    forward(q, k_cache, v_cache, page_table, seq_lens) -> (o, lse)

q, o (batch, heads, dim); query head h reads key head h // (heads // heads_kv).  The query is
sequence b's token seq_lens[b] - 1 and sees the tokens up to it, the last ``window`` of them if
given.  lse (batch, heads) float32 is in the log2 domain, as MultiHeadAttentionFwdOp's.  A
sequence without a token has o = 0 and lse = -inf.  Caches 16-byte aligned, their strides
multiples of 8.  Softmax statistics and sums are fp32; the weights meet the values as numbers of
``dtype``, with what those round off beside them where heads // heads_kv is at most 8.

Offsets that break their rule set the device error flag to 2; a token in use without a page in
[0, num_pages) sets it to 3 (its slot is not written, its key and value count as zeros), as does a
length that the table has no room for (attention takes it as the table's room).  Caches that share
an element are refused; k, v and q may not lie in slots that the call writes.  A
device's first call looks that flag up: make it outside a graph's capture.  The decode op keeps a
workspace of some MB for each of torch's streams that it is called on; captured calls and those on
other streams have their own.
"""

from __future__ import annotations

from typing import Dict, Optional, Sequence

import torch

from tileops.device import get_device_backend
from tileops.kernels.attention import PagedAttentionDecodeKernel, PagedKVAppendKernel
from tileops.kernels.attention._layouts import NO_PLAN, Layouts, layout_of, plan_of
from tileops.kernels.kernel_base import Kernel
from tileops.ops.attention._arguments import check_tensor
from tileops.ops.attention.rotary_embedding import rotary_frequencies
from tileops.ops.op_base import Op

__all__ = ["PagedAttentionDecodeOp", "PagedKVAppendOp"]


def _check_cache(dev, k_cache, v_cache, page_table, seq_lens, batch: int, slot: tuple,
                 dtype: torch.dtype) -> None:
    on_device = get_device_backend().is_device_tensor
    for name, t, dims in (("k_cache", k_cache, 4), ("page_table", page_table, 2)):
        if on_device(t) and t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    pages = k_cache.shape[0] if on_device(k_cache) else 0
    check_tensor(dev, "k_cache", k_cache, (pages, *slot), dtype)
    check_tensor(dev, "v_cache", v_cache, (pages, *slot), dtype)
    if not 1 <= pages < 2**31:
        raise ValueError(f"the cache must have between 1 and 2^31 - 1 pages, got {pages}")
    columns = page_table.shape[1] if on_device(page_table) else 0
    check_tensor(dev, "page_table", page_table, (batch, columns), torch.int32)
    check_tensor(dev, "seq_lens", seq_lens, (batch,), torch.int32)


class PagedKVAppendOp(Op):
    """New tokens into a paged cache of keys and values, the keys rotated on the way.

    Args:
        heads_kv, dim, page_size: The cache's.
        heads: Query heads, of ``q`` if it is passed.
        rotary_dim: Channels of a head that rotate, the first ones (0: none), even, up to 256.
        interleaved, frequencies, amplitude: As in RotaryEmbeddingFwdOp.
        dtype: float32, float16 or bfloat16.
        kernel_map: Optional override of ``"paged_kv_append"``.
    """

    def __init__(self, heads_kv: int, dim: int, page_size: int, heads: int = 0,
                 rotary_dim: int = 0, interleaved: bool = False,
                 frequencies: Optional[Sequence[float]] = None, amplitude: float = 1.0,
                 dtype: torch.dtype = torch.bfloat16,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.heads, self.heads_kv, self.dim, self.page_size = heads, heads_kv, dim, page_size
        self.rotary_dim = rotary_dim
        self.interleaved = interleaved
        self.frequencies = (rotary_frequencies(rotary_dim) if frequencies is None
                            else tuple(float(f) for f in frequencies))
        self.amplitude = amplitude
        self.dtype = dtype
        self._last = (0, 0, 0), False  # of the last call: k's shape, whether there were queries
        self._plans = Layouts()  # of the arguments that were found right
        self.dispatch_kernel(kernel_map)
        self.kernel = self.kernel_map["paged_kv_append"](
            heads_kv, dim, page_size, heads, rotary_dim, interleaved, self.frequencies, amplitude,
            dtype)

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"paged_kv_append": PagedKVAppendKernel}

    def forward(self, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                q: Optional[torch.Tensor] = None,
                cu_seqlens: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        layout = layout_of(k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens)
        plan = self._plans.get(layout)
        if plan is None:
            self._check(k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens)
            plan = self._plans.keep(layout, plan_of(self.kernel, k, v, k_cache, v_cache, page_table,
                                                    seq_lens, q, cu_seqlens))
        self._last = layout[0][0], q is not None
        if plan is NO_PLAN:
            return self.kernel(k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens)
        return self.kernel.forward(k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens, plan)

    def _check(self, k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens) -> None:
        dev = getattr(k, "device", None)
        if get_device_backend().is_device_tensor(k) and k.dim() not in (3, 4):
            raise ValueError("k must be (batch, heads_kv, dim), (batch, tokens, heads_kv, dim) or packed "
                             f"(tokens, heads_kv, dim), got shape {tuple(k.shape)}")
        rows = tuple(k.shape[:-2]) if hasattr(k, "shape") else ()
        check_tensor(dev, "k", k, (*rows, self.heads_kv, self.dim), self.dtype)
        check_tensor(dev, "v", v, (*rows, self.heads_kv, self.dim), self.dtype)
        if q is not None:
            check_tensor(dev, "q", q, (*rows, self.heads, self.dim), self.dtype)
        batch = rows[0]
        if cu_seqlens is not None:
            if len(rows) != 1:
                raise ValueError("k must be packed, (tokens, heads_kv, dim), when using `cu_seqlens`, "
                                 f"got shape {tuple(k.shape)}")
            offsets = cu_seqlens.numel() if get_device_backend().is_device_tensor(cu_seqlens) else 0
            check_tensor(dev, "cu_seqlens", cu_seqlens, (offsets,), torch.int32)
            if offsets < 1:
                raise ValueError("cu_seqlens must have at least one offset")
            batch = offsets - 1
        _check_cache(dev, k_cache, v_cache, page_table, seq_lens, batch,
                     (self.page_size, self.heads_kv, self.dim), self.dtype)
        if k.numel() // (self.heads_kv * self.dim) >= 2**31:
            raise ValueError(f"at most 2^31 - 1 tokens are supported, got shape {tuple(k.shape)}")

    def eval_roofline(self) -> tuple[int, int]:
        """``(3 * T * (H + Hkv) * rotary_dim, 2 * T * (H + 2 * Hkv) * dim * elem_bytes)`` of the T
        tokens of the last call, H 0 where it had no queries."""
        shape, queries = self._last
        tokens = shape[0] if len(shape) == 3 else shape[0] * shape[1]
        heads = self.heads if queries else 0
        return (3 * tokens * (heads + self.heads_kv) * self.rotary_dim,
                2 * tokens * (heads + 2 * self.heads_kv) * self.dim * self.dtype.itemsize)


class PagedAttentionDecodeOp(Op):
    """Attention of one new token of every sequence over a paged cache.

    Args:
        heads, heads_kv: Query heads and key heads (heads a multiple of heads_kv).
        dim: Head dimension, a multiple of 8 up to 256.
        page_size: Tokens of a page.
        scale: Factor on the scores (default: ``dim ** -0.5``).
        window: How many of the last tokens are seen (default: all).
        dtype: float16 or bfloat16.
        kernel_map: Optional override of ``"paged_attention_decode"``.
    """

    def __init__(self, heads: int, heads_kv: int, dim: int, page_size: int,
                 scale: Optional[float] = None, window: Optional[int] = None,
                 dtype: torch.dtype = torch.bfloat16,
                 kernel_map: Optional[Dict[str, Kernel]] = None) -> None:
        self.heads, self.heads_kv, self.dim, self.page_size = heads, heads_kv, dim, page_size
        self.scale = max(dim, 1)**-0.5 if scale is None else scale  # dim is checked by the kernel
        if window is not None and window < 1:
            raise ValueError(f"window must be at least 1 token, got {window}")
        self.window = window
        self.dtype = dtype
        self._last = 0, 0  # of the last call: sequences, columns of the page table
        self._seq_lens = None  # and their lengths, on the device
        self._plans = Layouts()  # of the arguments that were found right
        self.dispatch_kernel(kernel_map)
        self.kernel = self.kernel_map["paged_attention_decode"](
            heads, heads_kv, dim, page_size, self.scale, window or 0, dtype)

    @property
    def default_kernel_map(self) -> Dict[str, Kernel]:
        return {"paged_attention_decode": PagedAttentionDecodeKernel}

    def forward(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                page_table: torch.Tensor,
                seq_lens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        layout = layout_of(q, k_cache, v_cache, page_table, seq_lens)
        plan = self._plans.get(layout)
        if plan is None:
            self._check(q, k_cache, v_cache, page_table, seq_lens)
            plan = self._plans.keep(layout, plan_of(self.kernel, q, k_cache, v_cache, page_table,
                                                    seq_lens))
        self._last, self._seq_lens = layout[3][0], seq_lens
        if plan is NO_PLAN:
            return self.kernel(q, k_cache, v_cache, page_table, seq_lens)
        return self.kernel.forward(q, k_cache, v_cache, page_table, seq_lens, plan)

    def _check(self, q, k_cache, v_cache, page_table, seq_lens) -> None:
        dev = getattr(q, "device", None)
        batch = q.shape[0] if hasattr(q, "shape") and len(q.shape) else 0
        check_tensor(dev, "q", q, (batch, self.heads, self.dim), self.dtype)
        _check_cache(dev, k_cache, v_cache, page_table, seq_lens, batch,
                     (self.page_size, self.heads_kv, self.dim), self.dtype)
        if page_table.shape[1] * self.page_size >= 2**31 - 128:
            raise ValueError("page_table has room for at most 2^31 - 129 tokens a sequence, got "
                             f"{page_table.shape[1]} pages of {self.page_size}")

    def eval_roofline(self) -> tuple[int, int]:
        """``(4 * T * H * D, (2 * T * Hkv * D + 2 * B * H * D) * elem_bytes + 4 * B * H)``, T the
        tokens that the B queries of the last call see, by what its ``seq_lens`` holds now (read from
        the device; without it as many as the table has room for)."""
        batch, columns = self._last
        room = columns * self.page_size
        lens = [room] * batch if self._seq_lens is None else self._seq_lens.tolist()
        seen = sum(min(max(n, 0), room, self.window or room) for n in lens)
        return (4 * seen * self.heads * self.dim,
                (2 * seen * self.heads_kv * self.dim + 2 * batch * self.heads * self.dim)
                * self.dtype.itemsize + 4 * batch * self.heads)
