"""Paged-cache kernels: appending keys and values, attention of one new token.

Shims over ``tileops_paged_kv_append`` (``csrc/rotary.cu``) and
``tileops_paged_decode_fwd`` (``csrc/paged_attention.cu``).  A cache is
``(pages, page_size, heads_kv, dim)`` with contiguous channels and any other
strides: a head-major one, ``(pages, heads_kv, page_size, dim)``, is its
transposed view.
"""

from __future__ import annotations

import ctypes
import threading
from typing import Optional, Sequence

import torch

from tileops import _native
from tileops.kernels.attention._layouts import Apart, channels_last, overlaps, row_of
from tileops.kernels.attention.rotary_embedding import check_rotation, turns_array
from tileops.kernels.kernel_base import Kernel, check_dtype

__all__ = ["PagedAttentionDecodeKernel", "PagedKVAppendKernel"]

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
        self.init_config(config)

    def plan(self, k, v, k_cache, v_cache, page_table, seq_lens, q=None, cu_seqlens=None):
        """What a call of this layout needs, for ``forward``: device, which arguments have to be
        copied, the stride array, the table's stride, the rows, the queries' shape and whether the
        caches lie apart; refuses caches that cannot be written."""
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if not channels_last(c):
                raise ValueError(f"{name} must have contiguous channels, got strides {c.stride()}")
            if overlaps(c.shape, c.stride()):
                raise ValueError(f"{name} has slots that share memory: shape {tuple(c.shape)}, "
                                 f"strides {c.stride()}")
        copy, values = [], []
        for t, dense in ((q, False), (k, False), (v, False), (q, True)):
            if t is None:
                copy.append(False)
                values += (0, 0, 0)
                continue
            copy.append(not channels_last(t))
            dense |= copy[-1]
            *rows, heads, dim = t.shape
            if len(rows) == 2:
                values += (rows[1] * heads * dim, heads * dim, dim) if dense else t.stride()[:3]
                continue
            token, head = (heads * dim, dim) if dense else t.stride()[:2]
            values += (token, 0, head) if cu_seqlens is None else (0, token, head)
        values += k_cache.stride()[:3] + v_cache.stride()[:3]
        copy = (*copy[:3], page_table.stride(-1) != 1, seq_lens.stride(0) != 1,
                cu_seqlens is not None and cu_seqlens.stride(0) != 1)
        table_stride = page_table.shape[1] if copy[3] else page_table.stride(0)
        tokens = k.shape[0] if k.dim() == 3 else k.shape[0] * k.shape[1]
        return (k.device, copy if any(copy) else None, (ctypes.c_int64 * 18)(*values), table_stride,
                seq_lens.shape[0], tokens, k_cache.shape[0], page_table.shape[1],
                None if q is None else row_of(q), Apart(k_cache, v_cache))

    def forward(self, k, v, k_cache, v_cache, page_table, seq_lens, q=None, cu_seqlens=None,
                plan=None):
        """Write the caches; return the rotated queries (None without ``q``).  ``plan``: what
        ``plan()`` gave for arguments of the same layout."""
        if plan is None:
            plan = self.plan(k, v, k_cache, v_cache, page_table, seq_lens, q, cu_seqlens)
        device, copy, strides, table_stride, seqs, tokens, pages, columns, q_like, apart = plan
        if copy is not None:
            q, k, v, page_table, seq_lens, cu_seqlens = (
                t.contiguous() if c else t
                for t, c in zip((q, k, v, page_table, seq_lens, cu_seqlens), copy))
        k_at, v_at = k_cache.data_ptr(), v_cache.data_ptr()
        if not apart(k_at, v_at):
            raise ValueError("k_cache and v_cache share memory: they cannot both be written")
        q_out = None if q is None else torch.empty_like(q_like)
        _native.launch(
            "tileops_paged_kv_append", device, 0 if q is None else q.data_ptr(), k.data_ptr(),
            v.data_ptr(), 0 if q is None else q_out.data_ptr(), k_at, v_at, page_table.data_ptr(),
            seq_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(), self._turns, seqs,
            tokens, 0 if q is None else self.heads, self.heads_kv, self.dim, self.rotary_dim, pages,
            self.page_size, columns, table_stride, strides, self.interleaved, self.amplitude,
            self._code)
        return q_out


_workspaces: dict = {}  # (device, stream's number): the largest one that a call of it has needed
_of_thread = threading.local()  # the same for the thread's per-thread default stream
_PER_THREAD_DEFAULT = 2  # handle (and number) of that stream


def _workspace(device: torch.device, room: int):
    """Scratch of ``room`` bytes on the current stream, and whether its counters are zero.

    Calls of one stream run one after another and each leaves the counters at zero, so they share
    a workspace that is kept (2.3 us a call less than one of its own that has to be cleared).  That
    holds for torch's own streams, which live as long as the process: the default one, number 0, and
    those of its pool, of odd numbers.  Another stream's number is its handle, an even one, which the next
    stream may get while this one's last call still runs: a call there gets a workspace of its own, cleared.
    The per-thread default stream is a stream in each thread, and so is what is kept for it.  A graph
    under capture, which may be replayed on any stream, gets one of its own, cleared in the graph.
    """
    if device.type != "cuda" or torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(room, dtype=torch.uint8, device=device), False
    stream = torch._C._cuda_getCurrentStream(device.index)[0]
    kept = _workspaces
    if stream % 2 == 0 and stream != 0:
        if stream != _PER_THREAD_DEFAULT:
            return torch.empty(room, dtype=torch.uint8, device=device), False
        kept = _of_thread.__dict__
    key = device.index, stream
    found = kept.get(key)
    if found is None or found.numel() < room:
        found = kept[key] = torch.zeros(room, dtype=torch.uint8, device=device)
    return found, True


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
        self.init_config(config)

    def plan(self, q, k_cache, v_cache, page_table, seq_lens):
        """What a call of this layout needs, for ``forward``: device, which arguments have to be
        copied (never a cache), the stride array, the table's stride and sizes, the shapes of the
        outputs and the bytes of the workspace."""
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if not channels_last(c) or any(s % 8 for s, n in zip(c.stride()[:3], c.shape) if n > 1):
                raise ValueError(f"{name} must have contiguous channels and strides that are "
                                 f"multiples of 8, got {c.stride()}")
        batch, heads, dim = q.shape
        copy = (not channels_last(q) or q.stride(0) % 8 != 0 or q.stride(1) % 8 != 0,
                page_table.stride(-1) != 1, seq_lens.stride(0) != 1)
        strides = [heads * dim, dim] if copy[0] else [*q.stride()[:2]]
        for c in (k_cache, v_cache):  # what a single page, slot or head is apart has no say
            strides += [s if n > 1 else 0 for s, n in zip(c.stride()[:3], c.shape)]
        table_stride = page_table.shape[1] if copy[1] else page_table.stride(0)
        room = _native.lib().tileops_paged_decode_workspace_bytes(heads, self.heads_kv, dim)
        like = torch.empty(1, dtype=torch.float32, device=q.device)
        return (q.device, copy if any(copy) else None, (ctypes.c_int64 * 8)(*strides), table_stride,
                batch, k_cache.shape[0], page_table.shape[1], row_of(q),
                like.expand(batch, heads), room)

    def forward(self, q, k_cache, v_cache, page_table, seq_lens, plan=None):
        """Return ``(o, lse)``.  ``plan``: what ``plan()`` gave for arguments of the same layout."""
        if plan is None:
            plan = self.plan(q, k_cache, v_cache, page_table, seq_lens)
        device, copy, strides, table_stride, batch, pages, columns, o_like, lse_like, room = plan
        if device.type == "cuda" and torch._C._cuda_getDevice() != device.index:
            with torch.cuda.device(device):
                return self.forward(q, k_cache, v_cache, page_table, seq_lens, plan)
        if copy is not None:
            q, page_table, seq_lens = (t.contiguous() if c else t
                                       for t, c in zip((q, page_table, seq_lens), copy))
        at = q.data_ptr()
        if at % 16:  # strides of whole 16 bytes, but not its start
            q = q.clone()
            at = q.data_ptr()
            strides = (ctypes.c_int64 * 8)(*q.stride()[:2], *strides[2:])
        o, lse = torch.empty_like(o_like), torch.empty_like(lse_like)
        ws, counters_zero = _workspace(device, room)
        _native.launch(
            "tileops_paged_decode_fwd", device, at, k_cache.data_ptr(), v_cache.data_ptr(),
            page_table.data_ptr(), seq_lens.data_ptr(), o.data_ptr(), lse.data_ptr(),
            ws.data_ptr(), batch, self.heads, self.heads_kv, self.dim, pages, self.page_size,
            columns, table_stride, strides, self.window, counters_zero, self.scale, self._code)
        return o, lse
