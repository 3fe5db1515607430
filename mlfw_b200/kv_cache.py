"""The int8 key/value cache of one attention layer (``b200q_kv_*``): pages of tokens, quantized as they are written.

The page table, ``start`` and ``count`` are int32 arrays in device memory (``None`` for ``count``: every row is in use); the
shapes and rules stand in ``include/b200q.h``.  Which pages a sequence owns is the caller's bookkeeping.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import check
from .device import Context, _ptr as _address


def _ptr(b):
    return b if type(b) is int or b is None else _address(b)


class KVCache:
    """``pages`` pages of ``page_tokens`` tokens for ``heads`` heads of ``head_dim`` (64 or 128).

    Allocates its buffers (``k_codes``, ``v_codes``, ``k_scales``, ``v_scales``) unless ``buffers`` names four the caller holds."""

    def __init__(self, ctx: Context, pages: int, page_tokens: int, heads: int, head_dim: int, buffers=None):
        self.ctx, self.pages, self.page_tokens, self.heads, self.head_dim = ctx, pages, page_tokens, heads, head_dim
        self.handle = None
        if buffers is None:
            shape = (max(pages, 0), max(heads, 0), max(page_tokens, 0))
            buffers = [ctx.empty(shape + (max(head_dim, 0),), np.int8) for _ in range(2)] + [ctx.empty(shape, np.float32) for _ in range(2)]
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = buffers
        h = C.c_void_p()
        check(ctx.lib.b200q_kv_create(ctx.handle, pages, page_tokens, heads, head_dim, *(_ptr(b) for b in buffers), C.byref(h)), "b200q_kv_create")
        self.handle = h.value
        self._append, self._read, self._attention, self._keep = (getattr(ctx.lib, "b200q_kv_" + n) for n in ("append", "read", "attention", "keep"))

    def close(self) -> None:
        if self.handle and self.ctx.handle:
            check(self.ctx.lib.b200q_kv_destroy(self.ctx.handle, self.handle), "b200q_kv_destroy")
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # A decoding step is a handful of these calls per layer: the wrappers do as little as they can.
    def append(self, k, v, ld_k, ld_v, B, T, page_table, max_pages, start, count=None):
        """Quantizes rows k, v (f32; row (b, t) of head h at base + (b*T + t)*ld + h*head_dim) into positions start[b] + t."""
        code = self._append(self.ctx.handle, self.handle, _ptr(k), _ptr(v), ld_k, ld_v, B, T, _ptr(page_table), max_pages, _ptr(start), _ptr(count))
        if code:
            check(code, "b200q_kv_append")

    def read(self, B, T, page_table, max_pages, start, count, k_out, v_out, ld_k, ld_v):
        """code * scale of positions start[b] + t, t < count[b], as f32."""
        code = self._read(self.ctx.handle, self.handle, B, T, _ptr(page_table), max_pages, _ptr(start), _ptr(count), _ptr(k_out), _ptr(v_out), ld_k, ld_v)
        if code:
            check(code, "b200q_kv_read")

    def attention(self, q, ld_q, B, T, H, page_table, max_pages, start, count, tree, scale, out, ld_out):
        """softmax(scale q K^T) V for T new rows per sequence; ``tree``: uint64 [B*T], the drafted rows each row sees, or None for
        those up to itself."""
        code = self._attention(self.ctx.handle, self.handle, _ptr(q), ld_q, B, T, H, _ptr(page_table), max_pages, _ptr(start), _ptr(count), _ptr(tree),
                               scale, _ptr(out), ld_out)
        if code:
            check(code, "b200q_kv_attention")

    def keep(self, B, T, page_table, max_pages, start, keep, count):
        """Moves the accepted drafted rows start[b] + keep[b*T + i] to start[b] + i, i < count[b]."""
        code = self._keep(self.ctx.handle, self.handle, B, T, _ptr(page_table), max_pages, _ptr(start), _ptr(keep), _ptr(count))
        if code:
            check(code, "b200q_kv_keep")
