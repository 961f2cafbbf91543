"""Paged 8-bit K/V cache of several sequences (rbn_kv_* of include/ronn_bitnet_hip.h).

A row is the place of one sequence.  Rows, their lengths, the page table and the free pages live on
the device and are advanced by plan(); store() and attend() then run for every layer of the model.  The
reference has no K/V cache (its BitNet provider stops at the matmul,
crates/ronn-providers/src/bitnet/kernels.rs:134-178).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import check
from .device import Context, DeviceBuffer

FORMATS = {"i8": _lib.KV_I8, "e4m3": _lib.KV_E4M3}


class PagedKVCache:
    """Buffers of `layers` layers for `rows` sequences of at most `max_len` positions each, which share `pages`
    pages of 32 positions; a call takes at most `max_tokens` tokens.  fmt: "i8" or "e4m3"."""

    def __init__(self, ctx: Context, layers: int, kv_heads: int, head_dim: int, rows: int, pages: int, max_len: int,
                 max_tokens: int, fmt: str = "i8"):
        if fmt not in FORMATS:
            raise ValueError("fmt is one of %s" % ", ".join(sorted(FORMATS)))
        if layers < 1 or max_len < 1:
            raise ValueError("layers and max_len must be positive")
        lib = ctx.lib
        code, scale = lib.rbn_kv_code_bytes(pages, kv_heads, head_dim), lib.rbn_kv_scale_bytes(pages, kv_heads)
        opened = lib.rbn_kv_open_bytes(rows, kv_heads, head_dim)
        if not (code and scale and opened) or not 0 < max_tokens <= _lib.KV_MAX_TOKENS:
            raise ValueError("sizes outside the cache's ranges: kv_heads %d, head_dim %d, rows %d, pages %d, max_tokens %d"
                             % (kv_heads, head_dim, rows, pages, max_tokens))
        max_blocks = -(-max_len // _lib.KV_BLOCK)
        if max_blocks > _lib.KV_MAX_BLOCKS:
            raise ValueError("max_len %d is more than %d blocks" % (max_len, _lib.KV_MAX_BLOCKS))
        self.ctx, self.lib = ctx, lib
        self.layers, self.kv_heads, self.head_dim, self.fmt = layers, kv_heads, head_dim, fmt
        self.rows, self.pages, self.max_blocks, self.max_tokens = rows, pages, max_blocks, max_tokens
        i32 = lambda n, v: ctx.to_device(np.full(n, v, dtype=np.int32))  # noqa: E731
        self.d_table, self.d_len = i32(rows * max_blocks, -1), i32(rows, 0)
        self.d_ring = ctx.to_device(np.arange(pages, dtype=np.int32))
        self.d_ring_state = ctx.to_device(np.array([0, pages], dtype=np.int32))
        self.d_start, self.d_count = i32(rows + 1, 0), i32(2, 0)
        self.d_row, self.d_pos, self.d_slot, self.d_unit = (i32(max_tokens, -1) for _ in range(4))
        self.buffers = []          # per layer: K codes, V codes, K open, V open, K scales, V scales
        self._layers = []
        for _ in range(layers):
            b = [ctx.alloc(n) for n in (code, code, opened, opened, scale, scale)]
            self.buffers.append(b)
            self._layers.append(_lib.KvLayer(FORMATS[fmt], kv_heads, head_dim, 0, *(x.ptr for x in b)))
        self._table = _lib.KvTable(rows, max_blocks, pages, self.d_table.ptr, self.d_len.ptr, self.d_ring.ptr,
                                   self.d_ring_state.ptr)
        self._batch = _lib.KvBatch(max_tokens, self.d_start.ptr, self.d_row.ptr, self.d_pos.ptr, self.d_slot.ptr,
                                   self.d_unit.ptr, self.d_count.ptr)

    def batch(self, max_tokens: int) -> "_lib.KvBatch":
        """The cache's batch arrays for a call of at most max_tokens tokens (fewer than the cache's own
        maximum launch less)."""
        if not 0 < max_tokens <= self.max_tokens:
            raise ValueError("max_tokens must be in [1, %d]" % self.max_tokens)
        b = _lib.KvBatch.from_buffer_copy(self._batch)
        b.max_tokens = max_tokens
        return b

    def _held(self, what: str, buf: DeviceBuffer, nbytes: int):
        if buf.nbytes < nbytes:
            raise ValueError("%s holds %d bytes, %d are needed" % (what, buf.nbytes, nbytes))

    def _layer(self, layer: int):
        if not 0 <= layer < self.layers:
            raise ValueError("layer %d is outside [0, %d)" % (layer, self.layers))
        return self._layers[layer]

    def plan(self, d_new: DeviceBuffer, batch=None):
        """Advances the rows by d_new [rows] int32 (n > 0: n tokens, 0: none, < 0: the row ends)."""
        self._held("d_new", d_new, 4 * self.rows)
        check(self.lib.rbn_kv_plan(self.ctx.handle, self._table, d_new.ptr, batch or self._batch, self.d_len.ptr,
                                   self.d_ring_state.ptr))

    def store(self, layer: int, d_qkv: DeviceBuffer, heads: int, theta: float, d_q: DeviceBuffer, batch=None):
        """Rotates q into d_q and stores k and v of the planned tokens.  d_qkv and d_q have room for as many tokens as
        the batch may have."""
        batch, kv = batch or self._batch, self._layer(layer)
        self._held("d_qkv", d_qkv, 4 * batch.max_tokens * (heads + 2 * self.kv_heads) * self.head_dim)
        self._held("d_q", d_q, 4 * batch.max_tokens * heads * self.head_dim)
        check(self.lib.rbn_rope_kv_store_q8(self.ctx.handle, d_qkv.ptr, self._table, batch, kv, heads, float(theta), d_q.ptr))

    def attend(self, layer: int, d_q: DeviceBuffer, heads: int, max_new: int, d_out: DeviceBuffer, batch=None):
        """Causal attention of the planned tokens over their rows.  d_q and d_out have room for as many tokens as the
        batch may have."""
        batch, kv = batch or self._batch, self._layer(layer)
        for what, buf in (("d_q", d_q), ("d_out", d_out)):
            self._held(what, buf, 4 * batch.max_tokens * heads * self.head_dim)
        check(self.lib.rbn_attention_q8kv(self.ctx.handle, d_q.ptr, self._table, batch, kv, heads, max_new, d_out.ptr))

    def read(self, layer: int, rows, positions):
        """What the cache holds at the places (rows[i], positions[i]): K and V [n, kv_heads, head_dim] float16."""
        rows, positions = (np.ascontiguousarray(x, dtype=np.int32) for x in (rows, positions))
        if rows.shape != positions.shape or rows.ndim != 1 or rows.size == 0:
            raise ValueError("rows and positions must be vectors of the same length, not empty")
        n = rows.size * self.kv_heads * self.head_dim
        d_k, d_v = self.ctx.alloc(2 * n), self.ctx.alloc(2 * n)
        d_rows, d_pos = self.ctx.to_device(rows), self.ctx.to_device(positions)
        check(self.lib.rbn_kv_read_f16(self.ctx.handle, self._table, self._layer(layer), d_rows.ptr, d_pos.ptr,
                                       rows.size, d_k.ptr, d_v.ptr))
        shape = (rows.size, self.kv_heads, self.head_dim)
        return d_k.download(np.float16, n).reshape(shape), d_v.download(np.float16, n).reshape(shape)

    def lengths(self) -> np.ndarray:
        """Positions held by each row."""
        return self.d_len.download(np.int32, self.rows)

    def free_pages(self) -> int:
        return int(self.d_ring_state.download(np.int32, 2)[1])
