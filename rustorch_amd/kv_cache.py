"""Device-resident mirror of `KVCache` / `KVLayerCache` (crates/rustorch-nn/src/kv_cache.rs:49-256).

Same object protocol as the reference -- `append(layer, seq_added, new_k, new_v)` for every layer, then
`advance(seq_added)` -- with the per-layer `[batch, n_heads, max_seq, head_dim]` buffers living in HBM (bf16 by
default, the storage type of the decode kernels; f32 on request) and the copies enqueued on a stream.  The
buffers are what `LlmKernels.gqa_decode_batched_bf16` and `qk_norm_rope_kv_append_bf16` take as caches: nothing
is trimmed or copied out before attention.

With dtype "q4" a layer's buffers are `Q4Rows`, rows of 4 bits, which the `_q4` calls of `LlmKernels` take; `append` takes bf16
rows there and rounds them.

`PagedKVCache` (no counterpart in the reference) holds many sequences of different lengths in pages, which the `_paged` calls of
`LlmKernels` take.
"""
from __future__ import annotations

import numpy as np

from . import _lib as L
from .device import HipStorage
from .errors import LayerOutOfRange, Overflow, check
from .llm_kernels import KVPages, LlmKernels, Q4Rows

_ELEM = {"bf16": 2, "f32": 4, "q4": 2}  # bytes an element of what is appended


class KVCache:
    def __init__(self, num_layers: int, batch: int, n_heads: int, head_dim: int, max_seq: int, dtype: str = "bf16"):
        """`KVCache::new` (kv_cache.rs:131-146; note the argument order: head_dim before max_seq).  The buffers
        start zeroed, like the reference's `vec![0.0; n]`."""
        if dtype not in _ELEM:
            raise ValueError(f"dtype must be 'bf16', 'f32' or 'q4', got {dtype!r}")
        if dtype == "q4" and head_dim not in (64, 128, 256):
            raise ValueError(f"a 4-bit cache has head_dim 64, 128 or 256, got {head_dim}")
        self.dtype, self.elem_bytes = dtype, _ELEM[dtype]
        self._dims = (batch, n_heads, max_seq, head_dim)
        self._max_seq = max_seq
        self._current_len = 0
        if dtype == "q4":
            self._layers = [tuple(Q4Rows.zeros(batch, n_heads, max_seq, head_dim) for _ in range(2)) for _ in range(num_layers)]
            return
        n_bytes = batch * n_heads * max_seq * head_dim * self.elem_bytes
        self._layers = [(HipStorage.zeros(n_bytes), HipStorage.zeros(n_bytes)) for _ in range(num_layers)]

    def num_layers(self) -> int:
        return len(self._layers)

    def max_seq(self) -> int:
        return self._max_seq

    def current_len(self) -> int:
        return self._current_len

    def clear(self) -> None:
        """Length back to zero; contents become stale, the allocation stays (kv_cache.rs:165-167)."""
        self._current_len = 0

    def append(self, layer_idx: int, seq_added: int, new_k, new_v, stream=None) -> None:
        """kv_cache.rs:172-190 then :77-112.  new_k / new_v are device buffers (`HipStorage`) holding
        `[batch, n_heads, seq_added, head_dim]` elements of the cache's dtype (bf16 for "q4"); their element counts are
        checked like the reference checks slice lengths."""
        if not 0 <= layer_idx < len(self._layers):
            raise LayerOutOfRange(layer_idx, len(self._layers))
        batch, n_heads, max_seq, head_dim = self._dims
        k, v = self._layers[layer_idx]
        if self.dtype == "q4":
            LlmKernels.kv_cache_append_q4(stream, k, v, new_k, new_k.byte_len // self.elem_bytes, new_v,
                                          new_v.byte_len // self.elem_bytes, batch, n_heads, max_seq, head_dim,
                                          self._current_len, seq_added)
            return
        check(L.native.rt_kv_cache_append_dev(stream, k, v, new_k, new_k.byte_len // self.elem_bytes, new_v,
                                              new_v.byte_len // self.elem_bytes, batch, n_heads, max_seq, head_dim,
                                              self._current_len, seq_added, self.elem_bytes))

    def advance(self, seq_added: int) -> None:
        """kv_cache.rs:194-204."""
        new_len = self._current_len + seq_added
        if new_len > self._max_seq:
            raise Overflow(new_len, self._max_seq)
        self._current_len = new_len

    def k_buffer(self, layer_idx: int):
        """The full `[batch, n_heads, max_seq, head_dim]` device buffer of the layer (`Q4Rows` for "q4"), or None
        (kv_cache.rs:210-212)."""
        return self._layers[layer_idx][0] if 0 <= layer_idx < len(self._layers) else None

    def v_buffer(self, layer_idx: int):
        return self._layers[layer_idx][1] if 0 <= layer_idx < len(self._layers) else None

    def dims(self):
        """`(batch, n_heads, max_seq, head_dim)`, or None without layers (kv_cache.rs:223-226)."""
        return self._dims if self._layers else None


class PagedKVCache:
    """Sequences in pages: per layer a `KVPages`, and one page table for all of them.  A sequence has a row of the table from `add` to
    `remove`; `reserve` gives it pages ahead of the append, `advance` counts the rows that every layer has appended.  Whole pages of a
    prefix are shared (`add(prefix_of=..., shared=...)`) and live as long as a sequence has them."""

    def __init__(self, num_layers: int, max_sequences: int, n_heads: int, head_dim: int, n_pages: int, page_size: int = 64,
                 table_pages: int | None = None):
        self.page_size, self.n_pages = page_size, n_pages
        self.table_pages = n_pages if table_pages is None else table_pages
        self._layers = [KVPages.zeros(n_pages, n_heads, page_size, head_dim) for _ in range(num_layers)]
        self._free = list(range(n_pages - 1, -1, -1))
        self._uses = np.zeros(n_pages, dtype=np.int32)
        self._table = np.full((max_sequences, self.table_pages), -1, dtype=np.int32)
        self._lens = np.full(max_sequences, -1, dtype=np.int32)  # -1: no sequence

    def num_layers(self) -> int:
        return len(self._layers)

    def layer(self, layer_idx: int) -> KVPages:
        if not 0 <= layer_idx < len(self._layers):
            raise LayerOutOfRange(layer_idx, len(self._layers))
        return self._layers[layer_idx]

    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, seq: int):
        if not 0 <= seq < len(self._lens) or self._lens[seq] < 0:
            raise KeyError(f"no sequence {seq}")

    def add(self, prefix_of: int | None = None, shared: int = 0) -> int:
        """A new sequence, empty, or with the first `shared` rows of another, whose pages it has in common: whole pages."""
        if shared % self.page_size:
            raise ValueError(f"a shared prefix ends with a page: {shared} rows of pages of {self.page_size}")
        if shared:
            self._check(prefix_of)
            if not 0 < shared <= self._lens[prefix_of]:
                raise Overflow(shared, int(self._lens[prefix_of]))
        free = np.flatnonzero(self._lens < 0)
        if not free.size:
            raise Overflow(len(self._lens) + 1, len(self._lens))
        seq, n = int(free[0]), shared // self.page_size
        if n:
            self._table[seq, :n] = self._table[prefix_of, :n]
            self._uses[self._table[seq, :n]] += 1
        self._lens[seq] = shared
        return seq

    def reserve(self, seq: int, rows: int) -> None:
        """Pages for `rows` more rows; all of them or, with Overflow, none."""
        self._check(seq)
        if rows < 0:
            raise ValueError(f"rows must not be negative, got {rows}")
        have, need = int((self._table[seq] >= 0).sum()), -(-(int(self._lens[seq]) + rows) // self.page_size)
        if need > self.table_pages or need - have > len(self._free):
            raise Overflow(int(self._lens[seq]) + rows, min(self.table_pages, have + len(self._free)) * self.page_size)
        for c in range(have, need):
            self._table[seq, c] = page = self._free.pop()
            self._uses[page] = 1

    def advance(self, seq: int, rows: int) -> None:
        self._check(seq)
        end, room = int(self._lens[seq]) + rows, int((self._table[seq] >= 0).sum()) * self.page_size
        if rows < 0 or end > room:
            raise Overflow(end, room)
        self._lens[seq] = end

    def remove(self, seq: int) -> None:
        """The sequence's row of the table is free, and so are the pages that nobody else has."""
        self._check(seq)
        for page in self._table[seq][self._table[seq] >= 0].tolist():
            self._uses[page] -= 1
            if self._uses[page] == 0:
                self._free.append(page)
        self._table[seq], self._lens[seq] = -1, -1

    def length(self, seq: int) -> int:
        self._check(seq)
        return int(self._lens[seq])

    def table(self, seqs, write_from=None) -> np.ndarray:
        """int32 [len(seqs), table_pages], the `page_table` of a call for these sequences.  write_from: for each of them the row from which
        the call may write; whole pages ahead of it are left out, so that an append keeps off what is shared."""
        seqs = list(seqs)
        for seq in seqs:
            self._check(seq)
        table = self._table[seqs].copy()
        if write_from is not None:
            rows = list(write_from)
            if len(rows) != len(seqs) or any(row < 0 for row in rows):
                raise ValueError(f"write_from is a row for each of {len(seqs)} sequences, got {rows}")
            for i, row in enumerate(rows):
                table[i, :row // self.page_size] = -1
        return table

    def lengths(self, seqs) -> np.ndarray:
        """int32 [len(seqs)], the rows that each has."""
        seqs = list(seqs)
        for seq in seqs:
            self._check(seq)
        return self._lens[seqs].copy()
