"""Host-side mirror of the attention part of `LlmKernels`
(crates/rustorch-cuda/src/llm_kernels.rs:874-958): raw device addresses, i32 dims and a stream;
calls enqueue and return."""
from __future__ import annotations

import functools
import operator

import numpy as np

from . import _lib as L
from .device import HipStorage
from .errors import Overflow, PositionOverflow, RopeWrongInputLen, check


class Q4Rows:
    """One of K and V held in 4 bits, the cache argument of the `_q4` calls: `codes`, bytes [batch, n_kv, max_seq,
    head_dim / 2], and `pairs`, 32-bit words [batch, n_kv, head_dim / 64, max_seq] of a bf16 scale s (low half) and middle z for
    64 dims of a row; a value is z + s (code - 8).  Device buffers of any kind the calls take (include/rt_attn.h says how
    the codes lie)."""

    __slots__ = ("codes", "pairs")

    def __init__(self, codes, pairs):
        self.codes, self.pairs = codes, pairs

    @classmethod
    def zeros(cls, batch: int, n_kv: int, max_seq: int, head_dim: int, stream=None) -> "Q4Rows":
        """A cache of zeros (s = z = 0); the fills are enqueued on `stream`."""
        rows = batch * n_kv * max_seq
        return cls(HipStorage.zeros(rows * head_dim // 2, stream), HipStorage.zeros(rows * (head_dim // 64) * 4, stream))


class KVPages:
    """K and V of a cache in pages, the cache argument of the `_paged` calls: device buffers [n_pages, n_kv, page_size, head_dim]
    of bf16, page_size a power of two from 16 to 1024.  Row r of sequence b lies in page `page_table[b, r // page_size]` (device
    int32 [batch, table_pages]; an entry that is no page, such as -1, stands for rows that are not there)."""

    __slots__ = ("k", "v", "n_pages", "page_size")

    def __init__(self, k, v, n_pages: int, page_size: int):
        self.k, self.v, self.n_pages, self.page_size = k, v, n_pages, page_size

    @classmethod
    def zeros(cls, n_pages: int, n_kv: int, page_size: int, head_dim: int, stream=None) -> "KVPages":
        n_bytes = n_pages * n_kv * page_size * head_dim * 2
        return cls(HipStorage.zeros(n_bytes, stream), HipStorage.zeros(n_bytes, stream), n_pages, page_size)


def _host_i32(*values):
    """(address, count, what keeps it alive) of host int32 values."""
    a = np.array([int(x) if isinstance(x, float) and x.is_integer() else operator.index(x) for x in values], dtype=np.int32)
    return a.ctypes.data, a.size, a


@functools.lru_cache(maxsize=64, typed=True)
def _kept_i32(*values):
    """The same, kept by the values; None where one of them is no plain int and may change (a tensor's element is kept by which it is)."""
    return _host_i32(*values) if all(type(x) is int for x in values) else None


def _host_or_dev(x):
    """(device address, host value) of an argument that is an int for every sequence or a device int32[batch] buffer."""
    return (None, int(x)) if isinstance(x, (int, np.integer)) else (x, 0)


def _checked_position(positions, rows, rope, seq, max_seq):
    """The device positions, or a host one checked as the reference does (rope.rs:179-184, kv_cache.rs:88-95)."""
    ptr, pos = _host_or_dev(positions)
    if ptr is None:
        if pos < 0 or pos + seq > rope.max_seq:
            raise PositionOverflow(rope.max_seq, pos + seq)
        if rows is None and pos + seq > max_seq:
            raise Overflow(pos + seq, max_seq)
    return ptr, pos


class LlmKernels:
    def __init__(self):
        L.lib()  # fail here, loudly, if the HIP library is not built

    @staticmethod
    def kv_append_bf16(stream, k_cache, v_cache, k_in, v_in, pos, n_kv, head_dim, max_seq):
        check(L.native.rt_kv_append_bf16(stream, k_cache, v_cache, k_in, v_in, pos, n_kv, head_dim, max_seq))

    @staticmethod
    def qk_norm_rope_kv_append_bf16(stream, q, k_in, v_in, k_cache, v_cache, positions, rope, batch, n_heads, n_kv,
                                    head_dim, max_seq, q_gamma=None, k_gamma=None, eps=1e-6, seq=1):
        """Steps 2a, 2b, 3 of decode_step (crates/rustorch-llm/src/model.rs:575-636) in one launch: per-head
        RMSNorm of q and k (device f32 gammas, or None), half-split RoPE with `rope`'s tables, cache append.
        `seq` new tokens per sequence ([batch, heads, seq, head_dim] buffers; 1 when decoding).  `positions` is a
        device int32[batch] buffer (position of each sequence's first new token), or an int used for every
        sequence (checked on the host)."""
        if isinstance(positions, (int, np.integer)):
            pos_ptr, pos = None, int(positions)
            # the reference's checks, before anything touches the device (rope.rs:179-184, kv_cache.rs:88-95)
            if pos < 0 or pos + seq > rope.max_seq:
                raise PositionOverflow(rope.max_seq, pos + seq)
            if pos + seq > max_seq:
                raise Overflow(pos + seq, max_seq)
        else:
            pos_ptr, pos = positions, 0
        cos, sin = rope.device_tables()
        check(L.native.rt_qk_norm_rope_kv_append_bf16(
            stream, q, k_in, v_in, k_cache, v_cache, pos_ptr, pos, q_gamma, k_gamma, eps, cos, sin, rope.max_seq, batch, seq,
            n_heads, n_kv, head_dim, max_seq))

    @staticmethod
    def gqa_decode_online_bf16(stream, q, k_cache, v_cache, out, n_heads, n_kv, kv_len, head_dim, max_seq):
        check(L.native.rt_gqa_decode_online_bf16(stream, q, k_cache, v_cache, out, n_heads, n_kv, kv_len, head_dim,
                                                 max_seq))

    @staticmethod
    def gqa_decode_naive_bf16(stream, q, k_cache, v_cache, out, n_heads, n_kv, kv_len, head_dim, max_seq):
        """llm_kernels.rs:990-1042: the reference's three-pass decode launcher; same function, same kernels here."""
        check(L.native.rt_gqa_decode_naive_bf16(stream, q, k_cache, v_cache, out, n_heads, n_kv, kv_len, head_dim,
                                                max_seq))

    @staticmethod
    def gqa_decode_workspace_bytes(batch, n_heads, n_kv, head_dim, max_seq) -> int:
        return L.lib().rt_gqa_decode_workspace_bytes(batch, n_heads, n_kv, head_dim, max_seq)

    @staticmethod
    def gqa_decode_batched_bf16(stream, q, k_cache, v_cache, out, kv_lens, batch, n_heads, n_kv, head_dim, max_seq,
                                workspace, workspace_bytes):
        """Ragged batch: q/out [B,Hq,D], caches [B,Hkv,max_seq,D], kv_lens device int32[B]."""
        check(L.native.rt_gqa_decode_batched_bf16(stream, q, k_cache, v_cache, out, kv_lens, batch, n_heads, n_kv, head_dim,
                                                  max_seq, workspace, workspace_bytes))

    @staticmethod
    def gqa_decode_batched_bf16_noalloc(stream, q, k_cache, v_cache, out, kv_lens, batch, n_heads, n_kv, head_dim,
                                        max_seq):
        """gqa_decode_batched_bf16 without a workspace argument: the partials go to a fixed block of device memory
        inside the library, and the call allocates nothing (for callers under graph capture or in loops that must
        not call hipMalloc).  Calls that overlap on one GPU race."""
        check(L.native.rt_gqa_decode_batched_bf16_noalloc(stream, q, k_cache, v_cache, out, kv_lens, batch, n_heads, n_kv,
                                                          head_dim, max_seq))

    @staticmethod
    def gqa_decode_chunk_bf16(stream, q, k_cache, v_cache, out, kv_lens, batch, seq_new, n_heads, n_kv, head_dim,
                              max_seq):
        """`seq_new` consecutive new positions per sequence against the cache, causally masked (the bf16, batched form
        of gqa_decode_batched_f32, crates/rustorch-metal/src/kernels.rs:14432-14516): q/out [B,seq_new,Hq,D], caches
        [B,Hkv,max_seq,D] already holding the new positions; `kv_lens` a device int32[B] buffer of key counts that
        include the new positions, or an int used for every sequence."""
        if isinstance(kv_lens, (int, np.integer)):
            lens_ptr, kv_len = None, int(kv_lens)
        else:
            lens_ptr, kv_len = kv_lens, 0
        check(L.native.rt_gqa_decode_chunk_bf16(stream, q, k_cache, v_cache, out, lens_ptr, kv_len, batch, seq_new, n_heads,
                                                n_kv, head_dim, max_seq))

    # ---- caches that are kept small (no counterparts in the reference): 4-bit rows, and rows taken out ----

    @staticmethod
    def qk_norm_rope_kv_append_q4(stream, q, q_out, k_in, v_in, k_cache, v_cache, positions, rope, batch, n_heads, n_kv,
                                  head_dim, max_seq, q_gamma=None, k_gamma=None, eps=1e-6, seq=1, rows=None, slots=None,
                                  weights=None):
        """`qk_norm_rope_kv_append_bf16` into a 4-bit cache (`Q4Rows`); q goes to `q_out`, which may be q.  `rows`, a device
        int32[batch] buffer, is each sequence's first cache row where that is not its position (a cache that rows were
        evicted from); `slots` (int32) and `weights` (f32) [batch, n_kv, max_seq] then take the new tokens' positions
        and zeros."""
        ptr, pos = _checked_position(positions, rows, rope, seq, max_seq)
        cos, sin = rope.device_tables()
        check(L.native.rt_qk_norm_rope_kv_append_q4(
            stream, q, q_out, k_in, v_in, k_cache.codes, k_cache.pairs, v_cache.codes, v_cache.pairs, ptr, pos, rows, slots, weights,
            q_gamma, k_gamma, eps, cos, sin, rope.max_seq, batch, seq, n_heads, n_kv, head_dim, max_seq))

    @staticmethod
    def qk_norm_rope_kv_append_rows_bf16(stream, q, q_out, k_in, v_in, k_cache, v_cache, positions, rope, batch, n_heads,
                                         n_kv, head_dim, max_seq, q_gamma=None, k_gamma=None, eps=1e-6, seq=1, rows=None,
                                         slots=None, weights=None):
        """The same into a bf16 cache whose rows are not the positions."""
        ptr, pos = _checked_position(positions, rows, rope, seq, max_seq)
        cos, sin = rope.device_tables()
        check(L.native.rt_qk_norm_rope_kv_append_rows_bf16(
            stream, q, q_out, k_in, v_in, k_cache, v_cache, ptr, pos, rows, slots, weights, q_gamma, k_gamma, eps, cos, sin,
            rope.max_seq, batch, seq, n_heads, n_kv, head_dim, max_seq))

    @staticmethod
    def kv_cache_append_q4(stream, k_cache, v_cache, new_k, new_k_len, new_v, new_v_len, batch, n_heads, max_seq, head_dim,
                           current_len, seq_added):
        """`KVLayerCache::append` (crates/rustorch-nn/src/kv_cache.rs:77-112) of bf16 rows into a 4-bit cache; the lengths
        are in elements."""
        check(L.native.rt_kv_cache_append_q4_dev(stream, k_cache.codes, k_cache.pairs, v_cache.codes, v_cache.pairs, new_k,
                                                 new_k_len, new_v, new_v_len, batch, n_heads, max_seq, head_dim, current_len,
                                                 seq_added))

    @staticmethod
    def kv_cache_read_q4(stream, cache, out, batch, n_kv, head_dim, max_seq, rows, n_rows):
        """`n_rows` rows of a 4-bit cache as bf16, out [batch, n_kv, n_rows, head_dim]; `rows` is the first of them, an int
        or a device int32[batch] buffer."""
        ptr, row = _host_or_dev(rows)
        check(L.native.rt_kv_cache_read_q4(stream, cache.codes, cache.pairs, out, ptr, row, n_rows, batch, n_kv, head_dim, max_seq))

    @staticmethod
    def gqa_decode_q4_workspace_bytes(batch, seq_new, n_heads, n_kv, head_dim, max_seq) -> int:
        return L.lib().rt_gqa_decode_q4_workspace_bytes(batch, seq_new, n_heads, n_kv, head_dim, max_seq)

    @staticmethod
    def gqa_decode_q4(stream, q, k_cache, v_cache, out, kv_lens, batch, seq_new, n_heads, n_kv, head_dim, max_seq, workspace,
                      workspace_bytes):
        """`gqa_decode_chunk_bf16` over a 4-bit cache: q/out [batch, seq_new, n_heads, head_dim], `kv_lens` (keys including
        the new positions') a device int32[batch] buffer or an int; seq_new = 1 is a decode step."""
        ptr, kv_len = _host_or_dev(kv_lens)
        check(L.native.rt_gqa_decode_q4(stream, q, k_cache.codes, k_cache.pairs, v_cache.codes, v_cache.pairs, out, ptr, kv_len,
                                        batch, seq_new, n_heads, n_kv, head_dim, max_seq, workspace, workspace_bytes))

    @staticmethod
    def gqa_decode_weights_workspace_bytes(batch, n_heads, n_kv, head_dim, max_seq) -> int:
        return L.lib().rt_gqa_decode_weights_workspace_bytes(batch, n_heads, n_kv, head_dim, max_seq)

    @staticmethod
    def gqa_decode_weights_bf16(stream, q, k_cache, v_cache, out, weights_in, weights_out, kv_lens, batch, n_heads, n_kv,
                                head_dim, max_seq, workspace, workspace_bytes):
        """A decode step over a bf16 cache that also sums what each key draws: weights_out = weights_in (None: zeros) + the
        softmax weights of the kv head's query heads, f32 [batch, n_kv, max_seq], for the keys that exist."""
        check(L.native.rt_gqa_decode_weights_bf16(stream, q, k_cache, v_cache, out, weights_in, weights_out, kv_lens, batch, n_heads,
                                                  n_kv, head_dim, max_seq, workspace, workspace_bytes))

    @staticmethod
    def gqa_decode_weights_q4(stream, q, k_cache, v_cache, out, weights_in, weights_out, kv_lens, batch, n_heads, n_kv,
                              head_dim, max_seq, workspace, workspace_bytes):
        """The same over a 4-bit cache."""
        check(L.native.rt_gqa_decode_weights_q4(stream, q, k_cache.codes, k_cache.pairs, v_cache.codes, v_cache.pairs, out,
                                                weights_in, weights_out, kv_lens, batch, n_heads, n_kv, head_dim, max_seq,
                                                workspace, workspace_bytes))

    @staticmethod
    def kv_evict_workspace_bytes(batch, n_kv, max_seq, budget) -> int:
        return L.lib().rt_kv_evict_workspace_bytes(batch, n_kv, max_seq, budget)

    @staticmethod
    def kv_evict_bf16(stream, k_cache, v_cache, weights_in, slots_in, weights_out, slots_out, kv_lens, new_lens, batch, n_kv,
                      head_dim, max_seq, budget, recent, workspace, workspace_bytes):
        """Cuts every sequence to `budget` rows, per kv head the `recent` newest tokens and the largest sums of weights;
        kept rows behind the budget move into the freed ones.  weights/slots [batch, n_kv, max_seq] in and out may be the
        same buffers; `new_lens` (None, or device int32[batch], which may be kv_lens) takes the new lengths."""
        check(L.native.rt_kv_evict_bf16(stream, k_cache, v_cache, weights_in, slots_in, weights_out, slots_out, kv_lens, new_lens,
                                        batch, n_kv, head_dim, max_seq, budget, recent, workspace, workspace_bytes))

    @staticmethod
    def kv_evict_q4(stream, k_cache, v_cache, weights_in, slots_in, weights_out, slots_out, kv_lens, new_lens, batch, n_kv,
                    head_dim, max_seq, budget, recent, workspace, workspace_bytes):
        """The same of a 4-bit cache."""
        check(L.native.rt_kv_evict_q4(stream, k_cache.codes, k_cache.pairs, v_cache.codes, v_cache.pairs, weights_in, slots_in,
                                      weights_out, slots_out, kv_lens, new_lens, batch, n_kv, head_dim, max_seq, budget, recent,
                                      workspace, workspace_bytes))

    # ---- many requests side by side (no counterparts in the reference): packed tokens, and caches in pages ----

    @staticmethod
    def qk_norm_rope_kv_append_paged_bf16(stream, q, q_out, k_in, v_in, pages, page_table, table_pages, positions, rope, tokens,
                                          batch, n_heads, n_kv, head_dim, starts=None, k_out=None, q_gamma=None, k_gamma=None,
                                          eps=1e-6, axis_positions=None, sections=None):
        """`qk_norm_rope_kv_append_bf16` for packed tokens ([tokens, heads, head_dim]) and a cache in pages (`KVPages`); q goes to
        `q_out` and, where it is given, rotated k to `k_out`; each may be its input.  `starts`, device int32[batch + 1], are the
        sequences' first tokens (None: tokens / batch each); `positions`, an int or a device int32[batch] buffer, the row of a sequence's
        first token.  With `sections`, pairs of a head for each of up to four axes, a token's rotary positions are
        `axis_positions`, device int32[len(sections), tokens], and not its row.  `rope` is of heads of head_dim."""
        of = getattr(rope, "head_dim", head_dim)
        if of != head_dim and of // 2 != head_dim // 2 and head_dim > 0:
            raise RopeWrongInputLen(rope.max_seq * (head_dim // 2), rope.max_seq * (of // 2))
        ptr, pos = _host_or_dev(positions)
        at, n_axes, _ = None, 0, None
        if sections is not None:
            sections = tuple(sections)
            at, n_axes, _ = _kept_i32(*sections) or _host_i32(*sections)
        cos, sin = rope.device_tables()
        check(L.native.rt_qk_norm_rope_kv_append_paged_bf16(
            stream, q, q_out, k_in, k_out, v_in, pages.k, pages.v, page_table, starts, ptr, pos, axis_positions, at, n_axes, q_gamma, k_gamma, eps, cos, sin,
            rope.max_seq, tokens, batch, n_heads, n_kv, head_dim, pages.n_pages, pages.page_size, table_pages))

    @staticmethod
    def gqa_decode_paged_workspace_bytes(batch, n_heads, n_kv, head_dim, page_size, table_pages) -> int:
        return L.lib().rt_gqa_decode_paged_workspace_bytes(batch, n_heads, n_kv, head_dim, page_size, table_pages)

    @staticmethod
    def gqa_decode_paged_bf16(stream, q, pages, out, page_table, table_pages, kv_lens, batch, n_heads, n_kv, head_dim, workspace,
                              workspace_bytes, shared_len=0):
        """`gqa_decode_batched_bf16` over a cache in pages: q/out [batch, n_heads, head_dim], kv_lens device int32[batch].  The
        first `shared_len` keys (an int or a device int32[1] buffer) of every sequence that has as many are the same for all of
        these, and are read once where the call's sizes say that it is shorter (an int), or always (a buffer)."""
        ptr, shared = _host_or_dev(shared_len)
        check(L.native.rt_gqa_decode_paged_bf16(stream, q, pages.k, pages.v, out, page_table, kv_lens, ptr, shared, batch, n_heads, n_kv,
                                                head_dim, pages.n_pages, pages.page_size, table_pages, workspace, workspace_bytes))
