"""Caches in pages and packed tokens, from their definitions in numpy: what the tests of those entries compare with."""
import numpy as np

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values

F32 = np.float32
NAN_BITS = np.uint16(0x7FC1)


def dev(a):
    return ra.HipStorage.from_numpy(np.ascontiguousarray(a))


def normal_bits(rng, *shape):
    return bf16_bits(rng.standard_normal(shape, dtype=F32))


class Pages:
    """Sequences of `lens` rows in shuffled pages, with the first `common` pages of all of them the same.  What no sequence has
    holds NaN: rows behind a sequence's last in its last page, and pages that nobody has."""

    def __init__(self, rng, lens, n_kv, dim, page, shared=0, spare=3, more_columns=1):
        self.page, self.n_kv, self.dim, self.lens, self.shared = page, n_kv, dim, list(lens), shared
        b = len(lens)
        need = [-(-n // page) for n in lens]
        self.table_pages = max(need + [1]) + more_columns
        common = shared // page
        sharers = [i for i in range(b) if lens[i] >= shared]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((b, self.table_pages), -1, dtype=np.int32)
        at = 0
        for i in range(b):
            for c in range(need[i]):
                if c < common and i in sharers and i != sharers[0]:
                    self.table[i, c] = self.table[sharers[0], c]
                else:
                    self.table[i, c] = order[at]
                    at += 1
        self.k = np.full((self.n_pages, n_kv, page, dim), NAN_BITS, dtype=np.uint16)
        self.v = self.k.copy()
        self.rows_k = [normal_bits(rng, n_kv, n, dim) for n in lens]
        self.rows_v = [normal_bits(rng, n_kv, n, dim) for n in lens]
        for i in sharers[1:]:
            self.rows_k[i][:, :shared] = self.rows_k[sharers[0]][:, :shared]
            self.rows_v[i][:, :shared] = self.rows_v[sharers[0]][:, :shared]
        for i in range(b):
            for r in range(lens[i]):
                self.k[self.table[i, r // page], :, r % page] = self.rows_k[i][:, r]
                self.v[self.table[i, r // page], :, r % page] = self.rows_v[i][:, r]

    def dev(self):
        return ra.KVPages(dev(self.k), dev(self.v), self.n_pages, self.page)


def attention(q, k, v):
    """q [heads, d], k, v [kv heads, n, d] f64 -> (values, the same over |v|) [heads, d]; no keys: zeros."""
    h, d = q.shape
    g = h // k.shape[0]
    out, size = np.zeros((h, d)), np.zeros((h, d))
    for j in range(h):
        if k.shape[1]:
            x = k[j // g] @ q[j] / np.sqrt(d)
            p = np.exp(x - x.max())
            p /= p.sum()
            out[j], size[j] = p @ v[j // g], p @ np.abs(v[j // g])
    return out, size


def expect_decode(q_bits, pages, lens=None, hidden=None):
    """(values, sizes) [b, heads, d] of a decode step; hidden[b]: keys that are not seen."""
    q = bf16_values(q_bits).astype(np.float64)
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for i, n in enumerate(pages.lens if lens is None else lens):
        keep = np.ones(n, dtype=bool)
        if hidden is not None and i in hidden:
            keep[np.asarray(hidden[i], dtype=int)] = False
        k, v = (bf16_values(x[i][:, :n])[:, keep].astype(np.float64) for x in (pages.rows_k, pages.rows_v))
        out[i], size[i] = attention(q[i], k, v)
    return out, size


def run_decode(q_bits, pages, n_kv, shared=0, lens=None, table=None, stream=None, out=None, ws=None):
    """The entry on host arrays; returns bf16 bits [b, heads, d].  shared: as the entry takes it (on the device: always read once)."""
    b, h, d = q_bits.shape
    table = pages.table if table is None else table
    K = ra.LlmKernels
    n = K.gqa_decode_paged_workspace_bytes(b, h, n_kv, d, pages.page, table.shape[1])
    if ws is None:
        ws = dev(np.full(max(n, 256), 0xA5, dtype=np.uint8))  # a workspace holds anything
    dout = dev(np.full(q_bits.shape, 0x7B7B, dtype=np.uint16)) if out is None else out
    lens = np.asarray(pages.lens if lens is None else lens, dtype=np.int32)
    keep = dev(q_bits), pages.dev(), dev(table), dev(lens)
    K.gqa_decode_paged_bf16(stream, keep[0], keep[1], dout, keep[2], table.shape[1], keep[3], b, h, n_kv, d, ws, n, shared_len=shared)
    ra.synchronize(stream)
    return dout.download(np.uint16).reshape(q_bits.shape)
