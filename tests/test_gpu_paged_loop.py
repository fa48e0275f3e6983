"""Requests side by side, as a server runs them: prompts packed one behind the other, their rows in pages, conversations that go on from a
prompt that they share, and decode steps that are recorded once and replayed, with what the program does in between."""
import ctypes as C

import numpy as np
import pytest

import rustorch_amd as ra
from rustorch_amd import _lib as L
from _cache import bf16_values
from _gpu import assert_within_rounding
from _paged import Pages, attention, dev, normal_bits, run_decode
from test_gpu_decode_graph import NODE_TYPE_MEMSET, Hip
from test_gpu_packed_prompts import expect as expect_prompts
from test_gpu_paged_append import Tables, rotated

pytestmark = pytest.mark.gpu
K = ra.LlmKernels

HEADS, N_KV, DIM, PAGE, ROWS = 8, 2, 64, 32, 400


class Layer:
    """What the device has of one layer, and the rows of every sequence as they must be."""

    def __init__(self, rng, cache, index):
        self.rng, self.pages = rng, cache.layer(index)
        self.gammas = [rng.standard_normal(DIM, dtype=np.float32) for _ in range(2)]
        self.d_gammas = [dev(g) for g in self.gammas]
        self.rows = {}  # sequence: [k, v], bits [rows, n_kv, dim]

    def tokens(self, n):
        self.q, self.k, self.v = (normal_bits(self.rng, n, h, DIM) for h in (HEADS, N_KV, N_KV))
        return self.q, self.k, self.v

    def appended(self, rope, seqs, positions, counts):
        """The step's rotated q and k, and the rows that its sequences have now."""
        at = np.concatenate([p + np.arange(n) for p, n in zip(positions, counts)])
        q = rotated(self.q, self.gammas[0], 1e-6, rope.cos[at], rope.sin[at])
        k = rotated(self.k, self.gammas[1], 1e-6, rope.cos[at], rope.sin[at])
        first = np.concatenate([[0], np.cumsum(counts)])
        for i, seq in enumerate(seqs):
            new = [x[first[i]:first[i + 1]] for x in (k, self.v)]
            self.rows[seq] = [np.concatenate([a, b]) for a, b in zip(self.rows[seq], new)] if seq in self.rows else new
        return q, k

    def expect(self, q, seqs):
        out = [attention(bf16_values(q[i]).astype(np.float64), *(bf16_values(x).astype(np.float64).transpose(1, 0, 2) for x in self.rows[seq])) for i, seq in enumerate(seqs)]
        return np.stack([x[0] for x in out]), np.stack([x[1] for x in out])


@pytest.mark.parametrize("prefix", [64, 0])
def test_prompts_then_forks_then_recorded_steps(prefix):
    rng = np.random.default_rng(prefix)
    hip, stream, others = Hip(), ra.Stream(), ra.Stream()
    rope = Tables(rng, DIM, ROWS)
    cache = ra.PagedKVCache(2, 6, N_KV, DIM, n_pages=40, page_size=PAGE, table_pages=8)
    layers = [Layer(rng, cache, i) for i in range(2)]
    # prompts: one that will be shared, and two others
    lens = [100, 37, 1]
    prompts = [cache.add() for _ in lens]
    for seq, n in zip(prompts, lens):
        cache.reserve(seq, n)
    starts, t = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), sum(lens)
    d_starts, d_table, d_zero = dev(starts), dev(cache.table(prompts)), dev(np.zeros(3, dtype=np.int32))
    for x in layers:
        q, k, v = (dev(a) for a in x.tokens(t))
        out = ra.HipStorage(t * HEADS * DIM * 2)
        K.qk_norm_rope_kv_append_paged_bf16(stream.handle, q, q, k, v, x.pages, d_table, 8, d_zero, rope, t, 3, HEADS, N_KV, DIM, starts=d_starts,
                                            k_out=k, q_gamma=x.d_gammas[0], k_gamma=x.d_gammas[1])
        ra.flash_forward_packed_bf16_dev(ra.AttentionShape.new(3, HEADS, t, DIM), q, k, v, d_starts, out, n_kv_heads=N_KV, stream=stream.handle)
        stream.synchronize()
        want, sizes = expect_prompts(*x.appended(rope, prompts, [0, 0, 0], lens), x.v, starts)
        assert_within_rounding(bf16_values(out.download(np.uint16).reshape(want.shape)), want, sizes, "prompts")
    for seq, n in zip(prompts, lens):
        cache.advance(seq, n)
    # conversations that go on from the first prompt's first 64 rows, and the prompts' own; the short ones share nothing, and one of
    # them comes first
    forks = [cache.add(prefix_of=prompts[0], shared=64) for _ in range(2)]
    for x in layers:
        for seq in forks:
            x.rows[seq] = [a[:64] for a in x.rows[prompts[0]]]
    seqs, steps = [prompts[1], *forks, prompts[0], prompts[2]], 4
    for seq in seqs:
        cache.reserve(seq, steps)
    b, at = len(seqs), cache.lengths(seqs)
    d_table, d_pos, d_lens = dev(cache.table(seqs)), dev(at), dev(at + 1)
    n = K.gqa_decode_paged_workspace_bytes(b, HEADS, N_KV, DIM, PAGE, 8)
    state = [[ra.HipStorage(b * h * DIM * 2) for h in (HEADS, N_KV, N_KV, HEADS)] + [ra.HipStorage(n)] for _ in layers]

    def step(s, x, of, positions, lengths):
        K.qk_norm_rope_kv_append_paged_bf16(s, of[0], of[0], of[1], of[2], x.pages, d_table, 8, positions, rope, b, b, HEADS, N_KV, DIM,
                                            q_gamma=x.d_gammas[0], k_gamma=x.d_gammas[1])
        K.gqa_decode_paged_bf16(s, of[0], x.pages, of[3], d_table, 8, lengths, b, HEADS, N_KV, DIM, of[4], n, shared_len=shared)

    # a graph for each layer, with a workspace of its own: they may run side by side
    shared = dev(np.array([prefix], dtype=np.int32)) if prefix else 0
    graphs = [hip.capture(s.handle, lambda s=s, x=x, of=of: step(s.handle, x, of, d_pos, d_lens)) for s, x, of in zip((stream, others), layers, state)]
    for _, _, types in graphs:
        assert NODE_TYPE_MEMSET not in types and len(types) == (3 if prefix else 2)
    for i in range(steps):
        for x, of in zip(layers, state):
            for buf, a in zip(of, x.tokens(b)):
                buf.upload(a)
        ra.synchronize()
        for s, (_, exe, _) in zip((stream, others), graphs):
            hip.launch(exe, s.handle)
        stream.synchronize()
        others.synchronize()
        for which, (x, of) in enumerate(zip(layers, state)):
            q, _ = x.appended(rope, seqs, at + i, [1] * b)
            want, sizes = x.expect(q, seqs)
            got = of[3].download(np.uint16).reshape(b, HEADS, DIM)
            assert_within_rounding(bf16_values(got), want, sizes, f"step {i} layer {which}")
            # the same attention again, eagerly, with a workspace that holds something else: the same bits
            ws, out = dev(np.full(n, 0x5A, dtype=np.uint8)), ra.HipStorage(b * HEADS * DIM * 2)
            K.gqa_decode_paged_bf16(None, of[0], x.pages, out, d_table, 8, d_lens, b, HEADS, N_KV, DIM, ws, n, shared_len=shared)
            ra.synchronize()
            assert np.array_equal(out.download(np.uint16).reshape(got.shape), got)
        for buf in (d_pos, d_lens):
            ra.i32_add_dev(buf, b, 1)
    # every sequence's rows are in its pages, the shared ones as the prompt left them
    table = cache.table(seqs)
    for x in layers:
        for which, pool in enumerate((x.pages.k, x.pages.v)):
            pool = pool.download(np.uint16).reshape(40, N_KV, PAGE, DIM)
            for i, seq in enumerate(seqs):
                for r, row in enumerate(x.rows[seq][which]):
                    assert np.array_equal(pool[table[i, r // PAGE], :, r % PAGE], row), (i, r)
    for graph, exe, _ in graphs:
        hip.destroy(graph, exe)
    stream.destroy()
    others.destroy()


def test_calls_side_by_side_have_the_bits_of_calls_alone():
    rng = np.random.default_rng(11)
    streams, sets = [ra.Stream(), ra.Stream()], []
    for i, shared in enumerate((0, 500)):
        lens = [500 + int(x) for x in rng.integers(0, 900, 20)]
        pages, q = Pages(rng, lens, 4, 128, 16, shared), normal_bits(rng, 20, 16, 128)
        n = K.gqa_decode_paged_workspace_bytes(20, 16, 4, 128, 16, pages.table_pages)
        shared = dev(np.array([shared], dtype=np.int32)) if shared else 0
        sets.append((run_decode(q, pages, 4, shared), [dev(q), pages.dev(), ra.HipStorage(q.nbytes), dev(pages.table), pages.table_pages,
                                                       dev(np.array(lens, dtype=np.int32)), 20, 16, 4, 128, ra.HipStorage(n), n], shared))
    for _ in range(20):
        for s, (_, args, shared) in zip(streams, sets):
            K.gqa_decode_paged_bf16(s.handle, *args, shared_len=shared)
    for s, (want, args, _) in zip(streams, sets):
        s.synchronize()
        assert np.array_equal(args[2].download(np.uint16).reshape(want.shape), want)
        s.destroy()


def test_pages_behind_four_gigabytes():
    """The same rows in a small pool and in one of 5 GiB: the same bits; and an append finds its row there."""
    rng = np.random.default_rng(12)
    n_kv, dim, page, n_pages = 8, 128, 64, 40000
    lens = [300, 130]
    pages, q = Pages(rng, lens, n_kv, dim, page), normal_bits(rng, 2, 32, dim)
    want = run_decode(q, pages, n_kv)
    size = n_kv * page * dim * 2
    far = rng.permutation(np.concatenate([np.arange(n_pages - 4, n_pages), np.arange(32760, 32764), [0, 1, 2, 3]]))[:pages.n_pages]
    pool = ra.KVPages(ra.HipStorage(n_pages * size), ra.HipStorage(n_pages * size), n_pages, page)

    def copy(call, device, host):
        err = L.RtErr()
        a, b = (device, host.ctypes.data) if call == "rt_memcpy_h2d" else (host.ctypes.data, device)
        assert getattr(L.lib(), call)(a, b, size, None, C.byref(err)) == 0
        ra.synchronize()

    for i, p in enumerate(far):
        for buf, host in ((pool.k, pages.k), (pool.v, pages.v)):
            copy("rt_memcpy_h2d", buf.ptr + int(p) * size, host[i])
    table = np.where(pages.table >= 0, far[pages.table], -1).astype(np.int32)
    n = K.gqa_decode_paged_workspace_bytes(2, 32, n_kv, dim, page, table.shape[1])
    out, d_table, d_lens = ra.HipStorage(q.nbytes), dev(table), dev(np.array(lens, dtype=np.int32))
    K.gqa_decode_paged_bf16(None, dev(q), pool, out, d_table, table.shape[1], d_lens, 2, 32, n_kv, dim, ra.HipStorage(n), n)
    ra.synchronize()
    assert np.array_equal(out.download(np.uint16).reshape(want.shape), want)
    new = [normal_bits(rng, 2, h, dim) for h in (32, n_kv, n_kv)]
    keep = [dev(x) for x in new]
    rope = Tables(rng, dim, 400)
    K.qk_norm_rope_kv_append_paged_bf16(None, keep[0], keep[0], keep[1], keep[2], pool, d_table, table.shape[1], d_lens, rope, 2, 2, 32, n_kv, dim)
    ra.synchronize()
    k = rotated(new[1], None, 0.0, rope.cos[lens], rope.sin[lens])
    for i, at in enumerate(lens):
        p = int(table[i, at // page])
        for buf, host, row in ((pool.k, pages.k, k[i]), (pool.v, pages.v, new[2][i])):
            got, exp = np.empty((n_kv, page, dim), dtype=np.uint16), host[pages.table[i, at // page]].copy()
            exp[:, at % page] = row
            copy("rt_memcpy_d2h", buf.ptr + p * size, got)
            assert np.array_equal(got, exp)


def test_recorded_calls_that_share_a_workspace():
    """One behind the other on one stream: without a prefix, with one on the device and with one that the host gives, recorded, replayed in
    turn and mixed with calls that are not recorded.  What a call leaves in the workspace is nothing to the next, and lengths that change
    between replays are those that a replay finds."""
    rng = np.random.default_rng(16)
    hip, stream, calls = Hip(), ra.Stream(), []
    for batch, prefix, shared in ((20, 0, 0), (20, 500, dev(np.array([500], dtype=np.int32))), (48, 900, 900)):
        lens = [max(prefix, 400) + 4 + int(x) for x in rng.integers(0, 300, batch)]
        pages, q = Pages(rng, lens, 8, 128, 32, prefix), normal_bits(rng, batch, 16, 128)
        at = [[n - 3 + i for n in lens] for i in range(3)]  # three steps' lengths; some of them at a unit's end
        want = [run_decode(q, pages, 8, shared, lens=x) for x in at]
        n = K.gqa_decode_paged_workspace_bytes(batch, 16, 8, 128, 32, pages.table_pages)
        calls.append(dict(q=dev(q), pages=pages.dev(), out=ra.HipStorage(q.nbytes), table=dev(pages.table), columns=pages.table_pages, lens=ra.HipStorage(batch * 4), at=at, batch=batch,
                          n=n, shared=shared, want=want))
    ws = dev(np.full(max(c["n"] for c in calls), 0x5A, dtype=np.uint8))

    def call(c, s):
        K.gqa_decode_paged_bf16(s, c["q"], c["pages"], c["out"], c["table"], c["columns"], c["lens"], c["batch"], 16, 8, 128, ws, c["n"], shared_len=c["shared"])

    graphs = [hip.capture(stream.handle, lambda c=c: call(c, stream.handle)) for c in calls]
    assert [len(types) for _, _, types in graphs] == [1, 2, 2]
    for i in range(12):
        for j in rng.permutation(3):
            c = calls[j]
            c["lens"].upload(np.array(c["at"][i % 3], dtype=np.int32))
            if (i + j) % 4 == 3:
                call(c, stream.handle)
            else:
                hip.launch(graphs[j][1], stream.handle)
            if i % 2:  # (every other time the next call is enqueued behind this one)
                stream.synchronize()
        stream.synchronize()
        for c in calls:
            got = c["out"].download(np.uint16).reshape(c["want"][0].shape)
            assert np.array_equal(got, c["want"][i % 3])
    for graph, exe, _ in graphs:
        hip.destroy(graph, exe)
    stream.destroy()
