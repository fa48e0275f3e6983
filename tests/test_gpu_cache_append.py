"""rt_qk_norm_rope_kv_append_q4, rt_qk_norm_rope_kv_append_rows_bf16, rt_kv_cache_append_q4_dev and rt_kv_cache_read_q4 against
the definition of the 4-bit cache in numpy (f32, operation by operation) and the oracle's preparation: bit for bit."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values, prepare, q4_dev, quantise, scales, values

pytestmark = pytest.mark.gpu
K = ra.LlmKernels()


def rows_of(rng, *shape):
    """bf16 bits of rows as layers leave them: some channels larger, some rows tiny, some of one value."""
    x = rng.standard_normal(shape).astype(np.float32)
    x *= np.where(rng.random((*shape[:-2], 1, shape[-1])) < 0.05, 6, 1)
    x *= np.where(rng.random((*shape[:-1], 1)) < 0.1, 1e-3, 1)
    x[..., 0, :] = np.where(rng.random(shape[:-2])[..., None] < 0.3, 0.75, x[..., 0, :])
    return bf16_bits(x)


class Case:
    def __init__(self, seed, b, hq, hkv, d, n, seq, norms=(False, False), own_rows=False):
        rng = np.random.default_rng(seed)
        self.dims = b, hq, hkv, d, n, seq
        self.rope = ra.RoPE(d, n + 7)
        self.q, self.k, self.v = rows_of(rng, b, hq, seq, d), rows_of(rng, b, hkv, seq, d), rows_of(rng, b, hkv, seq, d)
        self.positions = rng.integers(0, n - seq + 1, b).astype(np.int32)
        self.positions[0], self.positions[-1] = 0, n - seq
        self.rows = rng.integers(0, n - seq + 1, b).astype(np.int32) if own_rows else None
        self.gamma = [(1 + 0.1 * rng.standard_normal(d)).astype(np.float32) if x else None for x in norms]
        cos, sin = self.rope.cos.reshape(-1, d // 2), self.rope.sin.reshape(-1, d // 2)
        self.want_q = bf16_bits(prepare(bf16_values(self.q), self.gamma[0], 1e-6, cos, sin, self.positions))
        self.want_k = prepare(bf16_values(self.k), self.gamma[1], 1e-6, cos, sin, self.positions)
        self.rng = rng

    def run(self, call, k_cache, v_cache, in_place=False, slots=None, weights=None, stream=None):
        b, hq, hkv, d, n, seq = self.dims
        dq = ra.HipStorage.from_numpy(self.q)
        out = dq if in_place else ra.HipStorage.from_numpy(np.full_like(self.q, 0x7B7B))
        dk, dv = ra.HipStorage.from_numpy(self.k), ra.HipStorage.from_numpy(self.v)
        gamma = [None if g is None else ra.HipStorage.from_numpy(g) for g in self.gamma]
        pos = ra.HipStorage.from_numpy(self.positions)
        rows = None if self.rows is None else ra.HipStorage.from_numpy(self.rows)
        call(stream, dq, out, dk, dv, k_cache, v_cache, pos, self.rope, b, hq, hkv, d, n, q_gamma=gamma[0], k_gamma=gamma[1], seq=seq, rows=rows,
             slots=slots, weights=weights)
        ra.synchronize(stream)
        assert np.array_equal(out.download(np.uint16).reshape(self.q.shape), self.want_q)
        if not in_place:
            assert np.array_equal(dq.download(np.uint16).reshape(self.q.shape), self.q)

    def at(self, i):
        return (self.positions if self.rows is None else self.rows)[i]


SHAPES = [(1, 4, 2, 64, 9, 1), (3, 8, 2, 128, 40, 1), (2, 2, 1, 256, 33, 1), (64, 32, 8, 128, 17, 1), (2, 3, 3, 64, 90, 67), (2, 4, 1, 128, 70, 33),
          (1, 1, 2, 256, 40, 19), (3, 7, 1, 128, 300, 130), (2, 0, 2, 128, 12, 5)]


@pytest.mark.parametrize("norms", [(False, False), (True, True), (False, True)])
@pytest.mark.parametrize("own_rows", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_4_bit_rows_have_the_definitions_bits(shape, own_rows, norms):
    c = Case(1, *shape, norms=norms, own_rows=own_rows)
    b, hq, hkv, d, n, seq = shape
    old_codes, old_pairs = c.rng.integers(0, 256, (b, hkv, n, d // 2)).astype(np.uint8), c.rng.integers(0, 2 ** 32, (b, hkv, d // 64, n)).astype(np.uint32)
    k, v = q4_dev(old_codes, old_pairs), q4_dev(old_codes, old_pairs)
    slots, weights = ra.HipStorage.from_numpy(np.full((b, hkv, n), -7, np.int32)), ra.HipStorage.from_numpy(np.full((b, hkv, n), 3.5, np.float32))
    c.run(K.qk_norm_rope_kv_append_q4, k, v, slots=slots, weights=weights)
    want_s, want_w = np.full((b, hkv, n), -7, np.int32), np.full((b, hkv, n), 3.5, np.float32)
    for i in range(b):
        at = slice(c.at(i), c.at(i) + seq)
        want_s[i, :, at], want_w[i, :, at] = c.positions[i] + np.arange(seq), 0
    assert np.array_equal(slots.download(np.int32).reshape(b, hkv, n), want_s)
    assert np.array_equal(weights.download(np.float32).reshape(b, hkv, n), want_w)
    for cache, new in ((k, c.want_k), (v, bf16_values(c.v))):
        codes, pairs = quantise(new)
        want_codes, want_pairs = old_codes.copy(), old_pairs.copy()
        for i in range(b):
            at = slice(c.at(i), c.at(i) + seq)
            want_codes[i, :, at], want_pairs[i, :, :, at] = codes[i], pairs[i]
        assert np.array_equal(cache.pairs.download(np.uint32).reshape(old_pairs.shape), want_pairs)
        assert np.array_equal(cache.codes.download(np.uint8).reshape(old_codes.shape), want_codes)
        # half a step of the scale, and of its own rounding to f32
        s, _ = scales(pairs)
        assert (np.abs(values(codes, pairs) - new) <= np.repeat(s, 64, -1) * 0.500001 + 2.0 ** -23 * np.abs(new)).all()
        # and read back: by device rows and, the first sequence's, by a host row
        at = c.positions if c.rows is None else c.rows
        out = ra.HipStorage.from_numpy(np.full((b, hkv, seq, d), 0x7B7B, np.uint16))
        K.kv_cache_read_q4(None, cache, out, b, hkv, d, n, ra.HipStorage.from_numpy(np.ascontiguousarray(at)), seq)
        ra.synchronize()
        assert np.array_equal(out.download(np.uint16).reshape(b, hkv, seq, d), bf16_bits(values(codes, pairs)))
        K.kv_cache_read_q4(None, cache, out, b, hkv, d, n, int(at[0]), seq)
        ra.synchronize()
        assert np.array_equal(out.download(np.uint16).reshape(b, hkv, seq, d)[0], bf16_bits(values(codes, pairs))[0])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("norms", [(False, False), (True, True)])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1]])
def test_bf16_rows_of_their_own(oracle, shape, norms, in_place):
    """With the rows at the positions, the bits of the oracle's preparation (those of rt_qk_norm_rope_kv_append_bf16); at
    rows of their own, the same rows there."""
    for own_rows in (False, True):
        c = Case(2, *shape, norms=norms, own_rows=own_rows)
        b, hq, hkv, d, n, seq = shape
        old = c.rng.integers(0, 2 ** 16, (b, hkv, n, d)).astype(np.uint16)
        k, v = ra.HipStorage.from_numpy(old), ra.HipStorage.from_numpy(old)
        c.run(K.qk_norm_rope_kv_append_rows_bf16, k, v, in_place=in_place)
        want_k, want_v = old.copy(), old.copy()
        if own_rows:
            for i in range(b):
                at = slice(c.rows[i], c.rows[i] + seq)
                want_k[i, :, at], want_v[i, :, at] = bf16_bits(c.want_k)[i], c.v[i]
        else:
            oro = oracle.RoPE(d, n + 7)
            oro.cos, oro.sin = c.rope.cos.copy(), c.rope.sin.copy()
            wk, wv = want_k.reshape(-1), want_v.reshape(-1)
            want_q = oracle.decode_prepare_bf16(c.q.reshape(-1), c.k.reshape(-1), c.v.reshape(-1), wk, wv, c.positions, *c.gamma, 1e-6, oro, b, hq, hkv, d, n, seq=seq)
            assert np.array_equal(want_q.reshape(c.want_q.shape), c.want_q)
        assert np.array_equal(k.download(np.uint16).reshape(old.shape), want_k)
        assert np.array_equal(v.download(np.uint16).reshape(old.shape), want_v)


def test_sequences_that_do_not_fit_are_left_untouched():
    b, hq, hkv, d, n, seq = 6, 2, 1, 64, 8, 3
    rng = np.random.default_rng(3)
    rope = ra.RoPE(d, 16)
    q = rows_of(rng, b, hq, seq, d)
    new = rows_of(rng, b, hkv, seq, d)
    positions = np.array([0, 14, -1, 5, 2 ** 31 - 1, 4], dtype=np.int32)  # 14: past the tables
    rows = np.array([5, 0, 0, 6, 0, -1], dtype=np.int32)  # 6: past the cache
    old = rng.integers(0, 256, (b, hkv, n, d // 2)).astype(np.uint8)
    pairs = np.zeros((b, hkv, 1, n), np.uint32)
    k, v = q4_dev(old, pairs), q4_dev(old, pairs)
    out = ra.HipStorage.from_numpy(np.full_like(q, 0x7B7B))
    dk = ra.HipStorage.from_numpy(new)
    K.qk_norm_rope_kv_append_q4(None, ra.HipStorage.from_numpy(q), out, dk, dk, k, v, ra.HipStorage.from_numpy(positions), rope, b, hq, hkv, d, n, seq=seq,
                                rows=ra.HipStorage.from_numpy(rows))
    ra.synchronize()
    got_q, got = out.download(np.uint16).reshape(q.shape), k.codes.download(np.uint8).reshape(old.shape)
    assert (got_q[1:] == 0x7B7B).all() and (got_q[0] != 0x7B7B).any()
    assert np.array_equal(got[1:], old[1:]) and np.array_equal(got[0, :, :5], old[0, :, :5])
    # ... nor read
    back = ra.HipStorage.from_numpy(np.full((b, hkv, seq, d), 0x7B7B, np.uint16))
    K.kv_cache_read_q4(None, v, back, b, hkv, d, n, ra.HipStorage.from_numpy(rows), seq)
    ra.synchronize()
    got = back.download(np.uint16).reshape(b, hkv, seq, d)
    assert (got[[3, 5]] == 0x7B7B).all() and (got[[0, 1, 2, 4]] != 0x7B7B).any()


def test_groups_that_are_not_finite_read_as_nan():
    """A NaN, an infinity or a range that f32 does not hold spoils its 64 dims and no others; zeros and one value are exact."""
    d, n = 128, 8
    x = np.random.default_rng(4).standard_normal((1, 1, n, d)).astype(np.float32)
    x[0, 0, 0, 3], x[0, 0, 1, 70], x[0, 0, 2, 5], x[0, 0, 3, 64:66] = np.nan, np.inf, -np.inf, (3.3e38, -3.3e38)
    x[0, 0, 4] = 0
    x[0, 0, 5] = -2.5
    x[0, 0, 6, :64] = 3.0e38  # one value: z holds it
    bits = bf16_bits(x)
    x = bf16_values(bits)
    cache = ra.Q4Rows.zeros(1, 1, n, d)
    other = ra.Q4Rows.zeros(1, 1, n, d)
    new = ra.HipStorage.from_numpy(bits)
    K.kv_cache_append_q4(None, cache, other, new, n * d, new, n * d, 1, 1, n, d, 0, n)
    out = ra.HipStorage(n * d * 2)
    K.kv_cache_read_q4(None, cache, out, 1, 1, d, n, 0, n)
    ra.synchronize()
    codes, pairs = quantise(x)
    assert np.array_equal(cache.pairs.download(np.uint32), pairs.ravel()) and np.array_equal(cache.codes.download(np.uint8), codes.ravel())
    got = bf16_values(out.download(np.uint16)).reshape(n, d)
    bad = np.isnan(got)
    assert bad[0, :64].all() and bad[1, 64:].all() and bad[2, :64].all() and bad[3, 64:].all() and bad.sum() == 4 * 64 + bad[6, :64].sum()
    assert (got[4] == 0).all() and (got[5] == -2.5).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_kv_cache_of_4_bits(d):
    """KVCache(dtype="q4"): the protocol of the reference, rows as the definition rounds them."""
    b, h, n = 2, 3, 21
    rng = np.random.default_rng(5)
    c = ra.KVCache(2, b, h, d, n, dtype="q4")
    want_k, want_v = np.zeros((b, h, n, d), np.float32), np.zeros((b, h, n, d), np.float32)
    cur = 0
    for seq in (5, 1, 1, 13):
        nk, nv = rows_of(rng, b, h, seq, d), rows_of(rng, b, h, seq, d)
        c.append(1, seq, ra.HipStorage.from_numpy(nk), ra.HipStorage.from_numpy(nv))
        c.advance(seq)
        want_k[:, :, cur:cur + seq], want_v[:, :, cur:cur + seq] = (values(*quantise(bf16_values(x))) for x in (nk, nv))
        cur += seq
        for cache, want in ((c.k_buffer(1), want_k), (c.v_buffer(1), want_v)):
            out = ra.HipStorage(b * h * n * d * 2)
            K.kv_cache_read_q4(None, cache, out, b, h, d, n, 0, n)
            ra.synchronize()
            assert np.array_equal(out.download(np.uint16).reshape(want.shape), bf16_bits(want))
    ra.synchronize()
    assert not c.k_buffer(0).codes.download(np.uint8).any()
    with pytest.raises(ra.Overflow):
        c.append(1, 2, ra.HipStorage(b * h * 2 * d * 2), ra.HipStorage(b * h * 2 * d * 2))
    with pytest.raises(ra.KVWrongInputLen):
        c.append(1, 1, ra.HipStorage(b * h * d * 2 - 2), ra.HipStorage(b * h * d * 2))
    assert c.k_buffer(2) is None and c.dims() == (b, h, n, d)
