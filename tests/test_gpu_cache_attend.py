"""rt_gqa_decode_q4 and rt_gqa_decode_weights_{bf16,q4} against attention in 64 bits over what the caches stand for."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values, expect_bf16, expect_q4, q4_dev, quantise

pytestmark = pytest.mark.gpu
K = ra.LlmKernels()
NAN_PAIR = np.uint32(0x7FC07FC0)


class Case:
    """q and caches of `lens` keys; behind them every row holds NaN."""

    def __init__(self, seed, lens, hq, hkv, d, n, new=1, spread=1.0):
        rng = np.random.default_rng(seed)
        b = len(lens)
        self.dims = b, new, hq, hkv, d, n
        self.lens = np.asarray(lens, dtype=np.int32)
        self.q = bf16_bits(spread * rng.standard_normal((b, new, hq, d)))
        self.k, self.v = (bf16_bits(rng.standard_normal((b, hkv, n, d)) * np.where(rng.random((hkv, 1, d)) < 0.05, 4, 1)) for _ in range(2))
        self.behind = np.arange(n) >= np.clip(self.lens, 0, n)[:, None]

    def q4(self):
        (kc, kp), (vc, vp) = quantise(bf16_values(self.k)), quantise(bf16_values(self.v))
        kp, vp = (np.where(self.behind[:, None, None, :], NAN_PAIR, x).astype(np.uint32) for x in (kp, vp))
        return kc, kp, vc, vp

    def bf16(self):
        return tuple(np.where(self.behind[:, None, :, None], 0x7FC0, x).astype(np.uint16) for x in (self.k, self.v))


def attend_q4(c, caches, stream=None, lens=None):
    b, new, hq, hkv, d, n = c.dims
    kc, kp, vc, vp = caches
    ws = ra.HipStorage.from_numpy(np.full(K.gqa_decode_q4_workspace_bytes(b, new, hq, hkv, d, n) // 4, np.nan, np.float32))
    out = ra.HipStorage.from_numpy(np.full((b, new, hq, d), 0x7B7B, np.uint16))
    K.gqa_decode_q4(stream, ra.HipStorage.from_numpy(c.q), q4_dev(kc, kp), q4_dev(vc, vp), out, ra.HipStorage.from_numpy(c.lens) if lens is None else lens,
                    b, new, hq, hkv, d, n, ws, ws.byte_len)
    ra.synchronize(stream)
    return bf16_values(out.download(np.uint16)).reshape(b, new, hq, d)


def weigh(c, caches, before="in place", stream=None):
    """(out, weights_out, what weights_out held behind the keys)."""
    b, _, hq, hkv, d, n = c.dims
    ws = ra.HipStorage.from_numpy(np.full(K.gqa_decode_weights_workspace_bytes(b, hq, hkv, d, n) // 4, np.nan, np.float32))
    out = ra.HipStorage.from_numpy(np.full((b, hq, d), 0x7B7B, np.uint16))
    sums = np.random.default_rng(9).random((b, hkv, n)).astype(np.float32)
    w_in = ra.HipStorage.from_numpy(sums)
    w_out = w_in if before == "in place" else ra.HipStorage.from_numpy(np.full((b, hkv, n), 77, np.float32))
    args = (w_in if before != "none" else None, w_out, ra.HipStorage.from_numpy(c.lens), b, hq, hkv, d, n, ws, ws.byte_len)
    dq = ra.HipStorage.from_numpy(c.q)
    if len(caches) == 4:
        K.gqa_decode_weights_q4(stream, dq, q4_dev(*caches[:2]), q4_dev(*caches[2:]), out, *args)
    else:
        K.gqa_decode_weights_bf16(stream, dq, *(ra.HipStorage.from_numpy(x) for x in caches), out, *args)
    ra.synchronize(stream)
    got = w_out.download(np.float32).reshape(b, hkv, n)
    stays = sums if before == "in place" else np.full((b, hkv, n), 77, np.float32)
    for i, x in enumerate(c.lens):
        assert np.array_equal(got[i, :, max(int(x), 0):], stays[i, :, max(int(x), 0):])  # behind the keys: as they were
    return bf16_values(out.download(np.uint16)).reshape(b, 1, hq, d), got, sums if before != "none" else np.zeros_like(sums)


HEADS = [(4, 4), (8, 2), (7, 1), (34, 2)]
LENS = [[0, 1, 2, 31, 32, 33], [64, 129, 700, 65], [1500]]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_one_position_over_4_bits(lens, heads, d):
    c = Case(11, lens, *heads, d, max(lens) + 3)
    caches = c.q4()
    expect_q4(bf16_values(c.q), *caches, c.lens).check(attend_q4(c, caches))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,heads", [(2, (8, 2)), (5, (4, 4)), (17, (8, 2)), (40, (6, 1)), (3, (32, 8))])
def test_several_positions_over_4_bits(new, heads, d):
    """Causal among themselves; sequences with fewer keys than new positions have rows of zeros."""
    lens = [new, new + 1, max(0, new - 2), 0, new + 31, 200 + new]
    c = Case(12, lens, *heads, d, max(lens) + 1, new)
    caches = c.q4()
    want = expect_q4(bf16_values(c.q), *caches, c.lens)
    got = attend_q4(c, caches)
    want.check(got)
    assert not got[3].any() and not got[2, :min(2, new)].any()


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS)
def test_weights_are_summed(lens, heads, d, cache):
    c = Case(13, lens, *heads, d, max(lens) + 2, spread=2.0)
    caches = c.q4() if cache == "q4" else c.bf16()
    want = (expect_q4 if cache == "q4" else lambda q, k, v, n: expect_bf16(q, bf16_values(k), bf16_values(v), n))(bf16_values(c.q), *caches, c.lens)
    for before in ("in place", "apart", "none"):
        out, sums, start = weigh(c, caches, before)
        want.check(out, before)
        want.check_weights(sums, start, c.lens, before)
        if before == "none":  # every head's weights are 1 together
            for i, n in enumerate(lens):
                assert np.allclose(sums[i, :, :n].sum(-1), heads[0] // heads[1] if n else 0, rtol=1e-5, atol=0)


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_every_key_counts(d, cache):
    """One key draws all of the attention, wherever it lies: at the ends of steps, of halves of them, of a wave's span, of the
    cache.  The output is its row, the weights are one there and nothing elsewhere."""
    n = 1300
    places = [0, 1, 15, 16, 17, 31, 32, 63, 64, 127, 128, 500, 1023, 1024, 1298, 1299]
    c = Case(14, [n] * len(places), 8, 2, d, n)
    q = bf16_values(c.q)
    k = bf16_values(c.k) * 0.01
    for i, at in enumerate(places):
        k[i, :, at] = q[i, 0, ::4] * (4000 / d)  # the first head of each group: a score far above all others'
    c.q = bf16_bits(np.repeat(q[:, :, ::4], 4, axis=2))
    c.k = bf16_bits(k)
    caches = c.q4() if cache == "q4" else c.bf16()
    out, sums, _ = weigh(c, caches, "none")
    if cache == "q4":
        from _cache import values
        v = values(*caches[2:])
        assert np.array_equal(attend_q4(c, caches), out)
    else:
        v = bf16_values(caches[1])
    for i, at in enumerate(places):
        want = np.repeat(v[i, :, at], 4, axis=0)
        # bf16 rounding, and f32's of the offsets of the codes (31 + 24 steps of a row's range over 16)
        assert (np.abs(out[i, 0] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -12 * np.abs(v[i]).max()).all(), at
        assert np.allclose(sums[i, :, at], 4, rtol=1e-5) and (np.delete(sums[i], at, axis=-1) < 1e-6).all(), at


def test_more_sequences_than_a_wave_has_lanes_and_lengths_out_of_range():
    """150 sequences; lengths above the cache are the cache, below zero nothing."""
    rng = np.random.default_rng(15)
    lens = rng.integers(0, 90, 150)
    lens[[3, 77]], lens[[5, 149]] = -4, 1000
    c = Case(16, lens, 4, 2, 64, 89)
    caches = c.q4()
    clipped = np.clip(lens, 0, 89)
    want = expect_q4(bf16_values(c.q), *caches, clipped)
    want.check(attend_q4(c, caches))
    out, sums, start = weigh(c, caches)
    want.check(out)
    want.check_weights(sums, start, clipped)


@pytest.mark.parametrize("new", [1, 6])
def test_one_length_on_the_host_is_that_length_on_the_device(new):
    c = Case(17, [900, 900], 8, 2, 128, 1000, new)
    caches = c.q4()
    assert np.array_equal(attend_q4(c, caches), attend_q4(c, caches, lens=900))


def test_what_is_not_finite_stays_where_it_is_seen():
    """A NaN row among the visible keys spoils the rows that see it and no others; behind the last key a row may hold anything."""
    d, n, new = 128, 100, 8
    c = Case(18, [80, 80, 80], 8, 2, d, n, new)
    kc, kp, vc, vp = c.q4()
    vp[0, 1, 1, 76] = NAN_PAIR  # seen from position 76 on: new position 4 of sequence 0, dims 64 on
    kp[1, 0, 0, 79] = NAN_PAIR  # the last key: the last position alone, all of its dims
    got = attend_q4(c, (kc, kp, vc, vp))
    bad = np.isnan(got)
    assert bad[0, 4:, 4:, 64:].all() and bad[1, 7, :4].all()
    assert bad.sum() == 4 * 4 * 64 + 4 * d
    clean = Case(18, [80, 80, 80], 8, 2, d, n, new)
    assert np.array_equal(got[~bad], attend_q4(clean, clean.q4())[~bad])
    # one position, bf16: an infinite key draws everything or nothing, a NaN spoils its kv head
    c = Case(19, [50], 8, 2, d, n)
    k, v = c.bf16()
    k[0, 0, 7] = 0x7F80
    v[0, 1, 9, 3] = 0x7FC0
    out, sums, _ = weigh(c, (k, v), "none")
    assert np.isnan(out[0, 0, 4:, 3]).all() and np.isfinite(out[0, 0, 4:, 4:]).all() and np.isfinite(sums[0, 1, :50]).all()
    assert np.isnan(out[0, 0, :4]).any()


def test_large_and_tiny_values():
    """Scores in the hundreds, values of 1e4 beside values of 1e-6: every sum is f32."""
    c = Case(20, [400, 33], 8, 2, 128, 410, spread=8.0)
    v = bf16_values(c.v)
    v *= np.where(np.random.default_rng(21).random(v.shape[:-1])[..., None] < 0.5, 1e4, 1e-6)
    c.v = bf16_bits(v)
    caches = c.q4()
    want = expect_q4(bf16_values(c.q), *caches, c.lens)
    want.check(attend_q4(c, caches))
    out, sums, start = weigh(c, c.bf16())
    want = expect_bf16(bf16_values(c.q), *(bf16_values(x) for x in c.bf16()), c.lens)
    want.check(out)
    want.check_weights(sums, start, c.lens)


def test_calls_on_two_streams_with_workspaces_of_their_own():
    cases = [Case(22, [700, 33, 129], 8, 2, 128, 800), Case(23, [65, 900], 32, 8, 64, 901)]
    want = [attend_q4(c, c.q4()) for c in cases]
    streams = [ra.Stream(), ra.Stream()]
    held, outs = [], []
    for _ in range(3):
        for c, s in zip(cases, streams):
            b, new, hq, hkv, d, n = c.dims
            kc, kp, vc, vp = c.q4()
            ws, out = ra.HipStorage(K.gqa_decode_q4_workspace_bytes(b, new, hq, hkv, d, n)), ra.HipStorage(c.q.nbytes)
            held.append((ra.HipStorage.from_numpy(c.q), q4_dev(kc, kp), q4_dev(vc, vp), ra.HipStorage.from_numpy(c.lens), ws))
            outs.append(out)
            K.gqa_decode_q4(s, *held[-1][:3], out, held[-1][3], b, new, hq, hkv, d, n, ws, ws.byte_len)
    for s in streams:
        s.synchronize()
    for i, out in enumerate(outs):
        assert np.array_equal(bf16_values(out.download(np.uint16)).reshape(want[i % 2].shape), want[i % 2])


def test_rows_past_32_bits():
    """One head of 2^27 + 40 rows of 32 bytes: offsets of 4 GiB.  All keys are zeros but the last, which draws everything."""
    d, n = 64, 2 ** 27 + 40
    k, v = ra.Q4Rows.zeros(1, 1, n, d), ra.Q4Rows.zeros(1, 1, n, d)
    rng = np.random.default_rng(24)
    q = bf16_bits(rng.standard_normal((1, 1, 2, d)))
    q[0, 0, 1] = q[0, 0, 0]
    row = bf16_bits(bf16_values(q[0, 0, 0]) * 40)
    value = bf16_bits(rng.standard_normal(d))
    K.kv_cache_append_q4(None, k, v, ra.HipStorage.from_numpy(row), d, ra.HipStorage.from_numpy(value), d, 1, 1, n, d, n - 1, 1)
    out = ra.HipStorage(2 * d * 2)
    ws = ra.HipStorage(K.gqa_decode_q4_workspace_bytes(1, 1, 2, 1, d, n))
    K.gqa_decode_q4(None, ra.HipStorage.from_numpy(q), k, v, out, n, 1, 1, 2, 1, d, n, ws, ws.byte_len)
    back = ra.HipStorage(d * 2)
    K.kv_cache_read_q4(None, v, back, 1, 1, d, n, n - 1, 1)
    ra.synchronize()
    want = bf16_values(back.download(np.uint16))
    got = bf16_values(out.download(np.uint16)).reshape(2, d)
    assert np.abs(want).max() > 1 and (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -12).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [(8, 2), (34, 2)])
@pytest.mark.parametrize("q_by,k_by,v_by", [(40, -40, 0), (-40, 40, 0), (-70, 70, 0), (90, -90, 0), (0, 0, 50), (0, 0, -50), (-30, 30, 40)])
def test_powers_of_two_in_q_k_and_v_leave_the_bits(q_by, k_by, v_by, heads, d):
    """q and K scaled against each other, V by itself: every scale and middle is so many times as large exactly, and so is the output.  (The products of codes
    and the other operand are scaled into a range of their own; it has to follow the values'.)"""
    lens = [333, 70]
    base, c = Case(25, lens, *heads, d, 340), Case(25, lens, *heads, d, 340)
    for name, by in (("q", q_by), ("k", k_by), ("v", v_by)):
        setattr(c, name, bf16_bits(bf16_values(getattr(base, name)) * np.float32(2.0 ** by)))
    a, b = base.q4(), c.q4()
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[2], b[2])
    out, sums, _ = weigh(base, a)
    got, got_sums, _ = weigh(c, b)
    assert np.array_equal(got, out * np.float32(2.0 ** v_by)) and np.array_equal(got_sums, sums)
    assert np.array_equal(attend_q4(c, b), got)


@pytest.mark.parametrize("spread", [0.0, 1.0, 40.0])
@pytest.mark.parametrize("by", [43, -50])
def test_v_at_the_ends_of_its_range_over_many_keys(by, spread):
    """8192 keys: values of up to 2^60 / 8192 (2^47: 4 x 4 times 2^43), and down to 2^-50."""
    base, c = Case(28, [8192], 8, 2, 128, 8192, spread=spread), Case(28, [8192], 8, 2, 128, 8192, spread=spread)
    v = np.clip(bf16_values(base.v), -16, 16)
    base.v, c.v = bf16_bits(v), bf16_bits(v * np.float32(2.0 ** by))
    out = attend_q4(base, base.q4())
    assert np.isfinite(out).all() and np.array_equal(attend_q4(c, c.q4()), out * np.float32(2.0 ** by))


def test_q_of_zeros_and_of_the_smallest_values():
    """All keys weigh alike where q is zero, and as good as alike where its values are subnormal numbers."""
    c = Case(26, [100], 4, 2, 128, 100)
    caches = c.q4()
    for bits in (0, 0x8000, 0x0001, 0x8055):
        c.q = np.full_like(c.q, bits)
        want = expect_q4(bf16_values(c.q), *caches, c.lens)
        want.check(attend_q4(c, caches))
        out, sums, start = weigh(c, caches, "none")
        want.check(out)
        want.check_weights(sums, start, c.lens)


@pytest.mark.parametrize("kind", ["q4", "weights q4", "weights bf16"])
def test_replays_over_long_caches(kind):
    """A segment in many workgroups' pieces, joined by the last of them: recorded once, replayed between eager calls on the same workspace and
    on another, over lengths that change in between."""
    from test_gpu_decode_graph import NODE_TYPE_MEMSET, Hip

    ra.init(0)
    hip, stream, d, n = Hip(), ra.Stream(), 128, 9000
    b, hq, hkv = 2, 8, 2
    c = Case(27, [n, n], hq, hkv, d, n)
    q = ra.HipStorage.from_numpy(c.q)
    caches = [ra.HipStorage.from_numpy(x) for x in (c.bf16() if kind == "weights bf16" else c.q4())]
    lens = ra.HipStorage.from_numpy(np.array([n, 17], np.int32))
    rows = caches if kind == "weights bf16" else [ra.Q4Rows(*caches[:2]), ra.Q4Rows(*caches[2:])]
    size = K.gqa_decode_q4_workspace_bytes(b, 1, hq, hkv, d, n) if kind == "q4" else K.gqa_decode_weights_workspace_bytes(b, hq, hkv, d, n)
    spaces = [ra.HipStorage.from_numpy(np.full(size // 4, np.nan, np.float32)) for _ in range(2)]
    results = [(ra.HipStorage(b * hq * d * 2), ra.HipStorage(b * hkv * n * 4)) for _ in range(2)]

    def call(which, space):
        out, sums = results[which]
        if kind == "q4":
            K.gqa_decode_q4(stream, q, *rows, out, lens, b, 1, hq, hkv, d, n, spaces[space], size)
        else:
            (K.gqa_decode_weights_q4 if kind == "weights q4" else K.gqa_decode_weights_bf16)(stream, q, *rows, out, None, sums, lens, b, hq, hkv, d, n, spaces[space], size)

    def seen(which, now):
        stream.synchronize()
        sums = results[which][1].download(np.float32).reshape(b, hkv, n)
        return results[which][0].download(np.uint16), [] if kind == "q4" else [sums[i, :, :x] for i, x in enumerate(now)]

    graph, exe, types = hip.capture(stream, lambda: call(0, 0))
    assert NODE_TYPE_MEMSET not in types
    for now in ([n, 17], [n, n], [4097, 8191], [0, n], [n, n]):
        lens.upload(np.array(now, np.int32))
        for space in (0, 1, 0):
            call(1, space)
            want = seen(1, now)
            for _ in range(2):
                hip.launch(exe, stream)
                got = seen(0, now)
                assert np.array_equal(got[0], want[0]), now
                assert all(np.array_equal(x, y) for x, y in zip(got[1], want[1])), now
    hip.destroy(graph, exe)


@pytest.mark.parametrize("value", [2.0 ** 112, -(2.0 ** 127), np.inf, -np.inf, np.nan])
def test_a_row_of_q_beyond_its_range_is_nan_and_no_other(value):
    c = Case(32, [150], 8, 2, 128, 150)
    caches = c.q4()
    out, sums, _ = weigh(c, caches, "none")
    c.q[0, 0, 2, 77] = bf16_bits(np.float32(value))
    got, got_sums, _ = weigh(c, caches, "none")
    assert np.isnan(got[0, 0, 2]).all() and np.isnan(got_sums[0, 0]).all()
    rest = np.delete(np.arange(8), 2)
    assert np.array_equal(got[0, 0, rest], out[0, 0, rest]) and np.array_equal(got_sums[0, 1], sums[0, 1])


def test_scores_far_below_zero_are_scores():
    """Scores of -2^62, -2^63, ...: the least of them in size draws everything."""
    c = Case(30, [40], 4, 2, 128, 40)
    c.q = bf16_bits(np.full(c.q.shape, 2.0 ** -60))
    c.k = bf16_bits(np.broadcast_to(-(2.0 ** 115) * (1 + np.arange(40, dtype=np.float64))[::-1][:, None], c.k.shape))
    caches = c.q4()
    out, sums, _ = weigh(c, caches, "none")
    from _cache import values
    want = np.repeat(values(*caches[2:])[0, :, 39], 2, axis=0)
    assert (np.abs(out[0, 0] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -12 * np.abs(want).max()).all()
    assert np.array_equal(sums[0, :, 39], [2, 2]) and not sums[0, :, :39].any()
    assert np.array_equal(attend_q4(c, caches), out)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_constant_rows_of_v_come_out_as_they_are(d):
    """A group of equal values has s = 0: zeros give zeros, not what a scale of next to nothing would leave."""
    c = Case(29, [300, 1, 33], 8, 2, d, 300)
    v = np.repeat(np.array([0.0, -3.0, 1.5, 0.0], np.float32)[: max(d // 64, 1)], 64)
    c.v = bf16_bits(np.broadcast_to(v, c.v.shape))
    out, _, _ = weigh(c, c.q4())
    assert np.array_equal(out, np.broadcast_to(v, out.shape)) and np.array_equal(attend_q4(c, c.q4()), out)


@pytest.mark.parametrize("d,b,hq,hkv", [(64, 16, 8, 4), (128, 10, 8, 4), (256, 6, 6, 2)])
def test_batches_that_fill_the_chip(d, b, hq, hkv):
    """More steps than workgroups take at their least: spans that end inside sequences, of which some are empty or short."""
    lens = [2600 + 17 * i for i in range(b)]
    lens[3], lens[b // 2] = 0, 5
    c = Case(31, lens, hq, hkv, d, 2900)
    caches = c.q4()
    want = expect_q4(bf16_values(c.q), *caches, c.lens)
    want.check(attend_q4(c, caches))
    out, sums, start = weigh(c, caches)
    want.check(out)
    want.check_weights(sums, start, c.lens)
    caches = c.bf16()
    want = expect_bf16(bf16_values(c.q), *(bf16_values(x) for x in caches), c.lens)
    out, sums, start = weigh(c, caches)
    want.check(out)
    want.check_weights(sums, start, c.lens)
