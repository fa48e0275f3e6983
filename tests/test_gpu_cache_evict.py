"""rt_kv_evict_{bf16,q4} against the definition, head by head: rows, sums and positions bit for bit, and everything else as
it was."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import evict, q4_dev

pytestmark = pytest.mark.gpu
K = ra.LlmKernels()


def state(seed, lens, hkv, n, ties=True):
    rng = np.random.default_rng(seed)
    b = len(lens)
    w = np.exp(2 * rng.standard_normal((b, hkv, n))).astype(np.float32)
    if ties:
        w = np.where(rng.random(w.shape) < 0.4, rng.integers(0, 3, w.shape), w).astype(np.float32)
    slots = np.stack([[rng.permutation(n + 5)[:n] for _ in range(hkv)] for _ in range(b)]).astype(np.int32)
    return w, slots, np.asarray(lens, dtype=np.int32), rng


def check(w, slots, lens, budget, recent, d, q4, rng, in_place=True, stream=None, lens_in_place=False):
    b, hkv, n = w.shape
    source, new = evict(w, slots, lens, budget, recent)
    if q4:
        k = [rng.integers(0, 256, (b, hkv, n, d // 2)).astype(np.uint8) for _ in range(2)]
        p = [rng.integers(0, 2 ** 32, (b, hkv, d // 64, n)).astype(np.uint32) for _ in range(2)]
        dk, dv = (q4_dev(x, y) for x, y in zip(k, p))
    else:
        k = [rng.integers(0, 2 ** 16, (b, hkv, n, d)).astype(np.uint16) for _ in range(2)]
        p = []
        dk, dv = (ra.HipStorage.from_numpy(x) for x in k)
    dw, ds, dl = ra.HipStorage.from_numpy(w), ra.HipStorage.from_numpy(slots), ra.HipStorage.from_numpy(lens)
    if in_place:
        ow, os_, want_w, want_s = dw, ds, w.copy(), slots.copy()
    else:
        want_w, want_s = np.full_like(w, 55), np.full_like(slots, -55)
        ow, os_ = ra.HipStorage.from_numpy(want_w), ra.HipStorage.from_numpy(want_s)
    nl = dl if lens_in_place else ra.HipStorage.from_numpy(np.full(b, -9, np.int32))
    ws = ra.HipStorage.from_numpy(np.full(max(K.kv_evict_workspace_bytes(b, hkv, n, budget), 4) // 4, 0x7B7B7B7B, np.uint32))
    (K.kv_evict_q4 if q4 else K.kv_evict_bf16)(stream, dk, dv, dw, ds, ow, os_, dl, nl, b, hkv, d, n, budget, recent, ws, ws.byte_len)
    ra.synchronize(stream)
    for i in range(b):
        for j in range(hkv):
            at, m = source[i, j, :new[i]], new[i]
            want_w[i, j, :m], want_s[i, j, :m] = w[i, j, at], slots[i, j, at]
            for x in k:
                x[i, j, :m] = x[i, j, at]
            for x in p:
                x[i, j, :, :m] = x[i, j][:, at]
    assert np.array_equal(nl.download(np.int32), new)
    assert np.array_equal(os_.download(np.int32).reshape(slots.shape), want_s)
    assert np.array_equal(ow.download(np.uint32).reshape(w.shape), want_w.view(np.uint32))
    for got, x in zip((dk, dv), k):
        assert np.array_equal((got.codes if q4 else got).download(x.dtype).reshape(x.shape), x)
    for got, x in zip((dk, dv), p):
        assert np.array_equal(got.pairs.download(np.uint32).reshape(x.shape), x)
    if not in_place:
        assert np.array_equal(dw.download(np.uint32), w.view(np.uint32).ravel()) and np.array_equal(ds.download(np.int32), slots.ravel())


@pytest.mark.parametrize("q4", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (7, 3), (64, 64), (100, 0), (300, 10), (1023, 200), (1500, 1)])
def test_rows_that_stay(budget, recent, d, q4):
    w, slots, lens, rng = state(31, [0, 1, budget, budget + 1, 1200, 2100], 2, 2111)
    lens = np.minimum(lens, 2111)
    check(w, slots, lens, budget, recent, d, q4, rng, in_place=d != 128, lens_in_place=d == 256)


def test_nothing_stays_and_everything_stays():
    w, slots, lens, rng = state(32, [5, 0, 40], 3, 40)
    check(w, slots, lens, 0, 0, 64, False, rng)
    check(w, slots, lens, 40, 12, 64, True, rng, in_place=False)
    check(w, slots, lens, 1000, 0, 64, False, rng)


def test_sums_that_are_no_numbers_zeros_and_infinite():
    w, slots, lens, rng = state(33, [600, 600], 2, 600, ties=False)
    w[:, :, rng.permutation(600)[:200]] = np.nan
    w[:, :, rng.permutation(600)[:150]] = -0.0
    w[:, :, rng.permutation(600)[:150]] = 0.0
    w[0, :, rng.permutation(600)[:90]] = np.inf
    w[1, :, rng.permutation(600)[:90]] = -np.inf
    w[1, 1, :50] = -w[1, 1, :50]
    for budget, recent in ((50, 0), (80, 30), (333, 5), (590, 0)):
        check(w, slots, lens, budget, recent, 128, False, rng)


def test_all_sums_alike():
    """The lower rows stay, but for the newest tokens."""
    w, slots, lens, rng = state(34, [1025, 3000], 1, 3000)
    w[:] = 1.5
    slots[:] = np.arange(3000)
    check(w, slots, lens, 1024, 100, 64, True, rng)
    check(w, slots, lens, 1024, 0, 64, False, rng)


def test_lengths_out_of_range_and_a_long_cache():
    w, slots, lens, rng = state(35, [-3, 70000], 1, 33000)
    check(w, slots, lens, 5000, 77, 64, True, rng, stream=ra.Stream())


def test_a_row_a_token():
    """At the budget, every token evicts one row: in place, call after call, the definition's state."""
    n, budget, recent, d = 40, 32, 4, 64
    w, slots, lens, rng = state(36, [33, 33], 2, n)
    for _ in range(5):
        check(w, slots, lens, budget, recent, d, False, rng)
        source, new = evict(w, slots, lens, budget, recent)
        for i in range(2):
            for j in range(2):
                w[i, j, :budget], slots[i, j, :budget] = w[i, j, source[i, j]], slots[i, j, source[i, j]]
                w[i, j, budget], slots[i, j, budget] = 0, slots[i, j, :budget].max() + 1
        w[:, :, :33] += rng.random((2, 2, 33)).astype(np.float32)


@pytest.mark.parametrize("n", [8191, 8192, 8193, 20000])
@pytest.mark.parametrize("budget", [1, 8000, 8191, 8192, 12000])
def test_around_the_slots_that_registers_hold(n, budget):
    """Threads of eight slots each, tiles of 8192, equal sums on both sides of their ends."""
    w, slots, lens, rng = state(37, [n, n - 3, min(budget + 1, n)], 1, n)
    check(w, slots, lens, budget, min(budget, 500), 64, True, rng, in_place=budget < 8192)


@pytest.mark.parametrize("n", [5000, 9000])
def test_sums_a_bit_apart_and_far_apart(n):
    """Every range that the counts divide: sums that differ in their last bit, beside some from all over f32."""
    w, slots, lens, rng = state(38, [n] * 4, 1, n, ties=False)
    near = (np.uint32(0x40490FDB) + rng.permutation(n).astype(np.uint32)).view(np.float32)
    w[0, 0] = near
    w[1, 0] = np.where(rng.random(n) < 0.3, np.ldexp(rng.standard_normal(n), rng.integers(-140, 120, n)), near)
    w[2, 0] = rng.integers(0, 2 ** 32, n, dtype=np.uint64).astype(np.uint32).view(np.float32)
    w[3, 0] = np.where(rng.random(n) < 0.5, np.float32(1), np.float32(1 + 2.0 ** -23))
    for budget, recent in ((1, 0), (n // 3, 40), (n - 1, 0)):
        check(w, slots, lens, budget, recent, 64, False, rng)


def test_positions_at_the_ends_of_32_bits():
    for low in (-2 ** 31, 2 ** 31 - 300):
        w, slots, lens, rng = state(39, [300, 200], 2, 300)
        slots[:] = (low + np.argsort(rng.random(slots.shape), axis=-1)).astype(np.int64)
        check(w, slots, lens, 120, 50, 64, False, rng)
    w, slots, lens, rng = state(40, [300], 1, 300)
    slots[0, 0, ::2] = -2 ** 31 + np.arange(150)
    slots[0, 0, 1::2] = 2 ** 31 - 150 + np.arange(150)
    check(w, slots, lens, 100, 30, 64, False, rng)
    check(w, slots, lens, 200, 160, 64, False, rng)
