"""Decode steps over a cache in pages, with and without a shared prefix, against attention in 64 bits."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values
from _gpu import assert_within_rounding
from _paged import NAN_BITS, Pages, dev, expect_decode, normal_bits, run_decode

pytestmark = pytest.mark.gpu

HEADS = [(8, 8), (32, 8), (28, 4), (16, 2), (40, 8), (34, 2), (20, 1), (5, 1), (16, 1), (17, 1)]


def on_device(n):
    return dev(np.array([n], dtype=np.int32))


def check(q, pages, n_kv, shared=0, label="", **more):
    """With a prefix: its length given by the host, which chooses, and on the device, which has it read once."""
    want, sizes = expect_decode(q, pages, more.get("lens"))
    for way in (shared, on_device(shared)) if shared else (0,):
        got = bf16_values(run_decode(q, pages, n_kv, way, **more))
        assert_within_rounding(got, want, sizes, label)


@pytest.mark.parametrize("dim", [64, 128, 256, 16, 80, 96, 112, 160, 192])
@pytest.mark.parametrize("page", [16, 64])
def test_lengths_around_pages_and_steps(dim, page):
    rng = np.random.default_rng(dim + page)
    lens = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 0, 300]
    pages = Pages(rng, lens, 2, dim, page)
    check(normal_bits(rng, len(lens), 8, dim), pages, 2)


@pytest.mark.parametrize("heads,n_kv", HEADS)
def test_query_heads_of_a_kv_head(heads, n_kv):
    rng = np.random.default_rng(heads)
    pages = Pages(rng, [70, 3, 260], n_kv, 64, 32)
    check(normal_bits(rng, 3, heads, 64), pages, n_kv)


@pytest.mark.parametrize("page", [16, 32, 128, 256, 512, 1024])
def test_every_page_size(page):
    rng = np.random.default_rng(page)
    pages = Pages(rng, [1500, page, page + 1, max(page - 1, 1)], 2, 64, page)
    check(normal_bits(rng, 4, 8, 64), pages, 2)


@pytest.mark.parametrize("batch,heads,n_kv,dim,longest", [(1, 32, 8, 128, 5000), (1, 8, 1, 64, 40000), (3, 16, 2, 256, 3000), (70, 8, 2, 64, 400), (200, 4, 1, 128, 90), (33, 32, 8, 128, 700), (700, 8, 4, 128, 60), (40, 16, 16, 112, 500)])
def test_long_contexts_and_many_sequences(batch, heads, n_kv, dim, longest):
    rng = np.random.default_rng(batch)
    lens = [longest] + [int(x) for x in rng.integers(0, longest + 1, batch - 1)]
    pages = Pages(rng, lens, n_kv, dim, 16)
    check(normal_bits(rng, batch, heads, dim), pages, n_kv)


@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("shared", [1, 16, 31, 32, 33, 100, 256])
def test_a_shared_prefix(dim, shared):
    rng = np.random.default_rng(dim + shared)
    lens = [shared + n for n in (0, 1, 15, 16, 31, 33, 90)] + [0, shared - 1, max(shared - 20, 0)]
    pages = Pages(rng, lens, 2, dim, 16, shared)
    q = normal_bits(rng, len(lens), 8, dim)
    check(q, pages, 2, shared)


@pytest.mark.parametrize("heads,n_kv", HEADS)
@pytest.mark.parametrize("batch", [1, 2, 40])
def test_a_shared_prefix_and_query_heads(heads, n_kv, batch):
    rng = np.random.default_rng(heads + batch)
    lens = [150 + int(x) for x in rng.integers(0, 70, batch)]
    pages = Pages(rng, lens, n_kv, 64, 32, 150)
    check(normal_bits(rng, batch, heads, 64), pages, n_kv, 150)


@pytest.mark.parametrize("batch,heads,n_kv,dim,shared,own", [(64, 32, 8, 128, 2000, 100), (1, 8, 1, 64, 9000, 50), (100, 4, 1, 64, 3000, 10), (24, 16, 16, 64, 1001, 700), (16, 16, 2, 256, 1500, 300), (130, 8, 2, 128, 64, 500)])
def test_long_prefixes(batch, heads, n_kv, dim, shared, own):
    rng = np.random.default_rng(batch)
    lens = [shared + int(x) for x in rng.integers(0, own, batch)]
    if batch > 3:
        lens[2], lens[3] = shared // 2, 0
    pages = Pages(rng, lens, n_kv, dim, 64, shared)
    check(normal_bits(rng, batch, heads, dim), pages, n_kv, shared)


@pytest.mark.parametrize("ahead", [1, 70])
def test_a_prefix_behind_sequences_that_do_not_have_it(ahead):
    """Idle slots and short sequences come first, with rows of the table of their own."""
    rng = np.random.default_rng(ahead)
    lens = [0 if i % 3 == 0 else 20 + i for i in range(ahead)] + [200, 99, 130, 100]
    pages = Pages(rng, lens, 2, 64, 16, 100)
    check(normal_bits(rng, len(lens), 8, 64), pages, 2, 100)


def test_a_prefix_that_nobody_has_whole():
    rng = np.random.default_rng(5)
    pages = Pages(rng, [10, 0, 99], 2, 64, 16)
    check(normal_bits(rng, 3, 8, 64), pages, 2, 100)


@pytest.mark.parametrize("shared", [0, 130])
def test_rows_that_have_no_page(shared):
    """Entries that are no page hide their keys, in the middle and at the end, of the prefix too; all of them: zeros."""
    rng = np.random.default_rng(9)
    lens, page = [300, 200, 260, 131], 32
    pages = Pages(rng, lens, 2, 128, page, shared)
    q = normal_bits(rng, 4, 8, 128)
    table, hidden = pages.table.copy(), {i: [] for i in range(4)}

    def hide(i, c, entry):
        table[i, c] = entry
        hidden[i] += list(range(c * page, min((c + 1) * page, lens[i])))

    hide(0, 7, -1)
    hide(1, 6, pages.n_pages)
    hide(2, 5, 2 ** 31 - 1)
    hide(2, 8, -2 ** 31)
    if shared:  # the prefix is read through the first sequence's row
        table[0, 1] = -5
        for i in range(4):
            hidden[i] += list(range(page, 2 * page))
    way = on_device(shared) if shared else 0
    got = bf16_values(run_decode(q, pages, 2, way, table=table))
    want, sizes = expect_decode(q, pages, hidden=hidden)
    assert_within_rounding(got, want, sizes)
    assert not run_decode(q, pages, 2, way, table=np.full_like(table, -1)).any()


def test_what_is_not_seen_does_not_count():
    """Rows behind a sequence's last, other sequences' pages and, where the prefix is read once, own copies of shared rows hold NaN or
    infinities."""
    rng = np.random.default_rng(3)
    lens, shared, page = [75, 90, 64, 71], 70, 16
    pages = Pages(rng, lens, 2, 64, page, shared)
    for i in (1, 3):  # the prefix's last page is everybody's own: only the first sequence's is read
        own = pages.table[i, shared // page]
        pages.k[own, :, :shared % page] = NAN_BITS
        pages.v[own, :, :shared % page] = 0x7F80
    q = normal_bits(rng, 4, 8, 64)
    want, sizes = expect_decode(q, pages)
    assert_within_rounding(bf16_values(run_decode(q, pages, 2, on_device(shared))), want, sizes)


def test_infinities_and_nan_that_are_seen():
    rng = np.random.default_rng(4)
    pages = Pages(rng, [40, 50, 60], 1, 64, 16)
    pages.v[pages.table[1, 2], 0, 3, 7] = NAN_BITS
    pages.v[pages.table[2, 0], 0, 1, 9] = 0x7F80
    q = normal_bits(rng, 3, 4, 64)
    got = bf16_values(run_decode(q, pages, 1))
    want, sizes = expect_decode(q, pages)
    # (an infinite one may come out NaN: a weight that is too small for f32 is zero)
    assert np.isnan(got[1, :, 7]).all() and not np.isfinite(got[2, :, 9]).any()
    got[1, :, 7], got[2, :, 9] = want[1, :, 7], want[2, :, 9]
    assert_within_rounding(got, want, sizes)


def test_scores_far_from_zero():
    """A common offset of all scores, and a maximum that keeps rising along the keys."""
    rng = np.random.default_rng(8)
    lens = [700, 300]
    pages = Pages(rng, lens, 1, 128, 16)
    q = normal_bits(rng, 2, 4, 128)
    q[..., 5] = 0x4100  # 8
    for i in range(2):
        ramp = (np.arange(lens[i], dtype=np.float32) - 300) * 2
        bits = ramp.view(np.uint32).astype(np.uint32)
        pages.rows_k[i][0, :, 5] = (bits >> 16).astype(np.uint16)
        for r in range(lens[i]):
            pages.k[pages.table[i, r // 16], 0, r % 16] = pages.rows_k[i][0, r]
    check(q, pages, 1)


def test_the_same_call_gives_the_same_bits_and_any_workspace_will_do():
    rng = np.random.default_rng(2)
    lens = [2100, 2001, 3000, 2500]
    pages = Pages(rng, lens, 4, 128, 16, 2000)
    q = normal_bits(rng, 4, 16, 128)
    n = ra.LlmKernels.gqa_decode_paged_workspace_bytes(4, 16, 4, 128, 16, pages.table_pages)
    for shared in (on_device(2000), 0):
        first = run_decode(q, pages, 4, shared)
        for fill in (0, 0xFF, 0x7F):
            ws = dev(np.full(n, fill, dtype=np.uint8))
            for _ in range(3):
                assert np.array_equal(run_decode(q, pages, 4, shared, ws=ws), first)


def test_lengths_outside_the_table_count_as_its_ends():
    rng = np.random.default_rng(6)
    pages = Pages(rng, [48, 48], 1, 64, 16, more_columns=0)
    q = normal_bits(rng, 2, 4, 64)
    got = bf16_values(run_decode(q, pages, 1, lens=[2 ** 31 - 1, -7]))
    want, sizes = expect_decode(q, pages, lens=[48, 0])
    assert_within_rounding(got, want, sizes)


@pytest.mark.parametrize("shared", [0, 40])
def test_caches_without_pages(shared):
    """No page at all, and no column in the table: nothing is seen."""
    rng = np.random.default_rng(10)
    q = normal_bits(rng, 3, 8, 64)
    for n_pages, columns in ((0, 4), (2, 0), (0, 0)):
        n = ra.LlmKernels.gqa_decode_paged_workspace_bytes(3, 8, 2, 64, 16, columns)
        out, pool = dev(np.full(q.shape, 0x7B7B, dtype=np.uint16)), dev(np.full((max(n_pages, 1), 2, 16, 64), NAN_BITS, dtype=np.uint16))
        keep = dev(q), dev(np.zeros((3, max(columns, 1)), dtype=np.int32)), dev(np.array([50, 64, 7], dtype=np.int32)), dev(np.full(n, 0xA5, dtype=np.uint8))
        ra.LlmKernels.gqa_decode_paged_bf16(None, keep[0], ra.KVPages(pool, pool, n_pages, 16), out, keep[1], columns, keep[2], 3, 8, 2, 64, keep[3], n,
                                            shared_len=on_device(shared) if shared else 0)
        ra.synchronize()
        assert not out.download(np.uint16).any(), (n_pages, columns)


def test_a_prefix_that_is_read_once_or_by_each():
    """The same call with the prefix's length from the host, below and above where it is read once, and on the device."""
    rng = np.random.default_rng(12)
    for batch, shared in ((6, 600), (48, 900)):
        lens = [shared + int(x) for x in rng.integers(0, 90, batch)]
        pages = Pages(rng, lens, 8, 128, 32, shared)
        check(normal_bits(rng, batch, 16, 128), pages, 8, shared)


@pytest.mark.parametrize("batch,shared,once", [(48, 900, True), (6, 600, False)])
def test_the_rows_that_a_prefix_is_read_through(batch, shared, once):
    """Every sequence has pages of its own for the rows that are the same for all.  NaN in some of them shows whose are read: the first
    sequence's, where the prefix is read once, or everybody's own."""
    rng = np.random.default_rng(batch)
    lens = [shared + 1 + int(x) for x in rng.integers(0, 90, batch)]
    pages = Pages(rng, lens, 8, 128, 32)
    full = shared // 32
    for rows, pool in ((pages.rows_k, pages.k), (pages.rows_v, pages.v)):
        for i in range(1, batch):
            rows[i][:, :shared] = rows[0][:, :shared]
            pool[pages.table[i, :full]] = pool[pages.table[0, :full]]
            pool[pages.table[i, full], :, :shared % 32] = pool[pages.table[0, full], :, :shared % 32]
    q = normal_bits(rng, batch, 16, 128)
    want, sizes = expect_decode(q, pages)
    assert_within_rounding(bf16_values(run_decode(q, pages, 8, 0)), want, sizes)
    others, first = [pages.table[i, 3] for i in range(1, batch)], pages.table[0, 3]
    for way, read_once in ((shared, once), (on_device(shared), True)):
        assert_within_rounding(bf16_values(run_decode(q, pages, 8, way)), want, sizes)
        for poisoned, seen in ((others, [] if read_once else range(1, batch)), (first, range(batch) if read_once else [0])):
            was = pages.v[poisoned].copy()
            pages.v[poisoned] = NAN_BITS
            got = bf16_values(run_decode(q, pages, 8, way))
            pages.v[poisoned] = was
            ill = np.isin(np.arange(batch), list(seen))
            assert np.isnan(got[ill]).all()
            if not ill.all():
                assert_within_rounding(got[~ill], want[~ill], sizes[~ill])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shared", [0, 70])
def test_scores_of_minus_infinity(dim, shared):
    """Keys that are seen and have no weight: beside others they count nothing, and of them alone the softmax is NaN, as in
    gqa_decode_batched_bf16; zeros are what sequences have that see no key."""
    rng = np.random.default_rng(dim + shared)
    least = np.uint16(0xFF80)
    # of each sequence the rows whose scores are -infinity (dim 3 of q is 1): with a prefix that is all of it, part of it, or none
    for pre in (shared, shared // 2, 0):
        lens = [shared + n for n in (1, 33, 100, 5000, 64)] + [0]
        own = [slice(shared, None), slice(shared, None), slice(shared, shared + 90), slice(shared, shared + 4900), slice(0, 0), slice(0, 0)]
        pages = Pages(rng, lens, 1, dim, 16, shared)
        q = normal_bits(rng, len(lens), 6, dim)
        q[..., 3] = 0x3F80
        for i, n in enumerate(lens):
            if n:
                pages.rows_k[i][0, :pre, 3] = least
                pages.rows_k[i][0, own[i], 3] = least
                for r in range(n):
                    pages.k[pages.table[i, r // 16], 0, r % 16, 3] = pages.rows_k[i][0, r, 3]
        table = pages.table.copy()
        table[4, shared // 16 + 1:] = -1  # (sees little beside the prefix, and nothing without: page shared / 16 is its own)
        hidden = {4: range((shared // 16 + 1) * 16, lens[4])}
        if not shared:
            table[4] = -1
            hidden = {4: range(lens[4])}
        with np.errstate(invalid="ignore"):
            want, sizes = expect_decode(q, pages, hidden=hidden)
        ill = np.isnan(want)
        assert ill[0].all() == (pre == shared) and not ill[4:].any()
        for way in (shared, on_device(shared)) if shared else (0, on_device(0)):
            got = bf16_values(run_decode(q, pages, 1, way, table=table))
            assert np.array_equal(np.isnan(got), ill)
            assert_within_rounding(got[~ill], want[~ill], sizes[~ill])
            assert not got[5].any() and (shared or not got[4].any())


@pytest.mark.parametrize("shared", [0, 70])
@pytest.mark.parametrize("power", [10, 31, 40, 77, 120])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_finite_size(shared, power, sign):
    """q and k of one dim alone, so that scores are exact: of two values, a 64th apart, of which the smaller has no weight."""
    rng = np.random.default_rng(power + shared)
    lens = [shared + n for n in (1, 40, 900, 6000)]
    pages = Pages(rng, lens, 1, 128, 16, shared)
    q = np.zeros((4, 6, 128), dtype=np.uint16)
    q[..., 5] = bf16_bits(np.float32(sign * 1.375 * 2.0 ** (power // 2)))
    for i, n in enumerate(lens):
        x = np.full(n, 1.5 * 2.0 ** (power - power // 2), dtype=np.float32)
        x[1::3] *= np.float32(1 - 2.0 ** -6)
        pages.rows_k[i][...] = 0
        pages.rows_k[i][0, :, 5] = bf16_bits(x)
        for r in range(n):
            pages.k[pages.table[i, r // 16], :, r % 16] = pages.rows_k[i][:, r]
    check(q, pages, 1, shared)
