"""Attention of prompts packed one behind the other, against attention in 64 bits of each sequence alone."""
import ctypes as C

import numpy as np
import pytest

import rustorch_amd as ra
from rustorch_amd import _lib as L
from _cache import bf16_values
from _gpu import assert_within_rounding
from _paged import dev, normal_bits

pytestmark = pytest.mark.gpu


def run(q, k, v, starts, batch=None, stream=None):
    t, h, d = q.shape
    out = dev(np.full(q.shape, 0x7B7B, dtype=np.uint16))
    starts = np.asarray(starts, dtype=np.int32)
    shape = ra.AttentionShape.new(len(starts) - 1 if batch is None else batch, h, t, d)
    keep = dev(q), dev(k), dev(v), dev(starts)
    ra.flash_forward_packed_bf16_dev(shape, *keep, out, n_kv_heads=k.shape[1], stream=stream)
    ra.synchronize(stream)
    return out.download(np.uint16).reshape(q.shape)


def expect(q, k, v, starts):
    """(values, the same over |v|); NaN for tokens of no sequence."""
    t, h, d = q.shape
    g = h // k.shape[1]
    q, k, v = (bf16_values(x).astype(np.float64) for x in (q, k, v))
    out, size = np.full(q.shape, np.nan), np.zeros(q.shape)
    for a, b in zip(starts[:-1], starts[1:]):
        for j in range(h):
            x = q[a:b, j] @ k[a:b, j // g].T / np.sqrt(d)
            x = np.where(np.tri(b - a, dtype=bool), x, -np.inf)
            p = np.exp(x - x.max(-1, keepdims=True)) if b > a else x
            p = p / p.sum(-1, keepdims=True)
            out[a:b, j], size[a:b, j] = p @ v[a:b, j // g], p @ np.abs(v[a:b, j // g])
    return out, size


def check(seed, lens, heads, n_kv, dim, tail=0, head=0):
    rng = np.random.default_rng(seed)
    starts = head + np.concatenate([[0], np.cumsum(lens)])
    t = int(starts[-1]) + tail
    q, k, v = normal_bits(rng, t, heads, dim), normal_bits(rng, t, n_kv, dim), normal_bits(rng, t, n_kv, dim)
    # what belongs to no sequence holds NaN, and is not written
    for x in (q, k, v):
        x[:head] = x[int(starts[-1]):] = 0x7FC1
    got = run(q, k, v, starts)
    free = np.ones(t, dtype=bool)
    free[head:int(starts[-1])] = False
    assert (got[free] == 0x7B7B).all()
    if sum(lens):
        want, size = expect(q, k, v, starts)
        assert_within_rounding(bf16_values(got)[~free], want[~free], size[~free])


@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 72, 80, 96, 112, 128, 136, 160, 192, 256])
@pytest.mark.parametrize("lens", [[1, 2, 31, 33, 64, 0, 65, 129, 5], [130, 260, 127, 128]])
def test_head_dims(dim, lens):
    check(dim, lens, 4, 2, dim, tail=7)


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (8, 8), (32, 8), (28, 4), (7, 1), (16, 2), (40, 8)])
def test_grouped_heads(heads, n_kv):
    check(heads, [100, 3, 70], heads, n_kv, 64)


@pytest.mark.parametrize("dim,heads,lens", [(64, 16, [700, 90, 1100]), (128, 8, [1300, 20, 900]), (256, 4, [600, 333]), (80, 4, [900, 1000]), (32, 2, [1500])])
def test_long_sequences(dim, heads, lens):
    check(dim, lens, heads, heads, dim)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_one_long_sequence_on_few_heads(dim):
    """The launch that cuts a walk in two halves."""
    check(dim, [1700], 2, 1, dim)


@pytest.mark.parametrize("dim,heads,lens", [(128, 32, [1300]), (64, 16, [900, 130, 1000]), (80, 40, [1200]), (256, 16, [100, 1700])])
def test_walks_in_halves_two_to_a_cu(dim, heads, lens):
    check(dim, lens, heads, heads // 4, dim)


@pytest.mark.parametrize("dim,heads", [(64, 32), (128, 32), (256, 16)])
def test_more_tiles_than_the_chip_holds(dim, heads):
    check(dim, [300, 10, 500, 129, 400, 257, 200, 380], heads, heads // 4, dim)


@pytest.mark.parametrize("dim,heads,n_kv,batch,longest", [(64, 32, 8, 40, 60), (128, 32, 8, 70, 40), (80, 40, 8, 20, 60), (256, 16, 2, 40, 30), (96, 32, 2, 43, 280), (32, 28, 4, 60, 100),
                                                          (128, 24, 8, 32, 300), (256, 12, 4, 16, 300), (16, 34, 2, 60, 50), (136, 20, 1, 22, 3), (64, 32, 8, 12, 700)])
def test_many_sequences_of_grouped_heads(dim, heads, n_kv, batch, longest):
    rng = np.random.default_rng(dim + batch)
    check(dim, [int(x) for x in rng.integers(0, longest + 1, batch)], heads, n_kv, dim, tail=9, head=3)


def test_nan_among_many_sequences_of_grouped_heads():
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(1, 60, 40)]
    starts = np.concatenate([[0], np.cumsum(lens)])
    t, at = int(starts[-1]), int(starts[7])
    q, k, v = normal_bits(rng, t, 32, 64), normal_bits(rng, t, 8, 64), normal_bits(rng, t, 8, 64)
    want, size = expect(q, k, v, starts)
    k[at, 3, 5], v[at + lens[7], 2, 9] = 0x7FC1, 0x7FC1  # its first token's key; the next sequence's first V row
    got = bf16_values(run(q, k, v, starts))
    ill = np.zeros(got.shape, dtype=bool)
    ill[at:at + lens[7], 12:16] = True
    ill[at + lens[7]:at + lens[7] + lens[8], 8:12, 9] = True
    assert np.isnan(got[ill]).all()
    assert_within_rounding(got[~ill], want[~ill], size[~ill])


@pytest.mark.parametrize("batch", [63, 64, 65, 150])
def test_many_sequences(batch):
    rng = np.random.default_rng(batch)
    check(batch, [int(x) for x in rng.integers(0, 200, batch)], 2, 1, 64, tail=3)


def test_tokens_of_no_sequence():
    check(1, [50, 200], 4, 2, 64, tail=300, head=77)
    check(2, [0, 0, 0], 4, 2, 64, tail=30)


def test_starts_that_are_out_of_range_stay_within_the_tensors():
    """Read as ascending and within the tokens there are."""
    rng = np.random.default_rng(3)
    q, k, v = (normal_bits(rng, 60, 2, 64) for _ in range(3))
    for starts, read in (([-5, 20, 90], [0, 20, 60]), ([0, 30, 10], [0, 30, 30]), ([2 ** 31 - 1, 2 ** 31 - 1], [60, 60]), ([-2 ** 31, 2 ** 31 - 1], [0, 60])):
        got = run(q, k, v, starts)
        want, size = expect(q, k, v, read)
        on = slice(read[0], read[-1])
        assert (got[read[-1]:] == 0x7B7B).all()
        if read[-1] > read[0]:
            assert_within_rounding(bf16_values(got)[on], want[on], size[on])


def test_the_rows_of_the_same_prompt_alone():
    """Against the entry for [batch, seq, heads, dim], each sequence by itself, both within their rounding."""
    rng = np.random.default_rng(4)
    lens, h, d = [257, 40], 8, 128
    starts = [0, 257, 297]
    q, k, v = normal_bits(rng, 297, h, d), normal_bits(rng, 297, 2, d), normal_bits(rng, 297, 2, d)
    got = bf16_values(run(q, k, v, starts))
    _, size = expect(q, k, v, starts)
    for a, n in zip(starts, lens):
        out = ra.HipStorage(n * h * d * 2)
        ra.flash_forward_bnhd_bf16_dev(ra.AttentionShape.new(1, h, n, d), dev(q[a:a + n]), dev(k[a:a + n]), dev(v[a:a + n]), out, ra.Mask.causal(), n_kv_heads=2)
        ra.synchronize()
        alone = bf16_values(out.download(np.uint16).reshape(n, h, d))
        assert (np.abs(got[a:a + n] - alone) <= (2.0 ** -7 + 2.0 ** -12) * 2 * size[a:a + n]).all()


def test_infinities_and_nan_stay_in_their_sequence():
    rng = np.random.default_rng(6)
    lens = [100, 150, 80]
    q, k, v = (normal_bits(rng, 330, 2, 64) for _ in range(3))
    want, size = expect(q, k, v, [0, 100, 250, 330])
    k[249, :, 3], v[249, :, 5], v[100, :, 6] = 0x7FC1, 0x7F80, 0x7FC1
    got = bf16_values(run(q, k, v, [0, 100, 250, 330]))
    for a, b in ((0, 100), (250, 330)):
        assert_within_rounding(got[a:b], want[a:b], size[a:b])
    assert np.isnan(got[100:250, :, 6]).all() and np.isnan(got[249]).all()


def test_the_strict_rule_for_non_finite_v():
    rng = np.random.default_rng(7)
    q, k, v = (normal_bits(rng, 900, 2, 64) for _ in range(3))
    v[699, 1, 5] = 0x7F80  # the second sequence's last token, which its others do not see
    was = ra.set_strict_non_finite_v(True)
    try:
        got = bf16_values(run(q, k, v, [0, 100, 700, 900]))
    finally:
        ra.set_strict_non_finite_v(was)
    want, size = expect(q, k, v, [0, 100, 700, 900])
    bad = np.zeros(got.shape, dtype=bool)
    bad[100:699, 1, 5] = True
    assert np.isnan(got[bad]).all() and np.isposinf(got[699, 1, 5])
    bad[699, 1, 5] = True
    assert_within_rounding(got[~bad], want[~bad], size[~bad])


@pytest.mark.parametrize("lens", [[60, 40], [5] * 20])
def test_rows_behind_four_gigabytes(lens):
    """Queries and outputs of 4.9 GB, of which the last tokens belong to sequences."""
    rng = np.random.default_rng(13)
    t, n, h, d = 600000, sum(lens), 32, 128
    starts = t - n + np.concatenate([[0], np.cumsum(lens)])
    q, k, v = normal_bits(rng, n, h, d), normal_bits(rng, n, 1, d), normal_bits(rng, n, 1, d)
    bufs = [ra.HipStorage(t * heads * d * 2) for heads in (h, 1, 1, h)]
    out = np.full(q.shape, 0x7B7B, dtype=np.uint16)

    def copy(call, buf, host):
        err, at = L.RtErr(), buf.ptr + buf.byte_len - host.nbytes
        a, b = (at, host.ctypes.data) if call == "rt_memcpy_h2d" else (host.ctypes.data, at)
        assert getattr(L.lib(), call)(a, b, host.nbytes, None, C.byref(err)) == 0
        ra.synchronize()

    for buf, host in zip(bufs, (q, k, v, out)):
        copy("rt_memcpy_h2d", buf, host)
    ra.flash_forward_packed_bf16_dev(ra.AttentionShape.new(len(lens), h, t, d), *bufs[:3], dev(starts.astype(np.int32)), bufs[3], n_kv_heads=1)
    copy("rt_memcpy_d2h", bufs[3], out)
    want, size = expect(q, k, v, starts - (t - n))
    assert_within_rounding(bf16_values(out), want, size)


@pytest.mark.parametrize("dim,heads,n_kv,lens", [(64, 16, 16, [77, 300, 150]), (128, 16, 4, [1300, 20, 900]), (64, 32, 8, [5] * 40), (256, 8, 2, [100, 700, 33]), (128, 2, 1, [1700])])
def test_the_same_call_gives_the_same_bits(dim, heads, n_kv, lens):
    """A head's rows, a group's, walks in halves: nothing depends on the order in which workgroups end."""
    rng = np.random.default_rng(15)
    starts = np.concatenate([[0], np.cumsum(lens)])
    t = int(starts[-1])
    q, k, v = normal_bits(rng, t, heads, dim), normal_bits(rng, t, n_kv, dim), normal_bits(rng, t, n_kv, dim)
    first = run(q, k, v, starts)
    for _ in range(4):
        assert np.array_equal(run(q, k, v, starts), first)
