"""Attention over caches against 64 bits to within what its arithmetic is made of: weights of 16 bits, exponentials and sums in f32, one
rounding to bf16 (`_cache_bounds`; test_cache_precision_cpu.py shows which faults that tells apart)."""
from types import SimpleNamespace

import numpy as np
import pytest

from _cache import bf16_bits, bf16_values, quantise
from _cache_bounds import LEAST, Near, exact_k_bf16, exact_k_q4, pair_words, score_slack, small_q, v_q4
from test_gpu_cache_attend import attend_q4, weigh

pytestmark = pytest.mark.gpu


def drawn(seed, cache, lens, heads, d, rows, new=1):
    rng = np.random.default_rng(seed)
    shape = (len(lens), heads[1], rows, d)
    c = SimpleNamespace(dims=(len(lens), new, *heads, d, rows), lens=np.asarray(lens, np.int32), q=small_q(rng, (len(lens), new, heads[0], d)))
    if cache == "q4":
        return c, (*exact_k_q4(rng, shape), *v_q4(rng, shape))
    return c, (exact_k_bf16(rng, shape), bf16_bits(rng.standard_normal(shape).astype(np.float32)))


HEADS = [(4, 4), (8, 2), (8, 1), (34, 2)]  # 1, 4, 8 and 17 query rows a kv head


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", [[1, 33, 300, 64], [700]])
def test_outputs_and_sums_where_scores_are_exact(lens, heads, d, cache):
    c, caches = drawn(51, cache, lens, heads, d, max(lens) + 5)
    near = Near(c.q, caches, lens)
    out, sums, before = weigh(c, caches)
    near.check(out)
    near.check_rows(out)
    near.check_weights(sums, before, lens)
    _, sums, before = weigh(c, caches, "none")
    near.check_weights(sums, before, lens, "from zeros")
    if cache == "q4":
        near.check(attend_q4(c, caches), "without sums")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,heads", [(2, (4, 4)), (5, (8, 2)), (19, (8, 1))])
def test_several_positions_where_scores_are_exact(new, heads, d):
    lens = [new, 250, 31 + new, 0]
    c, caches = drawn(52, "q4", lens, heads, d, 251, new)
    near = Near(c.q, caches, lens)
    got = attend_q4(c, caches)
    near.check(got)
    near.check_rows(got)


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_key_wherever_it_lies(d, cache):
    """A key that draws everything, at the ends of steps, of halves of them, of a wave's turn, of the cache: the output is its row, to within the
    steps of that row's own codes."""
    n, heads = 1300, (8, 2)
    places = [0, 1, 15, 16, 17, 31, 32, 63, 64, 127, 128, 500, 1023, 1024, 1298, 1299]
    c, caches = drawn(53, cache, [n] * len(places), heads, d, n)
    q = bf16_values(c.q)[:, :, ::4]
    c.q = bf16_bits(np.repeat(q, 4, axis=2))
    caches = [x.copy() for x in caches]
    if cache == "q4":
        codes, pairs = caches[:2]
        codes[:] = 0x88  # c - 8 = 0, and the middles are 0: scores of 0 but for one key
        pairs[:] = pair_words(np.full(pairs.shape, LEAST, np.float32), np.zeros(pairs.shape, np.float32))
        from _cache import chunk_of
        for i, at in enumerate(places):
            sign = np.where(q[i, 0] > 0, 15, 1).reshape(2, d // 32, 16, 2)  # 7 or -7 times 2^1
            for p in range(d // 32):
                two = sign[:, chunk_of(p, d // 32)]
                codes[i, :, at].reshape(2, 16, d // 32)[..., p] = two[..., 0] | two[..., 1] << 4
            pairs[i, :, :, at] = pair_words(np.float32(2), np.float32(0))
    else:
        caches[0][:] = 0
        for i, at in enumerate(places):
            caches[0][i, :, at] = bf16_bits(np.where(q[i, 0] > 0, 14, -14).astype(np.float32))
    near = Near(c.q, caches, c.lens)
    assert all((near.weights[i, :, at] > 4 - 1e-6).all() for i, at in enumerate(places))
    out, sums, before = weigh(c, caches, "none")
    near.check(out)
    near.check_weights(sums, before, c.lens)
    if cache == "q4":
        near.check(attend_q4(c, caches), "without sums")


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", HEADS)
def test_rows_of_ordinary_operands(heads, d, cache):
    lens = [300, 33, 1]
    rng = np.random.default_rng(54)
    k, v = (bf16_bits(rng.standard_normal((3, heads[1], 301, d)).astype(np.float32)) for _ in range(2))
    c = SimpleNamespace(dims=(3, 1, *heads, d, 301), lens=np.asarray(lens, np.int32), q=bf16_bits(rng.standard_normal((3, 1, heads[0], d)).astype(np.float32)))
    caches = (*quantise(bf16_values(k)), *quantise(bf16_values(v))) if cache == "q4" else (k, v)
    near = Near(c.q, caches, lens, score_slack(c.q, caches))
    out, sums, before = weigh(c, caches)
    near.check_rows(out)
    near.check_weights(sums, before, lens)


@pytest.mark.parametrize("cache", ["q4", "weights q4", "weights bf16"])
@pytest.mark.parametrize("d,heads,lens", [(64, (16, 16), [37, 3001, 900, 0, 2500, 1]), (128, (32, 8), [8192]), (128, (32, 8), [600, 5000, 33]), (256, (16, 2), [4000, 1000])])
def test_the_same_call_gives_the_same_bits(d, heads, lens, cache):
    """Over segments that one workgroup has and such as many join, whichever of them is last."""
    c, caches = drawn(55, "bf16" if cache == "weights bf16" else "q4", lens, heads, d, max(lens))
    first = None
    for _ in range(6):
        got = (attend_q4(c, caches),) if cache == "q4" else weigh(c, caches)[:2]
        first = first or got
        assert all(np.array_equal(x, y) for x, y in zip(got, first))
