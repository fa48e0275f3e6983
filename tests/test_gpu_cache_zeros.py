"""Attention over 4-bit rows where q holds zeros and subnormal numbers and K is large: what is 0 in q adds nothing to a score,
however large the keys."""
import numpy as np
import pytest

from _cache import bf16_bits, bf16_values, expect_q4
from test_gpu_cache_attend import Case, attend_q4, weigh

pytestmark = pytest.mark.gpu


def rows_of_q(rng, heads, d, by):
    """[heads, d] that make scores of a few units at most with keys of 2^by: all zeros of either sign, zeros between
    values, zeros in the last 64 dims, subnormal numbers, those beside zeros, ordinary values."""
    q = np.ldexp(rng.standard_normal((heads, d)), -by)
    subnormal = np.ldexp(rng.integers(-127, 128, (heads, d)).astype(np.float64), -133)
    odd, last = np.arange(d) % 2 == 1, np.arange(d) >= d - 64
    for h in range(heads):
        q[h] = (np.zeros(d), -np.zeros(d), np.where(odd, 0, q[h]), np.where(last, 0, q[h]), subnormal[h], np.where(odd, subnormal[h], 0), q[h])[h % 7]
    return bf16_bits(q.astype(np.float32))


def check(c):
    caches = c.q4()
    want = expect_q4(bf16_values(c.q), *caches, c.lens)
    want.check(attend_q4(c, caches))
    out, sums, start = weigh(c, caches, "none")
    want.check(out)
    want.check_weights(sums, start, c.lens)


@pytest.mark.parametrize("by", [60, 115, 122])
@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (34, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_zeros_and_subnormal_values_of_q(d, heads, by):
    """The bound of a score is in proportion to sum |q k|: nothing for a row of zeros."""
    lens = [70, 333]
    c = Case(41, lens, *heads, d, 340)
    c.k = bf16_bits(np.clip(bf16_values(c.k), -15, 15) * np.float32(2.0 ** by))  # (a group's spread stays below 2^127)
    rng = np.random.default_rng(42)
    c.q = np.stack([rows_of_q(rng, heads[0], d, by)[None] for _ in lens])
    check(c)


@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (34, 2)])
@pytest.mark.parametrize("d", [128, 256])
def test_zeros_beside_ordinary_values_over_keys_that_are_large_there(d, heads):
    """q of ordinary size in the first 64 dims and 0 in the others, where the keys are 2^122: the scores are the first dims'."""
    c = Case(43, [200], *heads, d, 200)
    k, q = bf16_values(c.k).copy(), bf16_values(c.q).copy()
    k[..., 64:] = np.clip(k[..., 64:], -15, 15) * np.float32(2.0 ** 122)
    q[..., 64:] = 0
    c.k, c.q = bf16_bits(k), bf16_bits(q)
    check(c)


@pytest.mark.parametrize("by", [60, 104, 112])
@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (34, 2)])
@pytest.mark.parametrize("d", [128, 256])
def test_tiny_values_beside_ordinary_ones_over_keys_that_are_large_there(d, heads, by):
    """q of ordinary size in the first 64 dims and of 2^-by in the others, where the keys are 2^by: both parts are of a score.  (Sums of products have
    multiples of 2^-149 as their values, which is 2^-132 of the largest |q| times the largest |k| at most: 2^-16 here, a thousandth of
    the bound.)"""
    c = Case(44, [200], *heads, d, 200)
    k, q = bf16_values(c.k).copy(), bf16_values(c.q).copy()
    k[..., 64:] = np.clip(k[..., 64:], -15, 15) * np.float32(2.0 ** by)
    q[..., 64:] *= np.float32(2.0 ** -by)
    c.k, c.q = bf16_bits(k), bf16_bits(q)
    check(c)
