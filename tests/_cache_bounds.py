"""How near attention over a cache has to come to 64 bits, element by element, for operands whose scores f32 holds exactly.

q is whole numbers of -3 .. 3.  A 4-bit K has scales that are powers of two and middles that are multiples of half the least scale;
a bf16 K is multiples of 2^-4 below 8.  Every sum of their products, in whatever order and with whatever offset taken off, is a
multiple of 2^-4 below 2^16: f32 holds all of them, so that the scores are exact and what is left is

  * the factor log2(e) / sqrt(dim) of an exponent, four roundings from its own, and the product with it: 2^-22 + 2^-24 of the exponent.  A weight is
    the product of a few exponentials (the key's, one for each rise of the running maximum behind it, one for each fold: columns, waves,
    workgroups), whose exponents are together D + 16 in size at most, D being how far the key lies below the largest score in powers
    of two: the running maximum lags by 8;
  * those exponentials and the products with them, ten at most, for the maximum rises by 8 at least, 2^-23 + 2^-24 each: 2^-19 together, the
    division by the sum included;
  * the sum of the weights, a chain of n / 16 + 40 additions at most;
  * the weights that meet V: two bf16 terms, each cut off and not rounded, 2^-7 2^-7 = 2^-14;
  * an output's chain of sums: of n / 128 products a wave two terms and, as the matrix cores may add a product's 32 terms in parts, eight
    roundings each, n / 8, and 40 for the folds;
  * one rounding to bf16.  It takes the nearer of two neighbours, so an output that was off by e before it is off from 64 bits by what the exact value's own
    rounding is off by and 2 e at most: where e does not lead over the border between two neighbours it changes nothing, and where it does both
    neighbours are within half a step + e."""
import numpy as np

from _cache import bf16_bits, bf16_values, offsets, scales, values

F32 = np.float32
LEAST = 2.0 ** -3  # of K's scales


def small_q(rng, shape):
    return bf16_bits(rng.integers(-3, 4, shape).astype(F32))


def exact_k_q4(rng, shape):
    """codes and pairs [batch, kv, rows, dim] for exact scores, some units in size."""
    b, h, n, d = shape
    codes = rng.integers(0, 256, (b, h, n, d // 2)).astype(np.uint8)
    s = np.ldexp(LEAST, rng.integers(0, 2, (b, h, d // 64, n))).astype(F32)
    z = (rng.integers(-4, 5, s.shape) * (LEAST / 2)).astype(F32)
    return codes, pair_words(s, z)


def pair_words(s, z):
    return (bf16_bits(s).astype(np.uint32) | bf16_bits(z).astype(np.uint32) << np.uint32(16)).astype(np.uint32)


def v_q4(rng, shape):
    """codes and pairs of any values: scales and middles of all bf16 mantissas, over a factor of 16."""
    b, h, n, d = shape
    codes = rng.integers(0, 256, (b, h, n, d // 2)).astype(np.uint8)
    s = np.exp2(rng.uniform(-4, 0, (b, h, d // 64, n)))
    return codes, pair_words(s.astype(F32), (2 * s * rng.standard_normal(s.shape)).astype(F32))


def exact_k_bf16(rng, shape):
    return bf16_bits((np.clip(np.rint(16 * rng.standard_normal(shape)), -127, 127) / 16).astype(F32))


class Near:
    """Attention of q [b, new, heads, d] in 64 bits, and the bounds above.  `caches`: (K codes, K pairs, V codes, V pairs), or bf16 bits (K, V).
    `slack` [b, new, heads, rows] or None: how far a score may be off where scores are not exact."""

    def __init__(self, q, caches, lens, slack=None):
        q = bf16_values(q).astype(np.float64)
        if len(caches) == 4:
            k, v = values(*caches[:2]).astype(np.float64), values(*caches[2:]).astype(np.float64)
            s, z = (np.repeat(np.abs(x.astype(np.float64)), 64, -1) for x in scales(caches[3]))
            size = s * np.abs(offsets(caches[2])) + z  # what a weight meets
            sums = s * (offsets(caches[2]) + 8.0 + 8.0) + z  # ... and what is added up: the codes of 0 .. 15 and 8 that are taken off
        else:
            k, v = (bf16_values(x).astype(np.float64) for x in caches)
            size = sums = np.abs(v)
        b, new, h, d = q.shape
        hkv, rows = k.shape[1:3]
        self.out, self.off = np.zeros((b, new, h, d)), np.zeros((b, new, h, d))
        self.weights, self.weights_off = np.zeros((b, hkv, rows)), np.zeros((b, hkv, rows))
        for i in range(b):
            for t in range(new):
                n = min(max(int(lens[i]), 0), rows) - new + t + 1
                for j in range(h if n > 0 else 0):
                    x = k[i, j * hkv // h, :n] @ q[i, t, j] / np.sqrt(d)
                    below = (x.max() - x) * np.log2(np.e)
                    p = np.exp2(-below)
                    p /= p.sum()
                    rel = np.log(2) * (below + 16) * (2.0 ** -22 + 2.0 ** -24) + 2.0 ** -19
                    if slack is not None:
                        rel = rel + slack[i, t, j, :n]
                    rel = rel + p @ rel + (n / 16 + 40) * 2.0 ** -24
                    self.weights[i, j * hkv // h, :n] += p
                    self.weights_off[i, j * hkv // h, :n] += p * rel
                    own = (slice(i, i + 1), slice(j * hkv // h, j * hkv // h + 1), slice(0, n))
                    self.out[i, t, j] = p @ v[own][0, 0]
                    self.off[i, t, j] = (p * (rel + 2.0 ** -14)) @ size[own][0, 0] + (n / 8 + 40) * 2.0 ** -24 * (p @ sums[own][0, 0])
        self.rounding = np.abs(bf16_values(bf16_bits(self.out.astype(F32))).astype(np.float64) - self.out)

    def check(self, got, label=""):
        got = np.asarray(got, dtype=np.float64).reshape(self.out.shape)
        assert np.isfinite(got).all(), label
        over = (np.abs(got - self.out) - self.rounding) / np.maximum(2 * self.off, 1e-300)
        over[got == self.out] = 0
        at = np.unravel_index(np.argmax(over), over.shape)
        assert over[at] <= 1, f"{label}: element {at} is {got[at]} and not {self.out[at]}, {over[at]:.2f} of what it may be off beside its rounding"

    def check_rows(self, got, label=""):
        """The same over whole rows, [b, new, heads]: what rounding leaves and twice what may come before it."""
        got = np.asarray(got, dtype=np.float64).reshape(self.out.shape)
        norm = lambda x: np.sqrt((x * x).sum(-1))  # noqa: E731
        over = norm(got - self.out) / np.maximum(norm(self.rounding) + 2 * norm(self.off), 1e-300)
        assert np.isfinite(got).all() and (over <= 1).all(), f"{label}: a row is off by {over.max():.2f} of its bound"

    def check_weights(self, got, before, lens, label=""):
        """`got` = before + the weights below the lengths; a sum over the heads of a group and one more."""
        for i, n in enumerate(lens):
            n = min(max(int(n), 0), got.shape[2])
            want = before[i, :, :n].astype(np.float64) + self.weights[i, :, :n]
            group = self.out.shape[2] / got.shape[1]
            over = np.abs(got[i, :, :n] - want) / (self.weights_off[i, :, :n] + (group + 1) * 2.0 ** -24 * np.abs(want) + 1e-37)
            assert (over <= 1).all(), f"{label}: sequence {i}, a sum of weights is off by {over.max():.2f} of its bound"


def score_slack(q, caches):
    """How far a score of ordinary random operands is off, [b, new, heads, rows]: of the 2 d roundings of 2^-24 of what has come together, in either direction as it
    falls, six times the root of their number; sums of products of random signs come together as three times the root of the sum of
    their squares, the codes' offset among them."""
    q = bf16_values(q).astype(np.float64)
    b, new, h, d = q.shape
    hkv = caches[0].shape[1]
    group = h // hkv
    if len(caches) == 4:
        s, z = (np.abs(x.astype(np.float64)) for x in scales(caches[1]))
        norm = np.sqrt((q.reshape(b, new, h, d // 64, 64) ** 2).sum(-1))  # [b, new, h, groups]
        per = 15.0 * s + 8.0 * s + z  # [b, kv, rows, groups]
        come = 3 * np.einsum("bthg,bhrg->bthr", norm, np.repeat(per, group, 1))
    else:
        k = np.repeat(bf16_values(caches[0]).astype(np.float64), group, 1)
        come = 3 * np.sqrt(np.einsum("bthd,bhrd->bthr", q * q, k * k))
    return 6 * np.sqrt(2 * d) * 2.0 ** -24 * come / np.sqrt(d)
