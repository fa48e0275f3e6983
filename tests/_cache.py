"""The 4-bit cache, attention over caches and eviction, from their definitions in numpy: what the tests of those entries
compare with."""
import numpy as np

import rustorch_amd as ra
from oracle import attn_oracle as oracle

F32 = np.float32


def bf16_bits(x):
    return oracle.f32_to_bf16(np.ascontiguousarray(x, dtype=F32)).reshape(np.shape(x))


def bf16_values(bits):
    return oracle.bf16_to_f32(np.ascontiguousarray(bits)).reshape(np.shape(bits))


def chunk_of(p, n):
    """The 32-dim chunk whose two values byte i n + p of a row holds."""
    return p if n == 2 else (p & ~3) | (p & 1) << 1 | (p >> 1 & 1)


def quantise(x):
    """f32 rows [..., rows, dim] -> (codes [..., rows, dim / 2] uint8, pairs [..., dim / 64, rows] uint32), every f32 operation as
    the definition has it."""
    x = np.asarray(x, dtype=F32)
    d = x.shape[-1]
    n = d // 32
    g = x.reshape(*x.shape[:-1], d // 64, 64)
    with np.errstate(all="ignore"):
        hi, lo = g.max(-1), g.min(-1)
        z = bf16_values(bf16_bits((hi + lo) * F32(0.5) + (hi - lo) * F32(1 / 32)))
        up = np.maximum((hi - z) / F32(7.5), (z - lo) / F32(8.5))
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(z) & (up < F32(3e38)))
        s = ((np.where(bad, F32(0), up).astype(F32).view(np.uint32) + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(F32)
        c = np.clip(np.rint((g - z[..., None]) / s[..., None]), -8, 7)
        c = np.where((s == 0)[..., None], 0, c).astype(np.int64) + 8
    c = c.reshape(*x.shape[:-1], n, 16, 2)  # chunk, i, parity
    codes = np.empty((*x.shape[:-1], 16, n), dtype=np.uint8)
    for p in range(n):
        two = c[..., chunk_of(p, n), :, :]
        codes[..., p] = two[..., 0] | two[..., 1] << 4
    pairs = np.where(bad, np.uint32(0x7FC00000), s.view(np.uint32) >> np.uint32(16) | z.view(np.uint32) & np.uint32(0xFFFF0000))
    return codes.reshape(*x.shape[:-1], d // 2), np.ascontiguousarray(np.swapaxes(pairs, -1, -2).astype(np.uint32))


def scales(pairs):
    """(s, z) of each row's groups, [..., rows, dim / 64] f32."""
    pairs = np.swapaxes(pairs, -1, -2)
    return (pairs << np.uint32(16)).view(F32), (pairs & np.uint32(0xFFFF0000)).view(F32)


def offsets(codes):
    """c - 8 of every value, [..., rows, dim]."""
    half = codes.shape[-1]
    n = half // 16
    b = codes.reshape(*codes.shape[:-1], 16, n)
    c = np.empty((*codes.shape[:-1], n, 16, 2), dtype=F32)
    for p in range(n):
        c[..., chunk_of(p, n), :, 0] = b[..., p] & 15
        c[..., chunk_of(p, n), :, 1] = b[..., p] >> 4
    return c.reshape(*codes.shape[:-1], 2 * half) - F32(8)


def values(codes, pairs):
    """What a 4-bit cache stands for, f32 [..., rows, dim]."""
    s, z = scales(pairs)
    c = offsets(codes)
    g = c.reshape(*c.shape[:-1], c.shape[-1] // 64, 64)
    return (z[..., None] + s[..., None] * g).reshape(c.shape)


def q4_dev(codes, pairs):
    return ra.Q4Rows(ra.HipStorage.from_numpy(codes), ra.HipStorage.from_numpy(pairs))


def prepare(x, gamma, eps, cos, sin, positions):
    """[batch, heads, seq, dim] f32: RMSNorm (the squares summed in index order) and half-split rotation, operation by
    operation in f32; cos, sin [positions, dim / 2]."""
    x = np.asarray(x, dtype=F32).copy()
    b, _, seq, d = x.shape
    if gamma is not None:
        sq = np.zeros(x.shape[:-1], dtype=F32)
        for i in range(d):
            sq = sq + x[..., i] * x[..., i]
        inv = F32(1) / np.sqrt(sq * (F32(1) / F32(d)) + F32(eps))
        x = x * inv[..., None] * gamma.astype(F32)
    at = np.asarray(positions)[:, None] + np.arange(seq)
    c, s = cos[at][:, None], sin[at][:, None]
    x0, x1 = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], -1).astype(F32)


class Expected:
    """Attention in 64 bits and, element by element, how far f32 sums of products may be from it."""

    def __init__(self, q, k, v, lens, k_size, v_size, v_offset):
        """q [b, new, heads, d], k, v [b, kv heads, rows, d] f64; k_size [b, kv, rows, d]: what a factor of q is multiplied with at most,
        in magnitude, on the way to a score; v_size and v_offset the same on the way to an output: with the values' own sign,
        and with offsets that are taken off again (summed exactly but for f32)."""
        b, new, h, d = q.shape
        hkv = k.shape[1]
        g = h // hkv
        self.out = np.zeros((b, new, h, d))
        self.bound = np.zeros((b, new, h, d))
        self.weights = np.zeros((b, hkv, k.shape[2]))
        self.weight_bound = np.zeros((b, hkv, k.shape[2]))
        for i in range(b):
            for t in range(new):
                n = min(max(int(lens[i]), 0), k.shape[2]) - new + t + 1
                if n <= 0:
                    continue
                for j in range(h):
                    kk, vv = k[i, j // g, :n], v[i, j // g, :n]
                    x = kk @ q[i, t, j] / np.sqrt(d)
                    with np.errstate(invalid="ignore"):
                        p = np.exp(x - x.max())
                    p /= p.sum()
                    self.out[i, t, j] = p @ vv
                    # a score is a chain of at most 2 d + 8 f32 operations (each 2^-23 of what has come together, were they
                    # cut off and not rounded), its exponent a product and a difference more, the exponential itself 2^-21
                    dx = (2 * d + 8) * 2.0 ** -23 * (k_size[i, j // g, :n] @ np.abs(q[i, t, j])) / np.sqrt(d)
                    rel = 2 * dx.max() + 2.0 ** -20 + 2.0 ** -22 * np.abs(x).max() + n * 2.0 ** -24
                    self.weights[i, j // g, :n] += p
                    self.weight_bound[i, j // g, :n] += p * rel
                    # an output: the weights' own error and their two bf16 terms (2^-14), and n / 32 products of two f32 additions each
                    # with the offsets, folded once a wave; rounded to bf16 once
                    size, offset = p @ v_size[i, j // g, :n], p @ v_offset[i, j // g, :n]
                    self.bound[i, t, j] = 2.0 ** -8 * np.abs(self.out[i, t, j]) + (rel + 2.0 ** -14) * size + (n / 16 + 40) * 2.0 ** -23 * (size + offset)

    def check(self, got, label=""):
        got = np.asarray(got, dtype=np.float64).reshape(self.out.shape)
        assert np.isfinite(got).all(), label
        over = np.abs(got - self.out) / np.maximum(self.bound, 1e-300)
        over = np.where(np.abs(got - self.out) == 0, 0, over)
        worst = np.unravel_index(np.argmax(over), over.shape)
        assert over[worst] <= 1, f"{label}: element {worst} is {got[worst]} and not {self.out[worst]}, {over[worst]:.2f} of the bound"

    def check_weights(self, got, before, lens, label=""):
        """`got` = before + the weights below the lengths (one more f32 rounding of the sum)."""
        for i, n in enumerate(lens):
            n = min(max(int(n), 0), got.shape[2])
            want = before[i, :, :n].astype(np.float64) + self.weights[i, :, :n]
            off = np.abs(got[i, :, :n] - want)
            bound = self.weight_bound[i, :, :n] + 2.0 ** -23 * np.abs(want)
            assert (off <= bound).all(), f"{label}: sequence {i}, {np.max(off / np.maximum(bound, 1e-300)):.2f} of the bound"


def expect_q4(q, kc, kp, vc, vp, lens):
    """Expected over 4-bit caches.  A code enters a product as 16 + c, and 24 times what it is multiplied with is taken off."""
    def sizes(codes, pairs):
        s, z = (np.repeat(np.abs(np.nan_to_num(x.astype(np.float64))), 64, -1) for x in scales(pairs))
        c = np.abs(offsets(codes)).astype(np.float64)
        return s * c + z, s * (24 + 24 + c)

    k, v = values(kc, kp).astype(np.float64), values(vc, vp).astype(np.float64)
    (k_own, k_off), (v_own, v_off) = sizes(kc, kp), sizes(vc, vp)
    return Expected(q.astype(np.float64), k, v, lens, k_own + k_off, v_own, v_off)


def expect_bf16(q, k, v, lens):
    k, v = k.astype(np.float64), v.astype(np.float64)
    return Expected(q.astype(np.float64), k, v, lens, np.abs(k), np.abs(v), np.zeros_like(v))


def evict(weights, slots, lens, budget, recent):
    """(rows [b, kv, budget] that the new rows are, new lengths): the definition, head by head."""
    b, hkv, n = weights.shape
    source = np.full((b, hkv, budget), -1, dtype=np.int64)
    new = np.minimum(np.clip(lens, 0, n), budget)
    for i in range(b):
        length = min(max(int(lens[i]), 0), n)
        for j in range(hkv):
            if length <= budget:
                source[i, j, :length] = np.arange(length)
                continue
            w, s = weights[i, j, :length].astype(np.float64), slots[i, j, :length].astype(np.int64)
            w = np.where(np.isnan(w), -np.inf, w)
            w = np.where(s > s.max() - recent, np.inf, w)
            order = sorted(range(length), key=lambda r: (-w[r], r))
            keep = np.zeros(length, dtype=bool)
            keep[order[:budget]] = True
            at = np.arange(budget)
            at[~keep[:budget]] = budget + np.nonzero(keep[budget:])[0]
            source[i, j] = at
    return source, new
