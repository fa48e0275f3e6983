"""The bounds of `_cache_bounds` against a model of the kernels in numpy: what is right passes, and small faults do not."""
import numpy as np
import pytest

from _cache import bf16_bits, bf16_values, offsets, scales, values
from _cache_bounds import F32, Near, exact_k_bf16, exact_k_q4, score_slack, small_q, v_q4

FAULTS = ["low terms dropped", "scores by 1.02", "scores by 1.005", "a key missing", "a key twice", "a group's scale of V", "a group's scale of K", "a middle of V", "output by 1.003"]


def cut(x):
    """The bf16 that is not above, by cutting bits off."""
    return (np.ascontiguousarray(x, dtype=F32).view(np.uint32) & np.uint32(0xFFFF0000)).view(F32).astype(np.float64)


def model(q, caches, lens, fault=None):
    """Outputs and sums of weights as the kernels have them, sums in 64 bits: weights cut to two bf16 terms, offsets and middles on the sums."""
    q = bf16_values(q).astype(np.float64)
    b, _, h, d = q.shape
    if len(caches) == 4:
        k = values(*caches[:2]).astype(np.float64)
        s, z = (np.repeat(x.astype(np.float64), 64, -1) for x in scales(caches[3]))
        c = offsets(caches[2]).astype(np.float64)
        if fault == "a group's scale of K":
            ks, kz = scales(caches[1])
            ks = ks.copy()
            ks[..., 0] *= F32(1 + 2.0 ** -7)
            k = (np.repeat(kz, 64, -1) + np.repeat(ks, 64, -1) * offsets(caches[0])).astype(np.float64)
    else:
        k, v = (bf16_values(x).astype(np.float64) for x in caches)
        if fault == "a group's scale of K":
            k[..., :64] *= 1 + 2.0 ** -7
        s, z, c = np.ones_like(v), np.zeros_like(v), v
    if fault == "a group's scale of V":
        s[..., -64:] *= 1 + 2.0 ** -7
    if fault == "a middle of V":
        z[..., -64:] += 2.0 ** -6 * s[..., -64:] if len(caches) == 4 else 2.0 ** -6
    hkv, rows = k.shape[1:3]
    out, sums = np.zeros_like(q), np.zeros((b, hkv, rows))
    for i, n in enumerate(lens):
        for j in range(h):
            e = j * hkv // h
            x = k[i, e, :n] @ q[i, 0, j] / np.sqrt(d)
            x = x * {"scores by 1.02": 1.02, "scores by 1.005": 1.005}.get(fault, 1)
            w = np.exp(x - x.max() + 1.0)  # (the running maximum lags)
            if fault == "a key missing":
                w[n - 1] = 0
            if fault == "a key twice":
                w[n // 2] *= 2
            hi = cut(w[:, None] * s[i, e, :n])
            lo = cut((w[:, None] * s[i, e, :n]).astype(F32) - hi.astype(F32))
            terms = hi + (0 if fault == "low terms dropped" else lo)
            out[i, 0, j] = ((terms * c[i, e, :n]).sum(0) + w @ z[i, e, :n]) / w.sum()
            sums[i, e, :n] += w / w.sum()
    if fault == "output by 1.003":
        out *= 1.003
    return bf16_values(bf16_bits(out.astype(F32))), sums.astype(F32)


def case(cache, d, lens, seed=1, hq=8, hkv=2):
    rng = np.random.default_rng(seed)
    shape = (len(lens), hkv, max(lens), d)
    q = small_q(rng, (len(lens), 1, hq, d))
    if cache == "q4":
        return q, (*exact_k_q4(rng, shape), *v_q4(rng, shape))
    return q, (exact_k_bf16(rng, shape), bf16_bits(rng.standard_normal(shape).astype(F32)))


@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[33, 300], [700]])
def test_what_is_right_passes(lens, d, cache):
    q, caches = case(cache, d, lens)
    near = Near(q, caches, lens)
    out, sums = model(q, caches, lens)
    near.check(out)
    near.check_rows(out)
    near.check_weights(sums, np.zeros_like(sums), lens)


@pytest.mark.parametrize("fault", FAULTS)
@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_fault_does_not(d, cache, fault):
    lens = [33, 300]
    q, caches = case(cache, d, lens)
    near = Near(q, caches, lens)
    out, sums = model(q, caches, lens, fault)
    with pytest.raises(AssertionError):
        near.check(out)
    if fault in ("scores by 1.02", "scores by 1.005", "a key missing", "a key twice", "a group's scale of K"):
        with pytest.raises(AssertionError):
            near.check_weights(sums, np.zeros_like(sums), lens)


@pytest.mark.parametrize("fault", ["scores by 1.02", "a key missing"])
@pytest.mark.parametrize("cache", ["q4", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_of_ordinary_operands(d, cache, fault):
    """Where scores are not exact: the bound of whole rows, with what random operands' scores are off by."""
    from _cache import quantise

    rng = np.random.default_rng(2)
    lens = [300, 33]
    k, v = (bf16_bits(rng.standard_normal((2, 2, 300, d)).astype(F32)) for _ in range(2))
    q = bf16_bits(rng.standard_normal((2, 1, 8, d)).astype(F32))
    caches = (*quantise(bf16_values(k)), *quantise(bf16_values(v))) if cache == "q4" else (k, v)
    near = Near(q, caches, lens, score_slack(q, caches))
    near.check_rows(model(q, caches, lens)[0])
    with pytest.raises(AssertionError):
        near.check_rows(model(q, caches, lens, fault)[0])


def test_scores_are_exact_in_f32():
    """In any order: partial sums from either end, and with the codes' offset taken off at the end."""
    rng = np.random.default_rng(3)
    d = 256
    q, (kc, kp, *_) = case("q4", d, [40], 4)
    qf = bf16_values(q)[0, 0, 0]
    s, z = scales(kp)
    c = offsets(kc)
    want = values(kc, kp).astype(np.float64) @ qf.astype(np.float64)
    for order in (np.arange(64), np.arange(64)[::-1], rng.permutation(64)):
        y = np.zeros(want.shape, F32)
        for g in range(d // 64):
            a = np.zeros(want.shape, F32)
            total = F32(0)
            for i in order:
                a = a + (c[..., 64 * g + i] + F32(8)) * qf[64 * g + i]
                total = total + qf[64 * g + i]
            y = y + (s[..., g] * (a - F32(8) * total) + z[..., g] * total)
        assert np.array_equal(y[0, 0].astype(np.float64), want[0, 0])
