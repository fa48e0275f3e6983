"""The entries of caches that are kept small: what they refuse, before any device is looked for, and their format's helper."""
import ctypes as C

import numpy as np
import pytest

import rustorch_amd as ra
from rustorch_amd import _lib as L
from _cache import bf16_bits, bf16_values, quantise, scales, values

P = 0x10000  # never dereferenced
OK = (L.RT_OK, L.RT_ERR_NO_DEVICE)


def call(name, *args):
    err = L.RtErr()
    return getattr(L.lib(), name)(*args, C.byref(err)), err


def append(name="rt_qk_norm_rope_kv_append_q4", q=P, q_out=2 * P, k_in=3 * P, k=4 * P, kp=5 * P, positions=None, pos=0, rows=None, cos=6 * P, table=16, batch=1,
           seq=1, hq=2, hkv=1, d=64, n=8):
    caches = (k, kp, k, kp) if name.endswith("q4") else (k, k)
    return call(name, None, q, q_out, k_in, k_in, *caches, positions, pos, rows, None, None, None, None, 1e-6, cos, cos, table, batch, seq, hq, hkv, d, n)


@pytest.mark.parametrize("name", ["rt_qk_norm_rope_kv_append_q4", "rt_qk_norm_rope_kv_append_rows_bf16"])
def test_append_refusals(name):
    for d in (32, 80, 96, 512, 1):
        rc, err = append(name, d=d)
        assert rc == L.RT_ERR_UNSUPPORTED and err.got == d
    assert append(name, d=0)[0] == L.RT_ERR_ZERO_DIM
    for bad in ({"batch": -1}, {"seq": -1}, {"hq": -1}, {"n": -1}, {"batch": 65536}, {"seq": 1 << 30, "positions": P}):
        assert append(name, **bad)[0] == L.RT_ERR_UNSUPPORTED
    rc, err = append(name, pos=16)
    assert rc == L.RT_ERR_ROPE_POSITION_OVERFLOW and (err.expected, err.got) == (16, 17)
    assert append(name, pos=-1)[0] == L.RT_ERR_ROPE_POSITION_OVERFLOW
    rc, err = append(name, pos=7, seq=2)
    assert rc == L.RT_ERR_KV_OVERFLOW and (err.expected, err.got) == (8, 9)
    assert append(name, pos=7, seq=2, rows=P)[0] in OK  # rows of their own are the device's
    assert append(name, batch=0)[0] == append(name, seq=0)[0] == L.RT_OK
    for missing in ("q", "q_out", "k_in", "k", "cos"):
        assert append(name, **{missing: None})[0] == L.RT_ERR_NULL_POINTER
    assert append(name, hq=0, q=None, q_out=None)[0] in OK
    for odd in ("q", "q_out", "k_in", "k"):
        rc, err = append(name, **{odd: 8 * P + 8})
        assert rc == L.RT_ERR_UNSUPPORTED and err.expected == 16
    assert append(name, q_out=P + 16)[0] == L.RT_ERR_UNSUPPORTED  # over part of q
    assert append(name, q_out=P)[0] in OK


def test_append_q4_without_pairs():
    assert append(kp=None)[0] == L.RT_ERR_NULL_POINTER


def test_cache_append_refusals():
    def f(cur=0, add=2, nk=128, nv=128, b=1, h=1, n=8, d=64, k=P, new=2 * P):
        return call("rt_kv_cache_append_q4_dev", None, k, P, k, P, new, nk, new, nv, b, h, n, d, cur, add)

    rc, err = f(cur=7, nk=1)
    assert rc == L.RT_ERR_KV_OVERFLOW and (err.expected, err.got) == (8, 9)  # before the lengths, as in the reference
    assert f(cur=2 ** 64 - 1)[0] == L.RT_ERR_KV_OVERFLOW
    rc, err = f(nk=127)
    assert rc == L.RT_ERR_KV_WRONG_INPUT_LEN and (err.expected, err.got, err.got2) == (128, 127, 128)
    assert f(d=96, nk=192, nv=192)[0] == L.RT_ERR_UNSUPPORTED
    assert f(add=0, nk=0, nv=0)[0] == L.RT_OK
    assert f(k=None)[0] == f(new=None)[0] == L.RT_ERR_NULL_POINTER
    assert f(k=P + 4)[0] == L.RT_ERR_UNSUPPORTED
    assert f()[0] in OK


def test_read_refusals():
    def f(row=0, n_rows=2, b=1, h=1, d=64, n=8, rows=None, codes=P, out=2 * P):
        return call("rt_kv_cache_read_q4", None, codes, P, out, rows, row, n_rows, b, h, d, n)

    rc, err = f(row=7)
    assert rc == L.RT_ERR_KV_OVERFLOW and (err.expected, err.got) == (8, 9)
    assert f(row=-1)[0] == f(n_rows=9, rows=P)[0] == L.RT_ERR_KV_OVERFLOW
    assert f(d=32)[0] == f(b=-1)[0] == f(out=2 * P + 2)[0] == L.RT_ERR_UNSUPPORTED
    assert f(codes=None)[0] == L.RT_ERR_NULL_POINTER
    assert f(n_rows=0)[0] == L.RT_OK and f(row=6)[0] in OK


def test_attend_refusals():
    big = 1 << 40

    def f(lens=P, kv_len=0, b=2, s=1, hq=8, hkv=2, d=128, n=100, ws=P, size=big, q=P, k=P, kp=P, out=2 * P):
        return call("rt_gqa_decode_q4", None, q, k, kp, k, kp, out, lens, kv_len, b, s, hq, hkv, d, n, ws, size)

    assert f(hkv=3)[0] == f(hkv=0)[0] == L.RT_ERR_HEAD_COUNT_MISMATCH
    assert f(d=0)[0] == L.RT_ERR_ZERO_DIM
    assert f(d=96)[0] == f(b=-1)[0] == f(b=65536)[0] == f(s=65536)[0] == f(q=P + 2)[0] == L.RT_ERR_UNSUPPORTED
    assert f(b=60000, n=2 ** 31 - 1)[0] == L.RT_ERR_UNSUPPORTED  # more steps than an int counts
    assert f(n=2 ** 29 + 1)[0] == f(b=1, s=65535, hq=512, hkv=1)[0] == L.RT_ERR_UNSUPPORTED
    assert f(b=1, hkv=1, n=2 ** 29)[0] in OK
    rc, err = f(lens=None, kv_len=101)
    assert rc == L.RT_ERR_KV_OVERFLOW and (err.expected, err.got) == (100, 101)
    assert f(lens=None, kv_len=2, s=3)[0] == L.RT_ERR_KV_OVERFLOW
    assert f(b=0)[0] == f(s=0)[0] == f(hq=0, hkv=1)[0] == L.RT_OK
    for missing in ("q", "k", "kp", "out"):
        assert f(**{missing: None})[0] == L.RT_ERR_NULL_POINTER
    need = L.lib().rt_gqa_decode_q4_workspace_bytes(2, 1, 8, 2, 128, 100)
    assert need > 0
    rc, err = f(size=need - 1)
    assert rc == L.RT_ERR_WORKSPACE_TOO_SMALL and (err.expected, err.got) == (need, need - 1)
    assert f(ws=None)[0] == f(ws=P + 8)[0] == L.RT_ERR_WORKSPACE_TOO_SMALL
    assert f(size=need)[0] in OK
    assert f(n=0, k=None, kp=None, lens=P)[0] in OK
    for args in ((0, 1, 8, 2, 128, 100), (2, 1, 8, 3, 128, 100), (2, 1, 8, 2, 96, 100), (2, 1, 8, 2, 128, -1)):
        assert L.lib().rt_gqa_decode_q4_workspace_bytes(*args) == 0


@pytest.mark.parametrize("name", ["rt_gqa_decode_weights_bf16", "rt_gqa_decode_weights_q4"])
def test_weights_refusals(name):
    def f(w_in=8 * P, w_out=9 * P, lens=P, hkv=2, d=128, size=1 << 40, k=P):
        caches = (k, P, k, P) if name.endswith("q4") else (k, k)
        return call(name, None, P, *caches, 2 * P, w_in, w_out, lens, 2, 8, hkv, d, 100, P, size)

    assert f(hkv=3)[0] == L.RT_ERR_HEAD_COUNT_MISMATCH
    assert f(d=80)[0] == L.RT_ERR_UNSUPPORTED
    assert f(w_out=None)[0] == f(lens=None)[0] == f(k=None)[0] == L.RT_ERR_NULL_POINTER
    assert f(w_out=8 * P + 4)[0] == L.RT_ERR_UNSUPPORTED  # over part of weights_in
    assert f(w_out=8 * P)[0] in OK and f(w_in=None)[0] in OK
    need = L.lib().rt_gqa_decode_weights_workspace_bytes(2, 8, 2, 128, 100)
    assert need >= 2 * 8 * 100 * 4
    assert f(size=need - 1)[0] == L.RT_ERR_WORKSPACE_TOO_SMALL and f(size=need)[0] in OK


@pytest.mark.parametrize("name", ["rt_kv_evict_bf16", "rt_kv_evict_q4"])
def test_evict_refusals(name):
    def f(w_in=8 * P, s_in=9 * P, w_out=10 * P, s_out=11 * P, lens=12 * P, new=13 * P, b=2, h=2, d=64, n=100, budget=10, recent=4, size=1 << 40, k=P, ws=P):
        caches = (k, P, k, P) if name.endswith("q4") else (k, k)
        return call(name, None, *caches, w_in, s_in, w_out, s_out, lens, new, b, h, d, n, budget, recent, ws, size)

    assert f(d=0)[0] == L.RT_ERR_ZERO_DIM
    assert f(d=32)[0] == f(b=-1)[0] == f(h=65536)[0] == f(k=P + 4)[0] == L.RT_ERR_UNSUPPORTED
    rc, err = f(recent=11)
    assert rc == L.RT_ERR_UNSUPPORTED and (err.expected, err.got) == (10, 11)
    assert f(budget=-1, recent=0)[0] == f(recent=-1)[0] == L.RT_ERR_UNSUPPORTED
    assert f(n=2 ** 29 + 1)[0] == L.RT_ERR_UNSUPPORTED and f(n=2 ** 29, w_in=1 << 50, s_in=1 << 51, w_out=1 << 52, s_out=1 << 53, size=1 << 50)[0] in OK
    assert f(b=0)[0] == L.RT_OK
    for missing in ("k", "w_in", "s_in", "w_out", "s_out", "lens"):
        assert f(**{missing: None})[0] == L.RT_ERR_NULL_POINTER
    assert f(new=None)[0] in OK and f(new=12 * P)[0] in OK and f(w_out=8 * P, s_out=9 * P)[0] in OK
    for shared in ({"w_out": 8 * P + 4}, {"s_out": 9 * P + 4}, {"w_out": 11 * P}, {"w_out": 9 * P}, {"s_out": 8 * P}, {"new": 12 * P + 4}):
        assert f(**shared)[0] == L.RT_ERR_UNSUPPORTED, shared
    need = L.lib().rt_kv_evict_workspace_bytes(2, 2, 100, 10)
    assert f(size=need - 1)[0] == L.RT_ERR_WORKSPACE_TOO_SMALL and f(size=need)[0] in OK and f(ws=P + 4)[0] == L.RT_ERR_WORKSPACE_TOO_SMALL


def test_python_checks_before_the_library():
    K, rope = ra.LlmKernels(), ra.RoPE(64, 16)
    cache = ra.Q4Rows(P, P)
    with pytest.raises(ra.PositionOverflow):
        K.qk_norm_rope_kv_append_q4(None, P, P, P, P, cache, cache, 15, rope, 1, 1, 1, 64, 32, seq=2)
    with pytest.raises(ra.Overflow):
        K.qk_norm_rope_kv_append_rows_bf16(None, P, P, P, P, P, P, 7, rope, 1, 1, 1, 64, 8, seq=2)
    with pytest.raises(ValueError):
        ra.KVCache(0, 1, 1, 96, 8, dtype="q4")
    with pytest.raises(ra.HeadCountMismatch):
        K.gqa_decode_q4(None, P, cache, cache, P, 4, 1, 1, 8, 3, 64, 16, P, 1 << 30)


def test_the_formats_error_is_half_a_step():
    """Of the tests' own quantiser: s / 2, whatever the values' offset and spread (and f32's rounding of the difference)."""
    rng = np.random.default_rng(1)
    for offset, spread in ((0, 1), (100, 1), (-3, 1e-3), (1e-8, 1e-9), (1e30, 1e28)):
        x = bf16_values(bf16_bits(offset + spread * rng.standard_normal((50, 128))))
        codes, pairs = quantise(x)
        s, _ = scales(pairs)
        assert (np.abs(values(codes, pairs).astype(np.float64) - x) <= np.repeat(s, 64, -1) * (0.5 + 1e-6) + 2.0 ** -23 * np.abs(x)).all()
        top, low = x.reshape(50, 2, 64).max(-1), x.reshape(50, 2, 64).min(-1)
        # a sixteenth of the range, and what z's rounding (2^-8 of it) and s's own (2^-7) add
        assert (s <= ((top - low) / 16 + 2.0 ** -8 * np.abs([top, low]).max(0) / 7.5) * (1 + 2.0 ** -7) * 1.0001).all()
