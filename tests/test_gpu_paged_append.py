"""New rows of packed tokens into pages: the bits that f32 arithmetic gives operation by operation."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values, prepare
from _paged import dev, normal_bits

pytestmark = pytest.mark.gpu


class Tables:
    """RoPE tables with values that no formula stands behind: an error of place shows."""

    def __init__(self, rng, dim, rows):
        self.max_seq = rows
        self.cos, self.sin = (rng.standard_normal((rows, dim // 2), dtype=np.float32) for _ in range(2))
        self._dev = dev(self.cos), dev(self.sin)

    def device_tables(self):
        return self._dev


def rotated(x_bits, gamma, eps, cos, sin):
    """[tokens, heads, dim] bits, cos and sin [tokens, dim / 2] of each token -> bits."""
    x = bf16_values(x_bits)
    t = x.shape[0]
    y = prepare(x[:, :, None, :], gamma, eps, cos, sin, np.arange(t))
    return bf16_bits(y[:, :, 0, :])


def run(rng, lens, heads, n_kv, dim, page, starts=True, positions=None, norm=True, sections=None, k_out=True, in_place=False, tokens=None,
        rows=600, table=None, n_pages=None):
    b = len(lens)
    first = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    t = int(first[-1]) if tokens is None else tokens
    positions = np.zeros(b, dtype=np.int32) if positions is None else np.asarray(positions, dtype=np.int32)
    q, k, v = normal_bits(rng, t, heads, dim), normal_bits(rng, t, n_kv, dim), normal_bits(rng, t, n_kv, dim)
    gammas = [rng.standard_normal(dim, dtype=np.float32) if norm else None for _ in range(2)]
    rope = Tables(rng, dim, rows)
    cols = max(1, max(-(-int(p + n) // page) for p, n in zip(positions, lens)) + 1)
    if table is None:
        n_pages = b * cols + 2
        table = rng.permutation(n_pages)[:b * cols].reshape(b, cols).astype(np.int32)
    axes = None if sections is None else rng.integers(0, rows, (len(sections), t)).astype(np.int32)
    kp, vp = normal_bits(rng, n_pages, n_kv, page, dim), normal_bits(rng, n_pages, n_kv, page, dim)
    # what is expected
    want = {"q": np.full_like(q, 0x1234), "k": np.full_like(k, 0x1234), "kp": kp.copy(), "vp": vp.copy()}
    if in_place:
        want["q"], want["k"] = q.copy(), k.copy()
    half = dim // 2
    axis = None if sections is None else np.repeat(np.arange(len(sections)), sections)
    for i in range(b):
        for s in range(lens[i]):
            at, row = int(first[i]) + s, int(positions[i]) + s
            if axes is None:
                if not 0 <= row < rows:
                    continue
                c, z = rope.cos[row], rope.sin[row]
            else:
                if not all(0 <= axes[a, at] < rows for a in range(len(sections))):
                    continue
                c, z = (x[axes[axis, at], np.arange(half)] for x in (rope.cos, rope.sin))
            want["q"][at] = rotated(q[at:at + 1], gammas[0], 1e-5, c[None], z[None])[0]
            turned = rotated(k[at:at + 1], gammas[1], 1e-5, c[None], z[None])[0]
            want["k"][at] = turned
            entry = table[i, row // page] if 0 <= row and row // page < table.shape[1] else -1
            if 0 <= entry < n_pages:
                want["kp"][entry, :, row % page], want["vp"][entry, :, row % page] = turned, v[at]
    dq, dk = dev(q), dev(k)
    dq_out = dq if in_place else dev(np.full_like(q, 0x1234))
    dk_out = (dk if in_place else dev(np.full_like(k, 0x1234))) if k_out else None
    pages = ra.KVPages(dev(kp), dev(vp), n_pages, page)
    ra.LlmKernels.qk_norm_rope_kv_append_paged_bf16(
        None, dq, dq_out, dk, dev(v), pages, dev(table), table.shape[1], dev(positions), rope, t, b, heads, n_kv, dim,
        starts=dev(first) if starts else None, k_out=dk_out, q_gamma=None if gammas[0] is None else dev(gammas[0]),
        k_gamma=None if gammas[1] is None else dev(gammas[1]), eps=1e-5, axis_positions=None if axes is None else dev(axes), sections=sections)
    ra.synchronize()
    got = {"q": dq_out, "k": dk_out, "kp": pages.k, "vp": pages.v}
    for name, x in got.items():
        if x is not None:
            y = x.download(np.uint16).reshape(want[name].shape)
            assert np.array_equal(y, want[name]), (name, np.argwhere(y != want[name])[:5])


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256])
@pytest.mark.parametrize("norm", [False, True])
def test_head_dims(dim, norm):
    run(np.random.default_rng(dim), [3, 17, 1, 0, 40], 6, 2, dim, 16, norm=norm)


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (8, 8), (32, 8), (28, 4), (7, 1), (40, 8)])
def test_heads(heads, n_kv):
    run(np.random.default_rng(heads), [5, 30], heads, n_kv, 64, 32)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 512, 1024])
def test_page_sizes_and_rows_in_the_middle(page):
    run(np.random.default_rng(page), [33, 16, 1], 4, 2, 64, page, positions=[page - 5, 15, 2 * page - 1], rows=2200)


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 200])
def test_a_token_of_each_sequence(batch):
    rng = np.random.default_rng(batch)
    run(rng, [1] * batch, 8, 2, 128, 16, starts=False, positions=rng.integers(0, 500, batch))


@pytest.mark.parametrize("batch", [64, 65, 130])
def test_many_sequences_some_of_them_empty(batch):
    rng = np.random.default_rng(batch)
    run(rng, [int(x) for x in rng.integers(0, 4, batch)], 4, 1, 64, 16, positions=rng.integers(0, 50, batch))


def test_several_tokens_of_each_without_starts():
    run(np.random.default_rng(1), [7, 7, 7], 4, 2, 128, 16, starts=False, positions=[0, 10, 200])


def test_long_prompts():
    run(np.random.default_rng(2), [290, 1, 333], 4, 2, 128, 64)


@pytest.mark.parametrize("dim,sections", [(128, [16, 24, 24]), (64, [8, 12, 12]), (64, [32]), (64, [5, 27]), (128, [1, 2, 3, 58]), (64, [0, 32, 0]), (256, [43, 43, 42]), (80, [10, 15, 15])])
@pytest.mark.parametrize("norm", [False, True])
def test_several_axes(dim, sections, norm):
    run(np.random.default_rng(dim), [9, 300, 2], 6, 2, dim, 16, sections=sections, norm=norm)


def test_outputs_in_their_inputs_places():
    run(np.random.default_rng(3), [50, 20], 8, 2, 128, 16, in_place=True)


def test_without_k_out():
    run(np.random.default_rng(4), [50, 20], 8, 2, 128, 16, k_out=False)


def test_tokens_behind_the_last_sequence_stay():
    run(np.random.default_rng(5), [5, 6], 4, 2, 64, 16, tokens=40)


def test_positions_that_the_tables_do_not_have():
    """Such tokens are left as they are; the others of their sequence are not."""
    run(np.random.default_rng(6), [4, 10, 6], 4, 2, 64, 16, positions=[-2, 95, 2 ** 31 - 4], rows=100, table=np.arange(60, dtype=np.int32).reshape(3, 20), n_pages=60)


def test_rows_without_a_page_are_rotated_and_not_stored():
    table = np.array([[0, -1, 2], [7, 3, 2 ** 31 - 1], [-2 ** 31, 4, 5]], dtype=np.int32)
    run(np.random.default_rng(7), [40, 48, 60], 4, 2, 64, 16, table=table, n_pages=7)


@pytest.mark.parametrize("dim,norm", [(64, True), (128, True), (128, False), (256, True), (96, True)])
def test_the_bits_of_the_append_to_a_plain_cache(dim, norm):
    """rt_qk_norm_rope_kv_append_bf16 on the same tokens, with its own layouts."""
    rng = np.random.default_rng(dim)
    b, s, h, hkv, page, rows = 3, 21, 8, 2, 32, 128
    q, k, v = normal_bits(rng, b, h, s, dim), normal_bits(rng, b, hkv, s, dim), normal_bits(rng, b, hkv, s, dim)
    g = [dev(rng.standard_normal(dim, dtype=np.float32)) if norm else None for _ in range(2)]
    rope, at = ra.RoPE(dim, rows), dev(np.array([0, 5, 90], dtype=np.int32))
    dq, kc, vc = dev(q), ra.HipStorage.zeros(b * hkv * rows * dim * 2), ra.HipStorage.zeros(b * hkv * rows * dim * 2)
    ra.LlmKernels.qk_norm_rope_kv_append_bf16(None, dq, dev(k), dev(v), kc, vc, at, rope, b, h, hkv, dim, rows, q_gamma=g[0], k_gamma=g[1], seq=s)
    packed = [np.ascontiguousarray(x.transpose(0, 2, 1, 3)).reshape(b * s, -1, dim) for x in (q, k, v)]
    dq2 = dev(packed[0])
    pages, table = ra.KVPages.zeros(b * rows // page, hkv, page, dim), np.arange(b * rows // page, dtype=np.int32).reshape(b, -1)
    ra.LlmKernels.qk_norm_rope_kv_append_paged_bf16(None, dq2, dq2, dev(packed[1]), dev(packed[2]), pages, dev(table), table.shape[1], at, rope, b * s, b, h,
                                                    hkv, dim, q_gamma=g[0], k_gamma=g[1])
    ra.synchronize()
    assert np.array_equal(dq2.download(np.uint16).reshape(b, s, h, dim), dq.download(np.uint16).reshape(b, h, s, dim).transpose(0, 2, 1, 3))
    for a, c in ((pages.k, kc), (pages.v, vc)):
        got = a.download(np.uint16).reshape(b, rows // page, hkv, page, dim).transpose(0, 2, 1, 3, 4).reshape(b, hkv, rows, dim)
        assert np.array_equal(got, c.download(np.uint16).reshape(b, hkv, rows, dim))


def test_without_kv_heads_q_is_rotated_and_nothing_else_is_asked_for():
    """No k, v, pages or table: a call whose heads are all query heads."""
    rng = np.random.default_rng(14)
    t, heads, dim, rows = 37, 5, 128, 40
    q, gamma, rope = normal_bits(rng, t, heads, dim), rng.standard_normal(dim, dtype=np.float32), Tables(rng, dim, rows)
    dq, out = dev(q), dev(np.full_like(q, 0x1234))
    ra.LlmKernels.qk_norm_rope_kv_append_paged_bf16(None, dq, out, None, None, ra.KVPages(None, None, 0, 16), None, 3, 0, rope, t, 1, heads, 0, dim, q_gamma=dev(gamma), eps=1e-5)
    ra.synchronize()
    assert np.array_equal(out.download(np.uint16).reshape(q.shape), rotated(q, gamma, 1e-5, rope.cos[:t], rope.sin[:t]))
