"""A decode loop over caches that are kept small, per layer and token: norm, rotation and append behind the last row, attention
that sums the keys' weights, and eviction down to the budget -- checked step by step against the definitions, and recorded
into a HIP graph whose replays have the bits of the eager loop."""
import numpy as np
import pytest

import rustorch_amd as ra
from _cache import bf16_bits, bf16_values, evict, expect_bf16, expect_q4, prepare, q4_dev, quantise
from test_gpu_decode_graph import NODE_TYPE_MEMSET, Hip

pytestmark = pytest.mark.gpu
K = ra.LlmKernels()

B, HQ, HKV, D, BUDGET, RECENT = 3, 8, 2, 64, 96, 16
N = BUDGET + 5


class Layer:
    def __init__(self, seed, q4):
        rng = np.random.default_rng(seed)
        self.q4 = q4
        rows = [bf16_bits(rng.standard_normal((B, HKV, N, D))) for _ in range(2)]
        if q4:
            self.k, self.v = (q4_dev(*quantise(bf16_values(x))) for x in rows)
        else:
            self.k, self.v = (ra.HipStorage.from_numpy(x) for x in rows)
        self.weights = ra.HipStorage.from_numpy(rng.random((B, HKV, N)).astype(np.float32))
        self.slots = ra.HipStorage.from_numpy(np.tile(np.arange(N, dtype=np.int32), (B, HKV, 1)))
        self.lens = ra.HipStorage.from_numpy(np.array([BUDGET, BUDGET, 3], np.int32))  # two at the budget, one far below
        self.gamma = ra.HipStorage.from_numpy((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
        self.q, self.q_out, self.out = (ra.HipStorage(B * HQ * D * 2) for _ in range(3))
        self.k_in, self.v_in = (ra.HipStorage(B * HKV * D * 2) for _ in range(2))
        self.ws = ra.HipStorage(max(K.gqa_decode_weights_workspace_bytes(B, HQ, HKV, D, N), K.kv_evict_workspace_bytes(B, HKV, N, BUDGET)))
        self.rng = np.random.default_rng(seed + 100)

    def new_token(self):
        self.token = [bf16_bits(self.rng.standard_normal((B, h, 1, D))) for h in (HQ, HKV, HKV)]
        for buf, x in zip((self.q, self.k_in, self.v_in), self.token):
            buf.upload(x)

    def step(self, stream, positions, rope):
        """What a program calls for one layer of one token."""
        append, attend, cut = ((K.qk_norm_rope_kv_append_q4, K.gqa_decode_weights_q4, K.kv_evict_q4) if self.q4 else
                               (K.qk_norm_rope_kv_append_rows_bf16, K.gqa_decode_weights_bf16, K.kv_evict_bf16))
        append(stream, self.q, self.q_out, self.k_in, self.v_in, self.k, self.v, positions, rope, B, HQ, HKV, D, N, q_gamma=self.gamma, k_gamma=self.gamma,
               rows=self.lens, slots=self.slots, weights=self.weights)
        ra.i32_add_dev(self.lens, B, 1, stream)
        attend(stream, self.q_out, self.k, self.v, self.out, self.weights, self.weights, self.lens, B, HQ, HKV, D, N, self.ws, self.ws.byte_len)
        cut(stream, self.k, self.v, self.weights, self.slots, self.weights, self.slots, self.lens, self.lens, B, HKV, D, N, BUDGET, RECENT, self.ws,
            self.ws.byte_len)

    def state(self):
        bufs = [self.k.codes, self.k.pairs, self.v.codes, self.v.pairs] if self.q4 else [self.k, self.v]
        return [x.download(np.uint8) for x in (*bufs, self.weights, self.slots, self.lens, self.out)]

    def shaped(self):
        if self.q4:
            cache = [y for x in (self.k, self.v) for y in (x.codes.download(np.uint8).reshape(B, HKV, N, D // 2), x.pairs.download(np.uint32).reshape(B, HKV, 1, N))]
        else:
            cache = [x.download(np.uint16).reshape(B, HKV, N, D) for x in (self.k, self.v)]
        return cache, self.weights.download(np.float32).reshape(B, HKV, N), self.slots.download(np.int32).reshape(B, HKV, N), self.lens.download(np.int32)


@pytest.mark.parametrize("q4", [False, True])
def test_each_step_is_the_definitions(q4):
    layer, rope, at = Layer(41, q4), ra.RoPE(D, 400), 150
    cos, sin = rope.cos.reshape(-1, D // 2), rope.sin.reshape(-1, D // 2)
    gamma = layer.gamma.download(np.float32)
    for t in range(4):
        layer.new_token()
        cache, weights, slots, lens = layer.shaped()
        pos = np.full(B, at + t, np.int32)
        layer.step(None, ra.HipStorage.from_numpy(pos), rope)
        ra.synchronize()
        after, w_after, s_after, l_after = layer.shaped()
        # the append, by definition, on what was there
        q, k = (prepare(bf16_values(x), gamma, 1e-6, cos, sin, pos) for x in layer.token[:2])
        for i in range(B):
            new = [*quantise(k[i]), *quantise(bf16_values(layer.token[2][i]))] if q4 else [bf16_bits(k[i]), layer.token[2][i]]
            for x, y in zip(cache, new):
                if x.shape[-1] == N and q4:
                    x[i, :, :, lens[i]] = y[:, :, 0]
                else:
                    x[i, :, lens[i]] = y[:, 0]
            weights[i, :, lens[i]], slots[i, :, lens[i]] = 0, at + t
        # attention over it
        q = bf16_values(bf16_bits(q)).reshape(B, 1, HQ, D)
        want = expect_q4(q, *cache, lens + 1) if q4 else expect_bf16(q, *(bf16_values(x) for x in cache), lens + 1)
        want.check(bf16_values(layer.out.download(np.uint16)).reshape(B, 1, HQ, D))
        # and what stays: by the sums as the device has them, which is told by the rows that did
        assert np.array_equal(l_after, np.minimum(lens + 1, BUDGET))
        for i in range(B):
            for j in range(HKV):
                m = l_after[i]
                row = {int(s): r for r, s in enumerate(slots[i, j, :lens[i] + 1])}
                source = np.array([row[int(s)] for s in s_after[i, j, :m]])
                assert len(set(source)) == m
                sums = weights[i, j] + want.weights[i, j]
                off = want.weight_bound[i, j] + 2.0 ** -22 * np.abs(sums)
                assert (np.abs(w_after[i, j, :m] - sums[source]) <= off[source]).all()
                gone = np.setdiff1d(np.arange(lens[i] + 1), source)
                assert len(gone) == lens[i] + 1 - m
                for g in gone:  # none of the newest, and no larger sum than any of the others
                    assert slots[i, j, g] <= at + t - RECENT
                    old = source[slots[i, j, source] <= at + t - RECENT]
                    assert (sums[old] + off[old] >= sums[g] - off[g]).all()
                for x, y in zip(cache, after):
                    if x.shape[-1] == N and q4:
                        assert np.array_equal(y[i, j][:, :m], x[i, j][:, source])
                    else:
                        assert np.array_equal(y[i, j, :m], x[i, j, source])


@pytest.mark.parametrize("q4", [False, True])
def test_the_loop_in_a_graph_has_the_bits_of_the_eager_one(q4):
    ra.init(0)
    hip, rope = Hip(), ra.RoPE(D, 400)
    rope.device_tables()
    stream = ra.Stream()

    def loop(run):
        """The layers' states behind each token; run(step): one token."""
        layers = [Layer(51 + i, q4) for i in range(2)]
        positions = ra.HipStorage.from_numpy(np.full(B, 150, np.int32))

        def token():
            for x in layers:
                x.step(stream, positions, rope)
            ra.i32_add_dev(positions, B, 1, stream)

        go, end = run(token)
        seen = []
        for _ in range(5):
            for x in layers:
                x.new_token()
            go()
            stream.synchronize()
            seen.append([x.state() for x in layers])
        end()
        return seen

    def recorded(token):
        graph, exe, types = hip.capture(stream, token)
        assert NODE_TYPE_MEMSET not in types
        return (lambda: hip.launch(exe, stream)), (lambda: hip.destroy(graph, exe))

    eager, replayed = loop(lambda token: (token, lambda: None)), loop(recorded)
    for a, b in zip(eager, replayed):
        for x, y in zip(a, b):
            for u, v in zip(x, y):
                assert np.array_equal(u, v)


def test_eviction_agrees_with_the_definition_at_the_ends():
    """`evict` of the tests itself, on a case worked by hand: the newest two and the largest sums, the lower of equals."""
    w = np.array([[[5, 1, 3, 3, 0, 9, 0, 0]]], np.float32)
    slots = np.array([[[0, 1, 2, 3, 4, 5, 6, 7]]], np.int32)
    source, new = evict(w, slots, np.array([8]), 5, 2)
    assert source[0, 0].tolist() == [0, 5, 2, 6, 7] and new[0] == 5
