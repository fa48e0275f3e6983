// Tests of the C++ host mirror's calls for caches that are kept small (include/rustorch_attn.hpp).
//   cache_mirror_test errors   what they refuse, and as what: needs no GPU
//   cache_mirror_test gpu      append, attention that sums the keys' weights, eviction, over both kinds of cache
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "rustorch_attn.hpp"

using namespace rustorch_attn;

static int g_failed = 0;
#define CHECK(cond)                                                     \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failed;                                                 \
        }                                                               \
    } while (0)

template <typename E, typename F>
static bool throws(F&& f) {
    try {
        f();
    } catch (const E&) {
        return true;
    } catch (...) {
    }
    return false;
}

static void errors() {
    alignas(16) static uint32_t some[64];
    const Q4Rows rows{some, some};
    RoPE rope(64, 16);
    const size_t many = (size_t)1 << 40;
    CHECK(throws<RoPEError>([&] { LlmKernels::qk_norm_rope_kv_append_q4(nullptr, some, some, some, some, rows, rows, nullptr, 16, nullptr, nullptr, nullptr, nullptr, nullptr, 1e-6f, rope, 1, 1, 1, 64, 32); }));
    CHECK(throws<KVCacheOverflow>([&] { LlmKernels::qk_norm_rope_kv_append_rows_bf16(nullptr, some, some, some, some, some, some, nullptr, 8, nullptr, nullptr, nullptr, nullptr, nullptr, 1e-6f, rope, 1, 1, 1, 64, 8); }));
    CHECK(throws<KVCacheOverflow>([&] { LlmKernels::kv_cache_append_q4(nullptr, rows, rows, some, 64, some, 64, 1, 1, 4, 64, 4, 1); }));
    CHECK(throws<KVCacheWrongInputLen>([&] { LlmKernels::kv_cache_append_q4(nullptr, rows, rows, some, 63, some, 64, 1, 1, 4, 64, 0, 1); }));
    CHECK(throws<KVCacheOverflow>([&] { LlmKernels::kv_cache_read_q4(nullptr, rows, some, nullptr, 3, 2, 1, 1, 64, 4); }));
    CHECK(throws<GQAError>([&] { LlmKernels::gqa_decode_q4(nullptr, some, rows, rows, some, nullptr, 4, 1, 1, 4, 3, 64, 4, some, many); }));
    CHECK(throws<GQAError>([&] { LlmKernels::gqa_decode_weights_bf16(nullptr, some, some, some, some, nullptr, (float*)some, nullptr, 1, 4, 3, 64, 4, some, many); }));
    CHECK(throws<GQAError>([&] { LlmKernels::gqa_decode_weights_q4(nullptr, some, rows, rows, some, nullptr, (float*)some, nullptr, 1, 4, 3, 64, 4, some, many); }));
    CHECK(throws<DeviceError>([&] { LlmKernels::kv_evict_bf16(nullptr, some, some, (float*)some, (int32_t*)some, (float*)some, (int32_t*)some, (int32_t*)some, nullptr, 1, 1, 64, 4, 2, 3, some, many); }));
    CHECK(throws<DeviceError>([&] { LlmKernels::kv_evict_q4(nullptr, rows, rows, (float*)some, (int32_t*)some, (float*)some, (int32_t*)some, (int32_t*)some, nullptr, 1, 1, 64, 4, -1, 0, some, many); }));
    CHECK(LlmKernels::gqa_decode_q4_workspace_bytes(1, 1, 4, 2, 64, 100) > 0 && LlmKernels::gqa_decode_weights_workspace_bytes(1, 4, 2, 64, 100) > 0 &&
          LlmKernels::kv_evict_workspace_bytes(1, 2, 100, 10) > 0);
}

template <typename T>
static std::vector<T> back(const HipStorage& s, size_t n) {
    std::vector<T> v(n);
    rt_err_detail e;
    detail::check_device(rt_memcpy_d2h(v.data(), s.ptr(), n * sizeof(T), nullptr, &e), e);
    return v;
}
static HipStorage zeros(size_t bytes) {
    HipStorage s(bytes);
    rt_err_detail e;
    detail::check_device(rt_buf_zero(s.ptr(), bytes, nullptr, &e), e);
    return s;
}
static uint16_t bits(float x) {  // of numbers that are bf16
    uint32_t u;
    std::memcpy(&u, &x, 4);
    return (uint16_t)(u >> 16);
}
static float value(uint16_t b) {
    const uint32_t u = (uint32_t)b << 16;
    float x;
    std::memcpy(&x, &u, 4);
    return x;
}

// Twelve tokens whose q and k are zeros, so that every key weighs the same, and whose V is the token's number in every dim: the output is
// the mean of the numbers, a key's sum what it has drawn by then.  From the eighth token on one row goes for each that comes: of the
// old ones that with the smallest sum, which is the youngest of them.
static void gpu(bool q4) {
    const int heads = 4, kv = 2, d = 64, n = 16, budget = 8, recent = 2, tokens = 12;
    RoPE rope(d, 32);
    HipStorage q = zeros(heads * d * 2), k_in = zeros(kv * d * 2), v_in(kv * d * 2), out(heads * d * 2), sums = zeros(kv * n * 4), slots = zeros(kv * n * 4), pos = zeros(4), rows = zeros(4),
               lens = zeros(4);
    HipStorage k = zeros(kv * n * d * 2), v = zeros(kv * n * d * 2), kp = zeros(kv * n * 4), vp = zeros(kv * n * 4);  // (codes take a quarter)
    const Q4Rows k4{k.ptr(), (uint32_t*)kp.ptr()}, v4{v.ptr(), (uint32_t*)vp.ptr()};
    const size_t attend_bytes = LlmKernels::gqa_decode_weights_workspace_bytes(1, heads, kv, d, n), evict_bytes = LlmKernels::kv_evict_workspace_bytes(1, kv, n, budget);
    HipStorage attend_space(attend_bytes), evict_space(evict_bytes);
    float* w = (float*)sums.ptr();
    int32_t* s = (int32_t*)slots.ptr();
    rt_err_detail e;
    std::vector<double> drawn;  // of the rows that are there, by the token
    std::vector<int> there;
    for (int t = 0; t < tokens; t++) {
        const std::vector<uint16_t> row(kv * d, bits((float)t));
        detail::check_device(rt_memcpy_h2d(v_in.ptr(), row.data(), row.size() * 2, nullptr, &e), e);
        if (q4) LlmKernels::qk_norm_rope_kv_append_q4(nullptr, q.ptr(), q.ptr(), k_in.ptr(), v_in.ptr(), k4, v4, (int32_t*)pos.ptr(), 0, (int32_t*)rows.ptr(), s, w, nullptr, nullptr, 1e-6f, rope, 1, heads, kv, d, n);
        else LlmKernels::qk_norm_rope_kv_append_rows_bf16(nullptr, q.ptr(), q.ptr(), k_in.ptr(), v_in.ptr(), k.ptr(), v.ptr(), (int32_t*)pos.ptr(), 0, (int32_t*)rows.ptr(), s, w, nullptr, nullptr, 1e-6f, rope, 1, heads, kv, d, n);
        LlmKernels::i32_add_dev(nullptr, (int32_t*)lens.ptr(), 1, 1);
        if (q4) LlmKernels::gqa_decode_weights_q4(nullptr, q.ptr(), k4, v4, out.ptr(), w, w, (int32_t*)lens.ptr(), 1, heads, kv, d, n, attend_space.ptr(), attend_bytes);
        else LlmKernels::gqa_decode_weights_bf16(nullptr, q.ptr(), k.ptr(), v.ptr(), out.ptr(), w, w, (int32_t*)lens.ptr(), 1, heads, kv, d, n, attend_space.ptr(), attend_bytes);
        there.push_back(t);
        drawn.push_back(0.0);
        double mean = 0.0;
        for (size_t i = 0; i < there.size(); i++) {
            mean += (double)there[i] / there.size();
            drawn[i] += 2.0 / there.size();  // two heads a kv head
        }
        for (uint16_t x : back<uint16_t>(out, heads * d)) CHECK(std::fabs(value(x) - mean) <= std::ldexp(mean, -8));
        if (q4) LlmKernels::kv_evict_q4(nullptr, k4, v4, w, s, w, s, (int32_t*)lens.ptr(), (int32_t*)lens.ptr(), 1, kv, d, n, budget, recent, evict_space.ptr(), evict_bytes);
        else LlmKernels::kv_evict_bf16(nullptr, k.ptr(), v.ptr(), w, s, w, s, (int32_t*)lens.ptr(), (int32_t*)lens.ptr(), 1, kv, d, n, budget, recent, evict_space.ptr(), evict_bytes);
        if ((int)there.size() > budget) {  // the third last: the youngest but `recent`; the last row takes its place
            const size_t goes = there.size() - 1 - recent;
            there.erase(there.begin() + goes);
            drawn.erase(drawn.begin() + goes);
        }
        const std::vector<int32_t> len = back<int32_t>(lens, 1), at = back<int32_t>(slots, kv * n);
        const std::vector<float> sum = back<float>(sums, kv * n);
        CHECK(len[0] == (int)there.size());
        for (int h = 0; h < kv; h++)
            for (size_t i = 0; i < there.size(); i++) {
                int found = 0;
                for (int j = 0; j < len[0]; j++)
                    if (at[h * n + j] == there[i]) {
                        found++;
                        CHECK(std::fabs(sum[h * n + j] - drawn[i]) <= 1e-5 * drawn[i]);
                    }
                CHECK(found == 1);
            }
        LlmKernels::i32_add_dev(nullptr, (int32_t*)pos.ptr(), 1, 1);
        detail::check_device(rt_memcpy_h2d(rows.ptr(), len.data(), 4, nullptr, &e), e);
    }
    if (q4) {
        HipStorage rows_back(kv * budget * d * 2);
        LlmKernels::kv_cache_read_q4(nullptr, v4, rows_back.ptr(), nullptr, 0, budget, 1, kv, d, n);
        const std::vector<uint16_t> x = back<uint16_t>(rows_back, kv * budget * d);
        const std::vector<int32_t> at = back<int32_t>(slots, kv * n);
        for (int h = 0; h < kv; h++)
            for (int j = 0; j < budget; j++) CHECK(value(x[(h * budget + j) * d]) == (float)at[h * n + j]);
    }
}

int main(int argc, char** argv) {
    if (argc > 1 && !std::strcmp(argv[1], "gpu")) {
        gpu(false);
        gpu(true);
    } else {
        errors();
    }
    std::printf(g_failed ? "%d failed\n" : "ok\n", g_failed);
    return g_failed != 0;
}
