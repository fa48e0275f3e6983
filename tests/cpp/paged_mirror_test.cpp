// Tests of the C++ host mirror's calls for packed tokens and caches in pages (include/rustorch_attn.hpp).
//   paged_mirror_test errors   what they refuse, and as what: needs no GPU
//   paged_mirror_test rows     what they say of a host position
//   paged_mirror_test gpu      append, attention of the prompts, decode steps with a shared prefix
//   paged_mirror_test prefix   which rows a prefix is read through
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
    alignas(16) static int32_t some[64];
    const KVPages pages{some, some, 4, 16};
    RoPE rope(64, 16);
    const size_t many = (size_t)1 << 40;
    CHECK(throws<RoPEError>([&] { LlmKernels::qk_norm_rope_kv_append_paged_bf16(nullptr, some, some, some, nullptr, some, pages, some, 4, nullptr, nullptr, 16, nullptr, {}, nullptr, nullptr, 1e-6f, rope, 1, 1, 1, 1, 64); }));
    CHECK(throws<KVCacheOverflow>([&] { LlmKernels::qk_norm_rope_kv_append_paged_bf16(nullptr, some, some, some, nullptr, some, KVPages{some, some, 4, 8}, some, 1, nullptr, nullptr, 8, nullptr, {}, nullptr, nullptr, 1e-6f, rope, 1, 1, 1, 1, 64); }));
    CHECK(throws<GQAError>([&] { LlmKernels::gqa_decode_paged_bf16(nullptr, some, pages, some, some, 4, some, nullptr, 0, 1, 4, 3, 64, some, many); }));
    CHECK(throws<AttentionError>([&] { LlmKernels::flash_forward_packed_bf16(nullptr, AttentionShape::make(1, 4, 8, 0), 4, some, some, some, some, some); }));
    CHECK(LlmKernels::gqa_decode_paged_workspace_bytes(2, 4, 2, 64, 16, 8) > 0 && LlmKernels::gqa_decode_paged_workspace_bytes(2, 4, 2, 64, 17, 8) == 0);
}

// A host position, with and without `starts`, against the last row of the tables and of the page table.
static void rows() {
    alignas(16) static int32_t some[64];
    RoPE rope(64, 16);
    auto call = [&](const int32_t* starts, int32_t pos, const KVPages& pages, int32_t table_pages) {
        LlmKernels::qk_norm_rope_kv_append_paged_bf16(nullptr, some, some, some, nullptr, some, pages, some, table_pages, starts, nullptr, pos, nullptr, {}, nullptr, nullptr, 1e-6f, rope, 2, 1, 1, 1, 64);
    };
    const KVPages wide{some, some, 4, 16}, narrow{some, some, 4, 8};
    CHECK(throws<RoPEError>([&] { call(some, 16, wide, 4); }) && throws<RoPEError>([&] { call(nullptr, 15, wide, 4); }));
    CHECK(throws<KVCacheOverflow>([&] { call(some, 8, narrow, 1); }) && throws<KVCacheOverflow>([&] { call(nullptr, 7, narrow, 1); }));
    // (page tables of 2^31 and 2^32 rows, which the entry refuses as too large: no position is behind them)
    for (int32_t table_pages : {1 << 27, 1 << 28}) CHECK(throws<DeviceError>([&] { call(nullptr, 3, wide, table_pages); }));
    // tables of another head dim than the heads'
    RoPE half(32, 16);
    for (int32_t dim : {64, 16})
        CHECK(throws<RoPEError>([&] { LlmKernels::qk_norm_rope_kv_append_paged_bf16(nullptr, some, some, some, nullptr, some, wide, some, 4, some, some, 0, nullptr, {}, nullptr, nullptr, 1e-6f, half, 2, 1, 1, 1, dim); }));
}

template <typename T>
static HipStorage up(const std::vector<T>& v) {
    HipStorage s(v.size() * sizeof(T));
    rt_err_detail e;
    detail::check_device(rt_memcpy_h2d(s.ptr(), v.data(), v.size() * sizeof(T), nullptr, &e), e);
    detail::check_device(rt_stream_synchronize(nullptr, &e), e);
    return s;
}
static std::vector<uint16_t> back(const HipStorage& s, size_t n) {
    std::vector<uint16_t> v(n);
    rt_err_detail e;
    detail::check_device(rt_memcpy_d2h(v.data(), s.ptr(), n * 2, nullptr, &e), e);
    detail::check_device(rt_stream_synchronize(nullptr, &e), e);
    return v;
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

// Two prompts of 40 and 21 tokens whose q and k are zeros, so that every key weighs the same, and whose V is the token's number in every dim: an
// output is the mean of the numbers up to it.  Then a step of each behind the first 16 tokens of the first prompt, which both share.
static void gpu() {
    const int heads = 4, kv = 2, d = 64, tokens = 61, page = 16;
    RoPE rope(d, 64);
    std::vector<uint16_t> v_in(tokens * kv * d);
    for (int t = 0; t < tokens; t++)
        for (int i = 0; i < kv * d; i++) v_in[t * kv * d + i] = bits((float)(t < 40 ? t : t - 40));
    HipStorage q = up(std::vector<uint16_t>(tokens * heads * d)), k = up(std::vector<uint16_t>(tokens * kv * d)), v = up(v_in), out(tokens * heads * d * 2);
    HipStorage starts = up(std::vector<int32_t>{0, 40, 61}), rows = up(std::vector<int32_t>{0, 0});
    HipStorage k_pages(5 * kv * page * d * 2), v_pages(5 * kv * page * d * 2);
    HipStorage write = up(std::vector<int32_t>{4, 0, 2, -1, 3, -1}), read = up(std::vector<int32_t>{4, 0, 2, 4, 3, -1});
    const KVPages pages{k_pages.ptr(), v_pages.ptr(), 5, page};
    LlmKernels::qk_norm_rope_kv_append_paged_bf16(nullptr, q.ptr(), q.ptr(), k.ptr(), k.ptr(), v.ptr(), pages, (int32_t*)write.ptr(), 3, (int32_t*)starts.ptr(), (int32_t*)rows.ptr(), 0, nullptr, {}, nullptr,
                                                  nullptr, 1e-6f, rope, tokens, 2, heads, kv, d);
    LlmKernels::flash_forward_packed_bf16(nullptr, AttentionShape::make(2, heads, tokens, d), kv, q.ptr(), k.ptr(), v.ptr(), (int32_t*)starts.ptr(), out.ptr());
    const std::vector<uint16_t> got = back(out, tokens * heads * d);
    for (int t = 0; t < tokens; t++)
        for (int i = 0; i < heads * d; i++) {
            const double mean = 0.5 * (t < 40 ? t : t - 40);
            CHECK(std::fabs(value(got[t * heads * d + i]) - mean) <= std::ldexp(mean, -7));
        }
    HipStorage lens = up(std::vector<int32_t>{40, 21}), one(2 * heads * d * 2), zero = up(std::vector<uint16_t>(2 * heads * d));
    const size_t bytes = LlmKernels::gqa_decode_paged_workspace_bytes(2, heads, kv, d, page, 3);
    HipStorage space(bytes);
    for (int shared : {0, 16}) {
        LlmKernels::gqa_decode_paged_bf16(nullptr, zero.ptr(), pages, one.ptr(), (int32_t*)read.ptr(), 3, (int32_t*)lens.ptr(), nullptr, shared, 2, heads, kv, d, space.ptr(), bytes);
        const std::vector<uint16_t> step = back(one, 2 * heads * d);
        for (int i = 0; i < 2 * heads * d; i++) {
            const double mean = i < heads * d ? 19.5 : 10.0;
            CHECK(std::fabs(value(step[i]) - mean) <= std::ldexp(mean, -7));
        }
    }
}

// Two sequences of 32 keys, whose first 16 are said to be the same, in pages of their own that hold 1 and 5 (then 3 and 7) in every dim of V: which of
// them a sequence's mean is made of is how the prefix was read.  On the device its length has it read once, through the first sequence; the host's
// is too short for that, and 0 is no prefix.
static void prefix() {
    const int heads = 4, kv = 2, d = 64, page = 16;
    std::vector<uint16_t> v(4 * kv * page * d);
    for (int p = 0; p < 4; p++)
        for (int i = 0; i < kv * page * d; i++) v[p * kv * page * d + i] = bits((float)(p == 0 ? 1 : p == 1 ? 3 : p == 2 ? 5 : 7));
    HipStorage k_pages = up(std::vector<uint16_t>(v.size())), v_pages = up(v), q = up(std::vector<uint16_t>(2 * heads * d)), out(2 * heads * d * 2);
    HipStorage table = up(std::vector<int32_t>{0, 1, 2, 3}), lens = up(std::vector<int32_t>{32, 32}), sixteen = up(std::vector<int32_t>{16}), none = up(std::vector<int32_t>{0});
    const KVPages pages{k_pages.ptr(), v_pages.ptr(), 4, page};
    const size_t bytes = LlmKernels::gqa_decode_paged_workspace_bytes(2, heads, kv, d, page, 2);
    HipStorage space(bytes);
    auto second = [&](const int32_t* shared_lens, int32_t shared) {  // the second sequence's mean; the first's is 2 whatever is read
        LlmKernels::gqa_decode_paged_bf16(nullptr, q.ptr(), pages, out.ptr(), (int32_t*)table.ptr(), 2, (int32_t*)lens.ptr(), shared_lens, shared, 2, heads, kv, d, space.ptr(), bytes);
        const std::vector<uint16_t> got = back(out, 2 * heads * d);
        for (int i = 0; i < heads * d; i++) CHECK(value(got[i]) == 2.0f && got[heads * d + i] == got[heads * d]);
        return value(got[heads * d]);
    };
    CHECK(second((int32_t*)sixteen.ptr(), 0) == 4.0f);
    CHECK(second((int32_t*)sixteen.ptr(), -3) == 4.0f);  // (the host's is not looked at there)
    CHECK(second((int32_t*)none.ptr(), 16) == 6.0f);
    CHECK(second(nullptr, 16) == 6.0f && second(nullptr, 0) == 6.0f);
}

int main(int argc, char** argv) {
    if (argc > 1 && !std::strcmp(argv[1], "gpu")) gpu();
    else if (argc > 1 && !std::strcmp(argv[1], "rows")) rows();
    else if (argc > 1 && !std::strcmp(argv[1], "prefix")) prefix();
    else errors();
    std::printf(g_failed ? "%d failed\n" : "ok\n", g_failed);
    return g_failed != 0;
}
