// The rows of a cache that stay when it is cut to a budget, by the attention that their keys have drawn: of every (sequence, kv head)
// with more rows than `budget`, the `recent` newest tokens' and those with the largest sums of weights.
//
// A row's place in a cache says nothing to attention (its position went into the key with the rotation), so what stays need not keep its
// order: the kept rows behind the new length take, in order, the slots that are freed below it.  Only they are read and written --
// after a cut to a quarter three of four kept rows, in a loop that evicts one row a token a single one, where rows moved
// together in order would all have to move -- and no row that is read lies where one is written, so a copy needs no order either.
//
//   cache_select_kernel  one workgroup a (sequence, kv head): the budget-th largest sum by counts, then one pass in slot order that
//                        numbers the freed slots and the rows that move
//   cache_move_kernel    copies them
#include <algorithm>

#include "cache_q4.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"

namespace rt {

namespace {

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64, kPer = 8, kTile = kSelect * kPer;  // a thread's neighbouring slots; slots of a tile
constexpr int kBins = 2048;
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes from any word

// The order of the sums as that of whole numbers: NaN counts as -infinity, -0 as 0, the newest tokens' as +infinity.  0 is no sum's.
constexpr uint32_t kNewest = 0xff800000u;
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f), x = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    return w != w ? 0x007fffffu : x;
}

__device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ uint32_t bits(int32_t x) { return (uint32_t)x; }

// A workgroup's largest of three numbers and its sums: in a wave, then over the waves' results in `room` (not those of the call
// before: one barrier is enough then), all of it within registers (lanes_step, cache_q4.hpp).
__device__ __forceinline__ void largest_of(uint32_t (&x)[3], uint32_t (*room)[kSelectWaves]) {
    auto f = [](uint32_t a, uint32_t b) __attribute__((always_inline)) { return max(a, b); };
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const uint32_t y = lanes_fold<6>(x[i], f);
        if ((threadIdx.x & 63) == 63) room[i][threadIdx.x >> 6] = y;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; i++) x[i] = __builtin_amdgcn_readlane(lanes_fold<4>(room[i][threadIdx.x & (kSelectWaves - 1)], f), kSelectWaves - 1);
}
// The sum over the threads before this one; `all`: over all.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* room, uint32_t* all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t end = lane_sums((int)x);
    if (lane == 63) room[wave] = end;
    __syncthreads();
    const uint32_t ends = lane_sums((int)(lane < kSelectWaves ? room[lane] : 0u));
    *all = __builtin_amdgcn_readlane(ends, kSelectWaves - 1);
    return end - x + (wave ? __builtin_amdgcn_readlane(ends, wave - 1) : 0u);
}

// One workgroup a (sequence, kv head), grid (kv heads, batch).  Thread t has the slots 8 t .. 8 t + 7 of a tile of 8192; up to there the keys are
// read once and stay in registers (kOne), longer heads are walked tile by tile again for every question.
// The budget-th largest key is found by counts: the range that the keys in question span is cut into 2048 bins, and the bin it falls in is
// the next range -- three times at most, since 2048^3 > 2^32, and twice as a rule, since bins that follow the keys' own range hold few of them.
// (By fixed bytes from the top most sums share a bin, and a wave's counts in one word wait for each other: 8192 keys 30 us.)
// 8192 slots of 8 heads to 2048: 8.4 us, of which 1.9 until the sums are there, 1.8 for the counts, 2.2 for the lists; bound by the instructions of the one CU that
// a head has and by its barriers (14.5 us with the sums over threads through LDS and a barrier on either side of each).
// kOne goes by the cache's rows, which the host knows, not by the lengths: with a cache of 8193 rows the whole eviction of those 8192 takes 15.0 us for
// 12.1, of 4096 rows in a cache of 16384 13.5 for 11.0, of 32 x 300 .. 4096 in such a cache 38 for 33.  Longer heads, 8 of them: 16384 rows to 4096
// 24.5 us, 65536 to 8192 68, by the one workgroup a head.
template <bool kOne>
__global__ __launch_bounds__(kSelect) void cache_select_kernel(CacheEvictParams p) {
    __shared__ uint32_t bins[kBins], chosen[2], above_all, room[6][kSelectWaves];
    __shared__ uint16_t listed[2 * kTile];  // of a tile, in order: the slots that are freed, and behind them the rows that move
    const int tid = threadIdx.x, b = blockIdx.y, head = b * p.n_kv + (int)blockIdx.x;
    const int len = min(max(p.kv_lens[b], 0), p.max_seq);
    const float* w_in = p.weights_in + (size_t)head * p.max_seq;
    const int32_t* s_in = p.slots_in + (size_t)head * p.max_seq;
    float* w_out = p.weights_out + (size_t)head * p.max_seq;
    int32_t* s_out = p.slots_out + (size_t)head * p.max_seq;
    const bool copy_w = w_in != w_out, copy_s = s_in != s_out;
    float w[kPer];
    int32_t s[kPer];
    auto load = [&](int tile) __attribute__((always_inline)) {
        const int j0 = tile * kTile + tid * kPer;
        if (j0 + kPer <= p.max_seq) {  // (whatever the length, which is still on its way)
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
                const u32x4_any a = *(const u32x4_any*)(w_in + j0 + e), c = *(const u32x4_any*)(s_in + j0 + e);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    w[e + i] = __uint_as_float(a[i]);
                    s[e + i] = (int32_t)c[i];
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            w[e] = j0 + e < p.max_seq ? w_in[j0 + e] : 0.0f;
            s[e] = j0 + e < p.max_seq ? s_in[j0 + e] : 0;
        }
    };
    uint32_t key[kPer];
    auto sums = [&](int tile) __attribute__((always_inline)) {  // 0 behind the last slot
        const int there = len - tile * kTile - tid * kPer;
#pragma unroll
        for (int e = 0; e < kPer; e++) key[e] = e < there ? key_of(w[e]) : 0u;
    };
    if (kOne) load(0);
    if (len <= p.budget || p.budget == 0) {  // all of it stays, or nothing
        for (int j = tid; j < min(len, p.budget); j += kSelect) {
            if (copy_w) w_out[j] = w_in[j];
            if (copy_s) s_out[j] = s_in[j];
        }
        if (tid == 0) {
            p.header[2 * head] = len;
            p.header[2 * head + 1] = 0;
        }
        return;
    }
    const int tiles = kOne ? 1 : (len + kTile - 1) / kTile;
    bins[tid] = bins[tid + kSelect] = 0;
    if (tid == 0) above_all = 0;
    // the newest token (positions as unsigned numbers in their order), and the range of the sums' keys
    uint32_t most[3] = {0, 0, 0};
    for (int t = 0; t < tiles; t++) {
        if (!kOne) load(t);
        sums(t);
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            most[0] = max(most[0], key[e] ? bits(s[e]) ^ 0x80000000u : 0u);
            most[1] = max(most[1], key[e]);
            most[2] = max(most[2], key[e] ? ~key[e] : 0u);
        }
    }
    largest_of(most, room);
    const uint32_t newest = most[0] ^ 0x80000000u;
    uint32_t high = most[1], low = ~most[2];
    auto newer = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < kPer; e++) key[e] = key[e] && newest - bits(s[e]) < (uint32_t)p.recent ? kNewest : key[e];
    };
    auto keys = [&](int tile) __attribute__((always_inline)) {
        if (kOne) return;
        load(tile);
        sums(tile);
        newer(tile);
    };
    if (kOne) newer(0);
    // The newest tokens' keys lie above the range, and are counted apart the first time.  Of the keys in [low, high] the left-th largest is the
    // threshold; where all of a bin's stay, what lies below it is one as well, of which none stays.
    uint32_t left = (uint32_t)p.budget, above_range = 0;
    for (bool first = true; first || low < high; first = false) {
        const int shift = max(0, 32 - __builtin_clz((high - low) | 1u) - 11);  // (high - low) >> shift < 2048
        const uint32_t width = high - low;
        for (int t = 0; t < tiles; t++) {
            keys(t);
            if (width) {
#pragma unroll
                for (int e = 0; e < kPer; e++) {
                    const uint32_t x = key[e] - low;
                    if (x <= width) atomicAdd(&bins[x >> shift], 1u);
                }
            }
            if (first) {
#pragma unroll
                for (int e = 0; e < kPer; e++) above_range += (uint32_t)__popcll(__ballot(key[e] > high));
            }
        }
        if (first && above_range && (tid & 63) == 0) atomicAdd(&above_all, above_range);
        __syncthreads();
        if (first) {
            above_range = above_all;
            if (left <= above_range) {
                low = kNewest;
                break;
            }
            left -= above_range;
            if (low == high) break;
        }
        // thread t has the bins 2047 - 2 t and 2046 - 2 t: those above it are those before it
        const uint32_t c0 = bins[kBins - 1 - 2 * tid], c1 = bins[kBins - 2 - 2 * tid];
        bins[kBins - 1 - 2 * tid] = bins[kBins - 2 - 2 * tid] = 0;
        uint32_t all;
        const uint32_t above = sum_before(c0 + c1, room[3], &all);
        if (above < left && left <= above + c0 + c1) {
            const bool second = left > above + c0;
            const uint32_t rest = left - above - (second ? c0 : 0u);
            chosen[0] = (uint32_t)(kBins - 1 - 2 * tid) - (second ? 1u : 0u);
            chosen[1] = rest == (second ? c1 : c0) ? 0u : rest;
        }
        __syncthreads();
        const uint32_t bin = chosen[0];
        left = chosen[1];
        high = min(high, low + ((bin + 1) << shift) - 1);  // (no further than the range: low + 2^32 does not come up)
        low += bin << shift;
        if (left == 0) {
            low--;
            break;
        }
    }
    // in slot order: keys above it stay, and the first `left` that equal it
    uint32_t equal = 0, freed = 0, moved = 0;
    int32_t* from = p.from + (size_t)head * p.most;
    int32_t* to = p.to + (size_t)head * p.most;
    for (int t = 0; t < tiles; t++) {
        keys(t);
        const int j0 = t * kTile + tid * kPer;
        uint32_t keep = 0, all;  // bits of the slots that stay
        if (left) {
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < kPer; e++) mine += key[e] == low;
            uint32_t rank = equal + sum_before(mine, room[4], &all);
            equal += all;
#pragma unroll
            for (int e = 0; e < kPer; e++) {
                keep |= (key[e] == low && rank < left ? 1u : 0u) << e;
                rank += key[e] == low;
            }
        }
#pragma unroll
        for (int e = 0; e < kPer; e++) keep |= (key[e] > low ? 1u : 0u) << e;
        const uint32_t below = (1u << min(max(p.budget - j0, 0), kPer)) - 1u, which = keep ^ below;  // (the budget is less than the length)
        const uint32_t before = sum_before((uint32_t)__popc(which & below) + ((uint32_t)__popc(which & ~below) << 16), room[5], &all);  // 8192 each at most
        uint32_t at_hole = before & 0xffffu, at_mover = kTile + (before >> 16);
#pragma unroll
        for (int e = 0; e < kPer; e++)
            if (which >> e & 1u) listed[below >> e & 1u ? at_hole++ : at_mover++] = (uint16_t)(tid * kPer + e);
        // (freed slots too: a row that moves comes over them later)
        auto put = [&](auto* to, const auto (&x)[kPer]) __attribute__((always_inline)) {
            if (j0 + kPer <= p.budget) {
#pragma unroll
                for (int e = 0; e < kPer; e += 4) *(u32x4_any*)(to + j0 + e) = u32x4_any{bits(x[e]), bits(x[e + 1]), bits(x[e + 2]), bits(x[e + 3])};
            } else {
#pragma unroll
                for (int e = 0; e < kPer; e++)
                    if (j0 + e < p.budget) to[j0 + e] = x[e];
            }
        };
        if (copy_w) put(w_out, w);
        if (copy_s) put(s_out, s);
        __syncthreads();
        for (uint32_t i = tid; i < (all & 0xffffu); i += kSelect) to[freed + i] = t * kTile + listed[i];
        for (uint32_t i = tid; i < all >> 16; i += kSelect) from[moved + i] = t * kTile + listed[kTile + i];
        freed += all & 0xffffu;
        moved += all >> 16;
    }
    if (tid == 0) {
        p.header[2 * head] = len;
        p.header[2 * head + 1] = (int32_t)moved;
    }
}

// Grid (p.move_rows moved rows, kv heads, batch).  A thread has two pieces of 16 bytes of K's rows and of V's, all four under way at once.
// 32 sequences of 300 .. 4096 rows to 1500, 8 heads of 128 in bf16: 26.6 us for 125 MB both ways (4.7 TB/s), a copy's rate.
constexpr int kMovePieces = 512;
__global__ __launch_bounds__(256) void cache_move_kernel(CacheEvictParams p) {
    const int tid = threadIdx.x, b = blockIdx.z, head = b * p.n_kv + (int)blockIdx.y;
    const int len = p.header[2 * head], moves = p.header[2 * head + 1];
    if (p.new_lens && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) p.new_lens[b] = min(len, p.budget);
    const int first = (int)blockIdx.x * p.move_rows, rows = min(p.move_rows, moves - first);
    if (rows <= 0) return;
    const int32_t* from = p.from + (size_t)head * p.most + first;
    const int32_t* to = p.to + (size_t)head * p.most + first;
    const size_t slab = (size_t)head * p.max_seq;
    const int shift = __builtin_ctz(p.row_bytes / 16);  // a row is a power of two of pieces
    u32x4_t* k = (u32x4_t*)(p.k + slab * p.row_bytes);
    u32x4_t* v = (u32x4_t*)(p.v + slab * p.row_bytes);
    u32x4_t a[2], c[2];
    size_t dst[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = min((tid + 256 * x) >> shift, rows - 1), u = (tid + 256 * x) & ((1 << shift) - 1);
        const size_t src = ((size_t)from[r] << shift) + u;
        dst[x] = ((size_t)to[r] << shift) + u;
        a[x] = k[src];
        c[x] = v[src];
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
        if ((tid + 256 * x) >> shift < rows) {
            k[dst[x]] = a[x];
            v[dst[x]] = c[x];
        }
    if (p.k_pairs) {
        for (int i = tid; i < rows * p.groups; i += 256) {
            const int g = i / rows, r = i - g * rows;
            const size_t plane = (slab * p.groups) + (size_t)g * p.max_seq;
            const uint32_t a = p.k_pairs[plane + from[r]], c = p.v_pairs[plane + from[r]];
            p.k_pairs[plane + to[r]] = a;
            p.v_pairs[plane + to[r]] = c;
        }
    }
    for (int i = tid; i < rows; i += 256) {
        const float w = p.weights_in[slab + from[i]];
        const int32_t s = p.slots_in[slab + from[i]];
        p.weights_out[slab + to[i]] = w;
        p.slots_out[slab + to[i]] = s;
    }
}

struct EvictPlan {
    int most;
    size_t header_bytes, list_bytes;
};
EvictPlan plan_evict(int32_t batch, int32_t n_kv, int32_t max_seq, int32_t budget) {
    EvictPlan a{};
    a.most = budget >= max_seq ? 0 : std::min(budget, max_seq - budget);
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    a.header_bytes = round((size_t)batch * n_kv * 8);
    a.list_bytes = round((size_t)batch * n_kv * a.most * 4);
    return a;
}

int evict_common(void* stream, CacheEvictParams& p, int head_dim, bool q4, void* workspace, size_t workspace_bytes, rt_err_detail* err) {
    clear_err(err);
    if (p.batch < 0 || p.n_kv < 0 || head_dim < 0 || p.max_seq < 0) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    if (head_dim == 0) return fail(err, RT_ERR_ZERO_DIM, -1, 0, 0, "head_dim must be > 0");
    if (!cache_q4_dim(head_dim)) return fail(err, RT_ERR_UNSUPPORTED, -1, 256, (uint64_t)head_dim, "these kernels cover head_dim 64, 128 and 256");
    if (p.batch > 65535 || p.n_kv > 65535 || (int64_t)p.batch * p.n_kv > 0x3fffffff || p.max_seq > (1 << 29)) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (p.budget < 0 || p.recent < 0 || p.recent > p.budget)
        return fail(err, RT_ERR_UNSUPPORTED, -1, (uint64_t)(int64_t)p.budget, (uint64_t)(int64_t)p.recent, "budget must be >= recent >= 0");
    if (p.batch == 0 || p.n_kv == 0) return RT_OK;
    if (!p.kv_lens || (p.max_seq > 0 && (!p.k || !p.v || (q4 && (!p.k_pairs || !p.v_pairs)) || !p.weights_in || !p.slots_in || !p.weights_out || !p.slots_out)))
        return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)p.k | (uintptr_t)p.v) & 15) return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "the caches must be 16-byte aligned");
    const size_t n = (size_t)p.batch * p.n_kv * p.max_seq * 4;
    auto apart = [](const void* a, const void* b, size_t bytes) { return a == b || !overlap(a, bytes, b, bytes); };
    if (!apart(p.weights_in, p.weights_out, n) || !apart(p.slots_in, p.slots_out, n) || overlap(p.weights_out, n, p.slots_out, n) ||
        overlap(p.weights_out, n, p.slots_in, n) || overlap(p.weights_in, n, p.slots_out, n) || (p.new_lens && !apart(p.kv_lens, p.new_lens, (size_t)p.batch * 4)))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "an output must be its input or share no memory with any");
    const EvictPlan a = plan_evict(p.batch, p.n_kv, p.max_seq, p.budget);
    const size_t need = a.header_bytes + 2 * a.list_bytes;
    if (!workspace || workspace_bytes < need) return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, need, workspace ? workspace_bytes : 0, "workspace too small");
    if ((uintptr_t)workspace & 15) return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, 16, (uint64_t)((uintptr_t)workspace & 15), "workspace must be 16-byte aligned");
    int rc = ensure_device(err);
    if (rc) return rc;
    p.header = (int32_t*)workspace;
    p.from = (int32_t*)((char*)workspace + a.header_bytes);
    p.to = (int32_t*)((char*)workspace + a.header_bytes + a.list_bytes);
    p.most = a.most;
    p.row_bytes = q4 ? head_dim / 2 : 2 * head_dim;
    p.groups = q4 ? head_dim / 64 : 0;
    p.move_rows = kMovePieces * 16 / p.row_bytes;
    const hipStream_t s = (hipStream_t)stream;
    if (p.max_seq <= kTile) hipLaunchKernelGGL(cache_select_kernel<true>, dim3(p.n_kv, p.batch), dim3(kSelect), 0, s, p);
    else hipLaunchKernelGGL(cache_select_kernel<false>, dim3(p.n_kv, p.batch), dim3(kSelect), 0, s, p);
    HIP_TRY(hipGetLastError(), "cache_select launch");
    hipLaunchKernelGGL(cache_move_kernel, dim3(std::max(1, (a.most + p.move_rows - 1) / p.move_rows), p.n_kv, p.batch), dim3(256), 0, s, p);
    HIP_TRY(hipGetLastError(), "cache_move launch");
    return RT_OK;
}

CacheEvictParams evict_params(void* k, uint32_t* k_pairs, void* v, uint32_t* v_pairs, const float* weights_in, const int32_t* slots_in,
                              float* weights_out, int32_t* slots_out, const int32_t* kv_lens, int32_t* new_lens, int32_t batch,
                              int32_t n_kv, int32_t max_seq, int32_t budget, int32_t recent) {
    CacheEvictParams p{};
    p.k = (uint8_t*)k;
    p.k_pairs = k_pairs;
    p.v = (uint8_t*)v;
    p.v_pairs = v_pairs;
    p.weights_in = weights_in;
    p.slots_in = slots_in;
    p.weights_out = weights_out;
    p.slots_out = slots_out;
    p.kv_lens = kv_lens;
    p.new_lens = new_lens;
    p.batch = batch;
    p.n_kv = n_kv;
    p.max_seq = max_seq;
    p.budget = budget;
    p.recent = recent;
    return p;
}

}  // namespace

}  // namespace rt

using namespace rt;

RT_API size_t rt_kv_evict_workspace_bytes(int32_t batch, int32_t n_kv, int32_t max_seq, int32_t budget) {
    if (batch <= 0 || n_kv <= 0 || max_seq < 0 || budget < 0) return 0;
    const EvictPlan a = plan_evict(batch, n_kv, max_seq, budget);
    return a.header_bytes + 2 * a.list_bytes;
}

RT_API int rt_kv_evict_bf16(void* stream, void* k_cache, void* v_cache, const float* weights_in, const int32_t* slots_in,
                            float* weights_out, int32_t* slots_out, const int32_t* kv_lens, int32_t* new_lens, int32_t batch,
                            int32_t n_kv, int32_t head_dim, int32_t max_seq, int32_t budget, int32_t recent, void* workspace,
                            size_t workspace_bytes, rt_err_detail* err) {
    CacheEvictParams p = evict_params(k_cache, nullptr, v_cache, nullptr, weights_in, slots_in, weights_out, slots_out, kv_lens, new_lens, batch, n_kv,
                                      max_seq, budget, recent);
    return evict_common(stream, p, head_dim, false, workspace, workspace_bytes, err);
}

RT_API int rt_kv_evict_q4(void* stream, void* k_codes, uint32_t* k_pairs, void* v_codes, uint32_t* v_pairs, const float* weights_in,
                          const int32_t* slots_in, float* weights_out, int32_t* slots_out, const int32_t* kv_lens,
                          int32_t* new_lens, int32_t batch, int32_t n_kv, int32_t head_dim, int32_t max_seq, int32_t budget,
                          int32_t recent, void* workspace, size_t workspace_bytes, rt_err_detail* err) {
    CacheEvictParams p = evict_params(k_codes, k_pairs, v_codes, v_pairs, weights_in, slots_in, weights_out, slots_out, kv_lens, new_lens, batch, n_kv,
                                      max_seq, budget, recent);
    return evict_common(stream, p, head_dim, true, workspace, workspace_bytes, err);
}
