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

// The order of the sums as that of whole numbers: NaN counts as -infinity, -0 as 0, the newest tokens' as +infinity.
constexpr uint32_t kNewest = 0xff800000u;
__device__ __forceinline__ uint32_t key_of(float w, int pos, long long newest_out) {
    if ((long long)pos > newest_out) return kNewest;
    if (w != w) return 0x007fffffu;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// A workgroup's reductions and sums: in a wave, then over the waves' results in `room` (kSelectWaves words), one barrier ahead of
// their writing and one behind it.
template <typename T, typename F>
__device__ __forceinline__ T all_of(T x, F f, T* room) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = f(x, __shfl_xor(x, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
    __syncthreads();
    T y = room[threadIdx.x & (kSelectWaves - 1)];
#pragma unroll
    for (int o = kSelectWaves / 2; o >= 1; o >>= 1) y = f(y, __shfl_xor(y, o, 64));
    return y;
}
// The sum over the threads before this one; `all`: over all.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* room, uint32_t* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t end = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(end, o, 64);
        if (lane >= o) end += y;
    }
    __syncthreads();
    if (lane == 63) room[wave] = end;
    __syncthreads();
    uint32_t y = room[lane & (kSelectWaves - 1)];
#pragma unroll
    for (int o = 1; o < kSelectWaves; o <<= 1) {
        const uint32_t z = __shfl_up(y, o, kSelectWaves);
        if ((lane & (kSelectWaves - 1)) >= o) y += z;
    }
    *all = __shfl(y, kSelectWaves - 1, 64);
    return end - x + (wave ? __shfl(y, wave - 1, 64) : 0u);
}

// One workgroup a (sequence, kv head), grid (kv heads, batch).  Thread t has the slots 8 t .. 8 t + 7 of a tile of 8192; up to there the keys are
// read once and stay in registers (kOne), longer heads are walked tile by tile again for every question.
// The budget-th largest key is found by counts: the range that the keys in question span is cut into 2048 bins, and the bin it falls in is
// the next range -- three times at most, since 2048^3 > 2^32, and twice as a rule, since bins that follow the keys' own range hold few of them.
// (By fixed bytes from the top most sums share a bin, and a wave's counts in one word wait for each other: 8192 keys 30 us.)
template <bool kOne>
__global__ __launch_bounds__(kSelect) void cache_select_kernel(CacheEvictParams p) {
    __shared__ uint32_t bins[kBins], room[kSelectWaves], chosen[2];
    const int tid = threadIdx.x, b = blockIdx.y, head = b * p.n_kv + (int)blockIdx.x;
    const int len = min(max(p.kv_lens[b], 0), p.max_seq);
    const float* w_in = p.weights_in + (size_t)head * p.max_seq;
    const int32_t* s_in = p.slots_in + (size_t)head * p.max_seq;
    float* w_out = p.weights_out + (size_t)head * p.max_seq;
    int32_t* s_out = p.slots_out + (size_t)head * p.max_seq;
    const bool copy_w = w_in != w_out, copy_s = s_in != s_out;
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
    float w[kPer];
    int32_t s[kPer];
    auto load = [&](int tile) __attribute__((always_inline)) {  // (slots behind the last: what its key is made of does not count)
        const int j0 = tile * kTile + tid * kPer;
        if (j0 + kPer <= len) {
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
            w[e] = j0 + e < len ? w_in[j0 + e] : 0.0f;
            s[e] = j0 + e < len ? s_in[j0 + e] : INT32_MIN;
        }
    };
    // the newest token
    int newest = INT32_MIN;
    for (int t = 0; t < tiles; t++) {
        load(t);
#pragma unroll
        for (int e = 0; e < kPer; e++) newest = max(newest, s[e]);
    }
    newest = all_of(newest, [](int x, int y) { return max(x, y); }, (int*)room);
    const long long out_from = (long long)newest - p.recent;
    uint32_t key[kPer];
    auto keys = [&](int tile) __attribute__((always_inline)) {
        if (!kOne) load(tile);
#pragma unroll
        for (int e = 0; e < kPer; e++) key[e] = key_of(w[e], s[e], out_from);
    };
    auto in = [&](int tile, int e) __attribute__((always_inline)) { return tile * kTile + tid * kPer + e < len; };
    // the newest tokens' keys, which are the largest, apart: they would stretch the range of the others
    uint32_t low = ~0u, high = 0, at_top = 0;
    for (int t = 0; t < tiles; t++) {
        keys(t);
#pragma unroll
        for (int e = 0; e < kPer; e++)
            if (in(t, e)) {
                at_top += key[e] == kNewest;
                if (key[e] != kNewest) {
                    low = min(low, key[e]);
                    high = max(high, key[e]);
                }
            }
    }
    low = all_of(low, [](uint32_t x, uint32_t y) { return min(x, y); }, room);
    high = all_of(high, [](uint32_t x, uint32_t y) { return max(x, y); }, room);
    at_top = all_of(at_top, [](uint32_t x, uint32_t y) { return x + y; }, room);
    uint32_t left = (uint32_t)p.budget;  // of the keys in [low, high], the left-th largest is the threshold
    if (left <= at_top) low = high = kNewest;
    else left -= at_top;
    while (low < high) {
        const int shift = max(0, 32 - __builtin_clz(high - low) - 11);  // (high - low) >> shift < 2048
        bins[tid] = bins[tid + kSelect] = 0;
        __syncthreads();
        for (int t = 0; t < tiles; t++) {
            if (!kOne) keys(t);
#pragma unroll
            for (int e = 0; e < kPer; e++)
                if (in(t, e) && key[e] >= low && key[e] <= high) atomicAdd(&bins[(key[e] - low) >> shift], 1u);
        }
        __syncthreads();
        // thread t has the bins 2047 - 2 t and 2046 - 2 t: those above it are those before it
        const uint32_t c0 = bins[kBins - 1 - 2 * tid], c1 = bins[kBins - 2 - 2 * tid];
        uint32_t all;
        const uint32_t above = sum_before(c0 + c1, room, &all);
        if (above < left && left <= above + c0 + c1) {
            const bool second = left > above + c0;
            chosen[0] = (uint32_t)(kBins - 1 - 2 * tid) - (second ? 1u : 0u);
            chosen[1] = left - above - (second ? c0 : 0u);
        }
        __syncthreads();
        const uint32_t bin = chosen[0];
        left = chosen[1];
        high = min(high, low + ((bin + 1) << shift) - 1);  // (no further than the range: low + 2^32 does not come up)
        low += bin << shift;
    }
    // in slot order: keys above it stay, and the first `left` that equal it
    uint32_t equal = 0, freed = 0, moved = 0;
    int32_t* from = p.from + (size_t)head * p.most;
    int32_t* to = p.to + (size_t)head * p.most;
    for (int t = 0; t < tiles; t++) {
        if (!kOne) keys(t);
        const int j0 = t * kTile + tid * kPer;
        uint32_t mine = 0, all;
#pragma unroll
        for (int e = 0; e < kPer; e++) mine += in(t, e) && key[e] == low;
        uint32_t rank = equal + sum_before(mine, room, &all);
        equal += all;
        uint32_t keep = 0, count = 0;  // count: freed slots in the low half, rows that move in the high one (8192 each at most)
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const bool eq = key[e] == low, stays = in(t, e) && (key[e] > low || (eq && rank < left));
            rank += in(t, e) && eq;
            keep |= (stays ? 1u : 0u) << e;
            count += in(t, e) && !stays && j0 + e < p.budget ? 1u : 0u;
            count += stays && j0 + e >= p.budget ? 1u << 16 : 0u;
        }
        const uint32_t before = sum_before(count, room, &all);
        uint32_t at_hole = freed + (before & 0xffffu), at_mover = moved + (before >> 16);
        freed += all & 0xffffu;
        moved += all >> 16;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const bool stays = keep >> e & 1u, below = j0 + e < p.budget;
            if (in(t, e) && !stays && below) to[at_hole++] = j0 + e;
            if (stays && !below) from[at_mover++] = j0 + e;
            if (stays && below) {
                if (copy_w) w_out[j0 + e] = w[e];
                if (copy_s) s_out[j0 + e] = s[e];
            }
        }
    }
    if (tid == 0) {
        p.header[2 * head] = len;
        p.header[2 * head + 1] = (int32_t)moved;
    }
}

constexpr int kMoveRows = 32;  // a workgroup

// Grid (kMoveRows moved rows, kv heads, batch).
__global__ __launch_bounds__(256) void cache_move_kernel(CacheEvictParams p) {
    const int tid = threadIdx.x, b = blockIdx.z, head = b * p.n_kv + (int)blockIdx.y;
    const int len = p.header[2 * head], moves = p.header[2 * head + 1];
    if (p.new_lens && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) p.new_lens[b] = min(len, p.budget);
    const int first = (int)blockIdx.x * kMoveRows, rows = min(kMoveRows, moves - first);
    if (rows <= 0) return;
    const int32_t* from = p.from + (size_t)head * p.most + first;
    const int32_t* to = p.to + (size_t)head * p.most + first;
    const size_t slab = (size_t)head * p.max_seq;
    const int units = p.row_bytes / 16;
    uint4* k = (uint4*)(p.k + slab * p.row_bytes);
    uint4* v = (uint4*)(p.v + slab * p.row_bytes);
    for (int i = tid; i < rows * units; i += 256) {
        const int r = i / units, u = i - r * units;
        const size_t src = (size_t)from[r] * units + u, dst = (size_t)to[r] * units + u;
        const uint4 a = k[src], c = v[src];
        k[dst] = a;
        v[dst] = c;
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
    if (tid < rows) {
        const float w = p.weights_in[slab + from[tid]];
        const int32_t s = p.slots_in[slab + from[tid]];
        p.weights_out[slab + to[tid]] = w;
        p.slots_out[slab + to[tid]] = s;
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
    if (p.batch > 65535 || p.n_kv > 65535 || (int64_t)p.batch * p.n_kv > 0x3fffffff) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
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
    const hipStream_t s = (hipStream_t)stream;
    if (p.max_seq <= kTile) hipLaunchKernelGGL(cache_select_kernel<true>, dim3(p.n_kv, p.batch), dim3(kSelect), 0, s, p);
    else hipLaunchKernelGGL(cache_select_kernel<false>, dim3(p.n_kv, p.batch), dim3(kSelect), 0, s, p);
    HIP_TRY(hipGetLastError(), "cache_select launch");
    hipLaunchKernelGGL(cache_move_kernel, dim3(std::max(1, (a.most + kMoveRows - 1) / kMoveRows), p.n_kv, p.batch), dim3(256), 0, s, p);
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
