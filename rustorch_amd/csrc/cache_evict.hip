// The rows of a cache that stay when it is cut to a budget, by the attention that their keys have drawn: of every (sequence, kv head)
// with more rows than `budget`, the `recent` newest tokens' and those with the largest sums of weights.
//
// A row's place in a cache says nothing to attention (its position went into the key with the rotation), so what stays need not keep its
// order: the kept rows behind the new length take, in order, the slots that are freed below it.  Only they are read and written --
// after a cut to a quarter three of four kept rows, in a loop that evicts one row a token a single one, where rows moved
// together in order would all have to move -- and no row that is read lies where one is written, so a copy needs no order either.
//
//   cache_select_kernel  one workgroup a (sequence, kv head): the budget-th largest sum by its bytes from the top (four counts of
//                        256), then one pass in slot order that numbers the freed slots and the rows that move
//   cache_move_kernel    copies them
#include <algorithm>

#include "cache_q4.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"

namespace rt {

namespace {

constexpr int kSelect = 1024, kSelectWaves = kSelect / 64;

// The order of the sums as that of whole numbers: NaN counts as -infinity, -0 as 0, the newest tokens' as +infinity.
__device__ __forceinline__ uint32_t key_of(float w, int pos, long long newest_out) {
    if ((long long)pos > newest_out) return 0xff800000u;
    if (w != w) return 0x007fffffu;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive sums over the workgroup's threads, in thread order, of a truth value; `all`: how many there are.  `room`: kSelectWaves ints.
__device__ __forceinline__ int count_before(bool x, int* room, int* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t mine = __ballot(x);
    __syncthreads();  // (the room may still be read)
    if (lane == 0) room[wave] = __popcll(mine);
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) {
        const int c = room[w];
        before += w < wave ? c : 0;
        sum += c;
    }
    *all = sum;
    return before + __popcll(mine & ((1ull << lane) - 1ull));
}

// Grid (kv heads, batch).
__global__ __launch_bounds__(kSelect) void cache_select_kernel(CacheEvictParams p) {
    __shared__ int bins[256], room[kSelectWaves], chosen[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.y, head = b * p.n_kv + (int)blockIdx.x;
    const int len = min(max(p.kv_lens[b], 0), p.max_seq);
    const float* w_in = p.weights_in + (size_t)head * p.max_seq;
    const int32_t* s_in = p.slots_in + (size_t)head * p.max_seq;
    float* w_out = p.weights_out + (size_t)head * p.max_seq;
    int32_t* s_out = p.slots_out + (size_t)head * p.max_seq;
    const bool copy_w = w_in != w_out, copy_s = s_in != s_out;
    if (len <= p.budget) {  // all of it stays
        for (int j = tid; j < len; j += kSelect) {
            if (copy_w) w_out[j] = w_in[j];
            if (copy_s) s_out[j] = s_in[j];
        }
        if (tid == 0) {
            p.header[2 * head] = len;
            p.header[2 * head + 1] = 0;
        }
        return;
    }
    // the newest token
    int newest = INT32_MIN;
    for (int j = tid; j < len; j += kSelect) newest = max(newest, s_in[j]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) newest = max(newest, __shfl_xor(newest, o, 64));
    if (lane == 0) room[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) newest = max(newest, room[w]);
    const long long out_from = (long long)newest - p.recent;

    // the budget-th largest key: its bytes from the top, each by a count of the keys that share those above it
    uint32_t prefix = 0;
    int left = p.budget;  // of the keys that share the prefix, the left-th largest is it
    for (int shift = 24; shift >= 0 && p.budget > 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelect) bins[i] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += kSelect) {
            const uint32_t k = key_of(w_in[j], s_in[j], out_from);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&bins[k >> shift & 255u], 1);
        }
        __syncthreads();
        if (wave == 0) {  // lane i has the bins 4 i .. 4 i + 3; those above count first
            const int c[4] = {bins[4 * lane], bins[4 * lane + 1], bins[4 * lane + 2], bins[4 * lane + 3]};
            int up = c[0] + c[1] + c[2] + c[3];
            const int own = up;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_down(up, o, 64);
                if (lane + o < 64) up += y;
            }
            int above = up - own;
#pragma unroll
            for (int e = 3; e >= 0; e--) {
                if (above < left && left <= above + c[e]) {
                    chosen[0] = 4 * lane + e;
                    chosen[1] = left - above;
                }
                above += c[e];
            }
        }
        __syncthreads();
        prefix |= (uint32_t)chosen[0] << shift;
        left = chosen[1];
    }
    // in slot order: keys above it stay, and the first `left` that equal it
    int equal = 0, freed = 0, moved = 0;
    int32_t* from = p.from + (size_t)head * p.most;
    int32_t* to = p.to + (size_t)head * p.most;
    for (int j0 = 0; j0 < len; j0 += kSelect) {
        const int j = j0 + tid;
        const bool in = j < len && p.budget > 0;
        const float w = in ? w_in[j] : 0.0f;
        const int s = in ? s_in[j] : 0;
        const uint32_t k = in ? key_of(w, s, out_from) : 0u;
        int all;
        const bool eq = in && k == prefix;
        const int rank = equal + count_before(eq, room, &all);
        equal += all;
        const bool keep = in && (k > prefix || (eq && rank < left));
        const bool hole = in && j < p.budget && !keep, mover = keep && j >= p.budget;
        const int at_hole = freed + count_before(hole, room, &all);
        freed += all;
        const int at_mover = moved + count_before(mover, room, &all);
        moved += all;
        if (hole) to[at_hole] = j;
        if (mover) from[at_mover] = j;
        if (keep && j < p.budget) {
            if (copy_w) w_out[j] = w;
            if (copy_s) s_out[j] = s;
        }
    }
    if (tid == 0) {
        p.header[2 * head] = len;
        p.header[2 * head + 1] = moved;
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
    hipLaunchKernelGGL(cache_select_kernel, dim3(p.n_kv, p.batch), dim3(kSelect), 0, s, p);
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
