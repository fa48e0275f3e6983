// New rows into a cache, 4-bit or bf16, at rows of their own: per-head RMSNorm of q and k, half-split RoPE and the append, as in
// prepare.hip (steps 2a, 2b, 3 of LlamaModel::decode_step, crates/rustorch-llm/src/model.rs:575-636), where a token's cache row
// need not be its position (a cache that rows were taken out of) and q may go to a buffer of its own; and 4-bit rows read back.
//
// The f32 arithmetic is the reference's, rounding for rounding (this file too is compiled without contraction): the sum of
// squares runs in index order, so that a bf16 row has the bits that prepare.hip gives it.
#include <algorithm>

#include "cache_q4.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"

#pragma clang fp contract(off)

namespace rt {

namespace {

// z and s of a group from its extremes, the definition's f32 operations one by one; a group with a value that is not finite,
// or whose range f32 does not hold, has z = NaN and reads back as NaN throughout.
struct Pair {
    float s, z;
};
__device__ __forceinline__ Pair pair_of(float hi, float lo, bool bad) {
    const float z = bf16_bits_to_f32(f32_to_bf16_bits((hi + lo) * 0.5f + (hi - lo) * 0.03125f));
    const float up = fmaxf((hi - z) / 7.5f, (z - lo) / 8.5f);
    const float s = __uint_as_float((__float_as_uint(up) + 0xffffu) & 0xffff0000u);
    if (bad || !(fabsf(z) < __builtin_inff()) || !(up < 3.0e38f)) return Pair{0.0f, quiet_nan()};
    return Pair{s, z};
}
__device__ __forceinline__ uint32_t word_of(Pair p) { return (__float_as_uint(p.s) >> 16) | (__float_as_uint(p.z) & 0xffff0000u); }
__device__ __forceinline__ uint32_t code_of(float x, Pair p) {
    const float t = rintf((x - p.z) / p.s);
    return p.s > 0.0f ? (uint32_t)((int)fminf(fmaxf(t, -8.0f), 7.0f) + 8) : 8u;
}

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes from any word

// dim / 16 lanes a row; lane j has the dims 8 j .. 8 j + 7 and their partners dim / 2 on, which the rotation mixes: 16 bytes a request.
// Bound by the bytes: 2 x 4096 tokens, 32 + 2 x 8 heads of 128, into 4 bits 177 MB in 44 us (4.0 TB/s; 69 us with 4 bytes a request), the inputs past the
// caches (45).  With a norm every lane of a row walks all of the row's squares, in the order that the bits ask for: the same prompt 52 us, a token 4.0 for 3.3
// (dim 64 26 for 24, dim 256 115 for 85); into a bf16 cache in place 43 for 37, where prepare.hip, which has a thread take a row's sum, needs 39 for 38.
// Grid (rows of 256 / lanes, batch): the rows of a sequence are (head, token) pairs of q, then k, then v, tokens fastest.
template <int D, bool Q4>
__global__ __launch_bounds__(256) void cache_append_kernel(CacheAppendParams p) {
    constexpr int kLanes = D / 16, kRows = 256 / kLanes, kPitch = D + 4, kGroups = D / 64, kHalf = D / 2;
    extern __shared__ __attribute__((aligned(16))) float squares[];  // kRows * kPitch, where there is a norm
    const int tid = threadIdx.x, j = tid % kLanes, r = tid / kLanes, b = blockIdx.y, S = p.seq;
    const int all = (p.n_heads + 2 * p.n_kv) * S, idx = (int)blockIdx.x * kRows + r;
    const int pos0 = p.positions ? p.positions[b] : p.pos;
    const int row0 = p.rows ? p.rows[b] : p.cos_table ? pos0 : p.row;
    // a sequence whose rows would leave the tables or the cache is left as it is
    const bool fits = row0 >= 0 && row0 <= p.max_seq - S && (!p.cos_table || (pos0 >= 0 && pos0 <= p.table_rows - S));
    const bool on = idx < all && fits;
    const int hh = S == 1 ? min(idx, all - 1) : min(idx, all - 1) / S, tok = min(idx, all - 1) - hh * S;
    const bool is_q = hh < p.n_heads, is_v = hh >= p.n_heads + p.n_kv;
    const int h = is_q ? hh : is_v ? hh - p.n_heads - p.n_kv : hh - p.n_heads;
    const bool turn = !is_v && p.cos_table;
    const float* gamma = !turn ? nullptr : is_q ? p.q_gamma : p.k_gamma;

    float x[2][8];  // the lane's dims, and their partners
    u32x4_t raw[2];
    {
        const uint16_t* src = (is_q ? p.q : is_v ? p.v_in : p.k_in) + (((size_t)b * (is_q ? p.n_heads : p.n_kv) + h) * S + tok) * D + 8 * j;
#pragma unroll
        for (int e = 0; e < 2; e++) raw[e] = __builtin_nontemporal_load((const u32x4_t*)(src + e * kHalf));
    }
    float cs[8], sn[8];
    if (turn && on) {
        const size_t at = (size_t)(pos0 + tok) * kHalf + 8 * j;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4_t c = *(const f32x4_any*)(p.cos_table + at + e), s = *(const f32x4_any*)(p.sin_table + at + e);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                cs[e + i] = c[i];
                sn[e + i] = s[i];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[e][2 * i] = bf16_lo(raw[e][i]);
            x[e][2 * i + 1] = bf16_hi(raw[e][i]);
        }
    if (p.q_gamma || p.k_gamma) {  // (the same for every thread of the launch)
        float* mine = squares + r * kPitch;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *(f32x4_t*)(mine + e * kHalf + 8 * j + i) = f32x4_t{x[e][i] * x[e][i], x[e][i + 1] * x[e][i + 1], x[e][i + 2] * x[e][i + 2], x[e][i + 3] * x[e][i + 3]};
        __syncthreads();
        if (gamma) {
            float sum = 0.0f;
#pragma unroll 8
            for (int i = 0; i < D; i += 4) {
                const f32x4_t t = *(const f32x4_t*)(mine + i);
#pragma unroll
                for (int e = 0; e < 4; e++) sum = sum + t[e];
            }
            const float inv_d = 1.0f / (float)D;
            const float inv_rms = 1.0f / sqrtf(sum * inv_d + p.eps);
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const f32x4_t g = *(const f32x4_any*)(gamma + e * kHalf + 8 * j + i);
#pragma unroll
                    for (int k = 0; k < 4; k++) x[e][i + k] = x[e][i + k] * inv_rms * g[k];
                }
        }
    }
    if (!on) return;
    if (turn) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x0 = x[0][e], x1 = x[1][e];
            x[0][e] = x0 * cs[e] - x1 * sn[e];
            x[1][e] = x1 * cs[e] + x0 * sn[e];
        }
    }
    if (is_q || !Q4) {
        uint16_t* dst = is_q ? p.q_out + (((size_t)b * p.n_heads + h) * S + tok) * D
                             : (uint16_t*)(is_v ? p.v : p.k) + (((size_t)b * p.n_kv + h) * (size_t)p.max_seq + (size_t)(row0 + tok)) * D;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            u32x4_t o = raw[e];
            if (turn)
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = pack_bf16x2(x[e][2 * i], x[e][2 * i + 1]);
            *(u32x4_t*)(dst + e * kHalf + 8 * j) = o;
        }
        if (is_q) {
            return;
        }
    }
    const size_t head = (size_t)b * p.n_kv + h;
    if (!is_v && j == 0) {
        if (p.slots) p.slots[head * p.max_seq + (size_t)(row0 + tok)] = pos0 + tok;
        if (p.weights) p.weights[head * p.max_seq + (size_t)(row0 + tok)] = 0.0f;
    }
    if constexpr (Q4) {
        // extremes over the lanes of a group: 4 lanes with both halves at dim 64, 8 lanes a half above
        float hi[2], lo[2];
        int bad[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            hi[e] = lo[e] = x[e][0];
            bad[e] = !(fabsf(x[e][0]) < __builtin_inff());
#pragma unroll
            for (int i = 1; i < 8; i++) {
                hi[e] = fmaxf(hi[e], x[e][i]);
                lo[e] = fminf(lo[e], x[e][i]);
                bad[e] |= !(fabsf(x[e][i]) < __builtin_inff());
            }
        }
        if (D == 64) {
            hi[0] = fmaxf(hi[0], hi[1]);
            lo[0] = fminf(lo[0], lo[1]);
            bad[0] |= bad[1];
        }
        constexpr int kSpan = D == 64 ? 4 : 8;
        Pair pr[2];
#pragma unroll
        for (int e = 0; e < (D == 64 ? 1 : 2); e++) {
#pragma unroll
            for (int o = 1; o < kSpan; o *= 2) {
                hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], o, 64));
                lo[e] = fminf(lo[e], __shfl_xor(lo[e], o, 64));
                bad[e] |= __shfl_xor(bad[e], o, 64);
            }
            pr[e] = pair_of(hi[e], lo[e], bad[e] != 0);
        }
        if (D == 64) pr[1] = pr[0];
        const size_t row = (size_t)(row0 + tok);
        if (j % kSpan == 0) {
            uint32_t* pairs = (is_v ? p.v_pairs : p.k_pairs) + head * kGroups * p.max_seq + row;
            pairs[(size_t)(j / kSpan) * p.max_seq] = word_of(pr[0]);
            if (D > 64) pairs[(size_t)(kGroups / 2 + j / kSpan) * p.max_seq] = word_of(pr[1]);
        }
        uint32_t t[2];  // a byte a pair of dims: i = 4 (j % 4) .. + 3 of the lane's chunk, j / 4, and of its partner's
#pragma unroll
        for (int e = 0; e < 2; e++) {
            t[e] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) t[e] |= (code_of(x[e][2 * i], pr[e]) | code_of(x[e][2 * i + 1], pr[e]) << 4) << (8 * i);
        }
        // bytes (a.0, b.0, a.1, b.1) and (a.2, b.2, a.3, b.3)
        auto low = [](uint32_t a, uint32_t c) { return __builtin_amdgcn_perm(c, a, 0x05010400u); };
        auto high = [](uint32_t a, uint32_t c) { return __builtin_amdgcn_perm(c, a, 0x07030602u); };
        uint32_t* codes = (uint32_t*)(is_v ? p.v : p.k) + (head * (size_t)p.max_seq + row) * (D / 8);
        if constexpr (D == 64) {  // two bytes an i: chunks 0 and 1, the lane's two
            *(uint2*)(codes + 2 * j) = uint2{low(t[0], t[1]), high(t[0], t[1])};
        } else {
            // a word an i and 128 dims: chunks 0, 2, 1, 3.  At dim 128 lane j % 8 < 4 has 0 and 2, the one 4 on 1 and 3, and each keeps two of
            // the four i; at dim 256 lanes 0-3, 4-7, 8-11, 12-15 have chunks 0, 1, 2, 3 of one 128 dims (t[0]) and of the other (t[1]).
            if constexpr (D == 128) {
                const bool second = j & 4;
                const uint32_t give = second ? low(t[0], t[1]) : high(t[0], t[1]), keep = second ? high(t[0], t[1]) : low(t[0], t[1]);
                const uint32_t got = __shfl_xor(give, 4, 64);
                const uint32_t a = second ? got : keep, c = second ? keep : got;  // of chunks 0 and 2, of 1 and 3: two i's bytes each
                *(uint2*)(codes + 4 * (j & 3) + (second ? 2 : 0)) = uint2{(a & 0xffffu) | c << 16, a >> 16 | (c & 0xffff0000u)};
            } else {
                // lane k (of the four with one j % 4) takes the i-th word k of both: byte k of every lane's
                const int k = j >> 2;
                uint2 o = {0u, 0u};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int src = (int)(threadIdx.x & 48) + (j & 3) + 4 * c, to = 8 * ((c & 1) << 1 | c >> 1);
                    o.x |= (__shfl(t[0], src, 64) >> (8 * k) & 0xffu) << to;
                    o.y |= (__shfl(t[1], src, 64) >> (8 * k) & 0xffu) << to;
                }
                *(uint2*)(codes + 2 * (4 * (j & 3) + k)) = o;
            }
        }
    }
}

constexpr int kReadRows = 64;  // a workgroup

// Four lanes a row: lane j has the bytes of i = 4 j .. 4 j + 3, eight neighbouring dims of each chunk, so that it writes 16 bytes a request.
// (A word a request, sixteen lanes a row: 8192 rows of 8 heads 7.9 us.)
template <int D>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadParams p) {
    constexpr int kN = D / 32;
    const int j = threadIdx.x & 3, b = blockIdx.z, h = blockIdx.y, at = (int)blockIdx.x * kReadRows + (int)(threadIdx.x >> 2);
    const int row0 = p.rows ? p.rows[b] : p.row;
    if (at >= p.n_rows || row0 < 0 || row0 > p.max_seq - p.n_rows) return;
    const size_t head = (size_t)b * p.n_kv + h, row = (size_t)(row0 + at);
    const uint8_t* src = p.codes + (head * (size_t)p.max_seq + row) * (D / 2) + 4 * kN * j;
    const uint32_t* pairs = p.pairs + head * (D / 64) * (size_t)p.max_seq + row;
    uint16_t* dst = p.out + (head * (size_t)p.n_rows + (size_t)at) * D + 8 * j;
    uint32_t w[kN], pr[D / 64];
    if constexpr (kN == 2) *(u32x2_t*)w = *(const u32x2_t*)src;
    else
#pragma unroll
        for (int k = 0; k < kN; k += 4) *(u32x4_t*)(w + k) = *(const u32x4_t*)(src + 4 * k);
#pragma unroll
    for (int g = 0; g < D / 64; g++) pr[g] = pairs[(size_t)g * p.max_seq];
#pragma unroll
    for (int c = 0; c < kN; c++) {
        const int q = kN == 2 ? c : (c & ~3) | (c & 1) << 1 | (c >> 1 & 1);
        const float s = bf16_lo(pr[c / 2]), z = bf16_hi(pr[c / 2]);
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t byte = w[(i * kN + q) / 4] >> (8 * ((i * kN + q) % 4)) & 0xffu;
            o[i] = pack_bf16x2(z + s * (float)((int)(byte & 15) - 8), z + s * (float)((int)(byte >> 4) - 8));
        }
        *(u32x4_t*)(dst + 32 * c) = o;
    }
}

template <bool Q4>
hipError_t launch_append(hipStream_t stream, const CacheAppendParams& p, int dim) {
    const dim3 block(256);
    const long long all = ((long long)p.n_heads + 2ll * p.n_kv) * p.seq;
    auto grid = [&](int rows) { return dim3((unsigned)((all + rows - 1) / rows), (unsigned)p.batch); };
    const int rows = 4096 / dim;  // a workgroup
    const unsigned lds = p.q_gamma || p.k_gamma ? (unsigned)(rows * (dim + 4) * 4) : 0u;
    if (dim == 64) hipLaunchKernelGGL((cache_append_kernel<64, Q4>), grid(rows), block, lds, stream, p);
    else if (dim == 128) hipLaunchKernelGGL((cache_append_kernel<128, Q4>), grid(rows), block, lds, stream, p);
    else hipLaunchKernelGGL((cache_append_kernel<256, Q4>), grid(rows), block, lds, stream, p);
    return hipGetLastError();
}

int check_dim(int64_t dim, rt_err_detail* err) {
    if (dim == 0) return fail(err, RT_ERR_ZERO_DIM, -1, 0, 0, "head_dim must be > 0");
    if (dim != 64 && dim != 128 && dim != 256)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 256, (uint64_t)dim, "these kernels cover head_dim 64, 128 and 256");
    return RT_OK;
}

int append_common(void* stream, CacheAppendParams& p, int head_dim, bool q4, rt_err_detail* err) {
    clear_err(err);
    if (p.batch < 0 || p.seq < 0 || p.n_heads < 0 || p.n_kv < 0 || head_dim < 0 || p.max_seq < 0 || p.table_rows < 0)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    int rc = check_dim(head_dim, err);
    if (rc) return rc;
    if (p.batch > 65535 || ((int64_t)p.n_heads + 2ll * p.n_kv) * p.seq > 0x7fffffffll - 65536)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (!p.positions) {  // rope.rs:179-184, then kv_cache.rs:84-89, as for a cache whose rows are the positions
        if (p.pos < 0 || (int64_t)p.pos + p.seq > p.table_rows)
            return fail(err, RT_ERR_ROPE_POSITION_OVERFLOW, -1, (uint64_t)p.table_rows, (uint64_t)((int64_t)p.pos + p.seq), "positions outside the RoPE tables");
        if (!p.rows && (int64_t)p.pos + p.seq > p.max_seq)
            return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)p.max_seq, (uint64_t)((int64_t)p.pos + p.seq), "rows outside the cache");
    }
    if (p.batch == 0 || p.seq == 0 || p.n_heads + p.n_kv == 0) return RT_OK;
    if ((p.n_heads > 0 && (!p.q || !p.q_out)) || (p.n_kv > 0 && (!p.k_in || !p.v_in || !p.k || !p.v || (q4 && (!p.k_pairs || !p.v_pairs)))) ||
        !p.cos_table || !p.sin_table)
        return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)p.q | (uintptr_t)p.q_out | (uintptr_t)p.k_in | (uintptr_t)p.v_in | (uintptr_t)p.k | (uintptr_t)p.v) & 15)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "q, k, v and the caches must be 16-byte aligned");
    const size_t q_bytes = (size_t)p.batch * p.n_heads * p.seq * head_dim * 2;
    if (p.q != p.q_out && overlap(p.q, q_bytes, p.q_out, q_bytes))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "q_out must be q or share no memory with it");
    rc = ensure_device(err);
    if (rc) return rc;
    HIP_TRY(q4 ? launch_append<true>((hipStream_t)stream, p, head_dim) : launch_append<false>((hipStream_t)stream, p, head_dim), "cache_append launch");
    return RT_OK;
}

CacheAppendParams append_params(const void* q, void* q_out, const void* k_in, const void* v_in, void* k, uint32_t* k_pairs, void* v,
                                uint32_t* v_pairs, const int32_t* positions, int32_t pos, const int32_t* rows, int32_t* slots,
                                float* weights, const float* q_gamma, const float* k_gamma, float eps, const float* cos_table,
                                const float* sin_table, int32_t table_rows, int32_t batch, int32_t seq, int32_t n_heads,
                                int32_t n_kv, int32_t max_seq) {
    CacheAppendParams p{};
    p.q = (const uint16_t*)q;
    p.q_out = (uint16_t*)q_out;
    p.k_in = (const uint16_t*)k_in;
    p.v_in = (const uint16_t*)v_in;
    p.k = k;
    p.k_pairs = k_pairs;
    p.v = v;
    p.v_pairs = v_pairs;
    p.positions = positions;
    p.rows = rows;
    p.q_gamma = q_gamma;
    p.k_gamma = k_gamma;
    p.cos_table = cos_table;
    p.sin_table = sin_table;
    p.slots = slots;
    p.weights = weights;
    p.eps = eps;
    p.pos = pos;
    p.batch = batch;
    p.seq = seq;
    p.n_heads = n_heads;
    p.n_kv = n_kv;
    p.max_seq = max_seq;
    p.table_rows = table_rows;
    return p;
}

}  // namespace

}  // namespace rt

using namespace rt;

RT_API int rt_qk_norm_rope_kv_append_q4(void* stream, const void* q, void* q_out, const void* k_in, const void* v_in, void* k_codes,
                                        uint32_t* k_pairs, void* v_codes, uint32_t* v_pairs, const int32_t* positions, int32_t pos,
                                        const int32_t* rows, int32_t* slots, float* weights, const float* q_gamma,
                                        const float* k_gamma, float eps, const float* cos_table, const float* sin_table,
                                        int32_t table_rows, int32_t batch, int32_t seq, int32_t n_heads, int32_t n_kv,
                                        int32_t head_dim, int32_t max_seq, rt_err_detail* err) {
    CacheAppendParams p = append_params(q, q_out, k_in, v_in, k_codes, k_pairs, v_codes, v_pairs, positions, pos, rows, slots, weights,
                                        q_gamma, k_gamma, eps, cos_table, sin_table, table_rows, batch, seq, n_heads, n_kv, max_seq);
    return append_common(stream, p, head_dim, true, err);
}

RT_API int rt_qk_norm_rope_kv_append_rows_bf16(void* stream, const void* q, void* q_out, const void* k_in, const void* v_in,
                                               void* k_cache, void* v_cache, const int32_t* positions, int32_t pos,
                                               const int32_t* rows, int32_t* slots, float* weights, const float* q_gamma,
                                               const float* k_gamma, float eps, const float* cos_table, const float* sin_table,
                                               int32_t table_rows, int32_t batch, int32_t seq, int32_t n_heads, int32_t n_kv,
                                               int32_t head_dim, int32_t max_seq, rt_err_detail* err) {
    CacheAppendParams p = append_params(q, q_out, k_in, v_in, k_cache, nullptr, v_cache, nullptr, positions, pos, rows, slots, weights,
                                        q_gamma, k_gamma, eps, cos_table, sin_table, table_rows, batch, seq, n_heads, n_kv, max_seq);
    return append_common(stream, p, head_dim, false, err);
}

RT_API int rt_kv_cache_append_q4_dev(void* stream, void* k_codes, uint32_t* k_pairs, void* v_codes, uint32_t* v_pairs,
                                     const void* new_k, size_t new_k_len, const void* new_v, size_t new_v_len, size_t batch,
                                     size_t n_heads, size_t max_seq, size_t head_dim, size_t current_len, size_t seq_added,
                                     rt_err_detail* err) {
    clear_err(err);
    if (current_len + seq_added > max_seq || current_len + seq_added < current_len)  // kv_cache.rs:84-89
        return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)max_seq, (uint64_t)(current_len + seq_added), "append beyond max_seq");
    const size_t bhsd = batch * n_heads * seq_added * head_dim;
    if (new_k_len != bhsd || new_v_len != bhsd)  // kv_cache.rs:90-97
        return fail(err, RT_ERR_KV_WRONG_INPUT_LEN, -1, (uint64_t)bhsd, (uint64_t)new_k_len, "new_k / new_v length", (uint64_t)new_v_len);
    int rc = check_dim((int64_t)std::min<size_t>(head_dim, 0x7fffffffu), err);
    if (rc) return rc;
    if (batch > 65535 || n_heads > 65535 || max_seq > 0x7fffffffu || 2 * n_heads * seq_added > 0x7fffffffu - 65536)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (bhsd == 0) return RT_OK;
    if (!k_codes || !k_pairs || !v_codes || !v_pairs || !new_k || !new_v) return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)new_k | (uintptr_t)new_v) & 15)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "k, v and the caches must be 16-byte aligned");
    rc = ensure_device(err);
    if (rc) return rc;
    CacheAppendParams p{};
    p.k_in = (const uint16_t*)new_k;
    p.v_in = (const uint16_t*)new_v;
    p.k = k_codes;
    p.k_pairs = k_pairs;
    p.v = v_codes;
    p.v_pairs = v_pairs;
    p.row = (int)current_len;
    p.batch = (int)batch;
    p.seq = (int)seq_added;
    p.n_kv = (int)n_heads;
    p.max_seq = (int)max_seq;
    HIP_TRY(launch_append<true>((hipStream_t)stream, p, (int)head_dim), "cache_append launch");
    return RT_OK;
}

RT_API int rt_kv_cache_read_q4(void* stream, const void* codes, const uint32_t* pairs, void* out, const int32_t* rows, int32_t row,
                               int32_t n_rows, int32_t batch, int32_t n_kv, int32_t head_dim, int32_t max_seq, rt_err_detail* err) {
    clear_err(err);
    if (batch < 0 || n_rows < 0 || n_kv < 0 || head_dim < 0 || max_seq < 0) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    int rc = check_dim(head_dim, err);
    if (rc) return rc;
    if (batch > 65535 || n_kv > 65535) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (n_rows > max_seq || (!rows && (row < 0 || row > max_seq - n_rows)))
        return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)max_seq, (uint64_t)((int64_t)(rows ? 0 : row) + n_rows), "rows outside the cache");
    if (batch == 0 || n_kv == 0 || n_rows == 0) return RT_OK;
    if (!codes || !pairs || !out) return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)codes | (uintptr_t)out) & 15) return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "the cache and out must be 16-byte aligned");
    rc = ensure_device(err);
    if (rc) return rc;
    CacheReadParams p{};
    p.codes = (const uint8_t*)codes;
    p.pairs = pairs;
    p.out = (uint16_t*)out;
    p.rows = rows;
    p.row = row;
    p.n_rows = n_rows;
    p.n_kv = n_kv;
    p.max_seq = max_seq;
    const dim3 grid((unsigned)(((int64_t)n_rows + kReadRows - 1) / kReadRows), (unsigned)n_kv, (unsigned)batch), block(256);
    if (head_dim == 64) hipLaunchKernelGGL(cache_read_kernel<64>, grid, block, 0, (hipStream_t)stream, p);
    else if (head_dim == 128) hipLaunchKernelGGL(cache_read_kernel<128>, grid, block, 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(cache_read_kernel<256>, grid, block, 0, (hipStream_t)stream, p);
    HIP_TRY(hipGetLastError(), "cache_read launch");
    return RT_OK;
}
