// New rows of packed tokens into a cache in pages: per-head RMSNorm of q and k, half-split RoPE with one position a token or one on each
// of several axes, and the append, as in prepare.hip (steps 2a, 2b, 3 of LlamaModel::decode_step,
// crates/rustorch-llm/src/model.rs:575-636), where the tokens of all sequences follow one another ([tokens, heads, dim], what the
// projections leave) and a row's place is looked up in its sequence's page table.
//
//   x' = gamma x / sqrt(mean x^2 + eps)        pair i (dims i and i + D / 2) turned by the angle table[position on the pair's axis, i]
//
// The f32 arithmetic is the reference's, rounding for rounding (this file too is compiled without contraction): the sum of squares
// runs in index order, so that a row has the bits that prepare.hip gives it.
//
// D / 16 lanes a row (4, 8 or 16 of them set aside), so that a wave has 16, 8 or 4 of a token's rows: lane j has the dims 8 j .. 8 j + 7
// and their partners D / 2 on, 16 bytes a request.  The sum of squares goes from lane to lane within registers: at stage i lane i's value
// is that of dims 0 .. 8 i + 7, added one by one, and moves on; what the other lanes add meanwhile is thrown away.
//
// Bound: HBM where there are many tokens, a chain of reads (sequence, place, angles) where there are few.  A wave looks all that up for
// its few rows alone and is gone: us in a recorded loop, one pass a wave / all passes of a token by one wave, two at a time: 1 token
// of 32 + 8 heads of 128 3.5 / 9.4, 256 5.0 / 10.9, 1000 9.8 / 13.6, 4 prompts up to 4096 66.8 / 69.3 (301 MB: 4.5 TB/s), 6 up to 2000
// of 16 + 16 heads of 64 on three axes 27.9 / 27.1.  The angles of three axes 16 bytes a request where all sections are multiples of
// four, or word by word: 27.9, 31.1 on the last.  (As it is, a call among others: the four prompts 64.9 to 65.9 on 2 to 8 sets of tensors in turn,
// the six 25.2 to 26.1 on 4 or 8 and 20.4 to 21.6 on one or two, which the memory-side cache of 256 MB holds.)
//
// Rows go past the caches to the pages, which the attention of the same prompt does not read (call alone and with that attention behind
// it, us, plainly / past: 8 prompts up to 300 of 32 + 8 heads of 128 12.6, 25.0 / 11.8, 24.2; 6 up to 2000 of 16 + 16 of 64 27.3, 63.9 / 26.8, 63.9;
// 16 up to 2000 of 32 + 8 100, 318 / 100, 316), and stay in them where it does: with q_out and k_out past them too the call is 2 to 15 %
// shorter (23.5 for 26.8) and the two together as long or longer (64.4; 4 up to 4096 338 -> 345).
#include <algorithm>

#include "cache_paged.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"

#pragma clang fp contract(off)

namespace rt {

namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes from any word

__device__ __forceinline__ float from_lane_below(float x) {  // within a row of sixteen lanes
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x111, 0xf, 0xf, true));
}

// Grid (tokens, passes over a token's rows), a wave each.
// kAxes: 0: a position a token; else the pairs of a lane that lie side by side, kAxes of them, turn with one axis.
template <int kLanes, int kAxes>
__global__ __launch_bounds__(64) void paged_append_kernel(PagedAppendParams p) {
    constexpr int kRows = 64 / kLanes;  // a wave's
    const int lane = threadIdx.x, j = lane % kLanes, r = lane / kLanes, t = blockIdx.x, hh = (int)blockIdx.y * kRows + r;
    const int D = p.dim, half = D / 2, nl = D / 16;
    // the lane's row
    const bool on = hh < p.n_heads + 2 * p.n_kv, is_q = hh < p.n_heads, is_v = hh >= p.n_heads + p.n_kv;
    const int h = is_q ? hh : is_v ? hh - p.n_heads - p.n_kv : hh - p.n_heads;
    const bool in_row = j < nl;  // (a head dim of no power of two leaves lanes over)
    const int d0 = in_row ? 8 * j : 0;

    u32x4_t raw[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (on && in_row) {
        const uint16_t* src = (is_q ? p.q + ((size_t)t * p.n_heads + h) * D : (is_v ? p.v_in : p.k_in) + ((size_t)t * p.n_kv + h) * D) + d0;
        raw[0] = *(const u32x4_t*)src;
        raw[1] = *(const u32x4_t*)(src + half);
    }

    // the token's sequence, row and page
    int b, first;
    if (p.starts) {
        b = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 64) {  // sequences that end ahead of it
            const int n = __popcll(__ballot(b0 + lane < p.batch && p.starts[min(b0 + lane, p.batch - 1) + 1] <= t));
            b += n;
            if (n < 64) break;
        }
        b = __builtin_amdgcn_readfirstlane(b);
        if (b >= p.batch) return;  // behind the last sequence
        first = p.starts[b];
        if (first > t) return;  // ahead of the first
    } else {
        b = t / p.each;
        first = b * p.each;
    }
    const long long row = (long long)(p.positions ? p.positions[b] : p.pos) + ((long long)t - first);
    const bool in_table = row >= 0 && row >> p.page_shift < p.table_pages;
    const int page = in_table ? p.page_table[(size_t)b * p.table_pages + (size_t)(row >> p.page_shift)] : -1;
    const bool stored = page >= 0 && page < p.n_pages;
    // its angles; a token whose position the tables do not have is left as it is
    float cs[8], sn[8];
    if constexpr (kAxes > 0) {
        int at[kMaxAxes];
#pragma unroll
        for (int a = 0; a < kMaxAxes; a++) at[a] = a < p.n_axes ? p.axes[(size_t)a * p.tokens + t] : 0;
        bool ok = true;
#pragma unroll
        for (int a = 0; a < kMaxAxes; a++) ok = ok && at[a] >= 0 && at[a] < p.table_rows;
        if (!ok) return;
        typedef float piece_t __attribute__((ext_vector_type(kAxes), aligned(4)));
#pragma unroll
        for (int e = 0; e < 8; e += kAxes) {
            const int i = d0 + e;
            int pos = at[0];
#pragma unroll
            for (int a = 1; a < kMaxAxes; a++) pos = i >= p.ends[a - 1] ? at[a] : pos;
            const piece_t c = *(const piece_t*)(p.cos_table + (size_t)pos * half + i), s = *(const piece_t*)(p.sin_table + (size_t)pos * half + i);
#pragma unroll
            for (int k = 0; k < kAxes; k++) {
                cs[e + k] = c[k];
                sn[e + k] = s[k];
            }
        }
    } else {
        if (row < 0 || row >= p.table_rows) return;
        const size_t at = (size_t)row * half + d0;
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
    const size_t page_row = stored ? (size_t)page * p.n_kv << p.page_shift : 0;  // of head 0's first row
    const size_t in_page = (size_t)(row & ((1ll << p.page_shift) - 1));

    float x[2][8];
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[e][2 * i] = bf16_lo(raw[e][i]);
            x[e][2 * i + 1] = bf16_hi(raw[e][i]);
        }
    const float* const gamma = !on || is_v ? nullptr : is_q ? p.q_gamma : p.k_gamma;
    if (__any(gamma != nullptr)) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float sq[8], at = sum;
#pragma unroll
            for (int i = 0; i < 8; i++) sq[i] = x[e][i] * x[e][i];
            for (int stage = 0; stage < nl; stage++) {
                sum = at;
#pragma unroll
                for (int i = 0; i < 8; i++) sum = sum + sq[i];
                at = from_lane_below(sum);
            }
            sum = __shfl(sum, r * kLanes + nl - 1, 64);
        }
        if (gamma) {
            const float inv_d = 1.0f / (float)D;
            const float inv_rms = 1.0f / sqrtf(sum * inv_d + p.eps);
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const f32x4_t g = *(const f32x4_any*)(gamma + e * half + d0 + i);
#pragma unroll
                    for (int k = 0; k < 4; k++) x[e][i + k] = x[e][i + k] * inv_rms * g[k];
                }
        }
    }
    if (!on || !in_row) return;
    u32x4_t o[2] = {raw[0], raw[1]};
    if (!is_v) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float y0[2], y1[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int e = 2 * i + k;
                y0[k] = x[0][e] * cs[e] - x[1][e] * sn[e];
                y1[k] = x[1][e] * cs[e] + x[0][e] * sn[e];
            }
            o[0][i] = pack_bf16x2(y0[0], y0[1]);
            o[1][i] = pack_bf16x2(y1[0], y1[1]);
        }
    }
    if (is_q || (!is_v && p.k_out)) {
        uint16_t* dst = (is_q ? p.q_out + ((size_t)t * p.n_heads + h) * D : p.k_out + ((size_t)t * p.n_kv + h) * D) + d0;
        *(u32x4_t*)dst = o[0];
        *(u32x4_t*)(dst + half) = o[1];
    }
    if (!is_q && stored) {
        uint16_t* dst = (is_v ? p.v_pages : p.k_pages) + (page_row + ((size_t)h << p.page_shift) + in_page) * D + d0;
        __builtin_nontemporal_store(o[0], (u32x4_t*)dst);
        __builtin_nontemporal_store(o[1], (u32x4_t*)(dst + half));
    }
}

template <int kLanes>
hipError_t launch_lanes(hipStream_t stream, const PagedAppendParams& p) {
    const dim3 grid((unsigned)p.tokens, (unsigned)((p.n_heads + 2 * p.n_kv + 64 / kLanes - 1) / (64 / kLanes))), block(64);
    if (!p.axes) hipLaunchKernelGGL((paged_append_kernel<kLanes, 0>), grid, block, 0, stream, p);
    else if ((p.ends[0] | p.ends[1] | p.ends[2]) % 4 == 0) hipLaunchKernelGGL((paged_append_kernel<kLanes, 4>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_append_kernel<kLanes, 1>), grid, block, 0, stream, p);
    return hipGetLastError();
}
hipError_t launch_paged_append(hipStream_t stream, const PagedAppendParams& p) {
    return p.dim <= 64 ? launch_lanes<4>(stream, p) : p.dim <= 128 ? launch_lanes<8>(stream, p) : launch_lanes<16>(stream, p);
}

}  // namespace

}  // namespace rt

using namespace rt;

RT_API int rt_qk_norm_rope_kv_append_paged_bf16(void* stream, const void* q, void* q_out, const void* k_in, void* k_out, const void* v_in,
                                                void* k_pages, void* v_pages, const int32_t* page_table, const int32_t* starts,
                                                const int32_t* positions, int32_t pos, const int32_t* axis_positions,
                                                const int32_t* sections, int32_t n_axes, const float* q_gamma, const float* k_gamma,
                                                float eps, const float* cos_table, const float* sin_table, int32_t table_rows,
                                                int32_t tokens, int32_t batch, int32_t n_heads, int32_t n_kv, int32_t head_dim,
                                                int32_t n_pages, int32_t page_size, int32_t table_pages, rt_err_detail* err) {
    clear_err(err);
    if (tokens < 0 || batch < 0 || n_heads < 0 || n_kv < 0 || head_dim < 0 || n_pages < 0 || table_pages < 0 || table_rows < 0 || n_axes < 0)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    if (head_dim == 0) return fail(err, RT_ERR_ZERO_DIM, -1, 0, 0, "head_dim must be > 0");
    if (!cache_paged_dim(head_dim)) return fail(err, RT_ERR_UNSUPPORTED, -1, 256, (uint64_t)head_dim, "pages have head_dim up to 256, a multiple of 16");
    if (!cache_page_size(page_size)) return fail(err, RT_ERR_UNSUPPORTED, -1, kPageMax, (uint64_t)(int64_t)page_size, "page_size must be a power of two, 16 to 1024");
    if (tokens > (1 << 25) || n_heads > 65535 || n_kv > 65535 || (int64_t)table_pages * page_size > 0x7fffffffll) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    PagedAppendParams p{};
    if (n_axes > 0) {
        if (n_axes > kMaxAxes) return fail(err, RT_ERR_UNSUPPORTED, -1, kMaxAxes, (uint64_t)n_axes, "at most four axes");
        if (!sections) return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL sections");
        int64_t sum = 0;
        for (int a = 0; a < n_axes; a++) {
            if (sections[a] < 0) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
            sum += sections[a];
            p.ends[a] = (int)std::min<int64_t>(sum, head_dim);
        }
        if (sum != head_dim / 2) return fail(err, RT_ERR_ROPE_WRONG_INPUT_LEN, -1, (uint64_t)(head_dim / 2), (uint64_t)sum, "the sections' sum must be head_dim / 2");
        for (int a = n_axes; a < kMaxAxes; a++) p.ends[a] = head_dim;
    }
    if (!starts && batch > 0 && tokens % batch != 0)
        return fail(err, RT_ERR_WRONG_INPUT_LEN, RT_WHICH_Q, (uint64_t)batch, (uint64_t)tokens, "without starts every sequence has tokens / batch tokens");
    if (!positions) {  // rope.rs:179-184, then kv_cache.rs:84-89
        const int64_t last = (int64_t)pos + (batch == 0 || tokens == 0 ? 0 : starts ? 1 : tokens / batch);  // (of `starts` no more is known here)
        if (pos < 0 || (n_axes == 0 && last > table_rows))
            return fail(err, RT_ERR_ROPE_POSITION_OVERFLOW, -1, (uint64_t)table_rows, (uint64_t)last, "positions outside the RoPE tables");
        if (n_kv > 0 && last > (int64_t)table_pages * page_size)
            return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)((int64_t)table_pages * page_size), (uint64_t)last, "rows behind the page table");
    }
    if (batch == 0 || tokens == 0 || n_heads + n_kv == 0) return RT_OK;
    if ((n_heads > 0 && (!q || !q_out)) || (n_kv > 0 && (!k_in || !v_in || ((!k_pages || !v_pages) && n_pages > 0) || (!page_table && table_pages > 0))) || !cos_table || !sin_table ||
        (n_axes > 0 && !axis_positions))
        return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k_in | (uintptr_t)k_out | (uintptr_t)v_in | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15)
        return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "q, k, v and the pages must be 16-byte aligned");
    const size_t q_bytes = (size_t)tokens * n_heads * head_dim * 2, kv_bytes = (size_t)tokens * n_kv * head_dim * 2;
    const size_t page_bytes = (size_t)n_pages * n_kv * page_size * head_dim * 2;
    if ((q != q_out && overlap(q, q_bytes, q_out, q_bytes)) || (k_out && k_out != k_in && overlap(k_in, kv_bytes, k_out, kv_bytes)))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "q_out must be q, and k_out k_in, or share no memory with it");
    const struct {
        const void* at;
        size_t n;
    } written[4] = {{q_out, q_bytes}, {k_out, k_out ? kv_bytes : 0}, {k_pages, page_bytes}, {v_pages, page_bytes}}, read[3] = {{q, q_bytes}, {k_in, kv_bytes}, {v_in, kv_bytes}};
    for (int i = 0; i < 4; i++) {
        for (int k = i + 1; k < 4; k++)
            if (overlap(written[i].at, written[i].n, written[k].at, written[k].n)) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "outputs and pages must share no memory");
        for (int k = 0; k < 3; k++)
            if ((i >= 2 || k != i) && overlap(written[i].at, written[i].n, read[k].at, read[k].n)) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "outputs and pages must share no memory with the inputs");
    }
    int rc = ensure_device(err);
    if (rc) return rc;
    p.q = (const uint16_t*)q;
    p.q_out = (uint16_t*)q_out;
    p.k_in = (const uint16_t*)k_in;
    p.k_out = (uint16_t*)k_out;
    p.v_in = (const uint16_t*)v_in;
    p.k_pages = (uint16_t*)k_pages;
    p.v_pages = (uint16_t*)v_pages;
    p.page_table = page_table;
    p.starts = starts;
    p.positions = positions;
    p.pos = pos;
    p.axes = n_axes > 0 ? axis_positions : nullptr;
    p.n_axes = n_axes;
    p.q_gamma = q_gamma;
    p.k_gamma = k_gamma;
    p.eps = eps;
    p.cos_table = cos_table;
    p.sin_table = sin_table;
    p.table_rows = table_rows;
    p.tokens = tokens;
    p.batch = batch;
    p.each = tokens / batch;
    p.n_heads = n_heads;
    p.n_kv = n_kv;
    p.dim = head_dim;
    p.n_pages = n_pages;
    p.table_pages = n_kv > 0 ? table_pages : 0;  // (without kv heads nothing is stored, and the table may be missing)
    p.page_shift = __builtin_ctz((unsigned)page_size);
    HIP_TRY(launch_paged_append((hipStream_t)stream, p), "paged_append launch");
    return RT_OK;
}
