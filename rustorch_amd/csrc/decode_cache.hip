// Attention of new positions over a cache held in 4 bits, and over a cache of either kind with the keys' weights summed:
//
//   out = softmax(q K^T / sqrt(dim)) V        weights_out[j] = weights_in[j] + sum over the heads of the group of their softmax weight of key j
//
// One wave walks steps of 32 keys of one kv head for up to 16 query rows (heads of the group x new positions) by the matrix cores,
// both products transposed: scores^T = K q^T leaves a lane with the scores of ONE query row for eight keys, which is the operand
// that out^T = V^T P^T takes, so that nothing of a step crosses lanes but the running maximum.
//
// 4-bit rows enter the products as codes: 16 + c is a bf16 whose mantissa the code's bits are (0x4180 | c << 3), and what follows
// from x = z + s (c - 8) is done on the sums, 64 dims at a time:
//   score = sum over groups of s (sum q (16 + c) - 24 sum q) + z sum q
//   out_d = sum over keys of (p s) (16 + c_d) - 24 sum over keys of (p s) + sum over keys of p z
// The weights p s are two bf16 terms (16 bits), as are those of a bf16 cache: with one the output's error is half as large again
// as its own rounding's.
//
// The keys of all (sequence, kv head, 16 query rows) segments form one list of steps that is cut into equal spans, one a wave; a wave that
// does not have a segment to itself leaves an unnormalised partial, which a second kernel folds.
#include <algorithm>

#include "cache_q4.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"
#include "rt_kernels.hpp"

namespace rt {

namespace {

constexpr int kStep = 32;       // keys a step
constexpr int kMaxWaves = 2048; // eight a CU
constexpr float kNoMax = -1.0e30f;

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ int len_of(const CacheAttendParams& p, int b) {
    return p.kv_lens ? min(max(p.kv_lens[b], 0), p.max_seq) : p.kv_len;
}
__device__ __forceinline__ int steps_of(int len) { return (len + kStep - 1) / kStep; }
__device__ __forceinline__ int wave_sum_int(int x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// Where a flat step lies: its sequence, and the first step of that sequence; `total`: steps of all.
struct Place {
    int total, b, first;
};
// Sum of the steps before sequence `upto` (all of them: batch).  Called by a whole wave.
__device__ __forceinline__ int steps_before(const CacheAttendParams& p, int upto, int lane) {
    int sum = 0;
    for (int b = lane; b < upto; b += 64) sum += steps_of(len_of(p, b));
    return wave_sum_int(sum) * (p.kv_heads * p.n_tiles);
}
// The sequence that holds flat step `at`, and its first step.
__device__ __forceinline__ void find_sequence(const CacheAttendParams& p, int at, int lane, int* seq, int* first) {
    const int per = p.kv_heads * p.n_tiles;
    int before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int mine = b0 + lane < p.batch ? steps_of(len_of(p, b0 + lane)) * per : 0;
        int end = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(end, o, 64);
            if (lane >= o) end += y;
        }
        const uint64_t past = __ballot(before + end > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            *seq = b0 + l;
            *first = before + __shfl(end - mine, l, 64);
            return;
        }
        before += __shfl(end, 63, 64);
    }
    *seq = p.batch;
    *first = before;
}
__device__ __forceinline__ int span_of(const CacheAttendParams& p, int total) { return max(p.span_min, (total + p.n_waves - 1) / p.n_waves); }

// ---- what a lane holds of 32 keys ----------------------------------------------------------------------------------
// As an operand of scores^T, keys are rows: lane (n, quad) has key n of either 16, and a quarter of each row.  As an operand of
// out^T, dims are rows and keys the products' inner index: lane (n, quad) has dims by n of the eight keys 4 quad + {0..3}, 16 + those, in the order
// in which scores^T leaves their weights.
template <int D, bool Q4>
struct Keys {
    static constexpr int kKw = Q4 ? D / 32 : D / 8, kVw = Q4 ? (D + 127) / 128 : D / 32, kG = Q4 ? D / 64 : 1;
    uint32_t k[2][kKw], v[8][kVw];
    uint32_t ks[2][kG][4], vs[2][kG][4];  // pairs of keys 4 quad + i of either 16
};

template <int D, bool Q4>
__device__ __forceinline__ void load_keys(Keys<D, Q4>& t, const uint8_t* k, const uint8_t* v, const uint32_t* kp, const uint32_t* vp, int max_seq, int key0, int len, int n, int quad) {
    using T = Keys<D, Q4>;
    constexpr int kRow = Q4 ? D / 2 : 2 * D;
    const int last = len - 1;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint8_t* row = k + (size_t)min(key0 + 16 * h + n, last) * kRow;
        if constexpr (Q4) {
#pragma unroll
            for (int i = 0; i < T::kKw; i++) t.k[h][i] = ((const uint32_t*)(row + quad * (D / 8)))[i];
        } else {
#pragma unroll
            for (int c = 0; c < D / 32; c++) *(u32x4_t*)(t.k[h] + 4 * c) = *(const u32x4_t*)(row + 64 * c + 16 * quad);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint8_t* row = v + (size_t)min(key0 + 16 * (e / 4) + 4 * quad + e % 4, last) * kRow;
        if constexpr (Q4 && D == 64) t.v[e][0] = *(const uint16_t*)(row + 2 * n);
        else
#pragma unroll
            for (int i = 0; i < T::kVw; i++) t.v[e][i] = ((const uint32_t*)(row + (kRow / 16) * n))[i];
    }
    if constexpr (Q4) {
#pragma unroll
        for (int g = 0; g < T::kG; g++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const size_t at = (size_t)g * max_seq + (size_t)min(key0 + 16 * h + 4 * quad + i, last);
                    t.ks[h][g][i] = kp[at];
                    t.vs[h][g][i] = vp[at];
                }
    }
}

constexpr uint32_t kCode = 0x00780078u, kSixteen = 0x41804180u;
// the codes at bits 4 nib of every second byte pair as two bf16 numbers 16 + c
template <int kNib>
__device__ __forceinline__ uint32_t codes_of(uint32_t w) {
    return ((kNib == 0 ? w << 3 : w >> (4 * kNib - 3)) & kCode) | kSixteen;
}

// The hi and lo terms of two weights: hi by truncation, what it leaves by truncation too (16 bits in all).
__device__ __forceinline__ void two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    hi = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    const float la = a - __uint_as_float(ua & 0xffff0000u), lb = b - __uint_as_float(ub & 0xffff0000u);
    lo = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302u);
}

template <int D, bool Q4, bool kWeigh>
__global__ __launch_bounds__(64) void cache_attend_kernel(CacheAttendParams p) {
    using T = Keys<D, Q4>;
    constexpr int kG = T::kG, kO = D / 16;
    const int lane = threadIdx.x, n = lane & 15, quad = lane >> 4;
    const int total = steps_before(p, p.batch, lane), span = span_of(p, total);
    const long long begin = (long long)blockIdx.x * span;
    if (begin >= total) return;
    int at = (int)begin;
    const int end = (int)min((long long)total, begin + span);
    int b, first;
    find_sequence(p, at, lane, &b, &first);

    while (at < end) {
        // the piece of a segment from here
        const int len = len_of(p, b), st = steps_of(len);
        if (st == 0 || at >= first + st * p.kv_heads * p.n_tiles) {  // the next sequence
            first += st * p.kv_heads * p.n_tiles;
            b++;
            continue;
        }
        const int seg = (at - first) / st, t0 = (at - first) - seg * st, t1 = min(st, t0 + (end - at));
        const int kvh = seg / p.n_tiles, tile = seg - kvh * p.n_tiles;
        at += t1 - t0;

        const int r = tile * 16 + n;  // the query row: position * group + head of the group
        const bool there = r < p.rows;
        const int s_new = there ? r / p.group : 0, head = kvh * p.group + (there ? r - s_new * p.group : 0);
        const int seen = len - p.seq_new + s_new + 1;  // keys that it sees
        const size_t q_at = (((size_t)b * p.seq_new + s_new) * p.heads + head) * D;

        // q as the operand that the keys' words pair with
        u32x4_t q[D / 32];
        float q_sum[kG];
        {
            u32x4_t nat[D / 32];
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                nat[c] = u32x4_t{0, 0, 0, 0};
                if (there) nat[c] = *(const u32x4_t*)(p.q + q_at + 32 * c + 8 * quad);
            }
            if constexpr (!Q4) {
#pragma unroll
                for (int c = 0; c < D / 32; c++) q[c] = nat[c];
            } else {
#pragma unroll
                for (int g = 0; g < kG; g++) {
                    float sum = 0.0f;
#pragma unroll
                    for (int c = 2 * g; c < 2 * g + 2; c++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sum += bf16_lo(nat[c][i]) + bf16_hi(nat[c][i]);
                    sum += __shfl_xor(sum, 16, 64);
                    sum += __shfl_xor(sum, 32, 64);
                    q_sum[g] = sum;
#pragma unroll
                    for (int par = 0; par < 2; par++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // dim 64: word (u, c) pairs i's of one chunk; above: chunks 2 g and 2 g + 1 at one i
                            const uint32_t a = D == 64 ? nat[i & 1][i & 2] : nat[2 * g][i], o = D == 64 ? nat[i & 1][(i & 2) + 1] : nat[2 * g + 1][i];
                            q[2 * g + par][i] = __builtin_amdgcn_perm(o, a, par ? 0x07060302u : 0x05040100u);
                        }
                }
            }
        }
        const size_t slab = ((size_t)b * p.kv_heads + kvh) * (size_t)p.max_seq;
        constexpr int kRow = Q4 ? D / 2 : 2 * D;
        const uint8_t* k = (const uint8_t*)p.k + slab * kRow;
        const uint8_t* v = (const uint8_t*)p.v + slab * kRow;
        const uint32_t* kp = Q4 ? p.k_pairs + slab * kG : nullptr;
        const uint32_t* vp = Q4 ? p.v_pairs + slab * kG : nullptr;
        const int all_see = len - p.seq_new + 1;  // keys that every row sees

        float m = kNoMax, l = 0.0f, pz[kG] = {};
        f32x4_t o[kO], ps[kG] = {};  // ps: the sums of the weights as they enter the products, by a row of ones
#pragma unroll
        for (int i = 0; i < kO; i++) o[i] = f32x4_t{0, 0, 0, 0};

        for (int t = t0; t < t1; t++) {
            const int key0 = t * kStep;
            T x;
            load_keys<D, Q4>(x, k, v, kp, vp, p.max_seq, key0, len, n, quad);
            // scores^T
            float y[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (Q4) {
#pragma unroll
                    for (int i = 0; i < 4; i++) y[4 * h + i] = 0.0f;
#pragma unroll
                    for (int g = 0; g < kG; g++) {
                        const float c0 = -24.0f * q_sum[g];
                        f32x4_t a = {c0, c0, c0, c0};
                        u32x4_t lo, hi;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // dim 64: word i / 2, chunk i % 2; above: word i of (dim 128 pairs) g / 2, its group g % 2
                            const uint32_t w = D == 64 ? x.k[h][i / 2] : x.k[h][i * (D / 128) + g / 2];
                            const bool upper = D == 64 ? i & 1 : g & 1;
                            lo[i] = upper ? codes_of<2>(w) : codes_of<0>(w);
                            hi[i] = upper ? codes_of<3>(w) : codes_of<1>(w);
                        }
                        a = mfma(lo, q[2 * g], a);
                        a = mfma(hi, q[2 * g + 1], a);
#pragma unroll
                        for (int i = 0; i < 4; i++) y[4 * h + i] += bf16_lo(x.ks[h][g][i]) * a[i] + bf16_hi(x.ks[h][g][i]) * q_sum[g];
                    }
                } else {
                    f32x4_t a = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < D / 32; c++) a = mfma(*(const u32x4_t*)(x.k[h] + 4 * c), q[c], a);
#pragma unroll
                    for (int i = 0; i < 4; i++) y[4 * h + i] = a[i];
                }
            }
            const bool cut = key0 + kStep > all_see;  // some row does not see all of them
            bool hid[8] = {};
            if (cut) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    hid[e] = key0 + 16 * (e / 4) + 4 * quad + e % 4 >= seen;
                    if (hid[e]) y[e] = neg_inf();
                }
            }
            if constexpr (kWeigh) {
                if (there) {
                    float* dst = p.scores + ((size_t)b * p.heads + head) * (size_t)p.max_seq + key0 + 4 * quad;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (!hid[e]) dst[16 * (e / 4) + e % 4] = y[e];
                }
            }
            // the running maximum, common to the four lanes of a query row
            float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m)) {
                const float m_new = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f((m - m_new) * p.scale_log2e);
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int g = 0; g < kG; g++) {
                    ps[g] *= alpha;  // (rows alike: one would do)
                    pz[g] *= alpha;
                }
#pragma unroll
                for (int i = 0; i < kO; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][e] *= alpha;
            }
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = __builtin_amdgcn_exp2f((y[e] - m) * p.scale_log2e);
                l += w[e];
            }
            // out^T
#pragma unroll
            for (int g = 0; g < kG; g++) {
                u32x4_t p_hi, p_lo;
                if constexpr (Q4) {
                    float s[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint32_t pr = x.vs[e / 4][g][e % 4];
                        s[e] = hid[e] ? 0.0f : w[e] * bf16_lo(pr);  // (what a hidden row holds stays out, were it NaN)
                        pz[g] += hid[e] ? 0.0f : w[e] * bf16_hi(pr);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t a, c;
                        two_terms(s[2 * i], s[2 * i + 1], a, c);
                        p_hi[i] = a;
                        p_lo[i] = c;
                    }
                    constexpr u32x4_t kOnes = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
                    ps[g] = mfma(kOnes, p_lo, mfma(kOnes, p_hi, ps[g]));
                    // the bytes whose chunks are of this group
#pragma unroll
                    for (int f = 0; f < 2; f++) {
                        const int byte = D == 64 ? f : (g & 1) + 2 * f, word = D == 64 ? 0 : g / 2;
                        u32x4_t lo, hi;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t z = __builtin_amdgcn_perm(x.v[2 * i + 1][word], x.v[2 * i][word], 0x0c000c00u | (uint32_t)(4 + byte) << 16 | (uint32_t)byte);
                            lo[i] = codes_of<0>(z);
                            hi[i] = codes_of<1>(z);
                        }
                        const int at_o = 8 * word + 2 * byte;
                        o[at_o] = mfma(lo, p_lo, mfma(lo, p_hi, o[at_o]));
                        o[at_o + 1] = mfma(hi, p_lo, mfma(hi, p_hi, o[at_o + 1]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t a, c;
                        two_terms(w[2 * i], w[2 * i + 1], a, c);
                        p_hi[i] = a;
                        p_lo[i] = c;
                    }
#pragma unroll
                    for (int d = 0; d < kO; d++) {  // dim n * (D / 16) + d
                        u32x4_t a;
#pragma unroll
                        for (int i = 0; i < 4; i++) a[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][d / 2], x.v[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
                        o[d] = mfma(a, p_lo, mfma(a, p_hi, o[d]));
                    }
                }
            }
        }

        // sums over the four lanes of a query row
        auto row_sum = [](float f) {
            f += __shfl_xor(f, 16, 64);
            return f + __shfl_xor(f, 32, 64);
        };
        l = row_sum(l);
        if constexpr (Q4) {
#pragma unroll
            for (int g = 0; g < kG; g++) {
                const float off = row_sum(pz[g]) - 24.0f * ps[g][0];
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    const int byte = D == 64 ? f / 2 : (g & 1) + 2 * (f / 2), i = 8 * (D == 64 ? 0 : g / 2) + 2 * byte + f % 2;
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][e] += off;
                }
            }
        }
        // a lane's eight dims in a row: of chunk c (dims 32 c + 8 quad on), or of lane row 4 quad + i
        const bool alone = t0 == 0 && t1 == st;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (there) {
            auto dims = [&](int c, float (&f)[8]) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if constexpr (Q4) {
                        const int byte = D == 64 ? c : (c & ~3) | (c & 1) << 1 | (c >> 1 & 1);
                        f[e] = o[2 * byte + e % 2][e / 2];
                    } else {  // dims (4 quad + i) * (D / 16) + d: 8 c on of the lane's D / 4
                        f[e] = o[(8 * c + e) % (D / 16)][(8 * c + e) / (D / 16)];
                    }
                }
            };
            auto dim_of = [&](int c) { return Q4 ? 32 * c + 8 * quad : quad * (D / 4) + 8 * c; };
            if (alone) {
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    float f[8];
                    dims(c, f);
                    *(u32x4_t*)(p.out + q_at + dim_of(c)) = u32x4_t{pack_bf16x2(f[0] * inv, f[1] * inv), pack_bf16x2(f[2] * inv, f[3] * inv), pack_bf16x2(f[4] * inv, f[5] * inv),
                                                                  pack_bf16x2(f[6] * inv, f[7] * inv)};
                }
                if (kWeigh && quad == 0) {
                    float* st_at = p.stats + ((size_t)b * p.heads + head) * 2;
                    st_at[0] = m;
                    st_at[1] = inv;
                }
            } else {
                const size_t segment = ((size_t)b * p.kv_heads + kvh) * p.n_tiles + tile;
                float* slot = p.part + ((size_t)blockIdx.x + segment) * p.part_rows * (D + 2);
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    float f[8];
                    dims(c, f);
                    float* dst = slot + n * D + dim_of(c);
                    *(f32x4_t*)dst = f32x4_t{f[0], f[1], f[2], f[3]};
                    *(f32x4_t*)(dst + 4) = f32x4_t{f[4], f[5], f[6], f[7]};
                }
                if (quad == 0) {
                    slot[p.part_rows * D + n] = m;
                    slot[p.part_rows * (D + 1) + n] = l;
                }
            }
        }
    }
}

// Folds the partials of a segment that more than one wave walked; rows without keys are zeros.  Grid (rows of a kv head, kv heads,
// batch), a thread a dim.
template <int D, bool kWeigh>
__global__ __launch_bounds__(D) void cache_merge_kernel(CacheAttendParams p) {
    const int d = threadIdx.x, lane = d & 63, r = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int total = steps_before(p, p.batch, lane), first = steps_before(p, b, lane), span = span_of(p, total);
    const int st = steps_of(len_of(p, b)), tile = r / 16, n = r % 16;
    const int s_new = r / p.group, head = kvh * p.group + r - s_new * p.group;
    const int seg = kvh * p.n_tiles + tile, at = first + seg * st;
    const size_t out_at = (((size_t)b * p.seq_new + s_new) * p.heads + head) * D + d;
    float* stats = kWeigh ? p.stats + ((size_t)b * p.heads + head) * 2 : nullptr;
    if (st == 0) {
        p.out[out_at] = 0;
        return;
    }
    const int w0 = at / span, w1 = (at + st - 1) / span;
    if (w0 == w1) return;  // the one wave has written it
    const size_t segment = (size_t)b * p.kv_heads * p.n_tiles + seg, slot_size = (size_t)p.part_rows * (D + 2);
    const float* slot = p.part + (w0 + segment) * slot_size;
    float m = kNoMax;
    for (int w = 0; w <= w1 - w0; w++) m = fmaxf(m, slot[w * slot_size + p.part_rows * D + n]);
    float o = 0.0f, l = 0.0f;
    for (int w = 0; w <= w1 - w0; w++) {
        const float* s = slot + w * slot_size;
        const float f = __builtin_amdgcn_exp2f((s[p.part_rows * D + n] - m) * p.scale_log2e);
        o += s[n * D + d] * f;
        l += s[p.part_rows * (D + 1) + n] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    p.out[out_at] = f32_to_bf16_bits(o * inv);
    if (kWeigh && d == 0) {
        stats[0] = m;
        stats[1] = inv;
    }
}

// The keys' weights from the scores and the rows' statistics.  Grid (1024 keys, kv heads, batch).
__global__ __launch_bounds__(256) void cache_weigh_kernel(CacheAttendParams p) {
    const int kvh = blockIdx.y, b = blockIdx.z, len = len_of(p, b);
    const size_t sums = ((size_t)b * p.kv_heads + kvh) * (size_t)p.max_seq;
    for (int j = (int)blockIdx.x * 1024 + (int)threadIdx.x, e = 0; e < 4 && j < len; e++, j += 256) {
        float w = p.weights_in ? p.weights_in[sums + j] : 0.0f, sum = 0.0f;
        for (int h = 0; h < p.group; h++) {
            const size_t row = (size_t)b * p.heads + kvh * p.group + h;
            sum += __builtin_amdgcn_exp2f((p.scores[row * p.max_seq + j] - p.stats[2 * row]) * p.scale_log2e) * p.stats[2 * row + 1];
        }
        p.weights_out[sums + j] = w + sum;
    }
}

template <int D, bool Q4, bool kWeigh>
hipError_t launch_attend_as(hipStream_t stream, const CacheAttendParams& p) {
    hipLaunchKernelGGL((cache_attend_kernel<D, Q4, kWeigh>), dim3(p.n_waves), dim3(64), 0, stream, p);
    hipLaunchKernelGGL((cache_merge_kernel<D, kWeigh>), dim3(p.rows, p.kv_heads, p.batch), dim3(D), 0, stream, p);
    if (kWeigh && p.max_seq > 0)
        hipLaunchKernelGGL(cache_weigh_kernel, dim3((p.max_seq + 1023) / 1024, p.kv_heads, p.batch), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <bool Q4, bool kWeigh>
hipError_t launch_attend(hipStream_t stream, const CacheAttendParams& p, int dim) {
    return dim == 64 ? launch_attend_as<64, Q4, kWeigh>(stream, p) : dim == 128 ? launch_attend_as<128, Q4, kWeigh>(stream, p) : launch_attend_as<256, Q4, kWeigh>(stream, p);
}

// Segments, steps and waves of a call at its longest.
struct AttendPlan {
    int64_t rows, n_tiles, segments, steps;
    int waves, part_rows;
    size_t part_bytes, score_bytes, stat_bytes;
};
AttendPlan plan_attend(int64_t batch, int64_t seq_new, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_seq, bool weigh) {
    AttendPlan a{};
    a.rows = seq_new * (heads / kv_heads);
    a.n_tiles = (a.rows + 15) / 16;
    a.segments = batch * kv_heads * a.n_tiles;
    a.steps = a.segments * ((max_seq + kStep - 1) / kStep);
    a.waves = (int)std::min<int64_t>(kMaxWaves, std::max<int64_t>(a.steps, 1));
    a.part_rows = (int)std::min<int64_t>(16, a.rows);
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    a.part_bytes = round(((size_t)a.waves + (size_t)a.segments) * (size_t)a.part_rows * (size_t)(dim + 2) * 4);
    if (weigh) {
        a.score_bytes = round((size_t)batch * (size_t)heads * (size_t)max_seq * 4);
        a.stat_bytes = round((size_t)batch * (size_t)heads * 8);
    }
    return a;
}

int attend_common(void* stream, CacheAttendParams& p, int head_dim, bool q4, bool weigh, void* workspace, size_t workspace_bytes, rt_err_detail* err) {
    clear_err(err);
    if (p.batch < 0 || p.heads < 0 || p.kv_heads < 0 || p.seq_new < 0 || head_dim < 0 || p.max_seq < 0) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    if (p.kv_heads == 0 || p.heads % p.kv_heads != 0)
        return fail(err, RT_ERR_HEAD_COUNT_MISMATCH, -1, (uint64_t)p.heads, (uint64_t)p.kv_heads, "n_heads not divisible by n_kv");
    if (head_dim == 0) return fail(err, RT_ERR_ZERO_DIM, -1, 0, 0, "head_dim must be > 0");
    if (!cache_q4_dim(head_dim)) return fail(err, RT_ERR_UNSUPPORTED, -1, 256, (uint64_t)head_dim, "these kernels cover head_dim 64, 128 and 256");
    if (p.batch > 65535 || p.heads > 65535 || p.seq_new > 65535) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (!p.kv_lens && (p.kv_len < p.seq_new || p.kv_len > p.max_seq))
        return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)p.max_seq, (uint64_t)(int64_t)p.kv_len, "kv_len must cover the new positions and fit the cache");
    if (p.batch == 0 || p.heads == 0 || p.seq_new == 0) return RT_OK;
    const AttendPlan a = plan_attend(p.batch, p.seq_new, p.heads, p.kv_heads, head_dim, p.max_seq, weigh);
    if (a.steps + a.segments > 0x7fffffffll - kMaxWaves || a.rows > 0x7fffffffll) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (!p.q || !p.out || (weigh && (!p.weights_out || !p.kv_lens)) || (p.max_seq > 0 && (!p.k || !p.v || (q4 && (!p.k_pairs || !p.v_pairs)))))
        return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.out) & 15) return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "q, out and the caches must be 16-byte aligned");
    const size_t sum_bytes = (size_t)p.batch * p.kv_heads * p.max_seq * 4;
    if (weigh && p.weights_in != p.weights_out && overlap(p.weights_in, p.weights_in ? sum_bytes : 0, p.weights_out, sum_bytes))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "weights_out must be weights_in or share no memory with it");
    const size_t need = a.part_bytes + a.score_bytes + a.stat_bytes;
    if (!workspace || workspace_bytes < need)
        return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, need, workspace ? workspace_bytes : 0, "workspace too small");
    if ((uintptr_t)workspace & 15) return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, 16, (uint64_t)((uintptr_t)workspace & 15), "workspace must be 16-byte aligned");
    int rc = ensure_device(err);
    if (rc) return rc;
    p.group = p.heads / p.kv_heads;
    p.rows = (int)a.rows;
    p.n_tiles = (int)a.n_tiles;
    p.n_waves = a.waves;
    p.span_min = 4;
    p.scale_log2e = (1.0f / sqrtf((float)head_dim)) * kLog2eHost;
    p.part = (float*)workspace;
    p.part_rows = a.part_rows;
    p.scores = (float*)((char*)workspace + a.part_bytes);
    p.stats = (float*)((char*)workspace + a.part_bytes + a.score_bytes);
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = !q4 ? launch_attend<false, true>(s, p, head_dim) : weigh ? launch_attend<true, true>(s, p, head_dim) : launch_attend<true, false>(s, p, head_dim);
    HIP_TRY(e, "cache_attend launch");
    return RT_OK;
}

size_t attend_bytes(int32_t batch, int32_t seq_new, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq, bool weigh) {
    if (batch <= 0 || seq_new <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || !cache_q4_dim(head_dim) || max_seq < 0) return 0;
    const AttendPlan a = plan_attend(batch, seq_new, n_heads, n_kv, head_dim, max_seq, weigh);
    return a.part_bytes + a.score_bytes + a.stat_bytes;
}

}  // namespace

}  // namespace rt

using namespace rt;

RT_API size_t rt_gqa_decode_q4_workspace_bytes(int32_t batch, int32_t seq_new, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq) {
    return attend_bytes(batch, seq_new, n_heads, n_kv, head_dim, max_seq, false);
}

RT_API int rt_gqa_decode_q4(void* stream, const void* q, const void* k_codes, const uint32_t* k_pairs, const void* v_codes,
                            const uint32_t* v_pairs, void* out, const int32_t* kv_lens, int32_t kv_len, int32_t batch,
                            int32_t seq_new, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq, void* workspace,
                            size_t workspace_bytes, rt_err_detail* err) {
    CacheAttendParams p{};
    p.q = (const uint16_t*)q;
    p.k = k_codes;
    p.k_pairs = k_pairs;
    p.v = v_codes;
    p.v_pairs = v_pairs;
    p.out = (uint16_t*)out;
    p.kv_lens = kv_lens;
    p.kv_len = kv_len;
    p.batch = batch;
    p.heads = n_heads;
    p.kv_heads = n_kv;
    p.seq_new = seq_new;
    p.max_seq = max_seq;
    return attend_common(stream, p, head_dim, true, false, workspace, workspace_bytes, err);
}

RT_API size_t rt_gqa_decode_weights_workspace_bytes(int32_t batch, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq) {
    return attend_bytes(batch, 1, n_heads, n_kv, head_dim, max_seq, true);
}

static int decode_weights(void* stream, const void* q, const void* k, const uint32_t* k_pairs, const void* v, const uint32_t* v_pairs,
                          void* out, const float* weights_in, float* weights_out, const int32_t* kv_lens, int32_t batch,
                          int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq, bool q4, void* workspace,
                          size_t workspace_bytes, rt_err_detail* err) {
    CacheAttendParams p{};
    p.q = (const uint16_t*)q;
    p.k = k;
    p.k_pairs = k_pairs;
    p.v = v;
    p.v_pairs = v_pairs;
    p.out = (uint16_t*)out;
    p.kv_lens = kv_lens;
    p.kv_len = 1;
    p.batch = batch;
    p.heads = n_heads;
    p.kv_heads = n_kv;
    p.seq_new = 1;
    p.max_seq = max_seq;
    p.weights_in = weights_in;
    p.weights_out = weights_out;
    return attend_common(stream, p, head_dim, q4, true, workspace, workspace_bytes, err);
}

RT_API int rt_gqa_decode_weights_q4(void* stream, const void* q, const void* k_codes, const uint32_t* k_pairs, const void* v_codes,
                                    const uint32_t* v_pairs, void* out, const float* weights_in, float* weights_out,
                                    const int32_t* kv_lens, int32_t batch, int32_t n_heads, int32_t n_kv, int32_t head_dim,
                                    int32_t max_seq, void* workspace, size_t workspace_bytes, rt_err_detail* err) {
    return decode_weights(stream, q, k_codes, k_pairs, v_codes, v_pairs, out, weights_in, weights_out, kv_lens, batch, n_heads, n_kv, head_dim,
                          max_seq, true, workspace, workspace_bytes, err);
}

RT_API int rt_gqa_decode_weights_bf16(void* stream, const void* q, const void* k_cache, const void* v_cache, void* out,
                                      const float* weights_in, float* weights_out, const int32_t* kv_lens, int32_t batch,
                                      int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq, void* workspace,
                                      size_t workspace_bytes, rt_err_detail* err) {
    return decode_weights(stream, q, k_cache, nullptr, v_cache, nullptr, out, weights_in, weights_out, kv_lens, batch, n_heads, n_kv, head_dim,
                          max_seq, false, workspace, workspace_bytes, err);
}
