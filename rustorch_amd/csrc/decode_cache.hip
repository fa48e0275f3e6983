// Attention of new positions over a cache held in 4 bits, and over a cache of either kind with the keys' weights summed:
//
//   out = softmax(q K^T / sqrt(dim)) V        weights_out[j] = weights_in[j] + sum over the heads of the group of their softmax weight of key j
//
// A wave walks steps of 32 keys of one kv head for up to 16 query rows (heads of the group x new positions) by the matrix cores,
// both products transposed: scores^T = K q^T leaves a lane with the scores of ONE query row for eight keys, which is the operand
// that out^T = V^T P^T takes, so that nothing of a step crosses lanes but the running maximum.
//
// 4-bit rows enter the products as the codes themselves: a byte below a byte of zeros is a bf16 of that many times 2^-133, subnormal or of
// the first binade (the matrix cores take both as they are, products and sums exact as ever), so that a mask, and for every second
// byte a shift, is all that a pair of codes costs; the high half of a byte stays where it is and counts 16-fold.  The other operand
// makes up for it: q scaled by the power of two that brings its row's largest value to 2^120 (and by 2^-4 where codes count
// 16-fold), the weights that meet V's codes by 2^60.  What follows from x = z + s (c - 8) is done on the sums, 64 dims at a time:
//   score = sum over groups of s (sum q c - 8 sum q) + z sum q
//   out_d = sum over keys of (p s) c_d - 8 sum over keys of (p s) + sum over keys of p z
// (With codes as the mantissa of 16 + c a pair of codes took a shift and an and-or, 144 of a step's 255 vector instructions at dim 128
// for 88 of 180 now.)  So V's scales have a range: below
// 2^-50 the products lose bits, and the sum of p s 2^60 has to stay below 2^127, where p is 2^8 at most.
// The weights p s are two bf16 terms (16 bits), as are those of a bf16 cache: with one the output's error is half as large again
// as its own rounding's.
//
// The steps of all (sequence, kv head, 16 query rows) segments form one list that is cut into equal spans, one a workgroup of four
// waves, which deal the steps of a segment among themselves and fold what they have through LDS.  A segment that lies in one span
// is written at once; of the others every workgroup leaves an unnormalised partial, and the one that finishes last folds them.
//
// Bound by the rows' bytes where there are many: 64 sequences of 8192 keys, 32 heads on 8 of 128, 604 MB in 97 us (6.2 TB/s), of 512 .. 8192 keys
// 322 MB in 59 us; by the start and the join where there are few: one sequence of 2048 keys 8.9 us, of which 2.8 pass before the
// first row is there and 2 in the join; by the steps' vector instructions where there are many query rows a kv head, since every sixteen
// of them walk, unpack and scale the same keys anew: 16 / 64 / 128 new positions over 8192 keys, 32 heads on 8 of 128, 19 / 36 / 59 us.
#include <algorithm>
#include <type_traits>

#include "cache_q4.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"
#include "rt_kernels.hpp"

namespace rt {

namespace {

constexpr int kStep = 32;       // keys a step
constexpr int kWaves = 4;        // a workgroup
constexpr int kCus = 256;
constexpr int kMaxPieces = 256;  // partials of a segment
constexpr float kNoMax = -3.0e38f;
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes from any word
typedef float f32x2_any __attribute__((ext_vector_type(2), aligned(4)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ int len_of(const CacheAttendParams& p, int b) {
    return p.kv_lens ? min(max(p.kv_lens[b], 0), p.max_seq) : p.kv_len;
}
__device__ __forceinline__ int steps_of(int len) { return (len + kStep - 1) / kStep; }
// x / d for 0 <= x < 2^31, 0 < d, by a reciprocal in f32 and what it is off by (nothing or one where the quotient is small).
__device__ __forceinline__ int quotient(int x, int d) {
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)d));
    int r = x - q * d;
    while (r < 0) {
        q--;
        r += d;
    }
    while (r >= d) {
        q++;
        r -= d;
    }
    return __builtin_amdgcn_readfirstlane(q);
}
// The list that the workgroups share: of every segment `kStart` places and its steps.  The places stand for what a segment costs
// besides its steps, so that a span of short sequences is no longer a walk than one of a long one: us for 0 / 4 / 8 / 16 / 32 places, 256
// sequences of up to 300 keys at dim 64 46 / 25.7 / 25.0 / 24.5 / 24.9, 16 of 37 .. 3001 21.1 / 18.1 / 17.9 / 15.7 / 16.3, 32 of 500 .. 4096 at dim 128
// - / 27.8 / 27.4 / 26.4 / 26.2.
constexpr int kStart = 16;
constexpr int kLong = 64;  // steps a sequence, see per_cu
__device__ __forceinline__ int places_of(int len) { return len ? kStart + steps_of(len) : 0; }
struct Span {
    int total, size;    // places of all; of a span
    int b, first, len;  // the sequence that holds the span's first place, the first place of that sequence, its length
    uint64_t empty;     // of the first 64 sequences, those without keys
};
// Places a span, of `total` and a longest sequence of `most` steps: what one of all workgroups gets, but no fewer than a join is worth --
// a segment of few spans is a long walk, one of many a long join: their sum is least around the root of its steps (p.span_root; one
// sequence of 8192 keys, 32 heads on 8 of 128, in 8 / 16 / 21 / 32 / 64 pieces 16.9 / 11.7 / 12.0 / 13.1 / 16.3 us) -- and
// never more of them than kMaxPieces (the steps of a segment touch at most most / size + 2).
__device__ __forceinline__ int span_size(const CacheAttendParams& p, int total, int most) {
    const int groups = total >= (long long)(kStart + kLong) * p.kv_heads * p.n_tiles * p.batch ? p.n_long : p.n_groups;
    const int root = __builtin_amdgcn_readfirstlane((int)(__builtin_amdgcn_sqrtf((float)most) * p.span_root + 0.5f * kWaves)) & -kWaves;
    return max(max(kWaves, quotient(total + groups - 1, groups)), max(root, (most + kMaxPieces - 3) / (kMaxPieces - 2)));
}
// Lengths 64 at a time, the first of them once for both walks.
__device__ __forceinline__ Span span_of(const CacheAttendParams& p, int group, int lane) {
    const int per = p.kv_heads * p.n_tiles;
    Span s;
    if (p.batch == 1) {  // (one scalar load)
        int len = p.kv_len;
        if (p.kv_lens) len = min(max(*(const __attribute__((address_space(4))) int32_t*)p.kv_lens, 0), p.max_seq);
        s.empty = len == 0;
        s.total = places_of(len) * per;
        const int most = steps_of(len);
        s.size = span_size(p, s.total, most);
        s.b = s.first = 0;
        s.len = len;
        return s;
    }
    auto len_at = [&](int b0) { return b0 + lane < p.batch ? len_of(p, b0 + lane) : 0; };
    const int len0 = len_at(0), ends0 = lane_sums(places_of(len0));
    s.empty = __ballot(len0 == 0);
    int sum = __builtin_amdgcn_readlane(ends0, 63), most = lane_max(len0);
    for (int b0 = 64; b0 < p.batch; b0 += 64) {
        const int len = len_at(b0);
        sum += __builtin_amdgcn_readlane(lane_sums(places_of(len)), 63);
        most = max(most, lane_max(len));
    }
    most = steps_of(most);
    s.total = sum * per;
    s.size = span_size(p, s.total, most);
    s.b = s.first = s.len = 0;
    const long long at = (long long)group * s.size;
    if (at >= s.total) return s;
    int before = 0, len = len0, ends = ends0;
    for (int b0 = 0;;) {
        const uint64_t past = __ballot((long long)before + (long long)ends * per > at);
        if (past) {  // (it is for one of them: `at` is below the total)
            const int l = __ffsll((unsigned long long)past) - 1;
            s.b = b0 + l;
            s.len = __builtin_amdgcn_readlane(len, l);
            s.first = before + (__builtin_amdgcn_readlane(ends, l) - places_of(s.len)) * per;
            return s;
        }
        before += __builtin_amdgcn_readlane(ends, 63) * per;
        b0 += 64;
        len = len_at(b0);
        ends = lane_sums(places_of(len));
    }
}

// ---- partials that another workgroup of the launch reads: device scope both ways, as in decode.hip --------------------------
constexpr int kScopeDevice = 16;  // sc1
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, kBufferFlags);
}
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t rs, uint32_t byte, f32x4_t v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), rs, byte, 0, kScopeDevice);
}
__device__ __forceinline__ void put2(__amdgpu_buffer_rsrc_t rs, uint32_t byte, float a, float b) {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{__float_as_uint(a), __float_as_uint(b)}, rs, byte, 0, kScopeDevice);
}
__device__ __forceinline__ f32x4_t get4(__amdgpu_buffer_rsrc_t rs, uint32_t byte) {
    return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, byte, 0, kScopeDevice));
}
__device__ __forceinline__ u32x2_t get2(__amdgpu_buffer_rsrc_t rs, uint32_t byte) { return __builtin_amdgcn_raw_buffer_load_b64(rs, byte, 0, kScopeDevice); }

// The word through which a segment's workgroups learn which of them is the last: (launch id | count).  It lies in the caller's
// workspace, which holds anything: every workgroup makes sure, ahead of its own count, that the word carries this launch's id.
// The last one leaves 0 there, so that a recorded launch, which brings its id along on every replay, finds none of its own counts.
typedef unsigned long long word_t;
constexpr int kWordPitch = 128;  // bytes: atomics on one line wait for each other
constexpr word_t kCountMask = 0xffff;
struct SegmentWord {
    word_t* at;
    word_t id, seen, got;
    __device__ __forceinline__ bool ours(word_t x) const { return ((x ^ id) & ~kCountMask) == 0; }
    // what is there, asked for ahead of the rows; it is replaced behind their requests, and whether that has held is looked at ahead
    // of the count: neither is waited for by itself
    __device__ __forceinline__ void request(void* word, word_t launch_id) {
        at = (word_t*)word;
        id = launch_id;
        seen = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ void replace() {
        got = seen;
        __hip_atomic_compare_exchange_strong(at, &got, ours(seen) ? seen : id, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ __forceinline__ void settle() {
        while (got != seen && !ours(got)) {  // (fails only if another workgroup was first, whose id is this one, or with another launch's word)
            seen = got;
            replace();
        }
    }
    // counts one finished partial of `n`; true for the one that completes the set
    __device__ __forceinline__ bool count(int n) {
        const word_t old = __hip_atomic_fetch_add(at, (word_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = (int)(old & kCountMask) + 1 == n;
        if (last) __hip_atomic_store(at, (word_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return last;
    }
};

// ---- what a lane holds of 32 keys ----------------------------------------------------------------------------------
// As an operand of scores^T, keys are rows: lane (n, quad) has key n of either 16, and a quarter of each row.  As an operand of
// out^T, dims are rows and keys the products' inner index: lane (n, quad) has dims by n of the eight keys 4 quad + {0..3}, 16 + those, in the order
// in which scores^T leaves their weights.
//
// Up to four or eight query rows leave most of the sixteen columns of a product idle, and what is done a (row, key) -- scales, exponentials,
// the weights' terms -- would be done for all sixteen.  There a row has C = 4 or 2 columns, n, n + 16 / C, ..., and each of them takes a
// C-th of a lane's eight keys: the others' weights are zeros in its operand, and its part of the row has a maximum and a sum of its own,
// folded with the waves' at the end.  (Scores of all eight are there anyway: selecting them costs less than finishing them.  Four rows
// with C = 1 / 2 / 4: 64 sequences of 512 .. 8192 keys, dim 128 91 / 78 / 77 us, 64 of 4096 at dim 64 40 / 35 / 33, 16 of 8192 at dim 256 138 / 70 / 67.)
template <int D, bool Q4, int C>
struct Keys {
    static constexpr int kKw = Q4 ? D / 32 : D / 8, kVw = Q4 ? (D + 127) / 128 : D / 32, kG = Q4 ? D / 64 : 1, kE = 8 / C;
    uint32_t k[2][kKw], v[8][kVw];
    uint32_t ks[kG][kE], vs[kG][kE];  // pairs of the lane's keys
};

// bf16 rows come through registers, K's of the next step as soon as this step's scores are there and V's as soon as its products are.  V's
// past the caches, whole lines a request (16 sequences of 4000 at dim 128 63 -> 49 us); K's, whose lines take two requests, through them.
template <int D, int C>
__device__ __forceinline__ void load_k(Keys<D, false, C>& t, const uint8_t* k, int key0, int len, int n, int quad) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint8_t* row = k + (size_t)min(key0 + 16 * h + n, len - 1) * (2 * D);
#pragma unroll
        for (int c = 0; c < D / 32; c++) *(u32x4_t*)(t.k[h] + 4 * c) = *(const u32x4_t*)(row + 64 * c + 16 * quad);
    }
}
template <int D, int C>
__device__ __forceinline__ void load_v(Keys<D, false, C>& t, const uint8_t* v, int key0, int len, int n, int quad) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint8_t* row = v + (size_t)min(key0 + 16 * (e / 4) + 4 * quad + e % 4, len - 1) * (2 * D);
#pragma unroll
        for (int i = 0; i < D / 128; i++) *(u32x4_t*)(t.v[e] + 4 * i) = __builtin_nontemporal_load((const u32x4_t*)(row + 256 * i + 16 * n));
        if constexpr (D == 64) *(u32x2_t*)t.v[e] = __builtin_nontemporal_load((const u32x2_t*)(row + 8 * n));
    }
}

// 4-bit rows go straight to LDS, kStages steps of a wave under way, and their pairs with them: in registers the pairs alone, of which
// sixteen lanes need each, were 32 a lane and step.  Rows lie there so that a wave's reads meet no bank twice: K's 16-byte pieces exchanged
// by the row (16 lanes read a piece each of 16 rows), V's rows 0, 4, 8, 12, 1, ... (four quads read rows 4 apart at once).
template <int D>
struct Ring {
    static constexpr int kRow = D / 2, kStages = 2, kG = D / 64;
    static constexpr int kRows = 32 * kRow, kPairs = D == 256 ? 512 : 256;  // bytes of K or V, of their pairs
    static_assert(kStages == 2, "the waits of the walk");
    static constexpr int kStage = 2 * kRows + 2 * kPairs;
    static constexpr int kLoads = 2 * (kRows / 1024) + 2 * (kPairs / 256);  // requests a stage
    // the source of what lands at byte `at` of 16 rows
    static __device__ __forceinline__ uint32_t k_source(uint32_t at) {
        const uint32_t r = at / kRow, c = at % kRow / 16;
        return r * kRow + 16 * (D == 64 ? c : D == 128 ? c ^ (r >> 2 & 3) : c ^ (r >> 1 & 7));
    }
    static __device__ __forceinline__ uint32_t v_source(uint32_t at) {
        const uint32_t slot = at / kRow;
        return (((slot & 3) << 2) + (slot >> 2)) * kRow + at % kRow;
    }
};

template <int D>
struct RingLanes {  // byte offsets of a lane's requests
    uint32_t k[D == 64 ? 1 : D == 128 ? 2 : 4], v[D == 64 ? 1 : D == 128 ? 2 : 4], pair;
    __device__ __forceinline__ RingLanes(int lane, int max_seq) {
        using R = Ring<D>;
#pragma unroll
        for (int i = 0; i < R::kRows / 1024; i++) {
            const uint32_t at = 1024u * i + 16u * lane, half = at / (16 * R::kRow);
            k[i] = half * (16 * R::kRow) + R::k_source(at % (16 * R::kRow));
            v[i] = half * (16 * R::kRow) + R::v_source(at % (16 * R::kRow));
        }
        pair = 4u * (uint32_t)(lane & 31) + (lane >= 32 ? 4u * (uint32_t)max_seq : 0u);  // (two groups a request)
    }
};

// The requests of one step: keys [key0, key0 + 32) of a slab of `len` keys.  What lies behind the last key lands as zeros, but for pairs
// of another group's first keys, which no visible key's place takes.  key0 < len.
// kOnce: past the caches, rows that no other workgroup asks for (64 sequences of 8192 keys 108 -> 98 us; with 64 query rows a head, whose
// keys four workgroups walk, 64 -> 69).
template <int D, bool kOnce>
__device__ __forceinline__ void ring_load(const RingLanes<D>& at, uint32_t lds, const uint8_t* k, const uint8_t* v, const uint32_t* kp, const uint32_t* vp, int max_seq, int key0, int len) {
    using R = Ring<D>;
    const int keys = min(kStep, len - key0);
    const size_t from = (size_t)key0;
    const uint32_t bytes = (uint32_t)keys * R::kRow;
    const u32x4_t krs = make_rsrc(k + from * R::kRow, bytes), vrs = make_rsrc(v + from * R::kRow, bytes);
#pragma unroll
    for (int i = 0; i < R::kRows / 1024; i++) {
        if constexpr (kOnce) {
            buffer_to_lds_past(krs, at.k[i], 0u, lds + 1024u * i);
            buffer_to_lds_past(vrs, at.v[i], 0u, lds + R::kRows + 1024u * i);
        } else {
            buffer_to_lds(krs, at.k[i], 0u, lds + 1024u * i);
            buffer_to_lds(vrs, at.v[i], 0u, lds + R::kRows + 1024u * i);
        }
    }
    const uint32_t pair_bytes = 4u * (uint32_t)keys + (D > 64 ? 4u * (uint32_t)max_seq : 0u);
#pragma unroll
    for (int i = 0; i < R::kPairs / 256; i++) {
        buffer_to_lds_b32(make_rsrc(kp + from + (size_t)(2 * i) * max_seq, pair_bytes), at.pair, 0u, lds + 2 * R::kRows + 256u * i);
        buffer_to_lds_b32(make_rsrc(vp + from + (size_t)(2 * i) * max_seq, pair_bytes), at.pair, 0u, lds + 2 * R::kRows + R::kPairs + 256u * i);
    }
}
// pairs of the lane's keys: of both sixteens, of one, or two of them
template <int D, int C>
__device__ __forceinline__ void ring_pairs(uint32_t (&to)[D / 64][8 / C], const unsigned char* pairs, int cls, int quad) {
#pragma unroll
    for (int g = 0; g < D / 64; g++) {
        const unsigned char* at = pairs + 128 * g + 16 * quad;
        if constexpr (C == 1) {
            *(u32x4_t*)to[g] = *(const u32x4_t*)at;
            *(u32x4_t*)(to[g] + 4) = *(const u32x4_t*)(at + 64);
        } else if constexpr (C == 2) {
            *(u32x4_t*)to[g] = *(const u32x4_t*)(at + 64 * cls);
        } else {
            *(u32x2_t*)to[g] = *(const u32x2_t*)(at + 64 * (cls >> 1) + 8 * (cls & 1));
        }
    }
}
template <int D, int C>
__device__ __forceinline__ void ring_k(Keys<D, true, C>& t, const unsigned char* stage, int n, int cls, int quad) {
    using R = Ring<D>;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const unsigned char* row = stage + (16 * h + n) * R::kRow;
        if constexpr (D == 64) {
            *(u32x2_t*)t.k[h] = *(const u32x2_t*)(row + 8 * quad);
        } else {
#pragma unroll
            for (int i = 0; i < D / 128; i++) {
                const int c = quad * (D / 128) + i;
                *(u32x4_t*)(t.k[h] + 4 * i) = *(const u32x4_t*)(row + 16 * (D == 128 ? c ^ (n >> 2 & 3) : c ^ (n >> 1 & 7)));
            }
        }
    }
    ring_pairs<D, C>(t.ks, stage + 2 * R::kRows, cls, quad);
}
template <int D, int C>
__device__ __forceinline__ void ring_v(Keys<D, true, C>& t, const unsigned char* stage, int n, int cls, int quad) {
    using R = Ring<D>;
    ring_pairs<D, C>(t.vs, stage + 2 * R::kRows + R::kPairs, cls, quad);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const unsigned char* row = stage + R::kRows + (16 * (e / 4) + 4 * (e % 4) + quad) * R::kRow + (D / 32) * n;
        if constexpr (D == 64) t.v[e][0] = *(const uint16_t*)row;
        else if constexpr (D == 128) t.v[e][0] = *(const uint32_t*)row;
        else *(u32x2_t*)t.v[e] = *(const u32x2_t*)row;
    }
}

// The codes at bits 4 nib of every second byte as two bf16 numbers, c or 16 c times 2^kCodeExp.  The masks stand in registers: as literals
// they would be a word more of every instruction.
constexpr int kCodeExp = -133, kScaleExp = 60;  // (kScaleExp: as 0x1p60f too)
struct Codes {
    uint32_t low, high;
    __device__ __forceinline__ Codes() {
        asm volatile("s_mov_b32 %0, 0xf000f" : "=s"(low));
        asm volatile("s_mov_b32 %0, 0xf000f0" : "=s"(high));
    }
    template <int kNib>
    __device__ __forceinline__ uint32_t of(uint32_t w) const {
        return (kNib >= 2 ? w >> 8 : w) & (kNib & 1 ? high : low);
    }
};

// The largest of the four lanes of a query row (rows of 16 lanes swapped, then halves of the wave).
__device__ __forceinline__ float quad_max(float x) {
    const u32x2_t a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const u32x2_t c = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
// A row of sixteen lanes turned by kBy, and what that makes of columns that lie 16 / C apart: their largest, their sum, in every one.
template <int kBy>
__device__ __forceinline__ float turned(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + kBy, 0xf, 0xf, true));
}
template <int C>
__device__ __forceinline__ float columns_max(float x) {
    if (C >= 2) x = fmaxf(x, turned<8>(x));
    if (C >= 4) x = fmaxf(x, turned<4>(x));
    if (C == 16) {
        x = fmaxf(x, turned<2>(x));
        x = fmaxf(x, turned<1>(x));
    }
    return x;
}
template <int C>
__device__ __forceinline__ float columns_sum(float x) {
    if (C >= 2) x += turned<8>(x);
    if (C >= 4) x += turned<4>(x);
    if (C == 16) {
        x += turned<2>(x);
        x += turned<1>(x);
    }
    return x;
}
__device__ __forceinline__ float quad_sum(float x) {
    const u32x2_t a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const u32x2_t c = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// The hi and lo terms of two weights: hi by truncation, what it leaves by truncation too (16 bits in all).  Returns the sum of the terms:
// what is taken off for the codes' offsets has to be what went in, or the truncation's bias comes back 8 times.
__device__ __forceinline__ float two_terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ha = __uint_as_float(__float_as_uint(a) & 0xffff0000u), hb = __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    hi = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    const float la = a - ha, lb = b - hb;
    lo = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302u);
    return (ha + __uint_as_float(__float_as_uint(la) & 0xffff0000u)) + (hb + __uint_as_float(__float_as_uint(lb) & 0xffff0000u));
}

// Waves that an SIMD can hold: as many as have their registers without spills.
template <int D, bool Q4, int C>
constexpr int per_simd() { return D == 64 ? 4 : !Q4 ? 256 / D : (D == 128 ? 3 : 2) - (C == 1 ? 1 : 0); }

// What a lane has of its query row over the keys it has walked.
template <int D, bool Q4>
struct State {
    static constexpr int kG = Q4 ? D / 64 : 1;
    float m, l, ps[kG], pz[kG];  // ps: the sum of the weights as they enter the products
    f32x4_t o[D / 16];
    __device__ __forceinline__ void reset() {
        m = kNoMax;
        l = 0.0f;
#pragma unroll
        for (int g = 0; g < kG; g++) {
            ps[g] = pz[g] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] = f32x4_t{0, 0, 0, 0};
    }
};

// One step.  kCut: not every row sees all of its keys.  scores: the lane's row from key0 + 4 quad on, or null.  k_done is called
// behind the last use of K, v_due ahead of V's first.
template <int D, bool Q4, int C, bool kCut, bool kWeigh, typename KDone, typename VDue>
__device__ __forceinline__ void step(State<D, Q4>& st, const Keys<D, Q4, C>& x, KDone k_done, VDue v_due, const Codes& codes, const u32x4_t (&q)[D / 32], const float (&q_sum)[Q4 ? D / 64 : 1],
                                     int cls, int first_key, int seen, float scale_log2e, float unscale, float* scores) {
    constexpr int kG = Keys<D, Q4, C>::kG, kO = D / 16, kE = 8 / C;
    float y[kE];
    // of both sixteens' scores, a column's
    auto own = [&](const f32x4_t (&a)[2], float (&to)[kE]) __attribute__((always_inline)) {
        if constexpr (C == 1) {
#pragma unroll
            for (int e = 0; e < 8; e++) to[e] = a[e / 4][e % 4];
        } else if constexpr (C == 2) {
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = cls ? a[1][e] : a[0][e];
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                // (of both sixteens first: two of one register group the compiler takes for an index into it, four selections)
                const float a0 = cls & 2 ? a[1][e] : a[0][e], a2 = cls & 2 ? a[1][2 + e] : a[0][2 + e];
                to[e] = cls & 1 ? a2 : a0;
            }
        }
    };
    if constexpr (Q4) {
#pragma unroll
        for (int g = 0; g < kG; g++) {
            const float c0 = -8.0f * q_sum[g];
            f32x4_t a[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                a[h] = f32x4_t{c0, c0, c0, c0};
                u32x4_t lo, hi;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // dim 64: word i / 2, chunk i % 2; above: word i of (dim 128 pairs) g / 2, its group g % 2
                    const uint32_t w = D == 64 ? x.k[h][i / 2] : x.k[h][i * (D / 128) + g / 2];
                    const bool upper = D == 64 ? i & 1 : g & 1;
                    lo[i] = upper ? codes.of<2>(w) : codes.of<0>(w);
                    hi[i] = upper ? codes.of<3>(w) : codes.of<1>(w);
                }
                a[h] = mfma(lo, q[2 * g], a[h]);
                a[h] = mfma(hi, q[2 * g + 1], a[h]);
            }
            float f[kE];
            own(a, f);
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const float z = bf16_hi(x.ks[g][e]) * q_sum[g];
                y[e] = fmaf(bf16_lo(x.ks[g][e]), f[e], g == 0 ? z : y[e] + z);
            }
            if (D > 64) __builtin_amdgcn_sched_barrier(0);  // (one group's words at a time in registers)
        }
    } else {
        f32x4_t a[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            a[h] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 32; c++) a[h] = mfma(*(const u32x4_t*)(x.k[h] + 4 * c), q[c], a[h]);
        }
        own(a, y);
    }
    k_done();
    // the lane's keys: first_key + place(e), of its eight slots
    auto place = [&](int e) __attribute__((always_inline)) { return C == 1 ? 16 * (e / 4) + e % 4 : C == 2 ? 16 * cls + e : 16 * (cls >> 1) + 2 * (cls & 1) + e; };
    bool hid[kE];
#pragma unroll
    for (int e = 0; e < kE; e++) {
        hid[e] = kCut && first_key + place(e) >= seen;
        if (hid[e]) y[e] = neg_inf();
    }
    if constexpr (kWeigh) {
        auto full = [&](float x) __attribute__((always_inline)) { return Q4 ? x * unscale : x; };
        if (scores) {
            if constexpr (kCut) {
#pragma unroll
                for (int e = 0; e < kE; e++)
                    if (!hid[e]) scores[place(e)] = full(y[e]);
            } else if constexpr (C == 4) {
                *(f32x2_any*)(scores + place(0)) = f32x2_any{full(y[0]), full(y[1])};
            } else {
#pragma unroll
                for (int e = 0; e < kE; e += 4) *(f32x4_any*)(scores + place(e)) = f32x4_any{full(y[e]), full(y[e + 1]), full(y[e + 2]), full(y[e + 3])};
            }
        }
    }
    // The running maximum, common to the four lanes of a column.  It follows the scores only where they have risen by 8 in the exponent
    // of two: up to there the weights, all of them f32 or two bf16 terms, are as exact, and sums are scaled once or twice a span
    // (64 query heads on 8, 64 sequences of 8192 keys: 137 us, 144 where every rise counts).
    float top = y[0];
#pragma unroll
    for (int e = 1; e < kE; e++) top = fmaxf(top, y[e]);
    top = quad_max(top);
    if (__any((top - st.m) * scale_log2e > 8.0f)) {
        const float m_new = fmaxf(st.m, top), alpha = __builtin_amdgcn_exp2f((st.m - m_new) * scale_log2e);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int g = 0; g < kG; g++) {
            st.ps[g] *= alpha;
            st.pz[g] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < kO; i++) st.o[i] *= alpha;
    }
    float w[kE];
#pragma unroll
    for (int e = 0; e < kE; e++) {
        w[e] = __builtin_amdgcn_exp2f((y[e] - st.m) * scale_log2e);
        st.l += w[e];
    }
    // pairs of weights as the operand's words, zeros in the other columns' places
    auto operand = [&](const float (&f)[kE], u32x4_t& hi, u32x4_t& lo) __attribute__((always_inline)) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kE / 2; i++) {
            uint32_t a, c;
            sum += two_terms(f[2 * i], f[2 * i + 1], a, c);
            if constexpr (C == 1) {
                hi[i] = a;
                lo[i] = c;
            } else {
#pragma unroll
                for (int j = 0; j < C; j++) {
                    hi[j * (kE / 2) + i] = cls == j ? a : 0u;
                    lo[j * (kE / 2) + i] = cls == j ? c : 0u;
                }
            }
        }
        return sum;
    };
    // out^T
    v_due();
    if constexpr (Q4) {
#pragma unroll
        for (int g = 0; g < kG; g++) {
            u32x4_t p_hi, p_lo;
            float s[kE];
#pragma unroll
            for (int e = 0; e < kE; e++) {
                s[e] = hid[e] ? 0.0f : w[e] * 0x1p60f * bf16_lo(x.vs[g][e]);  // (what a hidden row holds stays out, were it NaN)
                if (kCut) st.pz[g] += hid[e] ? 0.0f : w[e] * bf16_hi(x.vs[g][e]);
                else st.pz[g] = fmaf(w[e], bf16_hi(x.vs[g][e]), st.pz[g]);
            }
            st.ps[g] += operand(s, p_hi, p_lo);
            // the bytes whose chunks are of this group
#pragma unroll
            for (int f = 0; f < 2; f++) {
                const int byte = D == 64 ? f : (g & 1) + 2 * f, word = D == 64 ? 0 : g / 2;
                u32x4_t lo, hi;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t z = __builtin_amdgcn_perm(x.v[2 * i + 1][word], x.v[2 * i][word], 0x0c000c00u | (uint32_t)(4 + byte) << 16 | (uint32_t)byte);
                    lo[i] = codes.of<0>(z);
                    hi[i] = codes.of<1>(z);
                }
                const int at_o = 8 * word + 2 * byte;
                st.o[at_o] = mfma(lo, p_lo, mfma(lo, p_hi, st.o[at_o]));
                st.o[at_o + 1] = mfma(hi, p_lo, mfma(hi, p_hi, st.o[at_o + 1]));
                if (D > 64) __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else {
        u32x4_t p_hi, p_lo;
        operand(w, p_hi, p_lo);
#pragma unroll
        for (int d = 0; d < kO; d++) {  // dim n * (D / 16) + d; of 256, of the lower and of the upper 128 in turn
            u32x4_t a;
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][d / 2], x.v[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
            st.o[d] = mfma(a, p_lo, mfma(a, p_hi, st.o[d]));
        }
    }
}

template <int D, bool Q4, int C, bool kWeigh>
__global__ __launch_bounds__(64 * kWaves, (per_simd<D, Q4, C>())) void cache_attend_kernel(CacheAttendParams p) {
    constexpr int kG = Keys<D, Q4, C>::kG, NT = 64 * kWaves, kPitch = D + 4, kR = 16 / C;  // kR query rows
    constexpr int kRingBytes = Q4 ? kWaves * Ring<D>::kStages * Ring<D>::kStage : 0, kFold = kWaves * 16 * kPitch * 4, kFolds = kMaxPieces * 16 * 8 + NT * 16;
    constexpr int kLds = std::max(std::max(kRingBytes, kFold), kFolds);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kLds];
    __shared__ float red_m[kWaves][16], red_l[kWaves][16], inv_l[16];
    __shared__ int is_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, quad = lane >> 4, cls = n / kR, group = blockIdx.x;
    const int per = p.kv_heads * p.n_tiles;

    const Span span = span_of(p, group, lane);
    // sequences without keys, dealt to the workgroups: rows of zeros
    for (int b = group; b < p.batch; b += (int)gridDim.x)
        if (b < 64 ? (span.empty >> b & 1) != 0 : len_of(p, b) == 0)
            for (int i = tid; i < p.seq_new * p.heads * (D / 8); i += NT) *(u32x4_t*)(p.out + (size_t)b * p.seq_new * p.heads * D + 8 * i) = u32x4_t{0, 0, 0, 0};
    const long long begin = (long long)group * span.size;
    if (begin >= span.total) return;
    int at = (int)begin, b = span.b, first = span.first, len = span.len;
    const int end = (int)min((long long)span.total, begin + span.size);

    while (at < end) {
        // the piece of a segment from here
        const int places = places_of(len);
        if (at >= first + places * per) {  // the next sequence
            first += places * per;
            b++;
            len = len_of(p, b);
            continue;
        }
        const int seg = quotient(at - first, places), seg_first = first + seg * places;
        const int t0 = max(at - seg_first - kStart, 0), t1 = min(places, end - seg_first) - kStart;
        at = min(seg_first + places, end);
        if (t1 <= 0) continue;  // (places alone)
        const int kvh = p.n_tiles == 1 ? seg : quotient(seg, p.n_tiles), tile = seg - kvh * p.n_tiles;
        const int w0 = quotient(seg_first + kStart, span.size), pieces = quotient(seg_first + places - 1, span.size) - w0 + 1;  // workgroups that have some of its steps
        const size_t segment = (size_t)b * per + seg;

        const int r = tile * kR + n % kR;  // the query row: position * group + head of the group
        const bool there = r < p.rows;
        const int s_new = there ? r / p.group : 0, head = kvh * p.group + (there ? r - s_new * p.group : 0);
        const int seen = len - p.seq_new + s_new + 1;  // keys that it sees
        const size_t slab = ((size_t)b * p.kv_heads + kvh) * (size_t)p.max_seq;

        SegmentWord word;
        if (pieces > 1 && tid == 0) word.request(p.words + segment * kWordPitch, p.launch_id);
        // q as the operand that the keys' words pair with
        u32x4_t q[D / 32];
        float q_sum[kG] = {};
        int q_exp = 0;  // scores of 4-bit rows are 2^q_exp times their own
        u32x4_t nat[D / 32];
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            nat[c] = u32x4_t{0, 0, 0, 0};
            if (there) nat[c] = *(const u32x4_t*)(p.q + (((size_t)b * p.seq_new + s_new) * p.heads + head) * D + 32 * c + 8 * quad);
        }
        const RingLanes<D> lanes(lane, p.max_seq);
        constexpr int kRow = Q4 ? D / 2 : 2 * D;
        const uint8_t* k = (const uint8_t*)p.k + slab * kRow;
        const uint8_t* v = (const uint8_t*)p.v + slab * kRow;
        const uint32_t* kp = Q4 ? p.k_pairs + slab * kG : nullptr;
        const uint32_t* vp = Q4 ? p.v_pairs + slab * kG : nullptr;
        const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + (uint32_t)wave * (Q4 ? Ring<D>::kStages * Ring<D>::kStage : 0);
        const unsigned char* const ring_at = lds + wave * (Q4 ? Ring<D>::kStages * Ring<D>::kStage : 0);
        Keys<D, Q4, C> x;
        if constexpr (Q4) {
#pragma unroll
            for (int s = 0; s < Ring<D>::kStages; s++)
                if (t0 + wave + s * kWaves < t1) ring_load<D, (C > 1)>(lanes, ring + s * Ring<D>::kStage, k, v, kp, vp, p.max_seq, (t0 + wave + s * kWaves) * kStep, len);
        } else {
            if (t0 + wave < t1) {
                load_k<D, C>(x, k, (t0 + wave) * kStep, len, n, quad);
                load_v<D, C>(x, v, (t0 + wave) * kStep, len, n, quad);
            }
        }
        if (pieces > 1 && tid == 0) word.replace();
        if constexpr (!Q4) {
#pragma unroll
            for (int c = 0; c < D / 32; c++) q[c] = nat[c];
        } else {
            // the row's largest exponent, of 2^-60 at least (a score of 2^-133 times that much is as good as 0)
            u16x2_t most = {0, 0};
#pragma unroll
            for (int c = 0; c < D / 32; c++)
#pragma unroll
                for (int i = 0; i < 4; i++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, nat[c][i] & 0x7fff7fffu));
            const int field = max((int)quad_max((float)(max(most[0], most[1]) >> 7)), 67), up = 247 - field;
            q_exp = up + kCodeExp;
            // Through f32, exactly: 0 stays 0 and a subnormal number grows like the others.  (An addition to the exponents' bits is 0.1 us faster in
            // the smallest calls, but makes a 0 as much as 2^-127, and keys of 2^115 a score of that.)  A row with values above 2^110, or that
            // are no numbers, is NaN.
            auto scaled = [](float x, int by) __attribute__((always_inline)) { return __float_as_uint(__builtin_amdgcn_ldexpf(x, by)); };
#pragma unroll
            for (int g = 0; g < kG; g++) {
                float sum = field > 237 ? quiet_nan() : 0.0f;
#pragma unroll
                for (int c = 2 * g; c < 2 * g + 2; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) sum += bf16_lo(nat[c][i]) + bf16_hi(nat[c][i]);
                q_sum[g] = __builtin_amdgcn_ldexpf(quad_sum(sum), q_exp);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // dim 64: word (u, c) pairs i's of one chunk; above: chunks 2 g and 2 g + 1 at one i
                    const uint32_t a = D == 64 ? nat[i & 1][i & 2] : nat[2 * g][i], o = D == 64 ? nat[i & 1][(i & 2) + 1] : nat[2 * g + 1][i];
                    q[2 * g][i] = __builtin_amdgcn_perm(scaled(bf16_lo(o), up), scaled(bf16_lo(a), up), 0x07060302u);
                    q[2 * g + 1][i] = __builtin_amdgcn_perm(scaled(bf16_hi(o), up - 4), scaled(bf16_hi(a), up - 4), 0x07060302u);
                }
            }
        }
        const float scale_log2e = Q4 ? __builtin_amdgcn_ldexpf(p.scale_log2e, -q_exp) : p.scale_log2e, unscale = __builtin_amdgcn_ldexpf(1.0f, -q_exp);
        const int all_see = len - p.seq_new + 1;  // keys that every row sees
        float* const scores = kWeigh && there ? p.scores + ((size_t)b * p.heads + head) * (size_t)p.max_seq + 4 * quad : nullptr;

        const Codes codes;
        State<D, Q4> st;
        st.reset();
        // Steps that every row sees whole, then the others, in loops of their own: as two branches of one loop they would have the sums in
        // two sets of registers.
        const int t_whole = min(t1, max(all_see, 0) / kStep);
        int t = t0 + wave, stage = 0;
        auto take = [&](auto cut) __attribute__((always_inline)) {
            constexpr bool kCut = decltype(cut)::value;
            const int key0 = t * kStep;
            float* const to = kWeigh && there ? scores + key0 : nullptr;
            if constexpr (Q4) {
                // (this step's requests are there, if not the next one's)
                if (t + kWaves < t1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Ring<D>::kLoads) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                const unsigned char* const rows = ring_at + stage * Ring<D>::kStage;
                ring_k<D, C>(x, rows, n, cls, quad);
                step<D, Q4, C, kCut, kWeigh>(st, x, [] {}, [&]() __attribute__((always_inline)) { ring_v<D, C>(x, rows, n, cls, quad); }, codes, q, q_sum, cls, key0 + 4 * quad, seen, scale_log2e, unscale, to);
                const int next = t + Ring<D>::kStages * kWaves;
                if (next < t1) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (read before it is written again)
                    ring_load<D, (C > 1)>(lanes, ring + stage * Ring<D>::kStage, k, v, kp, vp, p.max_seq, next * kStep, len);
                }
                stage ^= 1;
            } else {
                const int next = t + kWaves;
                step<D, Q4, C, kCut, kWeigh>(st, x, [&]() __attribute__((always_inline)) { if (next < t1) load_k<D, C>(x, k, next * kStep, len, n, quad); }, [] {}, codes, q, q_sum, cls, key0 + 4 * quad, seen,
                                             scale_log2e, unscale, to);
                if (next < t1) load_v<D, C>(x, v, next * kStep, len, n, quad);
            }
            t += kWaves;
        };
        while (t < t_whole) take(std::false_type{});
        while (t < t1) take(std::true_type{});
        // ---- fold the four waves, and the columns of a row.  (The thread's number anew: what follows from it would be worked out
        // ahead of the steps otherwise, and take their registers.)
        int ft = threadIdx.x;
        asm volatile("" : "+v"(ft));
        const int tid = ft, lane = ft & 63, n = ft & 15, quad = lane >> 4;
        if (Q4 && st.m != kNoMax) st.m = __builtin_amdgcn_ldexpf(st.m, -q_exp);
        const float m = columns_max<C>(st.m), f = __builtin_amdgcn_exp2f((st.m - m) * p.scale_log2e);
        const float l = columns_sum<C>(quad_sum(st.l) * f);
        if constexpr (Q4) {
            static_assert(-kCodeExp - kScaleExp == 73);
            const float whole[2] = {0x1p73f * f, 0x1p69f * f};
#pragma unroll
            for (int g = 0; g < kG; g++) {
                const float off = (quad_sum(st.pz[g]) - __builtin_amdgcn_ldexpf(quad_sum(st.ps[g]), 3 - kScaleExp)) * f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int byte = D == 64 ? i / 2 : (g & 1) + 2 * (i / 2);
                    f32x4_t& o = st.o[8 * (D == 64 ? 0 : g / 2) + 2 * byte + i % 2];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = fmaf(o[e], whole[i % 2], off);
                }
            }
        }
        if (C > 1)
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) st.o[i][e] = columns_sum<C>(Q4 ? st.o[i][e] : st.o[i][e] * f);
        float* const red = (float*)lds;  // [wave][row][kPitch]
        if (n < kR && quad == 0) {
            red_m[wave][n] = m;
            red_l[wave][n] = l;
        }
        __syncthreads();  // also: every wave is done with the ring
        float m_wg = red_m[0][n % kR], l_wg = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; w++) m_wg = fmaxf(m_wg, red_m[w][n % kR]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) l_wg += red_l[w][n % kR] * __builtin_amdgcn_exp2f((red_m[w][n % kR] - m_wg) * p.scale_log2e);
        if (n < kR) {
            const float fw = __builtin_amdgcn_exp2f((m - m_wg) * p.scale_log2e);
            float* row = red + (wave * kR + n) * kPitch;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {  // eight dims in a row
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if constexpr (Q4) {
                        const int byte = D == 64 ? c : (c & ~3) | (c & 1) << 1 | (c >> 1 & 1);
                        y[e] = st.o[2 * byte + e % 2][e / 2] * fw;
                    } else {
                        y[e] = st.o[(8 * c + e) % (D / 16)][(8 * c + e) / (D / 16)] * fw;
                    }
                }
                float* dst = row + (Q4 ? 32 * c + 8 * quad : D == 256 ? 128 * (c & 1) + 32 * quad + 8 * (c >> 1) : quad * (D / 4) + 8 * c);
                *(f32x4_t*)dst = f32x4_t{y[0], y[1], y[2], y[3]};
                *(f32x4_t*)(dst + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
            }
            if (wave == 0 && quad == 0) inv_l[n] = l_wg == 0.0f ? 0.0f : 1.0f / l_wg;
        }
        __syncthreads();
        const int rows = min(kR, p.rows - tile * kR);
        const uint32_t slot_bytes = (uint32_t)p.part_rows * (D + 2) * 4;
        float* const slot = p.part + ((size_t)w0 + segment) * (slot_bytes / 4);  // of the segment's first piece; the others follow
        const uint32_t mine = (uint32_t)(group - w0) * slot_bytes;
        const __amdgpu_buffer_rsrc_t rs = rsrc_of(slot, (uint32_t)pieces * slot_bytes);
        auto out_row = [&](int row) {  // of the tile
            const int rr = tile * kR + row, s = rr / p.group;
            return (((size_t)b * p.seq_new + s) * p.heads + kvh * p.group + (rr - s * p.group)) * D;
        };
        for (int i = tid; i < rows * (D / 4); i += NT) {
            const int row = i / (D / 4), d = 4 * (i % (D / 4));
            f32x4_t o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; w++) o += *(const f32x4_t*)(red + (w * kR + row) * kPitch + d);
            if (pieces == 1) {
                o *= inv_l[row];
                *(u32x2_t*)(p.out + out_row(row) + d) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
            } else {
                put4(rs, mine + 4u * (uint32_t)(row * D + d), o);
            }
        }
        if (pieces == 1) {
            if (kWeigh && tid < rows) {
                float* to = p.stats + ((size_t)b * p.heads + kvh * p.group + tile * kR + tid) * 2;  // (one position: rows are heads)
                to[0] = m_wg;
                to[1] = inv_l[tid];
            }
            __syncthreads();  // (the next piece's requests land where the fold was)
            continue;
        }
        if (tid == 0) word.settle();
        if (tid < rows) put2(rs, mine + 4u * (uint32_t)(p.part_rows * D + 2 * tid), m_wg, l_wg);  // (tid < kR: n is tid)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) is_last = word.count(pieces) ? 1 : 0;
        __syncthreads();
        if (is_last) {
            // ---- the last workgroup of the segment: the weighted sum of its partials.  Items of four elements, kAhead pieces of each at a
            // time; where there are fewer items than threads, several threads an item, each with every sub-th piece.  The first are asked
            // for ahead of the (m, l) that their weights are made of.
            constexpr int kAhead = 8;
            float* const wgt = (float*)lds;  // [pieces][16]
            float* const wl = wgt + kMaxPieces * 16;
            f32x4_t* const part = (f32x4_t*)(wl + kMaxPieces * 16);
            const int items = rows * (D / 4), sub_n = items >= NT ? 1 : NT / items;
            const int x0 = sub_n == 1 ? tid : tid % items, sub = sub_n == 1 ? 0 : tid / items;
            f32x4_t a[kAhead];
            auto ask = [&](int i, int k0) __attribute__((always_inline)) {  // (row and element follow one another in a slot)
                const uint32_t from = 16u * (uint32_t)min(i, items - 1);
#pragma unroll
                for (int e = 0; e < kAhead; e++) a[e] = get4(rs, (uint32_t)min(k0 + e * sub_n, pieces - 1) * slot_bytes + from);
            };
            ask(x0, sub);
            {
                const int row = tid >> 4, col = tid & 15;  // sixteen lanes a row
                const bool on = row < rows;
                float top = kNoMax, sum = 0.0f;
                for (int k = col; on && k < pieces; k += 16) {
                    const u32x2_t ml = get2(rs, (uint32_t)k * slot_bytes + 4u * (uint32_t)(p.part_rows * D + 2 * row));
                    wgt[k * 16 + row] = __uint_as_float(ml[0]);
                    wl[k * 16 + row] = __uint_as_float(ml[1]);
                    top = fmaxf(top, __uint_as_float(ml[0]));
                }
                top = columns_max<16>(top);
                for (int k = col; on && k < pieces; k += 16) {
                    const float fk = __builtin_amdgcn_exp2f((wgt[k * 16 + row] - top) * p.scale_log2e);
                    wgt[k * 16 + row] = fk;
                    sum += wl[k * 16 + row] * fk;
                }
                sum = columns_sum<16>(sum);
                if (on && col == 0) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    inv_l[row] = inv;
                    if (kWeigh) {
                        float* to = p.stats + ((size_t)b * p.heads + kvh * p.group + tile * kR + row) * 2;
                        to[0] = top;
                        to[1] = inv;
                    }
                }
            }
            __syncthreads();
            for (int i0 = 0; i0 < items; i0 += NT) {
                const int i = i0 + x0;
                const bool on = i < items && sub < sub_n;
                const int row = on ? i / (D / 4) : 0, d = 4 * (i % (D / 4));
                f32x4_t o = {0, 0, 0, 0};
                for (int k0 = sub; on && k0 < pieces; k0 += kAhead * sub_n) {
                    if (i0 || k0 != sub) ask(i, k0);
#pragma unroll
                    for (int e = 0; e < kAhead; e++)
                        if (k0 + e * sub_n < pieces) o += a[e] * wgt[(k0 + e * sub_n) * 16 + row];
                }
                if (sub_n > 1) {  // (one round)
                    part[tid] = o;
                    __syncthreads();
                    if (on && sub == 0)
                        for (int e = 1; e < sub_n; e++) o += part[e * items + tid];
                }
                if (on && sub == 0) {
                    o *= inv_l[row];
                    *(u32x2_t*)(p.out + out_row(row) + d) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
                }
            }
        }
        __syncthreads();
    }
}

// The keys' weights from the scores and the rows' statistics.  Grid (1024 keys, kv heads, batch), four keys a thread; the heads' scores
// are asked for four at a time.  Bound by the launch and one chain of reads (one sequence of 8192 keys 4.0 us) or, in a batch, by the scores' bytes
// (32 of 300 .. 4096, 32 heads 5.8 us).  A launch of its own, since a weight needs its row's maximum over all spans.  (The workgroup that ends a
// segment has that maximum; with up to sixteen heads a kv head it could sum the segment's weights itself.  Not tried.)
__global__ __launch_bounds__(256) void cache_weigh_kernel(CacheAttendParams p) {
    const int kvh = blockIdx.y, b = blockIdx.z, len = len_of(p, b), j = (int)blockIdx.x * 1024 + 4 * (int)threadIdx.x;
    if (j >= len) return;
    const size_t sums = ((size_t)b * p.kv_heads + kvh) * (size_t)p.max_seq + j, row0 = (size_t)b * p.heads + kvh * p.group;
    const float* scores = p.scores + row0 * p.max_seq + j;
    const float* stats = p.stats + 2 * row0;
    auto part = [&](float y, int h) __attribute__((always_inline)) { return __builtin_amdgcn_exp2f((y - stats[2 * h]) * p.scale_log2e) * stats[2 * h + 1]; };
    if (j + 4 <= len) {
        f32x4_t w = {0, 0, 0, 0};
        if (p.weights_in) w = *(const f32x4_any*)(p.weights_in + sums);
        f32x4_t sum = {0, 0, 0, 0};
#pragma unroll 4
        for (int h = 0; h < p.group; h++) {
            const f32x4_t y = *(const f32x4_any*)(scores + (size_t)h * p.max_seq);
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += part(y[e], h);
        }
        *(f32x4_any*)(p.weights_out + sums) = w + sum;
        return;
    }
    for (int e = 0; j + e < len; e++) {
        float sum = 0.0f;
        for (int h = 0; h < p.group; h++) sum += part(scores[(size_t)h * p.max_seq + e], h);
        p.weights_out[sums + e] = (p.weights_in ? p.weights_in[sums + e] : 0.0f) + sum;
    }
}

template <int D, bool Q4, bool kWeigh>
hipError_t launch_attend_as(hipStream_t stream, const CacheAttendParams& p) {
    const dim3 grid(p.n_groups), block(64 * kWaves);
    if (p.rows <= 4) hipLaunchKernelGGL((cache_attend_kernel<D, Q4, 4, kWeigh>), grid, block, 0, stream, p);
    else if (p.rows <= 8) hipLaunchKernelGGL((cache_attend_kernel<D, Q4, 2, kWeigh>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((cache_attend_kernel<D, Q4, 1, kWeigh>), grid, block, 0, stream, p);
    if (kWeigh && p.max_seq > 0)
        hipLaunchKernelGGL(cache_weigh_kernel, dim3((p.max_seq + 1023) / 1024, p.kv_heads, p.batch), dim3(256), 0, stream, p);
    return hipGetLastError();
}
template <bool Q4, bool kWeigh>
hipError_t launch_attend(hipStream_t stream, const CacheAttendParams& p, int dim) {
    return dim == 64 ? launch_attend_as<64, Q4, kWeigh>(stream, p) : dim == 128 ? launch_attend_as<128, Q4, kWeigh>(stream, p) : launch_attend_as<256, Q4, kWeigh>(stream, p);
}

// Segments, steps and workgroups of a call at its longest, and what its workspace holds.
struct AttendPlan {
    int64_t rows, n_tiles, segments, steps;
    int groups, part_rows;
    size_t part_bytes, word_bytes, score_bytes, stat_bytes;
    size_t bytes() const { return part_bytes + word_bytes + score_bytes + stat_bytes; }
};
// Workgroups a CU, each with a wave on every SIMD: two steps under way a wave keep the memory busy with few waves, and each more is a
// span more to start and to join.  4-bit rows, a CU with 1 / 2 / 3 / 4: dim 128, 64 sequences of 512 .. 8192 keys 78 / 67 / 70 / 77 us, one
// with 16 query rows a head 19.5 / 20.4 / 25.5 / 25.5, 8 such 76 / 63 / 72 / 68; dim 256, 16 sequences of 8192 61 / 65 / 74 / 69;
// dim 64, 64 of 4096 43 / 29 / 34 / 34, but 16 of 37 .. 3001 19.2 / 16.5 / 17.5 / 15.5 and 256 of up to 300 38 / 27 / 24 / 24, where the starts of
// sequences count for more: two where they are of kLong steps on average, else four.  bf16 rows: dim 64, 16 sequences of 4000
// 32.2 / 30.4 / - / 31.4; dim 128 63.2 / 64.1 / 67.6.
constexpr int per_cu(int64_t dim, bool q4) { return q4 ? (dim == 64 ? 4 : dim == 128 ? 2 : 1) : dim == 64 ? 2 : 1; }
// (q4: the same workspace serves either kind of cache, so it is sized for the one with more workgroups)
AttendPlan plan_attend(int64_t batch, int64_t seq_new, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_seq, bool weigh, bool q4 = true) {
    AttendPlan a{};
    a.rows = seq_new * (heads / kv_heads);
    a.n_tiles = (a.rows + 15) / 16;
    a.segments = batch * kv_heads * a.n_tiles;
    a.steps = a.segments * ((max_seq + kStep - 1) / kStep + kStart);
    a.groups = (int)std::min<int64_t>(kCus * per_cu(dim, q4), std::max<int64_t>((a.steps + kWaves - 1) / kWaves, 1));
    a.part_rows = (int)std::min<int64_t>(16, a.rows);
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    a.part_bytes = round(((size_t)a.groups + (size_t)a.segments) * (size_t)a.part_rows * (size_t)(dim + 2) * 4);
    a.word_bytes = (size_t)a.segments * kWordPitch;
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
    const int groups = plan_attend(p.batch, p.seq_new, p.heads, p.kv_heads, head_dim, p.max_seq, weigh, q4).groups;
    if (a.steps + a.segments > 0x7fffffffll - 65536 || p.max_seq > (1 << 29) || (int64_t)p.seq_new * p.heads * head_dim > 0x7fffffffll) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (!p.q || !p.out || (weigh && (!p.weights_out || !p.kv_lens)) || (p.max_seq > 0 && (!p.k || !p.v || (q4 && (!p.k_pairs || !p.v_pairs)))))
        return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.out) & 15) return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "q, out and the caches must be 16-byte aligned");
    const size_t sum_bytes = (size_t)p.batch * p.kv_heads * p.max_seq * 4;
    if (weigh && p.weights_in != p.weights_out && overlap(p.weights_in, p.weights_in ? sum_bytes : 0, p.weights_out, sum_bytes))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "weights_out must be weights_in or share no memory with it");
    const size_t need = a.bytes();
    if (!workspace || workspace_bytes < need)
        return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, need, workspace ? workspace_bytes : 0, "workspace too small");
    if ((uintptr_t)workspace & 15) return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, 16, (uint64_t)((uintptr_t)workspace & 15), "workspace must be 16-byte aligned");
    int rc = ensure_device(err);
    if (rc) return rc;
    p.group = p.heads / p.kv_heads;
    p.rows = (int)a.rows;
    p.n_tiles = (int)a.n_tiles;
    p.n_groups = groups;
    p.n_long = q4 && head_dim == 64 ? std::min(groups, 2 * kCus) : groups;
    // Of four rows a piece's partial is short and is worth fewer steps than of sixteen.  us for 0.5 / 0.66 / 1 / 1.4 times the root, one sequence: 32 heads
    // on 8 of 128, 2048 keys 8.9 / 8.9 / 9.6 / 10.3, 8192 12.7 / 11.7 / 11.4 / 12.8, 32768 18.7 / 18.6 / 18.8 / 18.9; 16 heads of 64, 16384 keys
    // 12.1 / 12.1 / 12.8 / 13.6.  More rows, 8192 keys at dim 128: 8 rows 14.4 / 12.6 / 12.4 / 13.9, 16 18.6 / 15.7 / 14.9 / 16.5, 17 16.1 / 15.3 / 14.7 / 16.3,
    // 64 19.3 / 19.3 / 19.3 / 21.5.
    p.span_root = a.rows <= 4 ? 0.66f : 1.0f;
    p.scale_log2e = (1.0f / sqrtf((float)head_dim)) * kLog2eHost;
    p.part = (float*)workspace;
    p.part_rows = a.part_rows;
    p.words = (unsigned char*)workspace + a.part_bytes;
    p.launch_id = next_launch_id() << 8;
    p.scores = (float*)(p.words + a.word_bytes);
    p.stats = (float*)(p.words + a.word_bytes + a.score_bytes);
    const hipStream_t s = (hipStream_t)stream;
    const hipError_t e = !q4 ? launch_attend<false, true>(s, p, head_dim) : weigh ? launch_attend<true, true>(s, p, head_dim) : launch_attend<true, false>(s, p, head_dim);
    HIP_TRY(e, "cache_attend launch");
    return RT_OK;
}

size_t attend_bytes(int32_t batch, int32_t seq_new, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t max_seq, bool weigh) {
    if (batch <= 0 || seq_new <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || !cache_q4_dim(head_dim) || max_seq < 0) return 0;
    const AttendPlan a = plan_attend(batch, seq_new, n_heads, n_kv, head_dim, max_seq, weigh);
    return a.bytes();
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
