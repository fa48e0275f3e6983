// A decode step over a cache in pages, for a batch that may share a prefix:
//
//   out_b = softmax(q_b K_b^T / sqrt(dim)) V_b        K_b = [the prefix's rows; the sequence's own], looked up page by page
//
// A wave walks steps of 32 keys of one kv head by the matrix cores, both products transposed as in decode_cache.hip: scores^T = K q^T
// leaves a lane with the scores of ONE query row for eight keys, which is the operand that out^T = V^T P^T takes, so that nothing of
// a step crosses lanes but the running maximum.  A step's two sixteens of rows lie in a page each, whose place is looked up ahead; K
// and V come through descriptors that end with the last key's row, so that rows behind it are zeros and are not read.
//
// A sequence's own keys meet the up to sixteen query rows of one kv head, through registers.  The prefix's keys meet those of the whole
// batch, through LDS: the waves of a workgroup have 32 query rows each, of the sequences that share the prefix, in the larger matrix
// instruction's layout, and walk the same keys, which come straight to LDS once for all four (each wave with steps of its own through
// registers, sixteen rows an instruction: 36 us for 64 sequences behind 8192 keys alone, at 15 TB/s from the L2s).
// Both kinds of segments, (kv head, tile) of the prefix and (sequence, kv head), form one list of steps that is cut into equal
// spans, one a workgroup of four waves, which deal the steps of a segment among themselves and fold what they have through LDS.  What a
// workgroup finishes of a sequence it writes at once, where that is all there is; otherwise it leaves a partial (o, m, l).  Without a
// prefix the workgroup that finishes a sequence's kv head last folds its partials.  With one every sequence has at least two, and a
// prefix's tile is waited for by all of its sequences: there a second launch folds them, side by side.
//
// The weights meet V as one bf16 each, rounded to nearest, as in the prefill kernels: off by up to 2^-8 of a weight, and errors of many keys
// cancel (0.0023 of an output's size against 64 bits, 0.0017 where only the output is rounded).
//
// Bound: HBM; latency where there are few keys.  32 heads on 8 of 128: 64 sequences of 512 to 8192 keys 182 us, 6.3 TB/s; 1 of 2048 8.7 us; 64 of
// 8200 to 8704 of which 8192 are shared 37.8 us, 103 MB.
#include <algorithm>
#include <type_traits>

#include "cache_paged.hpp"
#include "flash_tile_lds.hpp"
#include "rt_common.hpp"
#include "rt_host.hpp"
#include "rt_kernels.hpp"

namespace rt {

namespace {

constexpr int kStep = 32;   // keys a step
constexpr int kWaves = 4;   // a workgroup
constexpr int kCus = 256;
constexpr int kMaxPieces = 256;  // partials of a sequence's kv head: half of the prefix, half of its own keys, or all of its own
// Maxima are of scores as the products leave them, and a weight is 2^((score - maximum) log2(e) / sqrt(dim)): scaled first, two scores of 2^31 that
// are the same would be a rounding of the scaled one apart, whose power of two is infinite or zero.
// The maximum of keys whose scores are all -infinity, which no finite score lies below; of no keys it is -infinity.  Where neither has a weight the one gives
// NaN, as the exponentials of -infinity less itself do, the other zeros.
constexpr float kNoMax = -__FLT_MAX__;
__device__ __forceinline__ float weight_of(float m, float top, float scale_log2e) { return __builtin_amdgcn_exp2f((m - (top == neg_inf() ? 0.0f : top)) * scale_log2e); }
__device__ __forceinline__ float inverse(float l, float top) { return l != 0.0f ? 1.0f / l : top == neg_inf() ? 0.0f : quiet_nan(); }
typedef float f32x2p __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2p __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {  // to nearest even
    const f32x2p x = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2p));
}
// x / d for 0 <= x < 2^31, 0 < d, by a reciprocal in f32 and what it is off by
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

// ---- over lanes, within registers (the steps of a prefix sum are those of cache_q4.hpp) ------------------------------------
template <int kStepNo>
__device__ __forceinline__ int lanes_from(int none, int x) {
    constexpr int kCtrl[6] = {0x111, 0x112, 0x114, 0x118, 0x142, 0x143}, kRows[6] = {0xf, 0xf, 0xf, 0xf, 0xa, 0xc};
    return __builtin_amdgcn_update_dpp(none, x, kCtrl[kStepNo], kRows[kStepNo], 0xf, false);
}
__device__ __forceinline__ int lane_sums(int x) {  // up to and with this lane
    x += lanes_from<0>(0, x);
    x += lanes_from<1>(0, x);
    x += lanes_from<2>(0, x);
    x += lanes_from<3>(0, x);
    x += lanes_from<4>(0, x);
    x += lanes_from<5>(0, x);
    return x;
}
__device__ __forceinline__ int lane_max(int x) {
    x = max(x, lanes_from<0>(x, x));
    x = max(x, lanes_from<1>(x, x));
    x = max(x, lanes_from<2>(x, x));
    x = max(x, lanes_from<3>(x, x));
    x = max(x, lanes_from<4>(x, x));
    x = max(x, lanes_from<5>(x, x));
    return __builtin_amdgcn_readlane(x, 63);
}
// of the four lanes of a query row (rows of 16 lanes swapped, then halves of the wave)
template <typename F>
__device__ __forceinline__ float over_quads(float x, F f) {
    const u32x2_t a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const u32x2_t c = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return f(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ __forceinline__ float quad_max(float x) {
    return over_quads(x, [](float a, float b) __attribute__((always_inline)) { return fmaxf(a, b); });
}
__device__ __forceinline__ float quad_sum(float x) {
    return over_quads(x, [](float a, float b) __attribute__((always_inline)) { return a + b; });
}
// of a row of sixteen lanes, in every one of them
template <int kBy>
__device__ __forceinline__ float turned(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + kBy, 0xf, 0xf, true));
}
__device__ __forceinline__ float sixteen_max(float x) {
    x = fmaxf(x, turned<8>(x));
    x = fmaxf(x, turned<4>(x));
    x = fmaxf(x, turned<2>(x));
    return fmaxf(x, turned<1>(x));
}
__device__ __forceinline__ float sixteen_sum(float x) {
    x += turned<8>(x);
    x += turned<4>(x);
    x += turned<2>(x);
    return x + turned<1>(x);
}

// ---- the list that the workgroups share -----------------------------------------------------------------------------------
// Of every segment kStart places, which stand for what it costs besides its steps, and its steps; of a prefix's step kPreCost places.
// us, 4 / 8 / 16 / 24 places a start, the next segment's rows being asked for ahead of a fold: 256 sequences of 100 to 700 keys 81.7 / 82.5 / 84.9 /
// 88.1, 32 of 100 to 900 without groups 20.7 / 19.4 / 21.1 / 23.0, 64 behind 8192 43.0 / 42.3 / 43.5 / 48.3, 4 of 1000 to 4000 15.0 / 13.9 / 13.9
// / -, 16 of 500 to 4000 on 2 kv heads 18.4 / 16.2 / 16.2 / 16.1.  1 / 2 / 3 places a prefix's step: 64 behind 8192 48.8 / 42.3 / 45.0, 32
// behind 4096 26.3 / 22.8 / 25.9, 128 behind 1000 40.9 / 31.4 / 28.3, 16 behind 2000 19.9 / 18.2 / 22.1.
constexpr int kStart = 8, kPreCost = 2;
__device__ __forceinline__ int steps_up_to(int key) { return (key + kStep - 1) / kStep; }
struct Own {  // a sequence's own keys
    int len, lo;  // [lo, len); lo: the prefix's length where it shares it, else 0
    __device__ __forceinline__ Own(int n, int shared) : len(n), lo(n >= shared ? shared : 0) {}
    __device__ __forceinline__ int first() const { return lo / kStep; }
    __device__ __forceinline__ int steps() const { return len > lo ? steps_up_to(len) - first() : 0; }
    __device__ __forceinline__ int places() const { return len > lo ? steps() + kStart : 0; }
};
__device__ __forceinline__ int len_of(const PagedDecodeParams& p, int b) { return min(max(p.kv_lens[b], 0), p.max_len); }

struct Span {
    int total, size;     // places of all; of a span
    int shared, owner;   // the prefix's length; 0: nobody shares one.  The sequence whose pages of it are read
    int pre_places;      // places of a (kv head, tile) of the prefix
    int pre_total;       // of all of them
    int b, first, len;   // the sequence that holds the span's first place, where it starts, its length
    uint64_t empty;      // of the first 64 sequences, those without keys
    int begin, end;
};
// The span of `group`, of workgroups that are numbered as they come.  A prefix's tiles read the same keys: their spans go to workgroups of
// one XCD, an eighth of the list each.
template <bool kShared>
__device__ __forceinline__ Span span_of(const PagedDecodeParams& p, int& group, int lane) {
    const int per = p.kv_heads * p.chunks;
    Span s;
    s.shared = !kShared ? 0 : min(max(p.shared_lens ? *(const __attribute__((address_space(4))) int32_t*)p.shared_lens : p.shared_len, 0), p.max_len);
    auto len_at = [&](int b0) { return b0 + lane < p.batch ? len_of(p, b0 + lane) : -1; };  // (behind the last: no sequence)
    auto places = [&](int len) { return len < 0 ? 0 : Own(len, s.shared).places(); };
    const int len0 = len_at(0), ends0 = lane_sums(places(len0));
    s.empty = __ballot(len0 == 0);
    int sum = __builtin_amdgcn_readlane(ends0, 63), most = lane_max(len0 < 0 ? 0 : Own(len0, s.shared).steps());
    auto sharer = [&](int len, int b0) {  // the first of 64 that has the prefix
        const uint64_t have = __ballot(len >= s.shared);
        return have ? b0 + __ffsll((unsigned long long)have) - 1 : -1;
    };
    s.owner = kShared ? sharer(len0, 0) : -1;
    for (int b0 = 64; b0 < p.batch; b0 += 64) {
        const int len = len_at(b0);
        sum += __builtin_amdgcn_readlane(lane_sums(places(len)), 63);
        most = max(most, lane_max(len < 0 ? 0 : Own(len, s.shared).steps()));
        if (kShared && s.owner < 0) s.owner = sharer(len, b0);
    }
    if (s.owner < 0) s.shared = 0;  // (then every `lo` was 0 already)
    s.pre_places = s.shared > 0 ? kStart + steps_up_to(s.shared) * kPreCost : 0;
    s.pre_total = s.pre_places * p.kv_heads * p.n_tiles;
    most = max(most, s.pre_places);
    s.total = s.pre_total + sum * per;
    // what one of all workgroups gets, but no fewer than a join is worth (a segment of few spans is a long walk, one of many a long join:
    // their sum is least around the root of its steps: span_root), and never more of them than a sequence may have
    const int pieces = s.shared > 0 ? kMaxPieces / 2 : kMaxPieces;
    const int root = __builtin_amdgcn_readfirstlane((int)(__builtin_amdgcn_sqrtf((float)most) * p.span_root + 0.5f * kWaves)) & -kWaves;
    s.size = max(max(kWaves, quotient(s.total + p.n_groups - 1, p.n_groups)), max(root, (most + pieces - 3) / (pieces - 2)));
    // more workgroups than CUs, but not about two for each: one for each, and spans that its waves share evenly (us, 1 sequence of 30000 keys
    // 31.4 -> 27.0, 4 of 1000 to 4000 15.0 -> 13.9, 16 behind 2000 20.5 -> 18.1; heads of 32 on 8 of 128)
    if (s.total < s.size * (p.n_groups / 8 * 7) && s.total > s.size * kCus) s.size = (quotient(s.total + kCus - 1, kCus) + kWaves - 1) & -kWaves;
    // long spans of dims 65 to 128 without a prefix: one for each too (us, two / one: 64 sequences of 512 to 8192 190.4 / 185.0, 512 of 100 to 1000 206 /
    // 198, 16 of 8000 100.8 / 98.5, of dim 96 79.8 / 78.7; but 64 without groups of 64 122 / 158; 64 of 200 to 512, spans of 19 places, 26.0
    // / 26.4)
    else if (!kShared && p.dim > 64 && p.dim <= 128 && s.size >= 32 && s.total > s.size * kCus) s.size *= 2;
    if (s.shared > 0) {
        const int active = quotient(s.total + s.size - 1, s.size), eighth = (active + 7) / 8;  // (n_groups divides by eight)
        group = group / 8 < eighth ? (group & 7) * eighth + group / 8 : 0x7fffffff;
    }
    s.b = s.first = s.len = 0;
    const long long at = (long long)group * s.size;
    s.begin = (int)min(at, (long long)s.total);
    s.end = (int)min((long long)s.total, at + s.size);
    if (s.begin >= s.total) return s;
    // the first sequence that has a place from `begin` on
    int before = s.pre_total, len = len0, ends = ends0;
    for (int b0 = 0;;) {
        const uint64_t past = __ballot(before + ends * per > max(s.begin, s.pre_total));
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s.b = b0 + l;
            s.len = __builtin_amdgcn_readlane(len, l);
            s.first = before + (__builtin_amdgcn_readlane(ends, l) - Own(s.len, s.shared).places()) * per;
            return s;
        }
        before += __builtin_amdgcn_readlane(ends, 63) * per;
        b0 += 64;
        if (b0 >= p.batch) return s;  // (a list of prefixes alone)
        len = len_at(b0);
        ends = lane_sums(places(len));
    }
}

// ---- partials: device scope both ways, as in decode_cache.hip.  (Where a second launch reads them they need none; without it 64 sequences
// behind 8192 keys took 44.5 us instead of 43.6.) ----------------------------------------------------------------------------------
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

// The word through which the workgroups of a (sequence, kv head, piece of its heads) learn which of them is the last: (launch id | count).
// It lies in the caller's workspace, which holds anything: every workgroup makes sure, ahead of its own count, that the word carries this
// launch's id.  The last one leaves 0 there, so that a recorded launch, which brings its id along on every replay, finds none of its own
// counts.  With a prefix the same line holds where the sequence's own partials are, for the launch that folds them.
typedef unsigned long long word_t;
constexpr int kWordPitch = 128;  // bytes: atomics on one line wait for each other
constexpr word_t kCountMask = 0xffff;
struct UnitWord {
    word_t* at;
    word_t id, seen, got;
    __device__ __forceinline__ bool ours(word_t x) const { return ((x ^ id) & ~kCountMask) == 0; }
    // what is there, asked for ahead of the rows; it is replaced behind their requests, and whether that has held is looked at ahead of
    // the count: neither is waited for by itself
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
// What the first launch leaves for the second: of the list, and of a unit's line.
struct ListHead {
    int size, shared, pre_places;
};
struct UnitLine {
    int w0, pieces;  // of its own keys' partials; none: pieces 0.  One alone, and no prefix: written already, pieces -1
};
__device__ __forceinline__ void* word_of(const PagedDecodeParams& p, int seq, int kvh, int piece) {
    return p.words + (((size_t)seq * p.kv_heads + kvh) * p.chunks + piece) * kWordPitch;
}

// ---- partials ----------------------------------------------------------------------------------------------------------------
// Slots of the prefix's come first, one a wave of a piece, then those of the sequences'.  A piece's number is (workgroup + segment): along
// the list each further piece advances one or the other.  A sequence's slot: rows of D floats, then their (m, l).  A wave's: o as the
// registers hold it, 16 bytes a lane and request, then the rows' (m, l).
constexpr int kWaveRows = 32;
template <int D>
struct Slots {
    static constexpr uint32_t kWave = (uint32_t)kWaveRows * (D + 2) * 4, kPre = kWaves * kWave;
    char *pre, *own;
    uint32_t own_bytes;
    __device__ __forceinline__ Slots(const PagedDecodeParams& p, bool shared)
        : pre((char*)p.part), own((char*)p.part + (shared ? (size_t)(p.n_groups + p.kv_heads * p.n_tiles) * kPre : 0)), own_bytes((uint32_t)p.rows * (D + 2) * 4) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t of_pre(int w0, int segment, int n) const { return rsrc_of(pre + ((size_t)w0 + segment) * kPre, (uint32_t)n * kPre); }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t of_own(int w0, size_t segment, int n) const { return rsrc_of(own + ((size_t)w0 + segment) * own_bytes, (uint32_t)n * own_bytes); }
    // Byte, in a wave's slot, of four dims from d on of row `row`; of its (m, l).
    static __device__ __forceinline__ uint32_t at(int row, int d) {  // lane (row, d / 4 % 2) has eight dims' half, d / 8 by d / 8
        return (uint32_t)(d / 8 * 1024 + ((d / 4 & 1) * 32 + row) * 16);
    }
    static __device__ __forceinline__ uint32_t at_ml(int row) { return (uint32_t)(kWaveRows * D * 4 + 8 * row); }
};
// Four dims of a row of the output.
__device__ __forceinline__ void put_out(const PagedDecodeParams& p, int dim, int seq, int head, int d, f32x4_t o) {
    if (d < dim) *(u32x2_t*)(p.out + ((size_t)seq * p.heads + head) * dim + d) = u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}
constexpr int kThreads = 64 * kWaves;
constexpr int join_lds(int pieces, int rows) { return kThreads * 16 + pieces * rows * 8; }
// All partials of `rows` heads from `head` on of sequence `seq`, by the whole workgroup: n_pre of the prefix, wave pre_wave's,
// rows of theirs from pre_row on, and n_own.  Items of four elements, kAhead pieces of each at a time (4 for 8: fewer registers, and
// fewer requests for nothing: 256 sequences behind 500 keys 69.3 -> 65.9 us, 8 of 2000 to 4000 of 64 15.9 -> 14.8); where there are
// fewer items than threads, several threads an item, each with every sub-th piece.  The first are asked for ahead of the (m, l) that
// their weights are made of.
template <int D, bool kShared>
__device__ __forceinline__ void join(const PagedDecodeParams& p, unsigned char* lds, float* inv_l, int dim, int seq, int head, int rows, __amdgpu_buffer_rsrc_t pre, int n_pre, int pre_wave, int pre_row, __amdgpu_buffer_rsrc_t own, int n_own) {
    constexpr int kAhead = 4, NT = kThreads, kMost = kMaxPieces;
    auto pre_at = [&](int k) __attribute__((always_inline)) { return (uint32_t)k * Slots<D>::kPre + (uint32_t)pre_wave * Slots<D>::kWave; };
    const uint32_t own_slot = (uint32_t)p.rows * (D + 2) * 4;
    f32x4_t* const part = (f32x4_t*)lds;
    float* const wgt = (float*)(part + NT);  // [pieces][p.rows]
    float* const wl = wgt + kMost * p.rows;
    const int tid = threadIdx.x, pieces = n_pre + n_own, items = rows * (D / 4), sub_n = items >= NT ? 1 : NT / items;
    const int x0 = sub_n == 1 ? tid : tid % items, sub = sub_n == 1 ? 0 : tid / items;
    f32x4_t a[kAhead];
    auto ask = [&](int i, int k0) __attribute__((always_inline)) {  // (row and element follow one another in a slot)
        const int it = min(i, items - 1);
        const uint32_t from = 16u * (uint32_t)it, from_pre = Slots<D>::at(pre_row + it / (D / 4), 4 * (it % (D / 4)));
#pragma unroll
        for (int e = 0; e < kAhead; e++) {
            const int k = min(k0 + e * sub_n, pieces - 1);
            a[e] = kShared && k < n_pre ? get4(pre, pre_at(k) + from_pre) : get4(own, (uint32_t)(k - n_pre) * own_slot + from);
        }
    };
    ask(x0, sub);
    {
        for (int x = tid; x < pieces * p.rows; x += NT) {
            const int k = x / p.rows, row = x - k * p.rows;
            const u32x2_t ml = kShared && k < n_pre ? get2(pre, pre_at(k) + Slots<D>::at_ml(pre_row + row))
                                                    : get2(own, (uint32_t)(k - n_pre) * own_slot + 4u * (uint32_t)(p.rows * D + 2 * row));
            wgt[x] = __uint_as_float(ml[0]);
            wl[x] = __uint_as_float(ml[1]);
        }
        __syncthreads();
        const int row = tid >> 4, col = tid & 15;  // sixteen lanes a row
        const bool on = row < rows;
        float top = neg_inf(), sum = 0.0f;
        for (int k = col; on && k < pieces; k += 16) top = fmaxf(top, wgt[k * p.rows + row]);
        top = sixteen_max(top);
        for (int k = col; on && k < pieces; k += 16) {
            const float fk = weight_of(wgt[k * p.rows + row], top, p.scale_log2e);
            wgt[k * p.rows + row] = fk;
            sum += wl[k * p.rows + row] * fk;
        }
        sum = sixteen_sum(sum);
        if (on && col == 0) inv_l[row] = inverse(sum, top);
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
                if (k0 + e * sub_n < pieces) o += a[e] * wgt[(k0 + e * sub_n) * p.rows + row];
        }
        if (sub_n > 1) {  // (one round)
            part[tid] = o;
            __syncthreads();
            if (on && sub == 0)
                for (int e = 1; e < sub_n; e++) o += part[e * items + tid];
        }
        if (on && sub == 0) put_out(p, dim, seq, head + row, d, o * inv_l[row]);
    }
}

// ---- what a lane holds of 32 keys ------------------------------------------------------------------------------------------
// As an operand of scores^T, keys are rows: lane (n, quad) has key n of either sixteen, and a quarter of each 32 dims.  As an operand of
// out^T, dims are rows and keys the products' inner index: lane (n, quad) has dims by n of the eight keys 4 quad + {0..3}, 16 + those, in the
// order in which scores^T leaves their weights.
//
// Up to four or eight query rows leave most of the sixteen columns of a product idle.  (Those columns put to use for the exponentials of the
// rows, with zeros in each other's weights, as decode_cache.hip does where codes have to be unpacked first, was no shorter: 64 sequences of 512
// to 8192 keys 189.3 us for 188.1, one of 2048 9.8 for 9.2, 16 heads of 64 without groups 25.1 for 24.9.)
template <int D>
struct Keys {
    uint32_t k[2][D / 8], v[8][D / 32];
};
// Byte offsets of a lane's requests from the first row of a sixteen.  kWhole: dim is D; else what lies behind a row's end is behind the
// descriptor's too.
constexpr uint32_t kNowhere = 0x80000000u;
template <int D, bool kWhole>
struct Lanes {
    static constexpr int kK = kWhole ? 1 : D / 32, kV = kWhole || D < 256 ? 1 : 2;
    uint32_t k[kK], v[4][kV];
    __device__ __forceinline__ Lanes(int n, int quad, uint32_t row_bytes) {
#pragma unroll
        for (int c = 0; c < kK; c++) k[c] = kWhole || 64u * c + 16u * quad < row_bytes ? n * row_bytes + 64u * c + 16u * quad : kNowhere;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int i = 0; i < kV; i++) {
                const uint32_t at = 256u * i + (D == 64 ? 8u : 16u) * n;
                v[e][i] = kWhole || at < row_bytes ? (4u * quad + e) * row_bytes + at : kNowhere;
            }
    }
};

// A walk over the keys [lo, hi) of one kv head of one sequence's pages, the wave's steps first, first + stride, ... below `end`.
template <int D, bool kWhole>
struct Walk {
    const PagedDecodeParams& p;
    const uint32_t row_bytes, page_bytes;
    const int32_t* table;  // the sequence's
    int lo, hi, first, end, stride, lane;
    const char *k_head, *v_head;  // the kv head's first row in page 0
    int entry[2];  // lane i: the pages of the two sixteens of the wave's i-th step from the last refill on
    __amdgpu_buffer_rsrc_t ks[2], vs[2];
    uint32_t seen;  // of the step whose place was taken last: a bit for every key that is there

    __device__ __forceinline__ Walk(const PagedDecodeParams& params, int every, int l)
        : p(params), row_bytes(2u * (uint32_t)(kWhole ? D : params.dim)), page_bytes(((uint32_t)params.kv_heads << params.page_shift) * row_bytes), stride(every), lane(l) {}
    __device__ __forceinline__ void over(const int32_t* row, int kv_head, int from, int to, int step0, int step1) {
        table = row;
        lo = from;
        hi = to;
        first = step0;
        end = step1;
        k_head = (const char*)p.k_pages + ((size_t)kv_head << p.page_shift) * row_bytes;
        v_head = (const char*)p.v_pages + ((size_t)kv_head << p.page_shift) * row_bytes;
    }
    // entries from step t on, and what has to stand between the request and the first use.  (Awaited there: behind a branch that requests
    // stand in, the compiler would wait in every step for whatever is under way.)
    __device__ __forceinline__ void request_entries(int t) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const long long row = ((long long)t + stride * lane) * kStep + 16 * h;
            entry[h] = table[(int)min(row >> p.page_shift, (long long)p.table_pages - 1)];
        }
    }
    __device__ __forceinline__ void await_entries() { asm volatile("" : "+v"(entry[0]), "+v"(entry[1])); }
    // The descriptors of step t, the wave's i-th.  (What they are made of is said to be the same in all lanes, which the compiler does not
    // see: it would ask for each lane's descriptor by itself.)
    __device__ __forceinline__ void place(int t, int i) {
        if (i && (i & 63) == 0) {
            request_entries(t);
            await_entries();
        }
        const int row = t * kStep;
        const uint32_t mask = (1u << p.page_shift) - 1;
        int rows[2], skip[2] = {0, 0};
        uint64_t at[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(entry[h], i & 63);
            const bool there = page < (uint32_t)p.n_pages;
            at[h] = (uint64_t)(there ? page : 0u) * page_bytes + (((uint32_t)row + 16u * h) & mask) * row_bytes;
            rows[h] = there ? 16 : 0;
        }
        seen = (rows[0] ? 0xffffu : 0u) | (rows[1] ? 0xffff0000u : 0u);
        if (row < lo || row + kStep > hi) {  // the first or last step of a sequence
            seen = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                rows[h] = min(max(hi - row - 16 * h, 0), rows[h]);
                skip[h] = min(max(lo - row - 16 * h, 0), 16);
                seen |= (((1u << rows[h]) - 1) & ~((1u << skip[h]) - 1)) << (16 * h);
            }
            seen = (uint32_t)__builtin_amdgcn_readfirstlane((int)seen);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at[h] >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at[h]);
            const uint32_t bytes = (uint32_t)__builtin_amdgcn_readfirstlane(rows[h]) * row_bytes;
            ks[h] = rsrc_of(k_head + from, bytes);
            vs[h] = rsrc_of(v_head + from, bytes);
        }
    }
    // The same of one of the two sixteens, as scalars, for rows that go to LDS; `seen` of both.  (lo is 0.)
    u32x4_t ring_k, ring_v;
    __device__ __forceinline__ void place_half(int t, int i, int h) {
        if (i && (i & 63) == 0) {
            request_entries(t);
            await_entries();
        }
        const int row = t * kStep;
        const uint32_t mask = (1u << p.page_shift) - 1;
        const uint32_t page0 = (uint32_t)__builtin_amdgcn_readlane(entry[0], i & 63), page1 = (uint32_t)__builtin_amdgcn_readlane(entry[1], i & 63);
        const int rows0 = page0 < (uint32_t)p.n_pages ? min(max(hi - row, 0), 16) : 0, rows1 = page1 < (uint32_t)p.n_pages ? min(max(hi - row - 16, 0), 16) : 0;
        seen = (uint32_t)__builtin_amdgcn_readfirstlane((int)(((1u << rows0) - 1) | ((1u << rows1) - 1) << 16));
        const int rows = h ? rows1 : rows0;
        const uint64_t at = (uint64_t)(rows ? h ? page1 : page0 : 0u) * page_bytes + (((uint32_t)row + 16u * h) & mask) * row_bytes;
        ring_k = make_rsrc(k_head + at, (uint32_t)rows * row_bytes);
        ring_v = make_rsrc(v_head + at, (uint32_t)rows * row_bytes);
    }
    __device__ __forceinline__ void load_k(Keys<D>& x, const Lanes<D, kWhole>& at) const {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                *(u32x4_t*)(x.k[h] + 4 * c) = __builtin_amdgcn_raw_buffer_load_b128(ks[h], kWhole ? at.k[0] + 64u * c : at.k[kWhole ? 0 : c], 0, 0);
    }
    // Past the caches: whole lines that no other workgroup asks for, but where a kv head has more than one piece of query heads, each of which
    // reads all keys by itself (64 sequences of 4096 keys of 128, 32 heads on 2 272 MB fetched, 49.4 us, 34 on 2 538 and 77.6; 16 on 1 141 and 30.0, 40 on 1 407 and 63.8).
    __device__ __forceinline__ void load_v(Keys<D>& x, const Lanes<D, kWhole>& at) const {
        constexpr int kAux = 2;  // nt
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (D == 64) {
                *(u32x2_t*)x.v[e] = __builtin_amdgcn_raw_buffer_load_b64(vs[e / 4], at.v[e % 4][0], 0, kAux);
            } else {
#pragma unroll
                for (int i = 0; i < D / 128; i++)
                    *(u32x4_t*)(x.v[e] + 4 * i) = __builtin_amdgcn_raw_buffer_load_b128(vs[e / 4], kWhole ? at.v[e % 4][0] + 256u * i : at.v[e % 4][kWhole || D < 256 ? 0 : i], 0, kAux);
            }
        }
    }
};

// What a lane has of its query row over the keys it has walked.
template <int D>
struct State {
    float m, l;
    f32x4_t o[D / 16];
    __device__ __forceinline__ void reset() {
        m = kNoMax;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; i++) o[i] = f32x4_t{0, 0, 0, 0};
    }
};

// One step.  k_done is called behind the last use of K.
template <int D, typename KDone>
__device__ __forceinline__ void step(State<D>& st, Keys<D>& x, const u32x4_t (&q)[D / 32], KDone k_done, uint32_t seen, int quad, float scale_log2e) {
    f32x4_t a[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int c = 0; c < D / 32; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) a[h] = mfma(*(const u32x4_t*)(x.k[h] + 4 * c), q[c], a[h]);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = a[e / 4][e % 4];
    // a key that is not there has no weight, and zeros in V, whatever lies there
    if (seen != ~0u) {
        const uint32_t mine = seen >> (4 * quad);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool hid = !(mine >> (16 * (e / 4) + e % 4) & 1);
            y[e] = hid ? neg_inf() : y[e];
#pragma unroll
            for (int w = 0; w < D / 32; w++) x.v[e][w] = hid ? 0u : x.v[e][w];
        }
    }
    k_done();
    // The running maximum, common to the four lanes of a column.  It follows the scores only where they have risen by 8 in the exponent of
    // two: up to there sums of weights in f32 and weights of 8 bits are as exact, and sums are scaled once or twice a span.
    float top = y[0];
#pragma unroll
    for (int e = 1; e < 8; e++) top = fmaxf(top, y[e]);
    top = quad_max(top);
    if (__any((top - st.m) * scale_log2e > 8.0f)) {
        const float m_new = fmaxf(st.m, top), alpha = __builtin_amdgcn_exp2f((st.m - m_new) * scale_log2e);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int d = 0; d < D / 16; d++) st.o[d] *= alpha;
    }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        f[e] = __builtin_amdgcn_exp2f((y[e] - st.m) * scale_log2e);
        st.l += f[e];
    }
    u32x4_t w;  // the weights, as the operand's words
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = two_bf16(f[2 * k], f[2 * k + 1]);
#pragma unroll
    for (int d = 0; d < D / 16; d++) {  // dim n * (D / 16) + d; of 256, of the lower and of the upper 128 in turn
        u32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][d / 2], x.v[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
        st.o[d] = mfma(v, w, st.o[d]);
    }
}

// x: the first step's rows, under way.
template <int D, bool kWhole>
__device__ __forceinline__ void walk(State<D>& st, Walk<D, kWhole>& at, Keys<D>& x, const Lanes<D, kWhole>& lanes, const u32x4_t (&q)[D / 32], int quad, float scale_log2e) {
    int i = 0;
    uint32_t any = 0;
    for (int t = at.first; t < at.end; t += at.stride) {
        const uint32_t seen = at.seen;
        any |= seen;
        const bool more = t + at.stride < at.end;
        step<D>(st, x, q, [&]() __attribute__((always_inline)) {
            if (more) {
                at.place(t + at.stride, ++i);
                at.load_k(x, lanes);
            }
        }, seen, quad, scale_log2e);
        if (more) at.load_v(x, lanes);
    }
    if (!any) st.m = neg_inf();
}

// ---- the prefix: 32 query rows a wave, keys in LDS ------------------------------------------------------------------------------
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
typedef short s16x4p __attribute__((ext_vector_type(4)));
// within each group of 16 lanes, lane j gets element j % 4 of the 8 bytes that lanes 4 e + j / 4 address, e = 0 .. 3
__device__ __forceinline__ u32x2_t lds_transposed(const unsigned char* p) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4p __attribute__((address_space(3)))*)p));
}
// kStages steps of K and V, as many as two workgroups a CU leave room for, rows as wide as they are (1 KB a request), their 16-byte pieces exchanged by the row so that neither K's reads (a
// piece each of 32 rows) nor V's transposing ones (four pieces each of four rows) meet a bank twice: the layout of the tile kernel.
template <int D, bool kWhole>
struct Ring {
    using L = TileLds<D>;
    static constexpr int kOwn = 32 / kWaves, kStages = D == 64 ? 8 : 4, kRow = 2 * D, kHalf = 32 * kRow, kStage = 2 * kHalf, kPieces = D / 8;
    static constexpr int kLoads = kHalf / 1024 / kWaves;  // requests of K, and of V, a wave and step
    uint32_t lds, k_at, v_at;
    uint32_t k_from[kLoads], v_from[kLoads];
    __device__ __forceinline__ Ring(unsigned char* space, int wave, int lane, uint32_t row_bytes) : lds((uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)space) {
        const int col = lane & 31, hh = lane >> 5, j = lane & 15, g = lane >> 4 & 1, v_row = (j >> 2) + 4 * hh;
        k_at = (uint32_t)(col * kRow + 16 * (hh ^ L::swz_k(col)));
        v_at = (uint32_t)(kHalf + v_row * kRow + 16 * ((2 * g + (j >> 1 & 1)) ^ L::swz_v(v_row)) + 8 * (j & 1));
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int at = 64 * i + lane, row = kOwn * wave + at / kPieces, k_piece = at % kPieces ^ L::swz_k(row), v_piece = at % kPieces ^ L::swz_v(row);
            k_from[i] = kWhole || 16u * k_piece < row_bytes ? (uint32_t)(row & 15) * row_bytes + 16u * k_piece : kNowhere;
            v_from[i] = kWhole || 16u * v_piece < row_bytes ? (uint32_t)(row & 15) * row_bytes + 16u * v_piece : kNowhere;
        }
    }
    // the wave's rows of K and of V of the step whose descriptors `at` has
    __device__ __forceinline__ void load(const Walk<D, kWhole>& at, int stage, int wave) const {
        const uint32_t to = lds + (uint32_t)(stage * kStage + wave * (kLoads * 1024));
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            buffer_to_lds(at.ring_k, k_from[i], 0u, to + 1024u * i);
            buffer_to_lds(at.ring_v, v_from[i], 0u, to + (uint32_t)kHalf + 1024u * i);
        }
    }
};
// What a lane has of its query row, lane % 32, over the keys walked; the row's other lane has the other eight of each sixteen.
template <int D>
struct PrefixState {
    float m, l;
    f32x16_t o[D / 32];  // o[t][4 j + e]: dim 32 t + 8 j + 4 (lane / 32) + e
};
// A step of 32 keys in `stage`.  scores^T leaves the lane keys 8 (i / 4) + 4 (lane / 32) + i % 4, i < 16; eight of them in a row are the
// operand of out^T for sixteen keys, in an order of keys that the transposing reads of V follow.
template <int D, bool kWhole>
__device__ __forceinline__ void prefix_step(PrefixState<D>& st, const u32x4_t (&q)[D / 16], const Ring<D, kWhole>& ring, const unsigned char* stage, uint32_t seen, int hh, float scale_log2e) {
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = 0.0f;
    {
        u32x4_t a[D / 16];  // (all asked for ahead of the first product)
#pragma unroll
        for (int k = 0; k < D / 16; k++) a[k] = *(const u32x4_t*)(stage + (ring.k_at ^ (uint32_t)(32 * k)));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < D / 16; k++) s = mfma32(a[k], q[k], s);
    }
    u32x4_t v[D / 32][2];  // under way during the softmax
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const unsigned char* const at = stage + (ring.v_at ^ (uint32_t)(64 * t)) + 16 * u * Ring<D, kWhole>::kRow;
            const u32x2_t lo = lds_transposed(at), hi = lds_transposed(at + 8 * Ring<D, kWhole>::kRow);
            v[t][u] = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
        }
    __builtin_amdgcn_sched_barrier(0);
    if (seen != ~0u) {
        const uint32_t mine = seen >> (4 * hh);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = mine >> (8 * (i / 4) + i % 4) & 1 ? s[i] : neg_inf();
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
    const u32x2_t both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
    if (__any((top - st.m) * scale_log2e > 8.0f)) {  // (as in step())
        const float m_new = fmaxf(st.m, top), alpha = __builtin_amdgcn_exp2f((st.m - m_new) * scale_log2e);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) st.o[t][i] *= alpha;
    }
    u32x4_t w[2];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float a = __builtin_amdgcn_exp2f((s[8 * u + 2 * i] - st.m) * scale_log2e), b = __builtin_amdgcn_exp2f((s[8 * u + 2 * i + 1] - st.m) * scale_log2e);
            st.l += a + b;
            w[u][i] = two_bf16(a, b);
        }
#pragma unroll
    for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int u = 0; u < 2; u++) st.o[t] = mfma32(v[t][u], w[u], st.o[t]);
}
// All four waves over the steps [at.first, at.end), each for its own rows (`rows`: it has some).
template <int D, bool kWhole>
__device__ __forceinline__ void prefix_walk(PrefixState<D>& st, Walk<D, kWhole>& at, unsigned char* space, u32x4_t (&q)[D / 16], bool rows, int wave, float scale_log2e) {
    using R = Ring<D, kWhole>;
    const R ring(space, wave, at.lane, at.row_bytes);
    constexpr int kAhead = R::kStages - 1;  // steps under way, beside the one that is read
    const int steps = at.end - at.first, hh = at.lane >> 5;
    int seen = 0;  // lane i % 64: of step i
    uint32_t any = 0;
    auto request = [&](int i) __attribute__((always_inline)) {
        at.place_half(at.first + i, i, wave * R::kOwn / 16);
        if (at.lane == (i & 63)) seen = (int)at.seen;
        ring.load(at, i & kAhead, wave);
    };
    // the wave's requests, but for as many later steps', and its reads of the last step, whose place is overwritten behind the barrier
    auto await = [&](auto others) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(others)::value * 2 * R::kLoads) : "memory");
    };
    static_assert((R::kStages & kAhead) == 0 && (kAhead - 1) * 2 * R::kLoads < 63);
    at.request_entries(at.first);
    __syncthreads();  // (what lay in LDS before has been read)
    at.await_entries();
    // q, awaited here: within the steps the compiler, which does not know of the requests to LDS, would wait for those under way with it
#pragma unroll
    for (int k = 0; k < D / 16; k++) asm volatile("" : "+v"(q[k]));
    for (int i = 0; i < min(kAhead, steps); i++) request(i);
    for (int i = 0; i < steps; i++) {
        // this step's rows are there, if not the next ones'; behind the barrier everybody's are, and nobody reads the last step's any more
        const int left = steps - 1 - i;
        if (left >= kAhead - 1) await(std::integral_constant<int, kAhead - 1>{});
        else if (left >= kAhead / 2) await(std::integral_constant<int, kAhead / 2>{});
        else if (left >= 1) await(std::integral_constant<int, 1>{});
        else await(std::integral_constant<int, 0>{});
        if (i + kAhead < steps) request(i + kAhead);
        const uint32_t now = (uint32_t)__builtin_amdgcn_readlane(seen, i & 63);
        any |= now;
        if (rows) prefix_step<D, kWhole>(st, q, ring, space + (i & kAhead) * R::kStage, now, hh, scale_log2e);
    }
    if (!any) st.m = neg_inf();
    __syncthreads();
}

template <int D, bool kWhole, bool kShared>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void paged_decode_kernel(PagedDecodeParams p) {
    constexpr int NT = kThreads, kPitch = D + 4;
    constexpr int kFold = kWaves * 16 * kPitch * 4, kLds = kShared ? std::max(kFold, Ring<D, kWhole>::kStages * Ring<D, kWhole>::kStage) : std::max(kFold, join_lds(kMaxPieces, 16));
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kLds];
    __shared__ float red_m[kWaves][16], red_l[kWaves][16], inv_l[16];
    __shared__ int is_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, quad = lane >> 4;
    const int per = p.kv_heads * p.chunks, dim = kWhole ? D : p.dim;
    int group = blockIdx.x;
    const Span span = span_of<kShared>(p, group, lane);
    // sequences without keys, dealt to the workgroups: rows of zeros
    for (int b = blockIdx.x; b < p.batch; b += (int)gridDim.x)
        if (b < 64 ? (span.empty >> b & 1) != 0 : len_of(p, b) == 0)
            for (int i = tid; i < p.heads * (dim / 8); i += NT) *(u32x4_t*)(p.out + (size_t)b * p.heads * dim + 8 * i) = u32x4_t{0, 0, 0, 0};
    if (kShared && blockIdx.x == 0 && tid == 0) *(ListHead*)p.head = ListHead{span.size, span.shared, span.pre_places};
    if (span.begin >= span.total) return;
    int at = span.begin, b = span.b, first = span.first, len = span.len;

    const Lanes<D, kWhole> lanes(n, quad, 2u * (uint32_t)dim);
    const Slots<D> slots(p, kShared);
    float* const red = (float*)lds;  // [wave][row][kPitch]

    // A tile's rows, folded over the waves of the workgroup: to_row(row, d, values of four dims, m, l).
    auto fold = [&](State<D>& st, int rows, auto to_row, auto to_ml) __attribute__((always_inline)) {
        const float l = quad_sum(st.l);
        if (quad == 0) {
            red_m[wave][n] = st.m;
            red_l[wave][n] = l;
        }
        __syncthreads();
        float m_wg = red_m[0][n], l_wg = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; w++) m_wg = fmaxf(m_wg, red_m[w][n]);
#pragma unroll
        for (int w = 0; w < kWaves; w++) l_wg += red_l[w][n] * weight_of(red_m[w][n], m_wg, p.scale_log2e);
        if (n < rows) {
            const float fw = weight_of(st.m, m_wg, p.scale_log2e);
            float* row = red + (wave * 16 + n) * kPitch;
#pragma unroll
            for (int c = 0; c < D / 32; c++) {  // eight dims in a row
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = st.o[(8 * c + e) % (D / 16)][(8 * c + e) / (D / 16)] * fw;
                float* dst = row + (D == 256 ? 128 * (c & 1) + 32 * quad + 8 * (c >> 1) : quad * (D / 4) + 8 * c);
                *(f32x4_t*)dst = f32x4_t{y[0], y[1], y[2], y[3]};
                *(f32x4_t*)(dst + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
            }
            if (wave == 0 && quad == 0) {
                inv_l[n] = inverse(l_wg, m_wg);
                to_ml(n, m_wg, l_wg);
            }
        }
        __syncthreads();
        for (int i = tid; i < rows * (D / 4); i += NT) {
            const int row = i / (D / 4), d = 4 * (i % (D / 4));
            f32x4_t o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; w++) o += *(const f32x4_t*)(red + (w * 16 + row) * kPitch + d);
            to_row(row, d, o);
        }
        __syncthreads();
    };
    // ---- pieces of the prefix
    if constexpr (kShared) {
        const int end = min(span.end, span.pre_total);
        while (at < end) {
            const int seg = quotient(at, span.pre_places), seg_first = seg * span.pre_places, to = min(seg_first + span.pre_places, end);
            // steps whose first place is in the span
            const int t0 = (max(at - seg_first - kStart, 0) + kPreCost - 1) / kPreCost, t1 = min(steps_up_to(span.shared), (max(to - seg_first - kStart, 0) + kPreCost - 1) / kPreCost);
            at = to;
            if (to - seg_first <= kStart) continue;  // (places alone: no piece)
            const int kvh = quotient(seg, p.n_tiles), tile = seg - kvh * p.n_tiles;
            // the wave's units, (sequence, piece of the kv head's query heads): row i of them is head i % rows of unit i / rows
            const int unit0 = tile * p.per_tile + wave * p.per_wave, units = min(p.per_wave, p.batch * p.chunks - unit0), col = lane & 31, hh = lane >> 5;
            u32x4_t q[D / 16];
            {
                const int u = col / p.rows, unit = min(unit0 + u, p.batch * p.chunks - 1), seq = unit / p.chunks, h = (unit - seq * p.chunks) * p.rows + col - u * p.rows;
                const bool there = u < units && h < p.group;
                const uint16_t* q_row = p.q + ((size_t)seq * p.heads + kvh * p.group + (there ? h : 0)) * dim;
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    q[k] = *(const u32x4_t*)(q_row + (kWhole ? 16 * k + 8 * hh : min(16 * k + 8 * hh, dim - 8)));
                    if (!there || (!kWhole && 16 * k >= dim)) q[k] = u32x4_t{0, 0, 0, 0};
                }
            }
            PrefixState<D> st;
            st.m = kNoMax;
            st.l = 0.0f;
#pragma unroll
            for (int t = 0; t < D / 32; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) st.o[t][i] = 0.0f;
            Walk<D, kWhole> w(p, 1, lane);
            w.over(p.page_table + (size_t)span.owner * p.table_pages, kvh, 0, span.shared, t0, t1);
            prefix_walk<D, kWhole>(st, w, lds, q, units > 0, wave, p.scale_log2e);
            if (units <= 0) continue;  // (a wave without rows has its share of the keys' way to LDS)
            const __amdgpu_buffer_rsrc_t rs = rsrc_of(slots.pre + ((size_t)group + seg) * Slots<D>::kPre + (size_t)wave * Slots<D>::kWave, Slots<D>::kWave);
            const u32x2_t l = __builtin_amdgcn_permlane32_swap(__float_as_uint(st.l), __float_as_uint(st.l), false, false);
            if (hh == 0) put2(rs, Slots<D>::at_ml(col), st.m, __uint_as_float(l[0]) + __uint_as_float(l[1]));
#pragma unroll
            for (int t = 0; t < D / 32; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) put4(rs, (uint32_t)((4 * t + j) * 1024 + lane * 16), f32x4_t{st.o[t][4 * j], st.o[t][4 * j + 1], st.o[t][4 * j + 2], st.o[t][4 * j + 3]});
        }
        if (at >= span.end) return;
    }
    // ---- pieces of sequences' own keys.  The next one's page entries are asked for ahead of a piece's steps, its q and first rows behind
    // them and ahead of the fold.
    struct Piece {
        int b, kvh, piece, lo, hi, t0, t1, w0, pieces;
    };
    int next_len = len_of(p, min(b + 1, p.batch - 1));
    auto next = [&](Piece& x) __attribute__((always_inline)) {  // false: there is none
        while (at < span.end) {
            const Own own(len, span.shared);
            const int places = own.places();
            if (at >= first + places * per) {  // the next sequence
                first += places * per;
                b++;
                len = next_len;
                next_len = len_of(p, min(b + 1, p.batch - 1));
                continue;
            }
            const int seg = quotient(at - first, places), seg_first = first + seg * places;
            const int t0 = max(at - seg_first - kStart, 0), t1 = min(places, span.end - seg_first) - kStart;
            at = min(seg_first + places, span.end);
            if (t1 <= 0) continue;  // (places alone)
            x.b = b;
            x.kvh = p.chunks == 1 ? seg : quotient(seg, p.chunks);
            x.piece = seg - x.kvh * p.chunks;
            x.lo = own.lo;
            x.hi = len;
            x.t0 = own.first() + t0;
            x.t1 = own.first() + t1;
            x.w0 = quotient(seg_first + kStart, span.size);
            x.pieces = quotient(seg_first + places - 1, span.size) - x.w0 + 1;
            return true;
        }
        return false;
    };
    Walk<D, kWhole> w(p, kWaves, lane);
    Keys<D> x;
    u32x4_t q[D / 32];
    auto over = [&](const Piece& c) __attribute__((always_inline)) {
        w.over(p.page_table + (size_t)c.b * p.table_pages, c.kvh, c.lo, c.hi, c.t0 + wave, c.t1);
        w.request_entries(min(w.first, w.end - 1));
    };
    auto rows_of = [&](const Piece& c) { return min(p.rows, p.group - c.piece * p.rows); };  // of the kv head's query heads
    auto begin = [&](const Piece& c) __attribute__((always_inline)) {
        const int rows = rows_of(c);
        const bool there = n < rows;
        const uint16_t* q_row = p.q + ((size_t)c.b * p.heads + c.kvh * p.group + c.piece * p.rows + (there ? n : 0)) * dim;
#pragma unroll
        for (int k = 0; k < D / 32; k++) {
            q[k] = *(const u32x4_t*)(q_row + (kWhole ? 32 * k + 8 * quad : min(32 * k + 8 * quad, dim - 8)));
            if (!there || (!kWhole && 32 * k + 8 * quad >= dim)) q[k] = u32x4_t{0, 0, 0, 0};
        }
        w.await_entries();
        if (w.first < w.end) {
            w.place(w.first, 0);
            w.load_k(x, lanes);
            w.load_v(x, lanes);
        }
    };
    Piece now, then;
    bool any = next(now);
    if (any) {
        over(now);
        begin(now);
    }
    while (any) {
        const bool alone = now.pieces == 1 && now.lo == 0;
        const int rows = rows_of(now), head = now.kvh * p.group + now.piece * p.rows;
        UnitWord word;
        if (!kShared && !alone && tid == 0) word.request(word_of(p, now.b, now.kvh, now.piece), p.launch_id);
        any = next(then);
        State<D> st;
        st.reset();
        walk<D, kWhole>(st, w, x, lanes, q, quad, p.scale_log2e);
        if (!kShared && !alone && tid == 0) word.replace();
        if (any) {
            over(then);
            begin(then);
        }
        const size_t segment = ((size_t)now.b * p.kv_heads + now.kvh) * p.chunks + now.piece;
        const __amdgpu_buffer_rsrc_t rs = slots.of_own(now.w0, segment, now.pieces);
        const uint32_t to = (uint32_t)(group - now.w0) * slots.own_bytes;
        if (kShared && tid == 0) *(UnitLine*)word_of(p, now.b, now.kvh, now.piece) = UnitLine{now.w0, alone ? -1 : now.pieces};
        fold(st, rows,
             [&](int row, int d, f32x4_t o) __attribute__((always_inline)) {
                 if (alone) put_out(p, dim, now.b, head + row, d, o * inv_l[row]);
                 else put4(rs, to + 4u * (uint32_t)(row * D + d), o);
             },
             [&](int row, float m, float l) __attribute__((always_inline)) {
                 if (!alone) put2(rs, to + 4u * (uint32_t)(p.rows * D + 2 * row), m, l);
             });
        if (!kShared && !alone) {
            if (tid == 0) word.settle();
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) is_last = word.count(now.pieces) ? 1 : 0;
            __syncthreads();
            if (is_last) join<D, false>(p, lds, inv_l, dim, now.b, head, rows, rs, 0, 0, 0, rs, now.pieces);
            __syncthreads();
        }
        now = then;
    }
}

// With a prefix: a workgroup for each unit, grid (pieces of a kv head's query heads, kv heads, batch).
template <int D>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedDecodeParams p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char join_space[];  // join_lds(kMaxPieces, p.rows)
    __shared__ float inv_l[16];
    const int piece = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    // (all three at once; what a unit's line holds counts where the sequence has keys of its own)
    const ListHead list = *(const ListHead*)p.head;
    const UnitLine left = *(const UnitLine*)word_of(p, b, kvh, piece);
    const Own own(len_of(p, b), list.shared);
    if (own.len == 0) return;  // (written already)
    const UnitLine line = own.steps() > 0 ? left : UnitLine{0, 0};
    if (line.pieces < 0) return;
    const Slots<D> slots(p, true);
    const int unit = b * p.chunks + piece, tile = quotient(unit, p.per_tile), segment = kvh * p.n_tiles + tile, head = piece * p.rows;
    const int in_tile = unit - tile * p.per_tile, row_wave = quotient(in_tile, p.per_wave), pre_row = (in_tile - row_wave * p.per_wave) * p.rows;
    int w0 = 0, n_pre = 0;
    if (own.lo > 0) {
        const int first = segment * list.pre_places;
        w0 = quotient(first + kStart, list.size);
        n_pre = quotient(first + list.pre_places - 1, list.size) - w0 + 1;
    }
    join<D, true>(p, join_space, inv_l, p.dim, b, kvh * p.group + head, min(p.rows, p.group - head), slots.of_pre(w0, segment, n_pre), n_pre, row_wave, pre_row,
                  slots.of_own(line.w0, ((size_t)b * p.kv_heads + kvh) * p.chunks + piece, line.pieces), line.pieces);
}

template <int D, bool kWhole, bool kShared>
hipError_t launch_as(hipStream_t stream, const PagedDecodeParams& p) {
    const dim3 grid(p.n_groups), block(kThreads);
    hipLaunchKernelGGL((paged_decode_kernel<D, kWhole, kShared>), grid, block, 0, stream, p);
    if (kShared) hipLaunchKernelGGL(paged_join_kernel<D>, dim3(p.chunks, p.kv_heads, p.batch), block, join_lds(kMaxPieces, p.rows), stream, p);
    return hipGetLastError();
}
template <int D>
hipError_t launch_dim(hipStream_t stream, const PagedDecodeParams& p, bool shared) {
    if (p.dim == D) return shared ? launch_as<D, true, true>(stream, p) : launch_as<D, true, false>(stream, p);
    return shared ? launch_as<D, false, true>(stream, p) : launch_as<D, false, false>(stream, p);
}

// Workgroups a CU, each with a wave on every SIMD (two of one: 16 heads of 64 without groups 24.9 us, one 32.9; 64 sequences behind 8192 keys 43.3,
// 48.6; at dim 256 the registers are one's).
constexpr int per_cu(int64_t dim) { return dim == 256 ? 1 : 2; }
// Segments, steps and workgroups of a call at its longest, and what its workspace holds.
struct Plan {
    int64_t chunks, rows, per_wave, per_tile, n_tiles, own_segments, pre_segments, places;
    int dim, groups;  // dim: the kernel's
    size_t part_bytes, word_bytes;
};
Plan plan_of(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_len) {
    Plan a{};
    const int64_t group = heads / kv_heads;
    a.dim = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
    a.chunks = (group + 15) / 16;
    a.rows = (group + a.chunks - 1) / a.chunks;
    a.per_wave = kWaveRows / a.rows;
    a.per_tile = kWaves * a.per_wave;
    a.n_tiles = (batch * a.chunks + a.per_tile - 1) / a.per_tile;
    a.own_segments = batch * kv_heads * a.chunks;
    a.pre_segments = kv_heads * a.n_tiles;
    const int64_t steps = max_len / kStep + 2;
    a.places = a.own_segments * (steps + kStart) + a.pre_segments * (steps * kPreCost + kStart);
    a.groups = (int)std::min<int64_t>(2 * kCus, std::max<int64_t>((a.places + kWaves - 1) / kWaves, 1));
    a.groups = (a.groups + 7) / 8 * 8;
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    a.part_bytes = round((size_t)(a.groups + a.pre_segments) * (size_t)(kWaves * kWaveRows) * (size_t)(a.dim + 2) * 4 + (size_t)(a.groups + a.own_segments) * (size_t)a.rows * (size_t)(a.dim + 2) * 4);
    a.word_bytes = (size_t)a.own_segments * kWordPitch + 256;
    return a;
}

// A prefix that the host knows is read once where that saves enough; else each sequence reads it with its own keys, and there is no second
// launch.  What reading it once costs is that launch, a walk that is cut into pieces by the root of its steps, and partials of all rows for every
// piece: it pays from 60 MB saved and as much more as the root of steps times rows, which at dim 256, with one workgroup a CU, weighs 4.5 times as
// much.  Over 530 calls of 1 to 32 kv heads, 2 to 256 sequences, prefixes of 64 to 16000 keys and own keys of up to 1000 the way so
// chosen takes 1 % more than the shorter one in the mean, 35 % at worst (from 40 MB saved, whatever the size: 9 %, twice as long).  us, once / by each, heads,
// kv heads, dim, batch, keys (MB saved): 32 8 128 64 8192 (2114) 36 / 193; 16 16 64 24 1001 and up to 2000 own (94) 28.3 / 33.4; 28 4 128 16 4096 (126) 27.0 / 24.4, 32 1024 (65)
// 18.4 / 16.5; 32 2 128 64 4096 (264) 39 / 32, 16 4096 (63) 33.7 / 20.3; 40 1 128 64 4096 (132) 37.7 / 44.2, 1024 (33) 25.9 / 20.1; 16 2 256 16 4096 (126) 38.0 / 27.2,
// 64 4096 (528) 42.3 / 59.3, 128 1024 (266) 33.3 / 40.7; 16 16 256 16 1024 (252) 25.8 / 40.4, 4 1024 (50) 18.3 / 17.5, but 200 64 (209) 108 / 106.
bool shares(const Plan& a, int64_t batch, int64_t kv_heads, int64_t dim, int64_t keys) {
    const double saved = (double)(batch - 1) * (double)keys * (double)(kv_heads * dim * 4), steps = (double)((keys + kStep - 1) / kStep);
    return keys >= 64 && saved >= 1e6 * (60.0 + (a.dim == 256 ? 4.5 : 1.0) * sqrt(steps * (double)a.rows));
}

}  // namespace

}  // namespace rt

using namespace rt;

RT_API size_t rt_gqa_decode_paged_workspace_bytes(int32_t batch, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t page_size, int32_t table_pages) {
    if (batch <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || !cache_paged_dim(head_dim) || !cache_page_size(page_size) || table_pages < 0) return 0;
    const Plan a = plan_of(batch, n_heads, n_kv, head_dim, (int64_t)table_pages * page_size);
    return a.part_bytes + a.word_bytes;
}

RT_API int rt_gqa_decode_paged_bf16(void* stream, const void* q, const void* k_pages, const void* v_pages, void* out, const int32_t* page_table,
                                    const int32_t* kv_lens, const int32_t* shared_lens, int32_t shared_len, int32_t batch, int32_t n_heads,
                                    int32_t n_kv, int32_t head_dim, int32_t n_pages, int32_t page_size, int32_t table_pages,
                                    void* workspace, size_t workspace_bytes, rt_err_detail* err) {
    clear_err(err);
    if (batch < 0 || n_heads < 0 || n_kv < 0 || head_dim < 0 || n_pages < 0 || table_pages < 0) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "negative dimension");
    if (n_kv == 0 || n_heads % n_kv != 0)
        return fail(err, RT_ERR_HEAD_COUNT_MISMATCH, -1, (uint64_t)n_heads, (uint64_t)n_kv, "n_heads not divisible by n_kv");
    if (head_dim == 0) return fail(err, RT_ERR_ZERO_DIM, -1, 0, 0, "head_dim must be > 0");
    if (!cache_paged_dim(head_dim)) return fail(err, RT_ERR_UNSUPPORTED, -1, 256, (uint64_t)head_dim, "pages have head_dim up to 256, a multiple of 16");
    if (!cache_page_size(page_size)) return fail(err, RT_ERR_UNSUPPORTED, -1, kPageMax, (uint64_t)(int64_t)page_size, "page_size must be a power of two, 16 to 1024");
    const int64_t max_len = (int64_t)table_pages * page_size;
    if (!shared_lens && (shared_len < 0 || shared_len > max_len))
        return fail(err, RT_ERR_KV_OVERFLOW, -1, (uint64_t)max_len, (uint64_t)(int64_t)shared_len, "a prefix behind the page table");
    if (batch == 0 || n_heads == 0) return RT_OK;
    const Plan a = plan_of(batch, n_heads, n_kv, head_dim, max_len);
    if (batch > 65535 || n_heads > 65535 || max_len > (1 << 28) || (int64_t)n_kv * page_size * head_dim >= (1ll << 30) || a.places > 0x7fffffffll - (1 << 20))
        return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "shape too large for the launch grid");
    if (!q || !out || !kv_lens || (max_len > 0 && (!page_table || (n_pages > 0 && (!k_pages || !v_pages))))) return fail(err, RT_ERR_NULL_POINTER, -1, 0, 0, "NULL buffer");
    if (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) return fail(err, RT_ERR_UNSUPPORTED, -1, 16, 0, "q, out and the pages must be 16-byte aligned");
    const size_t need = a.part_bytes + a.word_bytes;
    if (!workspace || workspace_bytes < need)
        return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, need, workspace ? workspace_bytes : 0, "workspace too small");
    if ((uintptr_t)workspace & 15) return fail(err, RT_ERR_WORKSPACE_TOO_SMALL, -1, 16, (uint64_t)((uintptr_t)workspace & 15), "workspace must be 16-byte aligned");
    // (a workgroup writes its rows while others read theirs, and the lengths and the table, which have to be the same for all of them)
    const size_t q_bytes = (size_t)batch * n_heads * head_dim * 2, page_bytes = (size_t)n_pages * n_kv * page_size * head_dim * 2;
    const size_t table_bytes = (size_t)batch * table_pages * 4, lens_bytes = (size_t)batch * 4;
    const struct {
        const void* at;
        size_t n;
    } written[2] = {{out, q_bytes}, {workspace, need}}, read[6] = {{q, q_bytes}, {k_pages, page_bytes}, {v_pages, page_bytes}, {page_table, table_bytes}, {kv_lens, lens_bytes}, {shared_lens, shared_lens ? 4u : 0u}};
    bool apart = !overlap(out, q_bytes, workspace, need);
    for (const auto& w : written)
        for (const auto& r : read) apart = apart && !overlap(w.at, w.n, r.at, r.n);
    if (!apart) return fail(err, RT_ERR_UNSUPPORTED, -1, 0, 0, "out and the workspace must share no memory with each other or with the inputs");
    int rc = ensure_device(err);
    if (rc) return rc;
    PagedDecodeParams p{};
    p.q = (const uint16_t*)q;
    p.k_pages = (const uint16_t*)k_pages;
    p.v_pages = (const uint16_t*)v_pages;
    p.out = (uint16_t*)out;
    p.page_table = page_table;
    p.kv_lens = kv_lens;
    p.shared_lens = shared_lens;
    p.shared_len = shared_len;
    p.batch = batch;
    p.heads = n_heads;
    p.kv_heads = n_kv;
    p.dim = head_dim;
    p.n_pages = n_pages;
    p.table_pages = table_pages;
    p.page_shift = __builtin_ctz((unsigned)page_size);
    p.max_len = (int)max_len;
    p.group = n_heads / n_kv;
    p.chunks = (int)a.chunks;
    p.rows = (int)a.rows;
    p.per_wave = (int)a.per_wave;
    p.per_tile = (int)a.per_tile;
    p.n_tiles = (int)a.n_tiles;
    // (a join's partials have `rows` rows.  us, 0.66 / 0.8 / 1: 1 sequence of 2048 keys, 32 heads on 8 of 128 9.2 / 10.5 / 10.5; 4 of 1756 to
    // 8783, 16 on 2 of 64 11.7 / 11.7 / 12.5, 1 of 12000, 32 on 4 of 128 15.7 / 15.7 / 16.5, 2 of 360 to 5412, 20 on 1 of 80 15.8 / 15.1 / 15.1, 8 of
    // 3010 to 4000, 16 on 1 of 128 15.3 / 15.3 / 14.9)
    p.span_root = a.rows <= 4 ? 0.66f : 0.8f;
    p.scale_log2e = (1.0f / sqrtf((float)head_dim)) * kLog2eHost;
    p.part = (float*)workspace;
    p.head = (unsigned char*)workspace + a.part_bytes;
    p.words = p.head + 256;
    p.launch_id = next_launch_id() << 8;  // (its low 16 bits zero)
    const bool shared = shared_lens || shares(a, batch, n_kv, head_dim, shared_len);
    p.n_groups = std::min(a.groups, kCus * per_cu(a.dim));
    const hipStream_t s = (hipStream_t)stream;
    HIP_TRY(a.dim == 64 ? launch_dim<64>(s, p, shared) : a.dim == 128 ? launch_dim<128>(s, p, shared) : launch_dim<256>(s, p, shared), "paged_decode launch");
    return RT_OK;
}
