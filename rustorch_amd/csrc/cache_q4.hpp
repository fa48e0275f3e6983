// Caches whose rows are held in 4 bits, and the parameter blocks of the kernels that write, read and shrink caches.
//
// A row of dim values (64, 128 or 256) has a pair of bf16 numbers for every 64 of them, a scale s and a middle z; a value is
// z + s (c - 8), c a code of 0 .. 15.  For the largest and smallest value of the 64, hi and lo,
//     z = bf16((hi + lo) / 2 + (hi - lo) / 32)        s = max((hi - z) / 7.5, (z - lo) / 8.5), up to the next bf16
//     c = 8 + clamp(nearest((x - z) / s), -8, 7)      (ties to even; 8 where s is 0)
// so that every code's interval is s wide and the sixteen of them cover lo .. hi whatever the two numbers' own rounding: a value
// is off by s / 2 at most.  Offsets from the middle, not from the smallest value, keep the sums of products that the codes go
// into as small as the values themselves.  64 values a pair: 4.5 bits a value; a pair for the whole row of 128 would save 3 % and lets
// one large channel coarsen all others, pairs for 32 cost 11 % more bytes.
//
// Codes: [batch, kv heads, max_seq, dim / 2] bytes.  Byte i n + p of a row, n = dim / 32, holds the dims 32 c + 2 i (low bits) and
// 32 c + 2 i + 1, where c is p with its two lowest bits exchanged (c = p for n = 2).  A lane of a matrix instruction that owns four
// consecutive i has the operand of a 64-dim group in the low bits of every second byte, so that two codes come out of a word with
// a mask, and a shift for the odd bytes.
// Pairs: [batch, kv heads, dim / 64, max_seq] words, s in the low half: a group's pairs of neighbouring rows are neighbours.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rt {

// Over the lanes of a wave within registers, where a shuffle goes through LDS and takes ten times as long: step i brings a lane the value
// from 1, 2, 4, 8 lanes down its row of 16, from the row before it (second and fourth row), from the lower half (upper half); `none`
// where there is none.
template <int kStep>
__device__ __forceinline__ int lanes_step(int none, int x) {
    constexpr int kCtrl[6] = {0x111, 0x112, 0x114, 0x118, 0x142, 0x143}, kRows[6] = {0xf, 0xf, 0xf, 0xf, 0xa, 0xc};
    return __builtin_amdgcn_update_dpp(none, x, kCtrl[kStep], kRows[kStep], 0xf, false);
}
// the sum up to and with this lane
__device__ __forceinline__ int lane_sums(int x) {
    x += lanes_step<0>(0, x);
    x += lanes_step<1>(0, x);
    x += lanes_step<2>(0, x);
    x += lanes_step<3>(0, x);
    x += lanes_step<4>(0, x);
    x += lanes_step<5>(0, x);
    return x;
}
// f over the lanes up to and with this one of its row of 16 (kSteps 4) or of the wave (6), in the last lane of each; f(x, x) = x
template <int kSteps, typename T, typename F>
__device__ __forceinline__ T lanes_fold(T x, F f) {
    x = f(x, (T)lanes_step<0>((int)x, (int)x));
    x = f(x, (T)lanes_step<1>((int)x, (int)x));
    x = f(x, (T)lanes_step<2>((int)x, (int)x));
    x = f(x, (T)lanes_step<3>((int)x, (int)x));
    if constexpr (kSteps == 6) {
        x = f(x, (T)lanes_step<4>((int)x, (int)x));
        x = f(x, (T)lanes_step<5>((int)x, (int)x));
    }
    return x;
}
__device__ __forceinline__ int lane_max(int x) {
    return __builtin_amdgcn_readlane(lanes_fold<6>(x, [](int a, int b) __attribute__((always_inline)) { return max(a, b); }), 63);
}

inline bool cache_q4_dim(int dim) { return dim == 64 || dim == 128 || dim == 256; }

// New rows into a cache, bf16 or 4-bit (cache_append.hip).
struct CacheAppendParams {
    const uint16_t* q;  // [batch, n_heads, seq, dim]
    uint16_t* q_out;    // the same shape; may be q
    const uint16_t* k_in;  // [batch, n_kv, seq, dim]
    const uint16_t* v_in;
    void* k;  // codes, or bf16 rows
    uint32_t* k_pairs;
    void* v;
    uint32_t* v_pairs;
    const int32_t* positions;  // device int32[batch]: position of a sequence's first new token; null: `pos`
    const int32_t* rows;       // device int32[batch]: its cache row; null: the position (or `row`, where nothing is rotated)
    const float* q_gamma;
    const float* k_gamma;
    const float* cos_table;  // null: rows as they come, no norm and no rotation
    const float* sin_table;
    int32_t* slots;   // optional [batch, n_kv, max_seq]: the position of the token that a row holds
    float* weights;   // optional [batch, n_kv, max_seq]: 0 for a new row
    float eps;
    int pos, row;
    int batch, seq, n_heads, n_kv, max_seq, table_rows;
};

struct CacheReadParams {
    const uint8_t* codes;
    const uint32_t* pairs;
    uint16_t* out;        // [batch, n_kv, n_rows, dim]
    const int32_t* rows;  // device int32[batch]: first row; null: `row`
    int row, n_rows, n_kv, max_seq;
};

// Attention over a cache of either kind (decode_cache.hip).
struct CacheAttendParams {
    const uint16_t* q;  // [batch, seq_new, heads, dim]
    const void* k;      // codes, or bf16 rows
    const uint32_t* k_pairs;
    const void* v;
    const uint32_t* v_pairs;
    uint16_t* out;           // the shape of q
    const int32_t* kv_lens;  // device int32[batch]; null: kv_len
    int kv_len;
    int batch, heads, kv_heads, seq_new, max_seq;
    int group;    // heads / kv_heads
    int rows;     // seq_new * group query rows of a kv head
    int n_tiles;  // of 16 of them
    int n_groups;  // workgroups launched
    int n_long;  // of them at work where sequences are long
    float span_root;  // one takes at least this many times the root of the longest sequence's steps of 32 keys
    float scale_log2e;
    float* part;    // partials: (n_groups + segments) slots of part_rows * (dim + 2) floats, the rows and behind them their (m, l)
    int part_rows;  // min(16, rows)
    unsigned char* words;  // a line a segment, see SegmentWord
    uint64_t launch_id;    // its low 16 bits zero
    // the weights' sums (seq_new = 1), or null
    float* scores;             // [batch, heads, max_seq]: unscaled scores
    float* stats;              // [batch, heads, 2]: the row's maximum (unscaled), 1 / sum
    const float* weights_in;   // [batch, kv_heads, max_seq] or null (zeros)
    float* weights_out;
};

// The rows of a cache that stay (cache_evict.hip).
struct CacheEvictParams {
    uint8_t* k;
    uint32_t* k_pairs;  // null: bf16 rows
    uint8_t* v;
    uint32_t* v_pairs;
    const float* weights_in;    // [batch, n_kv, max_seq]
    const int32_t* slots_in;
    float* weights_out;
    int32_t* slots_out;
    const int32_t* kv_lens;  // device int32[batch]
    int32_t* new_lens;       // device int32[batch] or null; may be kv_lens
    int32_t* header;  // [batch * n_kv, 2]: length, rows that move
    int32_t* from;    // [batch * n_kv, most]: the slots they leave
    int32_t* to;      // ... and take
    int batch, n_kv, max_seq, budget, recent;
    int row_bytes;    // of K and of V
    int groups;       // pairs a row has
    int move_rows;    // rows that a workgroup moves
    int most;         // min(budget, max_seq - budget): rows of a head that can move
};

}  // namespace rt
