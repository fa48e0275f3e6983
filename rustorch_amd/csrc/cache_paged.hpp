// Caches in pages, and the parameter blocks of the kernels that write and read them.
//
// K and V are [n_pages, kv heads, page_size, dim] of bf16, page_size a power of two from 16 on; row r of sequence b lies in page
// page_table[b, r / page_size], there in row r % page_size of each kv head.  An entry outside 0 .. n_pages - 1 is no page: rows that
// would go there are not written, and keys there are not seen.  A page holds a head's rows side by side, so that sixteen rows, or a
// multiple of them that starts at one, are one piece of memory: what a wave asks for at a time.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rt {

constexpr int kPageMin = 16, kPageMax = 1024, kMaxAxes = 4;
inline bool cache_page_size(int n) { return n >= kPageMin && n <= kPageMax && (n & (n - 1)) == 0; }
inline bool cache_paged_dim(int dim) { return dim >= 16 && dim <= 256 && dim % 16 == 0; }

// New rows of packed tokens into pages (paged_append.hip).
struct PagedAppendParams {
    const uint16_t* q;  // [tokens, n_heads, dim]
    uint16_t* q_out;    // the same shape; may be q
    const uint16_t* k_in;  // [tokens, n_kv, dim]
    uint16_t* k_out;       // the same shape, rotated; may be k_in; null: not wanted
    const uint16_t* v_in;
    uint16_t* k_pages;
    uint16_t* v_pages;
    const int32_t* page_table;  // device int32[batch, table_pages]
    const int32_t* starts;      // device int32[batch + 1]: first token of each sequence; null: tokens / batch of each
    const int32_t* positions;   // device int32[batch]: row of a sequence's first token; null: `pos`
    const int32_t* axes;        // device int32[n_axes, tokens], or null: a token's row is its position
    const float* q_gamma;
    const float* k_gamma;
    const float* cos_table;
    const float* sin_table;
    float eps;
    int pos, table_rows;
    int tokens, batch, each;  // each: tokens / batch where there are no starts
    int n_heads, n_kv, dim, n_pages, table_pages, page_shift;
    int n_axes, ends[kMaxAxes];  // pairs below ends[i], and not below ends[i - 1], turn with axis i
};

// A decode step over pages (decode_paged.hip).
struct PagedDecodeParams {
    const uint16_t* q;  // [batch, heads, dim]
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    uint16_t* out;              // the shape of q
    const int32_t* page_table;  // device int32[batch, table_pages]
    const int32_t* kv_lens;     // device int32[batch]
    const int32_t* shared_lens; // device int32[1]; null: shared_len
    int shared_len;
    int batch, heads, kv_heads, dim;
    int n_pages, table_pages, page_shift;
    int max_len;       // table_pages pages of rows
    int group;         // heads / kv_heads
    int chunks, rows;  // of a kv head's query heads: so many pieces of `rows` each (the last may have fewer), at most 16
    int per_wave, per_tile, n_tiles;  // (sequence, piece) pairs of a wave's rows and of a tile of the prefix; tiles of a kv head
    int n_groups;      // workgroups launched
    float span_root, scale_log2e;
    float* part;
    unsigned char* head;   // what one launch leaves for the next
    unsigned char* words;  // a line for each (sequence, kv head, piece)
    uint64_t launch_id;
};

}  // namespace rt
