// Paged KV cache of many sequences: what the kernels see, shared by paged_*.hip and capi_paged.cpp.
#pragma once

#include "larql_hip_internal.h"

namespace larql {

// Most positions of a sequence, and most rows of a call.
constexpr int kPagedMax = 1 << 30;

// n / d for n < 2^31 as n * mul / 2^(31 + shift): with 2^(shift - 1) < d <= 2^shift and mul =
// ceil(2^(31 + shift) / d) < 2^32 the product is above n / d by less than 1 / d.
inline void paged_divisor(int d, unsigned& mul, int& shift) {
    shift = 0;
    while ((1ll << shift) < d) shift++;
    mul = static_cast<unsigned>(((1ull << (31 + shift)) + d - 1) / d);
}

// Pages and batch on the device.  Strides in bytes; an element's address is 64-bit throughout (a
// cache passes 4 GiB).  Page of a position: paged_divisor.
struct PagedView {
    const char* k;
    const char* v;
    long long k_page, k_pos, k_head, v_page, v_pos, v_head;
    const float* k_scale;  // per kv head, or null
    const float* v_scale;
    const int* table;
    long long table_ld;
    const int* kv_len;
    const int* q_start;  // null: one token per sequence
    unsigned num_pages, page_mul;
    int page_shift, page_size, pages_per_seq;
    int num_seqs, num_tokens, num_kv, hd;
    int cap;  // positions a table row reaches
};

struct PagedAppendArgs {
    PagedView c;
    int kv_type, act_type;
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    long long q_ld, k_ld, v_ld, qo_ld;  // elements
    int num_q;  // 0: keys and values only
    int half;   // rotated pairs per head (0: none)
    double log2_base;
};

struct PagedAttnArgs {
    PagedView c;
    int kv_type, act_type;
    const void* q;
    void* out;
    long long q_ld, out_ld;  // elements
    int num_q, reps;
    unsigned rep_mul;  // row / reps = row * rep_mul / 2^(31 + rep_shift), as for pages
    int rep_shift;
    float scale, softcap;
    int window;  // 0: none
    // decode: the number of units, of workers with work and each segment's first unit, partial (m, l) and sums of the workers (two
    // each: the run's first and last segment)
    int groups;   // column groups per kv head: the most of a sequence
    int cols;     // columns a partial entry holds
    int join_cols;  // columns that a workgroup of the join takes
    int workers;
    int* seg;     // [2 + num_seqs * num_kv * groups]
    float* ml;
    float* part;
    // with q_start: sequences of up to `few` rows (tokens x query heads per kv head) are read as one
    // token is (few 0: none), the others in `tiles` tiles of rows (0: none can be), their positions in
    // `splits` parts
    int few, tiles, splits;
    float* tile_ml;
    float* tile_part;
};

// 16-column groups in a wave's hands: 1 for one token per sequence; 2 for several, where the sums fit.
constexpr int paged_nc(int hd, bool multi) { return multi && hd <= 128 ? 2 : 1; }
// Rows (tokens x query heads per kv head) of a sequence up to which its cache is read once per 32 of them
// rather than by a tile of 128.
constexpr int kPagedFew = 64;
// Rows of a call up to which all its sequences are, whatever their shares: the second kernel's launches
// cost what a prompt's few passes over its cache would save.
constexpr int kPagedFewAll = 256;
// Positions a table row reaches up to which tiles take the few rows as well: a run's change of segment costs
// more than a short cache read by a tile of mostly idle rows.  5 new tokens of 8-kv-head sequences, few / tiles: f16
// pages 64 sequences of 300 positions 80 / 23 us, 32 of 4000 126 / 89, 8 of 8000 47 / 55; e4m3 32 of 1000
// 48 / 31, 8 of 4000 29 / 33; head_dim 256 8 of 300 25 / 20, 8 of 2000 27 / 36.
constexpr int paged_short(int hd, int kv_type) { return hd > 128 ? 512 : kv_type == LARQL_ELEM_E4M3 ? 2048 : 6144; }
// Most rows of a sequence that is read as one token is, in a call of `rows` rows with q_start; 0: none is.
inline int paged_few(const PagedView& v, int kv_type, long long rows) {
    if (v.cap <= paged_short(v.hd, kv_type) || (v.num_seqs <= 1 && rows > kPagedFew)) return 0;
    return rows <= kPagedFewAll ? kPagedFewAll : kPagedFew;
}
// Waves of a worker.
constexpr int paged_wg(bool multi) { return multi ? 4 : 1; }
// Waves per SIMD that their registers leave room for (row: bytes of a head's row in the cache).
constexpr int paged_waves(int hd, int row, bool multi) {
    return multi ? ((hd <= 128 ? row > 192 : row > 448) ? 1 : 2) : hd <= 64 ? 3 : 2;
}

void launch_paged_append(const PagedAppendArgs& a, hipStream_t s);
// Work buffer bytes of one attention call, and the pointers of `a` into it (work null: sizes only).
size_t paged_attn_plan(PagedAttnArgs& a, void* work, int num_cus);
// What is enough for one call of every batch of no more sequences, tokens and positions over the same cache (with q_start:
// also without).  A prompt of fewer tokens takes more parts, so one call's own is not.
size_t paged_attn_most(PagedAttnArgs a, int num_cus);
void launch_paged_attention(const PagedAttnArgs& a, hipStream_t s);

// One launcher per head_dim (each compiled in a file of its own), by cache type and activation type.
#define LARQL_PAGED_HDS(X) X(32) X(64) X(96) X(128) X(160) X(192) X(224) X(256)
#define LARQL_PAGED_DECL(HD)                                             \
    void launch_paged_decode_##HD(const PagedAttnArgs& a, hipStream_t s); \
    void launch_paged_few_##HD(const PagedAttnArgs& a, hipStream_t s);    \
    void launch_paged_prompt_##HD(const PagedAttnArgs& a, hipStream_t s);
LARQL_PAGED_HDS(LARQL_PAGED_DECL)
#undef LARQL_PAGED_DECL

}  // namespace larql
