// Plan and dispatch of attention over the paged KV cache.
#include <algorithm>

#include "paged_prompt.h"

namespace larql {

namespace {

// Parts of a work buffer (null: their sizes only), 16-byte aligned.
struct Carve {
    char* p;
    size_t at;
    template <class T>
    T* take(size_t n) {
        char* r = p ? p + at : nullptr;
        at += (n * sizeof(T) + 15) & ~size_t{15};
        return reinterpret_cast<T*>(r);
    }
};

// The waves' part, for sequences of up to `rows` rows: one round of resident waves, and no more than there can be units.
// Grows with every shape.
void plan_waves(PagedAttnArgs& a, Carve& c, bool several, int rows, int num_cus) {
    const PagedView& v = a.c;
    const int per_simd = paged_waves(v.hd, v.hd * (a.kv_type == LARQL_ELEM_E4M3 ? 1 : 2), several);
    const int most = 16 * paged_nc(v.hd, several);
    a.groups = (rows + most - 1) / most;
    a.cols = std::min(most, rows);
    const size_t heads = static_cast<size_t>(v.num_kv) * a.groups;
    const size_t units = v.num_seqs * heads * static_cast<size_t>((v.cap + 31) / 32 + 1);
    a.workers = static_cast<int>(std::max<size_t>(1, std::min(units, static_cast<size_t>(num_cus) * 4 * per_simd / paged_wg(several))));
    // joins: about four workgroups per CU, a group of hd / 4 of their 256 threads to a column at least
    for (a.join_cols = 1; a.join_cols < (several && v.hd <= 128 ? 8 : 4) && a.join_cols < a.cols && v.num_seqs * heads * a.cols / a.join_cols > 4 * static_cast<size_t>(num_cus);)
        a.join_cols *= 2;
    const size_t entries = 2 * static_cast<size_t>(a.workers) * a.cols;
    a.seg = c.take<int>(2 + v.num_seqs * heads);
    a.ml = c.take<float>(entries * 2);
    a.part = c.take<float>(entries * v.hd);
}

// Parts of split tiles.
void plan_splits(PagedAttnArgs& a, Carve& c, size_t entries) {
    a.tile_ml = c.take<float>(entries * 2);
    a.tile_part = c.take<float>(entries * a.c.hd);
}

constexpr int kSplitsMost = 16;
// Workgroups of tiles that run at once; tiles of 64 positions that a table row reaches.
int tiles_resident(const PagedView& v, int num_cus) { return num_cus * (v.hd <= 128 ? 2 : 1); }
int tiles_reach(const PagedView& v) { return std::max(1, (v.cap + 63) / 64); }

}  // namespace

size_t paged_attn_plan(PagedAttnArgs& a, void* work, int num_cus) {
    const PagedView& v = a.c;
    Carve c{static_cast<char*>(work), 0};
    a.few = a.tiles = 0;
    a.splits = 1;
    if (!v.q_start) {
        plan_waves(a, c, false, a.reps, num_cus);
        return c.at;
    }
    // Several tokens: a short cache, few rows in all, or one sequence, tell which kernel they are for; else either
    // may have work.
    const long long rows = static_cast<long long>(v.num_tokens) * a.reps;
    a.few = paged_few(v, a.kv_type, rows);
    if (a.few) plan_waves(a, c, true, static_cast<int>(std::min<long long>(a.few, rows)), num_cus);
    if (rows > a.few) {
        a.tiles = static_cast<int>(rows / kPromptRows) + (a.few ? static_cast<int>(std::min<long long>(v.num_seqs, rows / a.few)) : v.num_seqs);
        // Splits by the modelled time (us): rounds of resident workgroups over tiles of 64 positions (2.5 with
        // f32 activations at head_dim 128, 4.4 at 256; the work buffer is the same for every type) and their start (6),
        // against the parts written and read (3.5 TB/s) and the join's launch (5).  One more than fills the
        // resident workgroups at most, which bounds the parts.
        const double tile = 2.5 * (v.hd <= 128 ? v.hd / 128.0 : v.hd / 145.0);
        const int resident = tiles_resident(v, num_cus), n = tiles_reach(v);
        const double groups = static_cast<double>(a.tiles) * v.num_kv;
        const double parts = 2.0 * v.num_tokens * a.num_q * v.hd * sizeof(float) / 3.5e6;
        double best = 0;
        for (int s = 1; s <= std::min(kSplitsMost, n) && (s - 1) * groups < resident; s++) {
            const double us = std::max(1.0, groups * s / resident) * ((n + s - 1) / s * tile + 6.0) + (s > 1 ? s * parts + 5.0 : 0.0);
            if (s == 1 || us < best) best = us, a.splits = s;
        }
        if (a.splits > 1) plan_splits(a, c, static_cast<size_t>(v.num_tokens) * a.num_q * a.splits);
    }
    return c.at;
}

size_t paged_attn_most(PagedAttnArgs a, int num_cus) {
    Carve several{nullptr, 0}, one{nullptr, 0};
    const long long rows = static_cast<long long>(a.c.num_tokens) * a.reps;
    if (a.c.q_start) {
        if (a.c.cap > paged_short(a.c.hd, a.kv_type)) plan_waves(a, several, true, static_cast<int>(std::min<long long>(kPagedFewAll, rows)), num_cus);
        // rows x kv heads are at most 128 times the tiles' workgroups, and (splits - 1) times those below the resident ones
        const size_t splits = static_cast<size_t>(std::min(kSplitsMost, tiles_reach(a.c)));
        if (splits > 1)
            plan_splits(a, several, std::min(static_cast<size_t>(a.c.num_tokens) * a.num_q * splits,
                                             size_t{2} * kPromptRows * tiles_resident(a.c, num_cus)));
    }
    a.c.num_seqs = std::min(a.c.num_seqs, a.c.num_tokens);
    plan_waves(a, one, false, a.reps, num_cus);
    return std::max(several.at, one.at);
}

void launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    if (a.c.num_seqs == 0) return;
    switch (a.c.hd) {
#define LARQL_PAGED_CASE(HD)                         \
    case HD:                                         \
        if (!a.c.q_start) launch_paged_decode_##HD(a, s); \
        if (a.few) launch_paged_few_##HD(a, s);      \
        if (a.tiles) launch_paged_prompt_##HD(a, s); \
        return;
        LARQL_PAGED_HDS(LARQL_PAGED_CASE)
#undef LARQL_PAGED_CASE
    }
    fail(LARQL_HIP_ERR_UNSUPPORTED, "paged KV: head_dim");
}

}  // namespace larql
