// Entry points of the paged KV cache of many sequences (no counterpart in the trait): new keys and
// values into pages, attention over pages.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "capi_util.h"
#include "paged.h"

using larql::fail;

namespace {

constexpr size_t kMax = static_cast<size_t>(larql::kPagedMax);

size_t elem_bytes(int type) { return type == LARQL_ELEM_F32 ? 4 : type == LARQL_ELEM_E4M3 ? 1 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void need(bool ok, const char* what) {
    if (!ok) fail(LARQL_HIP_ERR_INVALID, std::string("paged KV: ") + what);
}

void check_act(int type) {
    need(type == LARQL_ELEM_F32 || type == LARQL_ELEM_F16 || type == LARQL_ELEM_BF16,
         "activations must be F32, F16 or BF16");
}

// Token rows [rows][width] at p, `stride` elements apart.
void check_rows(const void* p, size_t stride, size_t width, int type, const char* what) {
    need(p, (std::string(what) + " is null").c_str());
    need(aligned16(p), (std::string(what) + " is not 16-byte aligned").c_str());
    need(stride >= width && stride < kMax && stride * elem_bytes(type) % 16 == 0,
         (std::string(what) + ": row stride below the row's width or not a multiple of 16 bytes").c_str());
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}
size_t rows_bytes(size_t rows, size_t stride, size_t width, int type) {
    return rows ? ((rows - 1) * stride + width) * elem_bytes(type) : 0;
}

// Whether [a, a + na) meets the pages at p: blocks of a page's positions and heads, `page` bytes apart (what lies between
// them, as in one allocation for several layers, is not theirs).
bool meets_pages(const void* p, size_t page, size_t pos, size_t head, const larql_paged_kv* kv, const void* a, size_t na) {
    using wide = unsigned __int128;
    const size_t es = elem_bytes(kv->type);
    const wide x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(a), stride = page * es;
    const wide block = ((kv->page_size - 1) * static_cast<wide>(pos) + (kv->num_kv_heads - 1) * static_cast<wide>(head) + kv->head_dim) * es;
    const wide all = (kv->num_pages - 1) * stride + block;
    if (na == 0 || y >= x + all || x >= y + na) return false;
    if (y <= x || kv->num_pages == 1 || block >= stride) return true;
    const wide at = (y - x) % stride;
    return at < block || ((y - x) / stride + 1 < kv->num_pages && at + na > stride);
}
void check_pages(const larql_paged_kv* kv, const void* a, size_t na, const char* what) {
    need(!meets_pages(kv->k, kv->k_page_stride, kv->k_pos_stride, kv->k_head_stride, kv, a, na) &&
             !meets_pages(kv->v, kv->v_page_stride, kv->v_pos_stride, kv->v_head_stride, kv, a, na),
         what);
}

// `pages`: the page memory itself is needed (else only the shapes).
larql::PagedView make_view(const larql_paged_kv* kv, const larql_paged_batch* bt, bool pages) {
    need(kv && bt, "null cache or batch");
    if (kv->type != LARQL_ELEM_F16 && kv->type != LARQL_ELEM_BF16 && kv->type != LARQL_ELEM_E4M3)
        fail(LARQL_HIP_ERR_INVALID, "paged KV: pages must be F16, BF16 or E4M3");
    need(kv->num_pages >= 1 && kv->num_pages < kMax && kv->page_size >= 1 && kv->page_size <= kMax,
         "num_pages or page_size out of range");
    need(kv->num_kv_heads >= 1 && kv->num_kv_heads <= 65535, "num_kv_heads out of range");
    need(kv->head_dim >= 1, "head_dim is 0");
    if (kv->head_dim % 32 || kv->head_dim > 256)
        fail(LARQL_HIP_ERR_UNSUPPORTED, "paged KV: head_dim must be a multiple of 32 up to 256");
    need(bt->num_seqs < kMax && bt->num_tokens < kMax, "num_seqs or num_tokens out of range");
    need(bt->q_start || bt->num_tokens == bt->num_seqs, "num_tokens must be num_seqs without q_start");
    need(bt->pages_per_seq <= bt->table_stride && bt->table_stride < kMax, "table_stride below pages_per_seq");
    need(bt->pages_per_seq * kv->page_size <= kMax, "page table reaches more than 2^30 positions");
    larql::PagedView v{};
    if (pages) {
        need(kv->k && kv->v, "null pages");
        need(aligned16(kv->k) && aligned16(kv->v), "pages are not 16-byte aligned");
        const size_t es = elem_bytes(kv->type);
        for (size_t s : {kv->k_page_stride, kv->k_pos_stride, kv->k_head_stride, kv->v_page_stride, kv->v_pos_stride,
                         kv->v_head_stride})
            need(s * es % 16 == 0 && s < (size_t{1} << 40), "a page stride is not a multiple of 16 bytes");
        need((kv->page_size == 1 || (kv->k_pos_stride >= kv->head_dim && kv->v_pos_stride >= kv->head_dim)) &&
                 (kv->num_kv_heads == 1 || (kv->k_head_stride >= kv->head_dim && kv->v_head_stride >= kv->head_dim)) &&
                 (kv->num_pages == 1 || (kv->k_page_stride >= kv->head_dim && kv->v_page_stride >= kv->head_dim)),
             "a page stride is below head_dim");
        need(bt->num_seqs == 0 || (bt->kv_len && (bt->page_table || bt->pages_per_seq == 0)), "null kv_len or page_table");
        v.k = static_cast<const char*>(kv->k);
        v.v = static_cast<const char*>(kv->v);
        v.k_page = static_cast<long long>(kv->k_page_stride * es);
        v.k_pos = static_cast<long long>(kv->k_pos_stride * es);
        v.k_head = static_cast<long long>(kv->k_head_stride * es);
        v.v_page = static_cast<long long>(kv->v_page_stride * es);
        v.v_pos = static_cast<long long>(kv->v_pos_stride * es);
        v.v_head = static_cast<long long>(kv->v_head_stride * es);
        need(kv->type == LARQL_ELEM_E4M3 || (!kv->k_scale && !kv->v_scale), "scales are for E4M3 pages");
        v.k_scale = kv->k_scale;
        v.v_scale = kv->v_scale;
        v.table = bt->page_table;
        v.kv_len = bt->kv_len;
    }
    v.q_start = bt->q_start;
    v.table_ld = static_cast<long long>(bt->table_stride);
    v.num_pages = static_cast<unsigned>(kv->num_pages);
    v.page_size = static_cast<int>(kv->page_size);
    v.pages_per_seq = static_cast<int>(bt->pages_per_seq);
    v.num_seqs = static_cast<int>(bt->num_seqs);
    v.num_tokens = static_cast<int>(bt->num_tokens);
    v.num_kv = static_cast<int>(kv->num_kv_heads);
    v.hd = static_cast<int>(kv->head_dim);
    v.cap = v.pages_per_seq * v.page_size;
    larql::paged_divisor(v.page_size, v.page_mul, v.page_shift);
    return v;
}

larql::PagedAttnArgs make_attn(const larql_paged_kv* kv, const larql_paged_batch* bt, size_t num_q, bool pages) {
    larql::PagedAttnArgs a{};
    a.c = make_view(kv, bt, pages);
    a.kv_type = kv->type;
    need(num_q >= 1 && num_q <= 65535 && num_q % kv->num_kv_heads == 0, "num_q_heads must be a multiple of num_kv_heads");
    need(bt->num_tokens * num_q < kMax && bt->num_seqs * num_q < kMax, "too many rows");
    a.num_q = static_cast<int>(num_q);
    a.reps = static_cast<int>(num_q / kv->num_kv_heads);
    larql::paged_divisor(a.reps, a.rep_mul, a.rep_shift);
    // units of 32 positions (counted in ints) of the groups of columns; with q_start of sequences of few rows
    const int most = 16 * larql::paged_nc(a.c.hd, bt->q_start);
    const double n = static_cast<double>(bt->num_seqs), rows = static_cast<double>(bt->num_tokens) * a.reps;
    const int few = larql::paged_few(a.c, a.kv_type, static_cast<long long>(rows));
    const double groups = bt->q_start ? std::min(n * ((few + most - 1) / most), n + rows / most) : n * ((a.reps + most - 1) / most);
    need(groups * kv->num_kv_heads * (a.c.cap / 32 + 1) < 2147483647.0, "too many positions in one call");
    // a launch counts its threads in 32 bits: 256 for each segment to join, and for each tile of rows
    const double segments = n * ((std::max(bt->q_start ? std::min<double>(larql::kPagedFewAll, rows) : a.reps, 1.0) + most - 1) / most);
    need(std::max(segments, bt->q_start ? n + rows / 128 : 0.0) * kv->num_kv_heads < 16777216.0, "too many rows in one call");
    return a;
}

}  // namespace

extern "C" int larql_hip_paged_append_dev(larql_hip_ctx* c, const larql_paged_kv* cache, const larql_paged_batch* batch,
                                          int type, const void* q, size_t q_stride, size_t num_q_heads, const void* k,
                                          size_t k_stride, const void* v, size_t v_stride, void* q_out,
                                          size_t q_out_stride, double rope_base, size_t rotary_dim, void* stream) {
    return guarded(c, [&] {
        larql::PagedAppendArgs a{};
        a.c = make_view(cache, batch, true);
        check_act(type);
        const size_t hd = cache->head_dim, kvd = cache->num_kv_heads * hd, qd = num_q_heads * hd, T = batch->num_tokens;
        need(num_q_heads <= 65535 && (T == 0 || (num_q_heads == 0) == (q == nullptr)), "q and num_q_heads must come together");
        need(rotary_dim <= hd && rotary_dim % 2 == 0, "rotary_dim must be even and at most head_dim");
        need(std::isfinite(rope_base) && rope_base >= 0.0, "rope_base must be positive, or 0 for no rotation");
        need(T < (size_t{1} << 26), "too many tokens in one call");  // (a launch counts its threads in 32 bits: 64 a token)
        if (T == 0) return;
        check_rows(k, k_stride, kvd, type, "k");
        check_rows(v, v_stride, kvd, type, "v");
        check_pages(cache, k, rows_bytes(T, k_stride, kvd, type), "k overlaps the pages");
        check_pages(cache, v, rows_bytes(T, v_stride, kvd, type), "v overlaps the pages");
        if (q) {
            check_rows(q, q_stride, qd, type, "q");
            check_rows(q_out, q_out_stride, qd, type, "q_out");
            const size_t no = rows_bytes(T, q_out_stride, qd, type);
            check_pages(cache, q, rows_bytes(T, q_stride, qd, type), "q overlaps the pages");
            check_pages(cache, q_out, no, "q_out overlaps the pages");
            // (rows of a packed projection interleave: equal strides whose rows do not meet are fine)
            auto rows_meet = [&](const void* p, size_t stride, size_t width) {
                if (!overlap(q_out, no, p, rows_bytes(T, stride, width, type))) return false;
                if (stride != q_out_stride) return true;
                const size_t es = elem_bytes(type), ld = stride * es;
                const uintptr_t x = reinterpret_cast<uintptr_t>(q_out), y = reinterpret_cast<uintptr_t>(p);
                const size_t at = x >= y ? (x - y) % ld : (ld - (y - x) % ld) % ld;  // q_out's start within p's rows
                return at < width * es || at + qd * es > ld;
            };
            need(q_out == q ? q_out_stride == q_stride : !rows_meet(q, q_stride, qd), "q_out overlaps q");
            need(!rows_meet(k, k_stride, kvd) && !rows_meet(v, v_stride, kvd), "q_out overlaps k or v");
        }
        a.kv_type = cache->type;
        a.act_type = type;
        a.q = q;
        a.k = k;
        a.v = v;
        a.q_out = q_out;
        a.q_ld = static_cast<long long>(q_stride);
        a.k_ld = static_cast<long long>(k_stride);
        a.v_ld = static_cast<long long>(v_stride);
        a.qo_ld = static_cast<long long>(q_out_stride);
        a.num_q = static_cast<int>(num_q_heads);
        a.half = rope_base > 0.0 ? static_cast<int>((rotary_dim ? rotary_dim : hd) / 2) : 0;
        a.log2_base = rope_base > 0.0 ? std::log2(rope_base) : 0.0;
        larql::launch_paged_append(a, pick_stream(c, stream));
    });
}

extern "C" int larql_hip_paged_attention_work_bytes(larql_hip_ctx* c, const larql_paged_kv* cache,
                                                    const larql_paged_batch* batch, size_t num_q_heads, size_t* bytes) {
    return guarded(c, [&] {
        need(bytes, "null bytes");
        larql::PagedAttnArgs a = make_attn(cache, batch, num_q_heads, false);
        *bytes = batch->num_tokens ? larql::paged_attn_most(a, c->num_cus) : 0;
    });
}

extern "C" int larql_hip_paged_attention_dev(larql_hip_ctx* c, const larql_paged_kv* cache,
                                             const larql_paged_batch* batch, int type, const void* q, size_t q_stride,
                                             size_t num_q_heads, void* out, size_t out_stride, float scale,
                                             size_t window, float softcap, void* work, size_t work_bytes, void* stream) {
    return guarded(c, [&] {
        larql::PagedAttnArgs a = make_attn(cache, batch, num_q_heads, true);
        check_act(type);
        need(std::isfinite(scale), "scale must be finite");
        need(std::isfinite(softcap) && softcap >= 0.f, "softcap must be positive, or 0 for none");
        const size_t T = batch->num_tokens, qd = num_q_heads * cache->head_dim;
        if (T == 0) return;
        check_rows(q, q_stride, qd, type, "q");
        check_rows(out, out_stride, qd, type, "out");
        const size_t nq = rows_bytes(T, q_stride, qd, type), no = rows_bytes(T, out_stride, qd, type);
        need(!overlap(q, nq, out, no), "out overlaps q");
        check_pages(cache, out, no, "out overlaps the pages");
        a.act_type = type;
        a.q = q;
        a.out = out;
        a.q_ld = static_cast<long long>(q_stride);
        a.out_ld = static_cast<long long>(out_stride);
        a.scale = scale;
        a.softcap = softcap;
        a.window = static_cast<int>(std::min(window, kMax));
        const size_t bytes = larql::paged_attn_plan(a, work, c->num_cus);
        need(bytes == 0 || (work && aligned16(work)), "work is null or not 16-byte aligned");
        need(work_bytes >= bytes, "work buffer too small (larql_hip_paged_attention_work_bytes)");
        need(!overlap(work, bytes, q, nq) && !overlap(work, bytes, out, no), "work overlaps q or out");
        check_pages(cache, work, bytes, "work overlaps the pages");
        larql::launch_paged_attention(a, pick_stream(c, stream));
    });
}
