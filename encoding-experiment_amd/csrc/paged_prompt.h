// Attention of several new tokens of every sequence over a paged KV cache (one head_dim per
// including file): a prompt's chunk behind what is cached, or a few drafted tokens.
//
// Row r of a sequence's n new tokens sits at position t = kv_len - n + r and attends positions
// (t - window, t].  Bound: the matrix cores and the softmax's vector work for long chunks, reading
// K and V for a few rows over a long cache.
//
// The query heads of a kv head share its K and V: rows (token, head of the group) are packed into
// tiles of 128, 32 to a wave (32 x 32 x 16 products).  Scores are K . Q^T: lane (h, n) = 32 h + n
// holds, for row n, positions 8 q + 4 h + i of 32 (q, i < 4), and registers 8 s .. 8 s + 7 are, as they
// lie, the B operand of V^T . P^T whose slots 4 q + i stand for positions 16 s + 8 q + 4 h + i.  V's
// operand comes from row-major LDS by the transposing read (4 positions of one dim per lane).
// K and V tiles of 64 positions lie in two LDS buffers: the next tile's loads are in flight over this
// tile's products, straight into LDS (e4m3: through registers, widened to f16).  At head_dim 256 the buffers take 132 KB,
// one workgroup per CU: tiles of 32, a barrier per half the work, took 215 us instead of 182 for 4000 tokens
// bf16.  16-byte pieces of a row are XORed with the row so that reads do not meet in a bank.
//
// Positions in a row's future, outside its window, behind the sequence or on no page get no weight
// whatever lies there: scores by select, V rows behind the sequence as zeros, and V elements that
// are not finite by a separate pass over tiles that some row masks (0 * inf is not 0).
//
// With few tiles the positions of a tile are split over several workgroups and joined in order.
//
// Measured, 32 query and 8 kv heads of 128: 8191 tokens bf16 630 us (870 TFLOP/s; its products alone 558,
// all but them 495), five chunks of up to 1200 tokens behind up to 2500 209 us, 512 tokens f32 over f16 32 us.  Two waves
// per SIMD of 32 rows each beat one of 64 rows (half the LDS reads, 732 us): one wave's softmax
// passes beside the other's products.
#pragma once

#include "paged_device.h"

namespace larql {

constexpr int kPromptRows = 128;

template <int HD, int KT, int NS>
struct PagedPrompt {
    static constexpr bool BF = KT == LARQL_ELEM_BF16, AF = NS == (BF ? 3 : 2);  // (AF: f32 activations)
    static constexpr int ES = KT == LARQL_ELEM_E4M3 ? 1 : 2;
    static constexpr int KV = 64;  // positions per tile: one to a lane
    // Scores held at once, in 32s: a whole tile's, or half of them where several parts of the rows leave no room.
    static constexpr int JN = (HD > (KT == LARQL_ELEM_E4M3 ? 64 : 96) && NS == 2) || (HD > 128 && NS == 3) ? 1 : KV / 32;
    static constexpr int NC = HD / 8;               // 16-byte pieces of an LDS row
    static constexpr int CH = KV * NC / 256;          // pieces per thread of one tile
    static constexpr bool DIRECT = ES == 2;           // pieces go from memory to LDS as they are
    static constexpr int KS = HD / 16, DT = HD / 32;
    static constexpr int W = 2 * ES;              // words of a piece in the cache
    using Weights = PagedWeights<BF, NS>;
    // Three parts of a wide row are more registers than the row itself: it stays f32, split per use.
    static constexpr bool QF = NS == 3 && HD > 192;

    static __device__ __forceinline__ int swz_k(int row, int cc) {
        return NC % 16 == 0 ? cc ^ (row & 15) : NC % 8 == 0 ? cc ^ (row & 7) : NC % 4 == 0 ? cc ^ (row >> 1 & 3) : cc;
    }
    static __device__ __forceinline__ int swz_v(int row, int cc) {
        return NC % 16 == 0 ? cc ^ (4 * (row & 3)) : NC % 8 == 0 ? cc ^ (4 * (row >> 1 & 1)) : cc;
    }
};

// Schedules N operands of R LDS reads and M products each: the reads of four operands before the
// products, so that their latency passes under as many products and not once per product.
template <int N, int R, int M>
__device__ __forceinline__ void lds_ahead() {
    constexpr int A = N < 4 ? N : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, R * A, 0);
#pragma unroll
    for (int i = 0; i < N - A; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, M * A, 0);
}

// Schedules the second half of a tile: the weights of 32 positions, then the products with them (N
// operands of two LDS reads and M products each), the next 32 positions' weights between them, so that the
// exponentials run beside the matrix cores; the reads four operands ahead.
template <int N, int M, int JN>
__device__ __forceinline__ void products_over_weights() {
    constexpr int V = M == 1 ? 5 : M == 2 ? 11 : 17;  // vector instructions per two weights
    constexpr int A = N < 4 ? N : 4;
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * A, 0);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < N * JN; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        if (i < N * JN - A) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        if (i < N * (JN - 1)) {
            __builtin_amdgcn_sched_group_barrier(0x002, V * 8 / N, 0);
            __builtin_amdgcn_sched_group_barrier(0x400, 16 / N, 0);
        }
    }
}

// A tile of rows: sequence, first packed row, rows, and the new tokens' first row and first position.
struct PagedTile {
    int b, r0, rows, row0, pos0, len;
};

// LDS of the search for a workgroup's tile.
struct PagedTileLds {
    int scan[4], find[2], len[256], tiles[256];
    unsigned char seq[256];
};

// Finds the tile `idx` (256 threads; all return the same).  b < 0: there is none.  The tiles that read most come
// first, or the last workgroups to start would end long after the others: sequences by their length
// (up to 256 of them; more stay in order), in each the last rows first.
__device__ __forceinline__ PagedTile paged_tile(const PagedAttnArgs& a, int idx, PagedTileLds& s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PagedView& v = a.c;
    const int per = (v.num_seqs + 255) / 256, b0 = min(tid * per, v.num_seqs), b1 = min(b0 + per, v.num_seqs);
    auto tiles = [&](int b) {
        int row0, n;
        paged_rows(v, b, row0, n);
        return n * a.reps <= a.few ? 0 : (n * a.reps + kPromptRows - 1) / kPromptRows;
    };
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += tiles(b);
    if (tid == 0) s.find[0] = -1;
    int first = b0;  // the first sequence of this thread's
    if (per == 1 && v.num_seqs > 1) {
        const int len = tid < v.num_seqs ? paged_len(v, tid) : 0;
        if (tid < v.num_seqs) s.len[tid] = len;
        __syncthreads();
        if (tid < v.num_seqs) {
            int rank = 0;
            for (int b = 0; b < v.num_seqs; b++) rank += s.len[b] > len || (s.len[b] == len && b < tid);
            s.tiles[rank] = mine;
            s.seq[rank] = static_cast<unsigned char>(tid);
        }
        __syncthreads();
        mine = tid < v.num_seqs ? s.tiles[tid] : 0;
        first = s.seq[min(tid, v.num_seqs - 1)];
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(incl, d, 64);
        if (lane >= d) incl += x;
    }
    if (lane == 63) s.scan[wave] = incl;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < 3; w++) before += w < wave ? s.scan[w] : 0;
    incl += before;
    if (idx >= incl - mine && idx < incl) {
        int b = first, left = idx - (incl - mine), n = per == 1 ? mine : tiles(b);
        for (; left >= n; n = tiles(++b)) left -= n;
        s.find[0] = b;
        s.find[1] = n - 1 - left;
    }
    __syncthreads();
    PagedTile t;
    t.b = __builtin_amdgcn_readfirstlane(s.find[0]);
    if (t.b < 0) return t;
    int n;
    paged_rows(v, t.b, t.row0, n);
    t.r0 = __builtin_amdgcn_readfirstlane(s.find[1]) * kPromptRows;
    t.rows = min(n * a.reps - t.r0, kPromptRows);
    t.pos0 = paged_kv_len(v, t.b) - n;
    t.len = paged_len(v, t.b);
    return t;
}

// grid (tiles x kv heads, splits), 256 threads.
template <int HD, int KT, int NS>
__global__ __launch_bounds__(256, HD <= 128 && NS <= 2 ? 2 : 1) void paged_prompt_kernel(PagedAttnArgs a) {
    using P = PagedPrompt<HD, KT, NS>;
    constexpr int KV = P::KV, JN = P::JN, NC = P::NC, CH = P::CH, KS = P::KS, DT = P::DT, W = P::W;
    constexpr bool BF = P::BF, AF = P::AF;
    __shared__ pg_u4 k_s[2][KV * NC];
    __shared__ pg_u4 v_s[2][KV * NC];
    __shared__ longlong2 row_s[4][KV];
    __shared__ uint32_t ok_s[4][2];
    __shared__ int bad_s[2];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % a.c.num_kv;
    // (the search is over before the first tile is loaded)
    const PagedTile t = paged_tile(a, blockIdx.x / a.c.num_kv, *reinterpret_cast<PagedTileLds*>(v_s));
    if (t.b < 0) return;
    if (tid == 0) bad_s[0] = bad_s[1] = -1;

    // this lane's row
    const int pr = t.r0 + min(32 * wave + n, t.rows - 1);
    const int tok = paged_div(pr, a.rep_mul, a.rep_shift), head = h * a.reps + pr - tok * a.reps;
    const bool live = 32 * wave + n < t.rows;
    const int tq = t.pos0 + tok;
    const int t_lo = t.pos0 + paged_div(t.r0, a.rep_mul, a.rep_shift),
              t_hi = t.pos0 + paged_div(t.r0 + t.rows - 1, a.rep_mul, a.rep_shift);  // of the tile
    int w_lo = tq, w_hi = tq;                                                               // of the wave
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        w_lo = min(w_lo, __shfl_xor(w_lo, d, 64));
        w_hi = max(w_hi, __shfl_xor(w_hi, d, 64));
    }
    w_lo = __builtin_amdgcn_readfirstlane(w_lo);
    w_hi = __builtin_amdgcn_readfirstlane(w_hi);
    const int win = a.window ? a.window : kPagedMax;
    const bool busy = 32 * wave < t.rows;

    // tiles of positions [i0, i1) of this split
    const int first = a.window ? max(0, t_lo - a.window + 1) / KV : 0;
    const int last = (min(t.len, t_hi + 1) + KV - 1) / KV;  // (t_hi + 1 <= 0: none)
    const int n_all = max(0, last - first), chunk = (n_all + a.splits - 1) / a.splits;
    const int i0 = first + min(n_all, static_cast<int>(blockIdx.y) * chunk);
    const int i1 = first + min(n_all, (static_cast<int>(blockIdx.y) + 1) * chunk);

    // queries as operands
    pg_u4 q[P::QF ? 1 : NS][P::QF ? 1 : KS];
    float qx[P::QF ? KS : 1][8];
    float qf;
    {
        const long long row = (t.row0 + tok) * a.q_ld + static_cast<long long>(head) * HD;
        float mx = 0.f;
        if constexpr (!BF) {
#pragma unroll
            for (int s = 0; s < KS; s++) {
                float x[8];
                act_load<AF, 8>(x, a.q, row + 16 * s + 8 * hh, a.act_type);
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[e]));
            }
        }
        const float ks = KT == LARQL_ELEM_E4M3 && a.c.k_scale ? a.c.k_scale[h] : 1.f;
        float up = 1.f, down = 1.f;
        if constexpr (!BF) {
            const int ex = query_exponent(max_x32(mx));
            up = ldexpf(1.f, ex);
            down = ldexpf(1.f, -ex);
        }
        up = ks * a.scale < 0.f ? -up : up;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            float x[8];
            act_load<AF, 8>(x, a.q, row + 16 * s + 8 * hh, a.act_type);
            if constexpr (P::QF) {
#pragma unroll
                for (int e = 0; e < 8; e++) qx[s][e] = x[e] * up;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t w[NS];
                    split2<BF, NS>(x[2 * e] * up, x[2 * e + 1] * up, w);
#pragma unroll
                    for (int p = 0; p < NS; p++) q[p][s][e] = w[p];
                }
            }
        }
        qf = score_factor(down * ks * a.scale * (a.softcap > 0.f ? 1.f : kLog2e));
    }

    // Where the rows of a tile lie: one lane of the last wave per position looks up its page two tiles
    // ahead, and writes the addresses of its K and V rows (and whether it exists) a tile later.
    unsigned id = 0;
    int off = 0;
    auto look = [&](int it) {
        if (wave == 3) id = paged_id(a.c, t.b, it * KV + lane, off);
    };
    auto place = [&](int it) {
        if (wave != 3) return;
        const bool have = id < a.c.num_pages && it * KV + lane < t.len;
        const long long pg = id < a.c.num_pages ? id : 0u;
        row_s[it & 3][lane] =
            make_longlong2(reinterpret_cast<long long>(a.c.k + pg * a.c.k_page + off * a.c.k_pos + h * a.c.k_head),
                           reinterpret_cast<long long>(a.c.v + pg * a.c.v_page + off * a.c.v_pos + h * a.c.v_head));
        const unsigned long long ok = __ballot(have);
        if (lane < 2) ok_s[it & 3][lane] = static_cast<uint32_t>(ok >> (32 * lane));
    };
    // LDS addresses are worked out where they are used: kept over the loop they would take the
    // registers of a second wave per SIMD.
    auto here = [](int x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    // Staging: LDS piece tid + 256 i of a tile (row, 16-byte place in it).
    uint32_t kr[P::DIRECT ? 1 : CH][W], vr[P::DIRECT ? 1 : CH][W];
    auto fetch = [&](int it) {
        const unsigned me = here(tid), r0 = me / NC;
        const uint32_t k_to = lds_address(&k_s[it & 1][64 * wave]), v_to = lds_address(&v_s[it & 1][64 * wave]);
        longlong2 at[CH];
        unsigned row[CH], cc[CH];
#pragma unroll
        for (int i = 0; i < CH; i++) {
            row[i] = 256 % NC ? (me + 256 * i) / NC : r0 + 256 / NC * i;
            cc[i] = 256 % NC ? me + 256 * i - row[i] * NC : me - r0 * NC;
            at[i] = row_s[it & 3][row[i]];
            if (256 % (16 * NC) == 0) row[i] = r0;  // (the same for the XOR)
        }
#pragma unroll
        for (int i = 0; i < CH; i++) {
            if constexpr (P::DIRECT) {
                load_lds16(at[i].x + 16 * P::swz_k(row[i], cc[i]), k_to + 4096 * i);
                load_lds16(at[i].y + 16 * P::swz_v(row[i], cc[i]), v_to + 4096 * i);
            } else {
                load_global<W>(kr[i], at[i].x + 4 * W * P::swz_k(row[i], cc[i]));
                load_global<W>(vr[i], at[i].y + 4 * W * P::swz_v(row[i], cc[i]));
            }
        }
    };
    auto widen = [&](const uint32_t* w) {
        return pg_u4{e4m3_f16<false>(w[0]), e4m3_f16<true>(w[0]), e4m3_f16<false>(w[1]), e4m3_f16<true>(w[1])};
    };
    auto stash = [&](int it) {
        const int buf = it & 1;
        if constexpr (P::DIRECT) {
            wait_vmcnt0();
        } else {
#pragma unroll
            for (int i = 0; i < CH; i++) {
                k_s[buf][tid + 256 * i] = widen(kr[i]);
                v_s[buf][tid + 256 * i] = widen(vr[i]);
            }
        }
        // a tile that some row masks: values without a position as zeros, and is one not finite?
        const uint32_t* ok = ok_s[it & 3];
        if (it * KV + KV - 1 > t_lo || it * KV <= t_hi - win || (ok[0] & ok[1]) != ~0u) {
            bool bad = false;
            for (int piece = tid; piece < KV * NC; piece += 256) {
                const int row = static_cast<unsigned>(piece) / NC;
                pg_u4 v = v_s[buf][piece];
                if (!(ok[row >> 5] >> (row & 31) & 1)) v_s[buf][piece] = v = pg_u4{0u, 0u, 0u, 0u};
                bad |= not_finite16(v[0], BF) || not_finite16(v[1], BF) || not_finite16(v[2], BF) || not_finite16(v[3], BF);
            }
            if (bad) bad_s[buf] = it;
        }
    };

    pg_f16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    // a tile's rows are placed two barriers before its products, its pieces loaded one before
    if (i0 < i1) {
        look(i0);
        place(i0);
        if (i0 + 1 < i1) look(i0 + 1);
    }
    __syncthreads();  // (and bad_s)
    if (i0 < i1) {
        fetch(i0);
        stash(i0);
        if (i0 + 1 < i1) place(i0 + 1);
    }
    __syncthreads();
    for (int it = i0; it < i1; it++) {
        const int buf = it & 1;
        const bool more = it + 1 < i1;
        if (it + 2 < i1) look(it + 2);
        if (more) fetch(it + 1);
        __builtin_amdgcn_sched_barrier(0);
        const int bad = bad_s[buf];
#pragma unroll
        for (int jb = 0; jb < KV / (32 * JN); jb++) {
            uint32_t seen[JN];  // positions that exist (read here, looked at after the products)
#pragma unroll
            for (int j = 0; j < JN; j++) seen[j] = ok_s[it & 3][JN * jb + j];
            const int j0 = 32 * JN * jb, p0 = it * KV + j0;  // rows of the tile, positions
            const bool go = busy && p0 <= w_hi && p0 + 32 * JN - 1 > w_lo - win;
            pg_f16 s[JN];  // 32 positions each
            float f, up;         // weights: 2^(s f + up)
            bool small = false;  // some are too small for the parts
            if (go) {
                const int row = here(n);
                pg_u4 kf[JN][KS];
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int j = 0; j < JN; j++)
                        if constexpr (!P::QF) kf[j][ks] = k_s[buf][(j0 + 32 * j + row) * NC + P::swz_k(row, 2 * ks + hh)];
#pragma unroll
                for (int j = 0; j < JN; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[j][e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    if constexpr (P::QF) {
                        __builtin_amdgcn_sched_barrier(0);  // (one piece's registers at a time)
                        pg_u4 qq[NS];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            // (opaque, or the parts would be kept over the loop)
                            float x0 = qx[ks][2 * e], x1 = qx[ks][2 * e + 1];
                            asm volatile("" : "+v"(x0), "+v"(x1));
                            uint32_t w[NS];
                            split2<BF, NS>(x0, x1, w);
#pragma unroll
                            for (int p = 0; p < NS; p++) qq[p][e] = w[p];
                        }
                        const pg_u4 kk = k_s[buf][(j0 + row) * NC + P::swz_k(row, 2 * ks + hh)];
#pragma unroll
                        for (int p = 0; p < NS; p++) s[0] = mfma32<BF>(kk, qq[p], s[0]);
                    } else {
#pragma unroll
                        for (int j = 0; j < JN; j++)
#pragma unroll
                            for (int p = 0; p < NS; p++) s[j] = mfma32<BF>(kf[j][ks], q[p][ks], s[j]);
                    }
                }
                if constexpr (!P::QF) lds_ahead<KS * JN, 1, NS>();
                __builtin_amdgcn_sched_barrier(0);
                uint32_t ok[JN], all = ~0u;
#pragma unroll
                for (int j = 0; j < JN; j++) {
                    ok[j] = __builtin_amdgcn_readfirstlane(seen[j]);
                    all &= ok[j];
                }
                if (a.softcap > 0.f) {
                    const float inv = qf / a.softcap, most = a.softcap * kLog2e;
#pragma unroll
                    for (int j = 0; j < JN; j++)
#pragma unroll
                        for (int e = 0; e < 16; e++) s[j][e] = tanhf(s[j][e] * inv) * most;
                }
                float mn = s[0][0];
                if (p0 + 32 * JN - 1 > w_lo || p0 <= w_hi - win || ~all) {
                    mn = INFINITY;
#pragma unroll
                    for (int j = 0; j < JN; j++) {
                        const int hi = tq - p0 - 32 * j - 4 * hh, lo = hi - win;
                        const uint32_t okh = ok[j] >> (4 * hh);
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int at = 8 * (e / 4) + e % 4;  // position p0 + 32 j + 4 hh + at
                            const bool in = at <= hi && at > lo && (okh >> at & 1);
                            if constexpr (!BF) mn = fminf(mn, in ? s[j][e] : INFINITY);
                            s[j][e] = in ? s[j][e] : -INFINITY;
                        }
                    }
                } else if constexpr (!BF) {
                    // (eight positions of the row, more than there may be larger weights: one of them tells)
                    static_assert(P::Weights::FEW < 8, "");
#pragma unroll
                    for (int e = 1; e < 4; e++) mn = fminf(mn, s[0][e]);
                }
                f = a.softcap > 0.f ? 1.f : qf;
                float mx = s[0][0];
#pragma unroll
                for (int j = 0; j < JN; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[j][e]);
                mx = max_x32(mx) * f;
                const bool under = P::Weights::under(mx, m);
                if (__any(under || P::Weights::above(mx, m))) {
                    const float was = m, room = P::Weights::room_weights(max_x32(l));
                    m = under ? was - fmaxf(0.f, fminf(was - ceilf(mx), room)) : P::Weights::reference(mx, was);
                    const int al = sums_move(was, m);
                    l = ldexpf(l, al);
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) o[d][e] = ldexpf(o[d][e], al);
                }
                up = P::Weights::offset(m);
                small = !BF && __any(P::Weights::tiny(mn, f, m));
            }
            if (__builtin_amdgcn_readfirstlane(bad) == it) {  // (the same for the workgroup)
                if (go)
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma nounroll
                        for (int at = j0; at < j0 + 32 * JN; at++) {
                            const int pos = it * KV + at;
                            const bool mine = pos <= tq && pos > tq - win && (ok_s[it & 3][at >> 5] >> (at & 31) & 1);
#pragma unroll
                            for (int e = 0; e < 16; e += 4) {
                                const int dim = 32 * d + 2 * e + 4 * hh;
                                const uint2 w = reinterpret_cast<const uint2*>(&v_s[buf][at * NC + P::swz_v(at, dim / 8)])[hh];
                                if (mine && not_finite16(w.x & 0xFFFFu, BF)) o[d][e] += unpack_lo<BF>(w.x);
                                if (mine && not_finite16(w.x >> 16, BF)) o[d][e + 1] += unpack_hi<BF>(w.x);
                                if (mine && not_finite16(w.y & 0xFFFFu, BF)) o[d][e + 2] += unpack_lo<BF>(w.y);
                                if (mine && not_finite16(w.y >> 16, BF)) o[d][e + 3] += unpack_hi<BF>(w.y);
                            }
                        }
                __syncthreads();
                for (int i = tid; i < 32 * JN * NC; i += 256) {
                    pg_u4 v = v_s[buf][j0 * NC + i];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = finite16(v[e], BF);
                    v_s[buf][j0 * NC + i] = v;
                }
                __syncthreads();
            }
            if (!BF && small) {
                // Weights too small for the parts, in rows where they are most of a tile's: summed here in f32, left out below.
                float larger = 0.f, seen = 0.f;
#pragma unroll
                for (int j = 0; j < JN; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        larger += __builtin_fmaf(s[j][e], f, up) < P::Weights::LEAST ? 0.f : 1.f;
                        seen += s[j][e] == -INFINITY ? 0.f : 1.f;
                    }
                const bool few = P::Weights::few(sum_x32(larger), sum_x32(seen));
                if (__any(few)) {
#pragma unroll
                    for (int j = 0; j < JN; j++)
#pragma nounroll
                        for (int e = 0; e < 16; e++) {
                            const float z = __builtin_fmaf(s[j][0], f, up);
                            const bool mine = few && z < P::Weights::LEAST;
                            const float p = exp2_hw(mine ? z : -INFINITY), y = mine ? -INFINITY : s[j][0];
                            l += p;
#pragma unroll
                            for (int i = 0; i < 15; i++) s[j][i] = s[j][i + 1];  // (registers have no index)
                            s[j][15] = y;
                            if (!__any(p > 0.f)) continue;
                            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(p), __float_as_uint(p), false, false);
                            float pk = __uint_as_float(both[0]), pn = __uint_as_float(both[1]);  // of the lanes' lower, upper half
#pragma nounroll
                            for (int k = 0; k < 2; k++) {
                                const int at = j0 + 32 * j + 8 * (e / 4) + e % 4 + 4 * k;
                                auto value = [&](int i) __attribute__((always_inline)) {  // dims 8 i + 4 hh ..
                                    return reinterpret_cast<const uint2*>(&v_s[buf][at * NC + P::swz_v(at, i)])[hh];
                                };
                                uint2 w[2][4];
#pragma unroll
                                for (int i = 0; i < 4; i++) w[0][i] = value(i);
#pragma unroll
                                for (int d = 0; d < DT; d++) {
#pragma unroll
                                    for (int i = 0; i < 4; i++)
                                        if (d + 1 < DT) w[(d + 1) & 1][i] = value(4 * (d + 1) + i);
#pragma unroll
                                    for (int i = 0; i < 4; i++) {
                                        const uint2 v = w[d & 1][i];
                                        o[d][4 * i] += pk * unpack_lo<BF>(v.x);
                                        o[d][4 * i + 1] += pk * unpack_hi<BF>(v.x);
                                        o[d][4 * i + 2] += pk * unpack_lo<BF>(v.y);
                                        o[d][4 * i + 3] += pk * unpack_hi<BF>(v.y);
                                    }
                                    __builtin_amdgcn_sched_barrier(0);  // (two blocks' values at a time)
                                }
                                pk = pn;
                            }
                        }
                }
            }
            if (go) {
                uint32_t pw[JN][NS][8];
                auto weights = [&](int j) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float x0 = exp2_hw(__builtin_fmaf(s[j][e], f, up)), x1 = exp2_hw(__builtin_fmaf(s[j][e + 1], f, up));
                        l += x0 + x1;
                        uint32_t w[NS];
                        split2<BF, NS>(x0, x1, w);
#pragma unroll
                        for (int p = 0; p < NS; p++) pw[j][p][e / 2] = w[p];
                    }
                };
                weights(0);
                const int ln = here(lane), grp = ln >> 4, i16 = ln & 15;
#pragma unroll
                for (int j = 0; j < JN; j++) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int s2 = 0; s2 < 2; s2++) {
                            typedef short s4 __attribute__((ext_vector_type(4)));
                            typedef __attribute__((address_space(3))) s4* lds_s4;
                            uint32_t vw[4];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const int r4 = 4 * (grp >> 1) + (i16 >> 2), row = j0 + 32 * j + 16 * s2 + 8 * u + r4;
                                const int cc = 4 * d + 2 * (grp & 1) + (i16 >> 1 & 1);
                                char* at = reinterpret_cast<char*>(&v_s[buf][row * NC + P::swz_v(r4, cc)]) + 8 * (i16 & 1);
                                const uint2 r = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at));
                                vw[2 * u] = r.x;
                                vw[2 * u + 1] = r.y;
                            }
                            const pg_u4 vv = {vw[0], vw[1], vw[2], vw[3]};
#pragma unroll
                            for (int p = 0; p < NS; p++) {
                                const pg_u4 pp = {pw[j][p][4 * s2], pw[j][p][4 * s2 + 1], pw[j][p][4 * s2 + 2], pw[j][p][4 * s2 + 3]};
                                o[d] = mfma32<BF>(vv, pp, o[d]);
                            }
                        }
                    if (j + 1 < JN) weights(j + 1);
                }
                if constexpr (!P::QF) products_over_weights<2 * DT, NS, JN>();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (more) stash(it + 1);
        if (it + 2 < i1) place(it + 2);
        __syncthreads();
    }

    l = sum_x32(l);
    if (!live) return;
    const long long row = t.row0 + tok;
    const float vs = KT == LARQL_ELEM_E4M3 && a.c.v_scale ? a.c.v_scale[h] : 1.f;
    if (a.splits == 1) {
        const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                act_store4<AF>(a.out, row * a.out_ld + static_cast<long long>(head) * HD + 32 * d + 2 * e + 4 * hh, a.act_type,
                           o[d][e] * f * vs, o[d][e + 1] * f * vs, o[d][e + 2] * f * vs, o[d][e + 3] * f * vs);
    } else {
        const long long at = (row * a.num_q + head) * a.splits + blockIdx.y;
        if (hh == 0) *reinterpret_cast<float2*>(a.tile_ml + 2 * at) = make_float2(m, l);
        if (l != 0.f) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<pg_f4*>(a.tile_part + at * HD + 32 * d + 2 * e + 4 * hh) =
                        pg_f4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
        }
    }
}

// Joins the splits of a (row, head) in order.  One lane per four dims; grid over rows x heads.
template <int HD, bool AF>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedAttnArgs a) {
    constexpr int L = HD / 4, G = 256 / L;
    const int k = threadIdx.x / L, d = threadIdx.x - k * L;
    const long long i = static_cast<long long>(blockIdx.x) * G + k;
    if (k >= G || i >= static_cast<long long>(a.c.num_tokens) * a.num_q) return;
    const int row = static_cast<int>(i / a.num_q), head = static_cast<int>(i - static_cast<long long>(row) * a.num_q);
    // rows of no sequence, and of sequences of a few rows, are not this kernel's
    int b = 0;
    for (int hi = a.c.num_seqs; hi - b > 1;) {  // the last sequence that starts at or before the row
        const int mid = (b + hi) >> 1;
        if (a.c.q_start[mid] <= row) b = mid;
        else hi = mid;
    }
    int row0, n;
    paged_rows(a.c, b, row0, n);
    if (row < row0 || row >= row0 + n || n * a.reps <= a.few) return;
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < a.splits; s++) m = fmaxf(m, a.tile_ml[2 * (i * a.splits + s)]);
    pg_f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; s++) {
        const float2 p = *reinterpret_cast<const float2*>(a.tile_ml + 2 * (i * a.splits + s));
        if (p.y == 0.f) continue;
        const int by = sums_move(p.x, m) - kJoinDown;
        l += ldexpf(p.y, by);
        o += ldexp4(*reinterpret_cast<const pg_f4*>(a.tile_part + (i * a.splits + s) * HD + 4 * d), by);
    }
    const float vs = a.kv_type == LARQL_ELEM_E4M3 && a.c.v_scale ? a.c.v_scale[head / a.reps] : 1.f;
    o *= l == 0.f ? 0.f : 1.f / l;
    act_store4<AF>(a.out, row * a.out_ld + static_cast<long long>(head) * HD + 4 * d, a.act_type, o[0] * vs, o[1] * vs, o[2] * vs,
               o[3] * vs);
}

template <int HD>
static void launch_paged_prompt(const PagedAttnArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.tiles * a.c.num_kv), static_cast<unsigned>(a.splits)), block(256);
    const int act = a.act_type;
    if (a.kv_type == LARQL_ELEM_F16) {
        if (act == LARQL_ELEM_F32) paged_prompt_kernel<HD, LARQL_ELEM_F16, 2><<<grid, block, 0, s>>>(a);
        else paged_prompt_kernel<HD, LARQL_ELEM_F16, 1><<<grid, block, 0, s>>>(a);
    } else if (a.kv_type == LARQL_ELEM_E4M3) {
        if (act == LARQL_ELEM_F32) paged_prompt_kernel<HD, LARQL_ELEM_E4M3, 2><<<grid, block, 0, s>>>(a);
        else paged_prompt_kernel<HD, LARQL_ELEM_E4M3, 1><<<grid, block, 0, s>>>(a);
    } else {
        if (act == LARQL_ELEM_F32) paged_prompt_kernel<HD, LARQL_ELEM_BF16, 3><<<grid, block, 0, s>>>(a);
        else if (act == LARQL_ELEM_F16) paged_prompt_kernel<HD, LARQL_ELEM_BF16, 2><<<grid, block, 0, s>>>(a);
        // (one part of the weights: rounded to 2^-8, results are off by 2.3e-3 where f32 weights give 1.6e-3, most of it
        // the output's own rounding; with two 8191 tokens take 980 us instead of 638.  Decode, bound by memory, has two.)
        else paged_prompt_kernel<HD, LARQL_ELEM_BF16, 1><<<grid, block, 0, s>>>(a);
    }
    LARQL_HIP_CHECK(hipGetLastError());
    if (a.splits == 1) return;
    const long long items = static_cast<long long>(a.c.num_tokens) * a.num_q;
    constexpr int G = 256 / (HD / 4);
    const dim3 jg(static_cast<unsigned>((items + G - 1) / G));
    if (act == LARQL_ELEM_F32) paged_prompt_join_kernel<HD, true><<<jg, block, 0, s>>>(a);
    else paged_prompt_join_kernel<HD, false><<<jg, block, 0, s>>>(a);
    LARQL_HIP_CHECK(hipGetLastError());
}

}  // namespace larql
