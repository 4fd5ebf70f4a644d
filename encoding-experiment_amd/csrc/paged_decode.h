// Attention of one or a few new tokens of every sequence over a paged KV cache (one head_dim per
// including file).
//
// out = softmax(scale q . k_j) v_j over the positions j <= t of a row's sequence (the last `window` of
// them), scores optionally capped by tanh.  Bound: reading K and V once.
//
// The cache is cut into units of 32 positions of one (sequence, kv head, group of columns), and every
// worker takes an equal run of them, so sequences of any lengths fill the GPU evenly.  The pieces of a
// run that are parts of a segment's units only go to the work buffer and are joined by a second
// launch; the whole ones are written out.  For one token per sequence a worker is a wave, which shares
// nothing with others: no barrier, and each runs on while others wait.  For several tokens, whose parts
// are as large as a unit or more, it is a workgroup of four waves that take a run's units in
// turn and join their sums in LDS first.  A column is a row (token, query head of the kv head): 16 of them to a
// wave, or 32 (two products per operand of the cache) for several tokens.
//
// A unit stays in registers from load to use.  Scores are K . Q^T (16 x 16 x 32 products), so lane
// (g, c) = 16 g + c holds, for column c, positions
// 16 j + 4 g + i (j < 2, i < 4): after the softmax those eight values are, as they lie, the B operand
// of V^T . P^T in which slot 4 j + i of lane group g stands for that position.  V's operand has the
// same slots: the lane reads hd / 16 consecutive dims of its eight positions' rows (16 lanes a whole
// row) and one byte permute per pair of rows transposes them.  No LDS and no cross-lane traffic but
// the maximum of a column over its four lane groups.
//
// Accuracy: the running maximum, sum and output are f32.  q and the weights go to the matrix cores as NS 16-bit
// parts (f32 activations: two f16 or three bf16 parts), q first scaled by a power of two into f16's range (22
// bits and more of a row's largest element), weights as PagedWeights says (19 bits and more of each); e4m3
// codes are exact in f16.
//
// Measured with the join, 8 kv heads of 128 with 4 query heads each: 1 sequence of 131071 positions bf16 106 us (5.1
// TB/s), 64 of up to 12000 e4m3 159 us (5.1 TB/s), 32 of up to 4096
// f16 with f32 activations 63 us, 1 of 517 12 us (two launches of 7.0 and 5.2).  8 sequences of 9 new tokens behind up to
// 15000 e4m3 positions 54 us, of which 20 are start, changes of segment and the join.
#pragma once

#include <type_traits>

#include "paged_device.h"

namespace larql {

// What a sequence's new rows read: positions [begin, len), units [t0, t0 + nt) for each of ct column
// groups of each kv head.  The group's columns are `rows` rows (token i, head) = (R / reps, R % reps) of
// the n tokens from row0 on, token i at position pos0 + i.
struct PagedRange {
    int begin, len, t0, nt, ct, rows, row0, n, pos0;
};
template <bool MULTI, int NC>
__device__ __forceinline__ PagedRange paged_range(const PagedAttnArgs& a, int b) {
    constexpr int COLS = 16 * NC;
    PagedRange r;
    const int kv = paged_kv_len(a.c, b);
    r.row0 = b;
    r.n = 1;
    if constexpr (MULTI) paged_rows(a.c, b, r.row0, r.n);
    r.rows = r.n * a.reps;
    r.pos0 = kv - r.n;
    r.len = min(kv, a.c.cap);
    r.begin = a.window ? max(0, r.pos0 - a.window + 1) : 0;
    r.t0 = r.begin >> 5;
    r.nt = r.len > r.begin ? ((r.len + 31) >> 5) - r.t0 : 0;
    r.ct = a.groups;
    if constexpr (MULTI) {
        r.ct = (r.rows + COLS - 1) / COLS;
        if (r.rows > a.few || r.rows == 0) r.nt = 0;  // (another kernel's, or nobody's)
    }
    return r;
}

// MULTI: several tokens per sequence (q_start); NC: groups of 16 columns in a wave's hands.
template <int HD, int KT, int NS, bool MULTI>
struct PagedDecode {
    static constexpr int NC = paged_nc(HD, MULTI);
    static constexpr bool BF = KT == LARQL_ELEM_BF16, AF = NS == (BF ? 3 : 2);  // (AF: f32 activations)
    static constexpr int E = HD / 16, KS = HD / 32, ES = KT == LARQL_ELEM_E4M3 ? 1 : 2;
    static constexpr int KW = 2 * ES, VB = E * ES, VW = (VB + 3) / 4;
    // Query operands in LDS where registers are short: two units in flight take 2 hd / 4 of them.
    static constexpr bool QL = HD > 128 || NS == 3 || MULTI;
    static constexpr int QS = QL ? NS * KS * NC * 64 : 1;
    // Two units in flight per wave where they fit beside the sums; else one, and two waves per SIMD.
    static constexpr bool TWO = HD <= 128;
    static constexpr int WAVES = paged_waves(HD, HD * ES, MULTI);
    static constexpr int WG = paged_wg(MULTI);  // waves of a worker
    using Weights = PagedWeights<BF, NS>;

    struct Unit {
        uint32_t k[2][KS][KW];
        uint32_t v[8][VW];
        uint32_t ok;  // slots whose page exists (bit 4 j + i)
    };

    // Page ids of a unit's two halves, for pages of whole 16-position groups.
    struct Ids {
        unsigned id[2];
        int off[2];
    };

    static __device__ __forceinline__ Ids ids(const PagedAttnArgs& a, int b, int t) {
        Ids r;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            r.id[j] = paged_id(a.c, b, 32 * t + 16 * j, r.off[j]);
        }
        return r;
    }

    static __device__ __forceinline__ void load(Unit& u, const PagedAttnArgs& a, int b, int h, int t, const Ids& ids,
                                                bool whole, int g, int c) {
        u.ok = 0xFF;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (whole) {
                const unsigned have = __builtin_amdgcn_readfirstlane(ids.id[j]);
                if (have >= a.c.num_pages) u.ok &= ~(0xFu << (4 * j));
                const long long id = have < a.c.num_pages ? have : 0u;
                const char* kp = a.c.k + (id * a.c.k_page + ids.off[j] * a.c.k_pos + h * a.c.k_head);
                const char* vp = a.c.v + (id * a.c.v_page + ids.off[j] * a.c.v_pos + h * a.c.v_head);
#pragma unroll
                for (int s = 0; s < KS; s++) load_bytes<4 * KW>(u.k[j][s], kp + c * a.c.k_pos + (32 * s + 8 * g) * ES);
#pragma unroll
                for (int i = 0; i < 4; i++) load_bytes<VB>(u.v[4 * j + i], vp + (4 * g + i) * a.c.v_pos + c * VB);
            } else {
                int off;
                const unsigned have = paged_id(a.c, b, 32 * t + 16 * j + c, off);
                const long long id = have < a.c.num_pages ? have : 0u;
                const char* kp = a.c.k + (id * a.c.k_page + off * a.c.k_pos + h * a.c.k_head);
#pragma unroll
                for (int s = 0; s < KS; s++) load_bytes<4 * KW>(u.k[j][s], kp + (32 * s + 8 * g) * ES);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    int vo;
                    const unsigned vi = paged_id(a.c, b, 32 * t + 16 * j + 4 * g + i, vo);
                    if (vi >= a.c.num_pages) u.ok &= ~(1u << (4 * j + i));
                    load_bytes<VB>(u.v[4 * j + i],
                                   a.c.v + ((vi < a.c.num_pages ? vi : 0ll) * a.c.v_page + vo * a.c.v_pos + h * a.c.v_head) + c * VB);
                }
            }
        }
    }

    struct State {
        pg_u4 q[QL ? 1 : NS][QL ? 1 : KS];
        float qf[NC];     // score = product * qf (log2 units, or the natural score with softcap)
        float m[NC], l[NC];     // running maximum (log2 units) of the column; this lane's part of the sum
        pg_f4 o[NC][E];   // o[.][e][i] = dim (4 g + i) E + e of column c
    };

    // Token, query head (of the kv head) and attended positions [lo, hi) of column c of 16-column group jg;
    // rows past the last repeat it (and are not written).
    struct Column {
        int tok, rep, lo, hi;
    };
    static __device__ __forceinline__ Column column(const PagedAttnArgs& a, const PagedRange& r, int jg, int c) {
        Column k;
        const int R = min(16 * jg + c, r.rows - 1);
        k.tok = MULTI ? paged_div(R, a.rep_mul, a.rep_shift) : 0;
        k.rep = R - k.tok * a.reps;
        k.lo = MULTI && a.window ? max(0, r.pos0 + k.tok - a.window + 1) : r.begin;
        k.hi = MULTI ? min(r.len, r.pos0 + k.tok + 1) : r.len;
        return k;
    }

    static __device__ __forceinline__ void load_q(ActRaw<AF> (*x)[KS], const PagedAttnArgs& a, const PagedRange& r, int h, int cg,
                                                  int g, int c) {
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const Column k = column(a, r, NC * cg + j, c);
            const long long row = (r.row0 + k.tok) * a.q_ld + static_cast<long long>(h * a.reps + k.rep) * HD;
#pragma unroll
            for (int s = 0; s < KS; s++) act_raw<AF>(x[j][s], a.q, row + 32 * s + 8 * g);
        }
    }

    template <bool H>
    static __device__ __forceinline__ void start(State& st, pg_u4* q_s, const ActRaw<AF> (*x)[KS], const PagedAttnArgs& a,
                                                 int h, int wave, int g, int c) {
        const float ks = KT == LARQL_ELEM_E4M3 && a.c.k_scale ? a.c.k_scale[h] : 1.f;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            float up = 1.f, down = 1.f;
            if constexpr (!BF) {
                float mx = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(act_value<AF, H>(x[j][s], e)));
                const int ex = query_exponent(max_x32(max_x16(mx)));
                up = ldexpf(1.f, ex);
                down = ldexpf(1.f, -ex);
            }
            up = ks * a.scale < 0.f ? -up : up;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                pg_u4 q[NS];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t w[NS];
                    split2<BF, NS>(act_value<AF, H>(x[j][s], 2 * e) * up, act_value<AF, H>(x[j][s], 2 * e + 1) * up, w);
#pragma unroll
                    for (int n = 0; n < NS; n++) q[n][e] = w[n];
                }
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    if constexpr (!QL)
                        st.q[n][s] = q[n];
                    else if (s % WG == wave)
                        q_s[((n * KS + s) * NC + j) * 64 + 16 * g + c] = q[n];
                }
            }
            st.qf[j] = score_factor(down * ks * a.scale * (a.softcap > 0.f ? 1.f : kLog2e));
            st.m[j] = -INFINITY;
            st.l[j] = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) st.o[j][e] = pg_f4{0.f, 0.f, 0.f, 0.f};
        }
    }

    static __device__ __forceinline__ pg_u4 k_operand(const uint32_t* w) {
        if constexpr (KT == LARQL_ELEM_E4M3)
            return pg_u4{e4m3_f16<false>(w[0]), e4m3_f16<true>(w[0]), e4m3_f16<false>(w[1]), e4m3_f16<true>(w[1])};
        else
            return pg_u4{w[0], w[1], w[2], w[3]};
    }

    // Dim e of the lane's eight rows as an operand: slots 2d, 2d + 1 in word d.
    template <int EE>
    static __device__ __forceinline__ pg_u4 v_operand(const Unit& u) {
        pg_u4 r;
#pragma unroll
        for (int d = 0; d < 4; d++) {
            if constexpr (KT == LARQL_ELEM_E4M3) {
                // bytes {row 2d, row 2d + 1} of two dims, then one conversion per dim
                const uint32_t lo = u.v[2 * d][EE / 4], hi = u.v[2 * d + 1][EE / 4];
                const uint32_t w = __builtin_amdgcn_perm(hi, lo, (EE / 2) % 2 ? 0x07030602u : 0x05010400u);
                r[d] = EE % 2 ? e4m3_f16<true>(w) : e4m3_f16<false>(w);
            } else {
                r[d] = __builtin_amdgcn_perm(u.v[2 * d + 1][EE / 2], u.v[2 * d][EE / 2],
                                             EE % 2 ? 0x07060302u : 0x05040100u);
            }
        }
        return r;
    }

    // Sums of V's dims.  Where an element is not finite in a unit that a column does not attend whole
    // (0 * inf is not 0), pv_odd first adds such elements position by position to the columns that
    // attend it, and drop_odd leaves the others.
    template <int EE>
    static __device__ __forceinline__ void pv(State& st, const Unit& u, const pg_u4 (*p)[NS]) {
        if constexpr (EE < E) {
            const pg_u4 v = v_operand<EE>(u);
#pragma unroll
            for (int j = 0; j < NC; j++)
#pragma unroll
                for (int n = 0; n < NS; n++) st.o[j][EE] = mfma16<BF>(v, p[j][n], st.o[j][EE]);
            pv<EE + 1>(st, u, p);
        }
    }
    // Whether the unit's values hold an infinity or NaN (e4m3: the codes 127 and 255).
    static __device__ __forceinline__ bool odd_values(const Unit& u) {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int w = 0; w < VW; w++) {
                const uint32_t x = u.v[e][w];
                if constexpr (KT == LARQL_ELEM_E4M3)
                    odd |= (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
                else
                    odd |= not_finite16(x, BF);
            }
        return odd;
    }
    // Those elements as zeros.
    static __device__ __forceinline__ void drop_odd(Unit& u) {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int w = 0; w < VW; w++) {
                const uint32_t x = u.v[e][w];
                if constexpr (KT == LARQL_ELEM_E4M3)
                    u.v[e][w] = x & ~(((((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu);
                else
                    u.v[e][w] = finite16(x, BF);
            }
    }
    // (operands worked out again from here on: kept over the positions they would not fit)
    static __device__ __forceinline__ void again(Unit& u) {
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int w = 0; w < VW; w++) asm volatile("" : "+v"(u.v[e][w]));
    }
    template <int EE>
    static __device__ __forceinline__ void pv_odd(State& st, const Unit& u, unsigned sees, int at, int g) {
        if constexpr (EE < E) {
            pg_u4 v = v_operand<EE>(u);
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const int s = 16 * (d / 2) + 4 * g + 2 * (d % 2);  // position of slot 2 d in the unit
                v[d] = (v[d] ^ finite16(v[d], BF)) & ((s == at ? 0xFFFFu : 0u) | (s + 1 == at ? 0xFFFF0000u : 0u));
            }
            const uint32_t one = pack2<BF>(1.f, 1.f);
            const pg_f4 w = mfma16<BF>(v, pg_u4{one, one, one, one}, pg_f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int j = 0; j < NC; j++) {
#pragma unroll
                for (int i = 0; i < 4; i++) st.o[j][EE][i] += sees >> j & 1 ? w[i] : 0.f;
            }
            __builtin_amdgcn_sched_barrier(0);  // (one dim's registers at a time)
            pv_odd<EE + 1>(st, u, sees, at, g);
        }
    }
    static __device__ __forceinline__ void scale(State& st, int j, int by) {  // by 2^by
        st.l[j] = ldexpf(st.l[j], by);
#pragma unroll
        for (int e = 0; e < E; e++) st.o[j][e] = ldexp4(st.o[j][e], by);
    }
    // By how much group j's sums may rise, `want` at most.
    static __device__ __forceinline__ float room(const State& st, int j, float want) {
        float sum = max_x32(max_x16(st.l[j])), r = Weights::room_weights(sum);
        if (__any(r < want)) {
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) sum = fmaxf(sum, fabsf(st.o[j][e][i]));
            r = Weights::room(max_x32(max_x16(sum)));
        }
        return fmaxf(0.f, fminf(r, want));
    }

    static __device__ __forceinline__ void step(State& st, const pg_u4* q_s, Unit& u, const PagedAttnArgs& a,
                                                const PagedRange& r, int cg, int t, int g, int c) {
        pg_f4 s[NC][2];
#pragma unroll
        for (int j = 0; j < NC; j++) s[j][0] = s[j][1] = pg_f4{0.f, 0.f, 0.f, 0.f};
        int ql = 16 * g + c;
        if constexpr (QL) asm volatile("" : "+v"(ql));  // (read per unit, not kept in registers over the loop)
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const pg_u4 k0 = k_operand(u.k[0][k]), k1 = k_operand(u.k[1][k]);
#pragma unroll
            for (int j = 0; j < NC; j++)
#pragma unroll
                for (int n = 0; n < NS; n++) {
                    pg_u4 q;
                    if constexpr (QL)
                        q = q_s[((n * KS + k) * NC + j) * 64 + ql];
                    else
                        q = st.q[n][k];
                    s[j][0] = mfma16<BF>(k0, q, s[j][0]);
                    s[j][1] = mfma16<BF>(k1, q, s[j][1]);
                }
        }
        // a unit that some column does not attend whole: [hi of the first token, lo of the last)
        const int first_hi = MULTI ? min(r.len, r.pos0 + 1) : r.len;
        const int last_lo = MULTI && a.window ? max(0, r.pos0 + r.n - a.window) : r.begin;
        const bool edge = 32 * t < last_lo || 32 * t + 32 > first_hi || __any(u.ok != 0xFF);
        if (edge) {
            // what lies behind the sequence, before its window or on no page may be anything
            const int lo = r.begin - 32 * t - 4 * g, hi = r.len - 32 * t - 4 * g;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at = 16 * (e / 4) + e % 4;  // position 32 t + 4 g + at
                if (!(at >= lo && at < hi && (u.ok >> e & 1))) {
                    u.ok &= ~(1u << e);
#pragma unroll
                    for (int w = 0; w < VW; w++) u.v[e][w] = 0u;
                }
            }
        }
        if constexpr (MULTI) {
            if (edge && __any(odd_values(u))) {
#pragma nounroll
                for (int at = 0; at < 32; at++) {
                    again(u);
                    unsigned sees = 0;
#pragma unroll
                    for (int j = 0; j < NC; j++) {
                        const Column k = column(a, r, NC * cg + j, c);
                        sees |= (32 * t + at >= k.lo && 32 * t + at < k.hi ? 1u : 0u) << j;
                    }
                    pv_odd<0>(st, u, sees, at, g);
                }
                drop_odd(u);
            }
        }
        float x[NC][8], least[NC];
        bool small = false, bands = false;  // weights that are too small for the parts; taken apart
#pragma unroll
        for (int j = 0; j < NC; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[j][e] = s[j][e / 4][e % 4];
            if (a.softcap > 0.f) {
                const float inv = st.qf[j] / a.softcap, most = a.softcap * kLog2e;
#pragma unroll
                for (int e = 0; e < 8; e++) x[j][e] = tanhf(x[j][e] * inv) * most;
            }
            const float f = a.softcap > 0.f ? 1.f : st.qf[j];
            if (edge) {
                int cc = c;
                asm volatile("" : "+v"(cc));  // (worked out here, not kept over the loop)
                const Column k = column(a, r, NC * cg + j, cc);
                const int lo = k.lo - 32 * t - 4 * g, hi = k.hi - 32 * t - 4 * g;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int at = 16 * (e / 4) + e % 4;
                    x[j][e] = (!MULTI || (at >= lo && at < hi)) && (u.ok >> e & 1) ? x[j][e] : -INFINITY;
                }
            }
            float mx = x[j][0];
#pragma unroll
            for (int e = 1; e < 8; e++) mx = fmaxf(mx, x[j][e]);
            mx = max_x32(max_x16(mx)) * f;
            // (of a whole unit eight positions of the column, more than there may be larger weights: one of them tells)
            static_assert(Weights::FEW < 8, "");
            float mn = fminf(x[j][0], x[j][1]);
            if (!BF && edge) {
                mn = INFINITY;
#pragma unroll
                for (int e = 0; e < 8; e++) mn = fminf(mn, x[j][e] == -INFINITY ? INFINITY : x[j][e]);
            }
            const bool under = Weights::under(mx, st.m[j]), moves = under || Weights::above(mx, st.m[j]);
            if (__any(moves || Weights::tiny(mn, f, st.m[j]))) {
                if (__any(moves)) {
                    const float was = st.m[j];
                    st.m[j] = Weights::reference(mx, was);
                    if (__any(under)) {
                        const float d = room(st, j, under ? was - ceilf(mx) : 0.f);
                        if (under) st.m[j] = was - d;
                    }
                    scale(st, j, sums_move(was, st.m[j]));
                }
                small |= __any(Weights::tiny(mn, f, st.m[j]));
            }
        }
        if (!BF && small) {
#pragma unroll
            for (int j = 0; j < NC; j++) {
                const float f = a.softcap > 0.f ? 1.f : st.qf[j], up = Weights::offset(st.m[j]);
                float mn = INFINITY, larger = 0.f, seen = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool in = x[j][e] != -INFINITY;
                    mn = fminf(mn, in ? x[j][e] : INFINITY);
                    seen += in ? 1.f : 0.f;
                    larger += __builtin_fmaf(x[j][e], f, up) < Weights::LEAST ? 0.f : 1.f;
                }
                least[j] = Weights::far(st.m[j]) ? INFINITY : __builtin_fmaf(mn, f, up);
                larger = sum_x32(sum_x16(larger));  // (by all lanes: those without a position have no small weight)
                seen = sum_x32(sum_x16(seen));
                bands |= __any(least[j] < Weights::LEAST && Weights::few(larger, seen));
            }
        }
        // The weights from 2^LEAST on; then, with the sums raised, those below, a band at a time (rare: PagedWeights).
        float most[NC], raise = 0.f;  // by how much the sums of this lane's columns rise in the end; by now at most
#pragma unroll
        for (int j = 0; j < NC; j++) most[j] = bands ? Weights::wanted(max_x32(max_x16(-least[j]))) : 0.f;
        for (;;) {
            pg_u4 p[NC][NS];
#pragma unroll
            for (int j = 0; j < NC; j++) {
                const float f = a.softcap > 0.f ? 1.f : st.qf[j], up = Weights::offset(st.m[j]) + raise;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = x[j][e];
                if (bands) {
                    const float before = Weights::before(up, raise, most[j]);
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = Weights::other(x[j][e], f, up, before) ? -INFINITY : x[j][e];
                }
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const float p0 = exp2_hw(__builtin_fmaf(y[2 * d], f, up)), p1 = exp2_hw(__builtin_fmaf(y[2 * d + 1], f, up));
                    st.l[j] += p0 + p1;
                    uint32_t w[NS];
                    split2<BF, NS>(p0, p1, w);
#pragma unroll
                    for (int n = 0; n < NS; n++) p[j][n][d] = w[n];
                }
            }
            pv<0>(st, u, p);
            if (!bands) break;
            bool more = false;
#pragma unroll
            for (int j = 0; j < NC; j++) {
                if (raise == 0.f) most[j] = Weights::whole(room(st, j, most[j]));
                more |= raise < most[j];
            }
            if (!__any(more)) break;
            again(u);
#pragma unroll
            for (int j = 0; j < NC; j++) scale(st, j, raise < most[j] ? static_cast<int>(Weights::BAND) : 0);
            raise += Weights::BAND;
        }
        if (bands) {
#pragma unroll
            for (int j = 0; j < NC; j++) scale(st, j, -static_cast<int>(most[j]));
        }
    }
};

// The runs of W <= n workers over n units: n / W each, one more for the first n % W.
struct PagedRuns {
    int q, rem;
    __device__ __forceinline__ PagedRuns(int n, int workers) : q(n / workers), rem(n - q * workers) {}
    __device__ __forceinline__ int start(int w) const { return w * q + min(w, rem); }
    __device__ __forceinline__ int of(int u) const {  // the worker of unit u
        const int longer = rem * (q + 1);
        return u < longer ? u / (q + 1) : rem + (u - longer) / q;
    }
};
// Workers that have work: a unit for each of their waves, but no more segments in turn than that takes (16
// sequences of two tokens behind four positions: 35 -> 13.7 us).
template <bool MULTI>
__device__ __forceinline__ int paged_workers(const PagedAttnArgs& a, int total, int segments) {
    return min(a.workers, max((total + paged_wg(MULTI) - 1) / paged_wg(MULTI), segments));
}

template <int HD, int KT, int NS, bool MULTI>
__global__ __launch_bounds__(64 * paged_wg(MULTI), (PagedDecode<HD, KT, NS, MULTI>::WAVES)) void paged_decode_kernel(PagedAttnArgs a) {
    using D = PagedDecode<HD, KT, NS, MULTI>;
    constexpr int E = D::E, NC = D::NC, WG = D::WG;
    // The queries' operands, and (WG > 1) in their place the waves' sums at a segment's end, a column's
    // row padded by 16 bytes so that 16 columns do not meet in a bank.
    constexpr int OP = HD + 4;
    __shared__ pg_u4 lds[WG > 1 ? (D::QS > WG * 4 * NC * OP ? D::QS : WG * 4 * NC * OP) : D::QS];
    __shared__ float2 ml_s[WG][16 * NC];
    pg_u4* q_s = lds;
    float* o_s = reinterpret_cast<float*>(lds);
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int wave = WG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    auto units = [&](int b) {
        const PagedRange r = paged_range<MULTI, NC>(a, b);
        return r.nt * r.ct * a.c.num_kv;
    };
    // units of all sequences, and this worker's run [u, u1)
    const int per = (a.c.num_seqs + 63) / 64, b0 = min(lane * per, a.c.num_seqs), b1 = min(b0 + per, a.c.num_seqs);
    int mine = 0, segments = 0;
#pragma unroll 4
    for (int b = b0; b < b1; b++) {
        const PagedRange r = paged_range<MULTI, NC>(a, b);
        mine += r.nt * r.ct * a.c.num_kv;
        if (MULTI && r.nt) segments += r.ct * a.c.num_kv;
    }
    if constexpr (MULTI) segments = __builtin_amdgcn_readfirstlane(wave_sum_i(segments));
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d, 64);
        if (lane >= d) incl += v;
    }
    const int total = __builtin_amdgcn_readlane(incl, 63);
    const int workers = paged_workers<MULTI>(a, total, segments);
    if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<int2*>(a.seg) = make_int2(total, workers);
    if (static_cast<int>(blockIdx.x) >= workers) return;
    const PagedRuns runs(total, workers);
    int u = runs.start(blockIdx.x);
    const int u1 = runs.start(blockIdx.x + 1);
    int b = b0, at = u - (incl - mine);
    const bool holds = at >= 0 && u < incl;
    if (holds)
        for (int n; at >= (n = units(b)); b++) at -= n;
    const int src = __builtin_ctzll(__ballot(holds));
    b = __builtin_amdgcn_readlane(b, src);
    at = __builtin_amdgcn_readlane(at, src);
    const bool whole = (a.c.page_size & 15) == 0;
    const int u_first = u;
    while (u < u1) {
        const PagedRange r = paged_range<MULTI, NC>(a, b);
        if (r.nt == 0) {
            b++;
            continue;
        }
        const int hh = at / r.nt, ta = at - hh * r.nt, n = min(r.nt - ta, u1 - u);
        const int h = hh / r.ct, cg = hh - h * r.ct;
        if (ta == 0 && threadIdx.x == 0) a.seg[2 + (b * a.c.num_kv + h) * a.groups + cg] = u;
        typename D::State st;
        int t = r.t0 + ta + wave;
        const int te = r.t0 + ta + n - 1;
        const bool busy = WG == 1 || t <= te;
        typename D::Unit ua;
        typename D::Ids ia, ib;
        if (busy) {
            ia = D::ids(a, b, t);
            ib = D::ids(a, b, min(t + WG, te));
        }
        {
            ActRaw<D::AF> x[NC][D::KS];
            D::load_q(x, a, r, h, cg, g, c);
            if (D::TWO && busy) D::load(ua, a, b, h, t, ia, whole, g, c);
            __builtin_amdgcn_sched_barrier(0);  // (the query's waits behind the unit's loads)
            if (a.act_type == LARQL_ELEM_F16)
                D::template start<true>(st, q_s, x, a, h, wave, g, c);
            else
                D::template start<false>(st, q_s, x, a, h, wave, g, c);
            if constexpr (WG > 1) lds_barrier();
        }
        if (busy) {
            if constexpr (D::TWO) {
                // (the last unit is loaded again rather than branching round its loads)
                typename D::Unit ub;
                for (;;) {
                    ia = D::ids(a, b, min(t + 2 * WG, te));
                    D::load(ub, a, b, h, min(t + WG, te), ib, whole, g, c);
                    D::step(st, q_s, ua, a, r, cg, t, g, c);
                    if ((t += WG) > te) break;
                    ib = D::ids(a, b, min(t + 2 * WG, te));
                    D::load(ua, a, b, h, min(t + WG, te), ia, whole, g, c);
                    D::step(st, q_s, ub, a, r, cg, t, g, c);
                    if ((t += WG) > te) break;
                }
            } else {
                for (;;) {
                    D::load(ua, a, b, h, t, ia, whole, g, c);
                    ia = ib;
                    ib = D::ids(a, b, min(t + 2 * WG, te));
                    D::step(st, q_s, ua, a, r, cg, t, g, c);
                    if ((t += WG) > te) break;
                }
            }
        }
        const float vs = KT == LARQL_ELEM_E4M3 && a.c.v_scale ? a.c.v_scale[h] : 1.f;
        const bool done = n == r.nt;
        const int slot = 2 * blockIdx.x + (ta != 0 || u == u_first ? 0 : 1);
        if constexpr (WG == 1) {
            const float l = sum_x32(sum_x16(st.l[0]));
            if (16 * cg + c < r.rows) {
                const float f = done ? (l == 0.f ? 0.f : 1.f / l) : 1.f, fv = done ? vs : 1.f;
                const long long entry = static_cast<long long>(slot) * a.cols + c;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = st.o[0][e][i] * f * fv;
                    constexpr int V = E % 8 == 0 ? 8 : E % 4 == 0 ? 4 : 2;
                    const int d = (4 * g + i) * E;
                    if (done) {
                        const long long o = r.row0 * a.out_ld + static_cast<long long>(h * a.reps + 16 * cg + c) * HD + d;
#pragma unroll
                        for (int e = 0; e < E; e += V) act_store<D::AF, V>(a.out, o + e, a.act_type, x + e);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; e += V) act_store<true, V>(a.part, entry * HD + d + e, LARQL_ELEM_F32, x + e);
                    }
                }
                if (!done && g == 0) *reinterpret_cast<float2*>(a.ml + 2 * entry) = make_float2(st.m[0], l);
            }
        } else {
            lds_barrier();  // (the queries are read)
#pragma unroll
            for (int j = 0; j < NC; j++) {
                const float l = sum_x32(sum_x16(st.l[j]));
                if (g == 0) ml_s[wave][16 * j + c] = make_float2(st.m[j], l);
                constexpr int V = E % 4 == 0 ? 4 : 2;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = st.o[j][e][i];
                    float* at = o_s + ((wave * NC + j) * 16 + c) * OP + (4 * g + i) * E;
#pragma unroll
                    for (int e = 0; e < E; e += V) act_store<true, V>(at, e, LARQL_ELEM_F32, x + e);
                }
            }
            lds_barrier();
            const int cols = min(16 * NC, r.rows - 16 * NC * cg);
            for (int i = threadIdx.x; i < cols * (HD / 4); i += 64 * WG) {
                const int col = i / (HD / 4), d = 4 * (i - col * (HD / 4));
                float m = -INFINITY, l = 0.f;
#pragma unroll
                for (int w = 0; w < WG; w++) m = fmaxf(m, ml_s[w][col].x);
                pg_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < WG; w++) {
                    const float2 ml = ml_s[w][col];
                    const int by = sums_move(ml.x, m);
                    l += ldexpf(ml.y, by);
                    o += ldexp4(*reinterpret_cast<const pg_f4*>(o_s + (w * NC * 16 + col) * OP + d), by);
                }
                if (done) {
                    const int R = 16 * NC * cg + col, tok = paged_div(R, a.rep_mul, a.rep_shift);
                    o *= l == 0.f ? 0.f : 1.f / l;
                    act_store4<D::AF>(a.out, (r.row0 + tok) * a.out_ld + static_cast<long long>(h * a.reps + R - tok * a.reps) * HD + d,
                                      a.act_type, o[0] * vs, o[1] * vs, o[2] * vs, o[3] * vs);
                } else {
                    const long long entry = static_cast<long long>(slot) * a.cols + col;
                    *reinterpret_cast<pg_f4*>(a.part + entry * HD + d) = o;
                    if (d == 0) *reinterpret_cast<float2*>(a.ml + 2 * entry) = make_float2(m, l);
                }
            }
        }
        if constexpr (WG > 1) lds_barrier();  // (the sums are read)
        u += n;
        at += n;
        if (at == r.nt * r.ct * a.c.num_kv) {
            at = 0;
            b++;
        }
    }
}

// Joins the parts of segments that several workers shared, and writes zeros for rows without
// positions.  A workgroup takes `join_cols` columns of a segment: HD / 4 threads (four dims each) times as
// many groups as there are threads for sum a column's parts, each group every so many of them in
// worker order, then the groups in theirs.  grid (sequences x kv heads x column groups, columns / join_cols).
template <int HD, bool AF, bool MULTI, int TH>
__global__ __launch_bounds__(TH) void paged_decode_join_kernel(PagedAttnArgs a) {
    constexpr int L = HD / 4, G = TH / L, NC = paged_nc(HD, MULTI), COLS = 16 * NC;
    __shared__ pg_f4 o_s[G][L];
    __shared__ float2 ml_s[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = a.c.num_kv * a.groups;
    const int b = blockIdx.x / per, hh = blockIdx.x - b * per, h = hh / a.groups, cg = hh - h * a.groups;
    const int c0 = blockIdx.y * a.join_cols;
    const PagedRange r = paged_range<MULTI, NC>(a, b);
    const int total = a.seg[0], workers = a.seg[1], u = a.seg[2 + blockIdx.x];
    const int cols = min(min(a.join_cols, COLS - c0), r.rows - COLS * cg - c0);  // of this workgroup
    if (cols <= 0 || (MULTI && r.rows > a.few)) return;
    const int k = tid / L, d = tid - k * L, col = k % a.join_cols, pg = k / a.join_cols, PG = G / a.join_cols;
    const int R = COLS * cg + c0 + min(col, cols - 1), tok = MULTI ? paged_div(R, a.rep_mul, a.rep_shift) : 0;
    const bool mine = col < cols && pg < PG;
    const long long out = (r.row0 + tok) * a.out_ld + static_cast<long long>(h * a.reps + R - tok * a.reps) * HD + 4 * d;
    if (r.nt == 0) {
        if (mine && pg == 0) act_store4<AF>(a.out, out, a.act_type, 0.f, 0.f, 0.f, 0.f);
        return;
    }
    const PagedRuns runs(total, workers);
    const int w0 = runs.of(u), n = runs.of(u + r.nt - 1) - w0 + 1;
    if (n == 1) return;
    // the first worker holds the segment's start in its slot 1 unless its run begins there
    const int first = runs.start(w0) == u ? 0 : 1;
    auto part = [&](int i, int c) { return (2 * (w0 + i) + (i == 0 ? first : 0)) * a.cols + c0 + c; };
    auto ml = [&](int i, int c) { return *reinterpret_cast<const float2*>(a.ml + 2 * part(i, c)); };
    // maximum and sum of each column, a wave at a time
    for (int c = wave; c < cols; c += TH / 64) {
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < n; i += 64) m = fmaxf(m, ml(i, c).x);
        m = wave_max(m);
        for (int i = lane; i < n; i += 64) l += ldexpf(ml(i, c).y, sums_move(ml(i, c).x, m) - kJoinDown);
        l = wave_sum(l);
        if (lane == 0) ml_s[c] = make_float2(m, l);
    }
    __syncthreads();
    pg_f4 o = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
        const float m = ml_s[col].x;
#pragma unroll 4
        for (int i = pg; i < n; i += PG)
            o += ldexp4(*reinterpret_cast<const pg_f4*>(a.part + static_cast<long long>(part(i, col)) * HD + 4 * d),
                        sums_move(ml(i, col).x, m) - kJoinDown);
        o_s[k][d] = o;
    }
    __syncthreads();
    if (!mine || pg) return;
#pragma unroll 4
    for (int j = 1; j < PG; j++) o += o_s[k + j * a.join_cols][d];
    const float l = ml_s[col].y;
    const float vs = a.kv_type == LARQL_ELEM_E4M3 && a.c.v_scale ? a.c.v_scale[h] : 1.f;
    o *= l == 0.f ? 0.f : 1.f / l;
    act_store4<AF>(a.out, out, a.act_type, o[0] * vs, o[1] * vs, o[2] * vs, o[3] * vs);
}

template <int HD, bool MULTI>
static void launch_paged_waves(const PagedAttnArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.workers)), block(64 * paged_wg(MULTI));
    const bool f32 = a.act_type == LARQL_ELEM_F32;
    if (a.kv_type == LARQL_ELEM_F16) {
        if (f32) paged_decode_kernel<HD, LARQL_ELEM_F16, 2, MULTI><<<grid, block, 0, s>>>(a);
        else paged_decode_kernel<HD, LARQL_ELEM_F16, 1, MULTI><<<grid, block, 0, s>>>(a);
    } else if (a.kv_type == LARQL_ELEM_E4M3) {
        if (f32) paged_decode_kernel<HD, LARQL_ELEM_E4M3, 2, MULTI><<<grid, block, 0, s>>>(a);
        else paged_decode_kernel<HD, LARQL_ELEM_E4M3, 1, MULTI><<<grid, block, 0, s>>>(a);
    } else {
        if (f32) paged_decode_kernel<HD, LARQL_ELEM_BF16, 3, MULTI><<<grid, block, 0, s>>>(a);
        else paged_decode_kernel<HD, LARQL_ELEM_BF16, 2, MULTI><<<grid, block, 0, s>>>(a);
    }
    LARQL_HIP_CHECK(hipGetLastError());
    const int segments = a.c.num_seqs * a.c.num_kv * a.groups;
    const dim3 jg(static_cast<unsigned>(segments), static_cast<unsigned>((a.cols + a.join_cols - 1) / a.join_cols));
    auto join = [&](auto af) {
        constexpr bool AF = decltype(af)::value;
        // few segments have many parts each
        if (a.workers > 16 * segments) paged_decode_join_kernel<HD, AF, MULTI, 1024><<<jg, 1024, 0, s>>>(a);
        else paged_decode_join_kernel<HD, AF, MULTI, 256><<<jg, 256, 0, s>>>(a);
    };
    if (f32) join(std::true_type{});
    else join(std::false_type{});
    LARQL_HIP_CHECK(hipGetLastError());
}

}  // namespace larql
