// Device helpers of the paged KV cache kernels: page lookup, 16-bit operand splits, MFMA by type.
#pragma once

#include "device_common.h"
#include "paged.h"

namespace larql {

typedef _Float16 pg_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_half2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_bf2 __attribute__((ext_vector_type(2)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int paged_div(int n, unsigned mul, int shift) {
    return static_cast<int>(__umulhi(2u * static_cast<unsigned>(n), mul) >> shift);
}
__device__ __forceinline__ int paged_page(const PagedView& c, int pos) { return paged_div(pos, c.page_mul, c.page_shift); }

// A sequence's positions (at most 2^30, so that differences of positions stay in range), and those
// that its table row reaches.
__device__ __forceinline__ int paged_kv_len(const PagedView& c, int b) { return min(max(c.kv_len[b], 0), kPagedMax); }
__device__ __forceinline__ int paged_len(const PagedView& c, int b) { return min(paged_kv_len(c, b), c.cap); }

// The token rows of sequence b: n from row0 on (inside the call's rows whatever q_start holds).
__device__ __forceinline__ void paged_rows(const PagedView& c, int b, int& row0, int& n) {
    row0 = min(max(c.q_start[b], 0), c.num_tokens);
    n = min(max(c.q_start[b + 1], row0), c.num_tokens) - row0;
}

// The page that holds position `pos` of sequence b and the position's place in it; not below
// num_pages (as unsigned) where the table names no page of the cache.  Positions the table row does not reach
// read its last entry: callers mask them by the length.
__device__ __forceinline__ unsigned paged_id(const PagedView& c, int b, int pos, int& off) {
    const int pi = paged_page(c, pos);
    off = pos - pi * c.page_size;
    return static_cast<unsigned>(c.table[b * c.table_ld + min(pi, c.pages_per_seq - 1)]);
}

// N bytes at p (a multiple of the largest power of two in N) into 32-bit words.
template <int N>
__device__ __forceinline__ void load_bytes(uint32_t* r, const char* p) {
    constexpr int A = (N & -N) > 16 ? 16 : (N & -N);
    if constexpr (N % 4) r[N / 4] = 0;
    __builtin_memcpy(r, __builtin_assume_aligned(p, A), N);
}

// W words (2 or 4) at a global address that went through LDS.
template <int W>
__device__ __forceinline__ void load_global(uint32_t* r, long long at) {
    typedef uint32_t v __attribute__((ext_vector_type(W)));
    const v x = *reinterpret_cast<const __attribute__((address_space(1))) v*>(at);
#pragma unroll
    for (int i = 0; i < W; i++) r[i] = x[i];
}

// 16 bytes per lane from global memory straight into LDS, lane i's at LDS address `to` + 16 i (to the same for
// the wave).  The caller waits (wait_vmcnt0) before its barrier.  The compiler does not see the load: it would
// wait for it before any later LDS read that it cannot tell apart, those of the other buffer among them.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p)));
}
__device__ __forceinline__ void load_lds16(long long at, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory", "m0");
}
__device__ __forceinline__ void wait_vmcnt0() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Activations are f32 (AF) or one of the 16-bit types, told apart when the kernel runs: the values are
// selected, not branched for.
__device__ __forceinline__ float act_lo(uint32_t w, bool h) { return h ? h2f(w) : __uint_as_float(w << 16); }
__device__ __forceinline__ float act_hi(uint32_t w, bool h) { return h ? h2f(w >> 16) : __uint_as_float(w & 0xFFFF0000u); }

// W consecutive elements (8, 4 or 2: aligned to their size up to 16 bytes; 1: one) as f32.
template <bool AF, int W>
__device__ __forceinline__ void act_load(float* x, const void* p, long long i, int type) {
    if constexpr (AF) {
        const float* f = static_cast<const float*>(p) + i;
        if constexpr (W == 1) {
            x[0] = f[0];
        } else {
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                const pg_f4 v = *reinterpret_cast<const pg_f4*>(f + j);
#pragma unroll
                for (int e = 0; e < 4; e++) x[j + e] = v[e];
            }
        }
    } else {
        const bool h = type == LARQL_ELEM_F16;
        const uint16_t* u = static_cast<const uint16_t*>(p) + i;
        if constexpr (W == 1) {
            x[0] = act_lo(u[0], h);
        } else {
            uint32_t w[W / 2];
            __builtin_memcpy(w, __builtin_assume_aligned(u, 2 * W), 2 * W);
#pragma unroll
            for (int j = 0; j < W / 2; j++) {
                x[2 * j] = act_lo(w[j], h);
                x[2 * j + 1] = act_hi(w[j], h);
            }
        }
    }
}

// Two f32 as f16 / bf16 bits (round to nearest even), low half first.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF) {
        const pg_bf2 r = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        return __builtin_bit_cast(uint32_t, r);
    } else {
        const pg_half2 r = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(uint32_t, r);
    }
}
template <bool BF>
__device__ __forceinline__ float unpack_lo(uint32_t w) {
    return BF ? __uint_as_float(w << 16) : static_cast<float>(__builtin_bit_cast(pg_half2, w)[0]);
}
template <bool BF>
__device__ __forceinline__ float unpack_hi(uint32_t w) {
    return BF ? __uint_as_float(w & 0xFFFF0000u) : static_cast<float>(__builtin_bit_cast(pg_half2, w)[1]);
}

// (a, b) as N 16-bit parts whose sum is the value to N times the type's significand.
template <bool BF, int N>
__device__ __forceinline__ void split2(float a, float b, uint32_t* w) {
#pragma unroll
    for (int n = 0; n < N; n++) {
        w[n] = pack2<BF>(a, b);
        if (n + 1 < N) {
            a -= unpack_lo<BF>(w[n]);
            b -= unpack_hi<BF>(w[n]);
        }
    }
}

// W consecutive activations (8 or 4: aligned to their size up to 16 bytes; 1: one) as they lie, and their
// values (H: f16, else bf16).
template <bool AF, int W = 8>
struct ActRaw {
    uint32_t w[AF ? W : (W + 1) / 2];
};
template <bool AF, int W = 8>
__device__ __forceinline__ void act_raw(ActRaw<AF, W>& r, const void* p, long long i) {
    constexpr int N = W * (AF ? 4 : 2);
    const char* at = static_cast<const char*>(p) + i * (AF ? 4 : 2);
    if constexpr (N > 16) {
        load_bytes<16>(r.w, at);
        load_bytes<16>(r.w + 4, at + 16);
    } else {
        load_bytes<N>(r.w, at);
    }
}
template <bool AF, bool H, int W>
__device__ __forceinline__ float act_value(const ActRaw<AF, W>& r, int e) {
    if constexpr (AF) return __uint_as_float(r.w[e]);
    const uint32_t w = r.w[AF ? 0 : e / 2];
    if constexpr (H) return h2f(e % 2 ? w >> 16 : w);
    return __uint_as_float(e % 2 ? w & 0xFFFF0000u : w << 16);
}

// W values as activations (alignment as for act_load).
template <bool AF, int W>
__device__ __forceinline__ void act_store(void* p, long long i, int type, const float* x) {
    if constexpr (AF) {
        float* f = static_cast<float*>(p) + i;
        if constexpr (W == 1) {
            f[0] = x[0];
        } else if constexpr (W == 2) {
            *reinterpret_cast<float2*>(f) = make_float2(x[0], x[1]);
        } else {
#pragma unroll
            for (int j = 0; j < W; j += 4) *reinterpret_cast<pg_f4*>(f + j) = pg_f4{x[j], x[j + 1], x[j + 2], x[j + 3]};
        }
    } else {
        const bool h = type == LARQL_ELEM_F16;
        uint16_t* u = static_cast<uint16_t*>(p) + i;
        if constexpr (W == 1) {
            u[0] = static_cast<uint16_t>(h ? pack2<false>(x[0], x[0]) : pack2<true>(x[0], x[0]));
        } else {
            uint32_t w[W / 2];
#pragma unroll
            for (int j = 0; j < W / 2; j++) w[j] = h ? pack2<false>(x[2 * j], x[2 * j + 1]) : pack2<true>(x[2 * j], x[2 * j + 1]);
            __builtin_memcpy(__builtin_assume_aligned(u, 2 * W), w, 2 * W);
        }
    }
}
template <bool AF>
__device__ __forceinline__ void act_store4(void* p, long long i, int type, float a, float b, float c, float d) {
    const float x[4] = {a, b, c, d};
    act_store<AF, 4>(p, i, type, x);
}

template <bool BF>
__device__ __forceinline__ pg_f4 mfma16(const pg_u4& a, const pg_u4& b, const pg_f4& c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf8, a), __builtin_bit_cast(pg_bf8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_half8, a), __builtin_bit_cast(pg_half8, b),
                                                      c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ pg_f16 mfma32(const pg_u4& a, const pg_u4& b, const pg_f16& c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pg_bf8, a), __builtin_bit_cast(pg_bf8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pg_half8, a), __builtin_bit_cast(pg_half8, b),
                                                      c, 0, 0, 0);
}

// Two e4m3 codes (the low or high half of w) as f16, exact.
template <bool HI>
__device__ __forceinline__ uint32_t e4m3_f16(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// Whether one of two 16-bit elements is an infinity or NaN, and the two with those as 0.
__device__ __forceinline__ bool not_finite16(uint32_t w, bool bf) {
    const uint32_t m = bf ? 0x7F80u : 0x7C00u;
    return (w & m) == m || (w & m << 16) == m << 16;
}
__device__ __forceinline__ uint32_t finite16(uint32_t w, bool bf) {
    const uint32_t m = bf ? 0x7F80u : 0x7C00u;
    return ((w & m) == m ? 0u : w & 0xFFFFu) | ((w & m << 16) == m << 16 ? 0u : w & 0xFFFF0000u);
}

// max / sum over the two lanes 32 apart, and 16 apart.
__device__ __forceinline__ float max_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_x32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_x16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_x16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^x on the hardware's unit (1 ulp; results below 2^-126 become 0).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's weights 2^(s - m) (s: its scores in log2, m: its reference) on their way to the matrix cores as NS 16-bit
// parts.  m is a whole number, so that rescaling the sums rounds nothing, and follows the row's largest score only where
// that rose by more than LAZY, so that most tiles rescale nothing.
//
// bf16 parts have f32's range.  f16 ends at 2^-24, so there weights are taken as 2^(z = s - m + UP) (the sums l too: it
// cancels in the end), and the parts hold those from 2^LEAST on: two of them to half a step of 2^-24, 2^-19 of the
// weight; one to its own rounding (the least normal number is 2^-14).  Smaller ones are held to 2^-25, 2^-39 of the
// row's largest.  That is too little where the larger ones meet values near zero, as an attention sink's are:
// - a tile whose largest weight is below 2^LOW lets m fall to its largest score (the sums rise with it, exactly, up to
//   2^MOST), so the tiles behind a position that dominates a row are like any others;
// - in a tile where FEW weights or a quarter of them (one at least) are not too small, the others are summed apart: decode in
//   bands of BAND, each with the sums raised as far; prompts, where a second set of products next to the first cost
//   every tile 10-40%, in f32 without the matrix cores.
// With more of them the others stay as they are: taking those apart too cost rows whose scores are spread widely (3 nats
// deviation) 2 to 5 times the time, for a case in which all of the larger values would have to be near zero.
// 512 tokens f32 over f16 32 us, 41 with a sink 18 nats above the rest, 40 with scores of 3 nats deviation; 32 sequences'
// decode 63 us, 1 more with a sink.  Without any of it 30 us and 62, and errors of 1e-3 behind a sink of 12 nats, 0.4 at 18.
template <bool BF, int NS>
struct PagedWeights {
    static constexpr float UP = BF ? 0.f : 14.f, LAZY = BF ? 8.f : 1.98f;  // (2^15.98 is f16's largest)
    static constexpr float LEAST = NS == 1 ? -14.f : -6.f, BAND = UP - LEAST, LOW = 5.f, FEW = 4.f;
    static constexpr float MOST = 122.f;  // (four lanes' or waves' sums of that stay finite)

    // Scores past 2^16 round by more than there is room above the largest weight: theirs start lower, and rise by nothing.
    static __device__ __forceinline__ bool far(float m) { return fabsf(m) > 65536.f; }
    // Whether a tile's largest score mx calls for a higher reference, and that one; or for a lower one.
    static __device__ __forceinline__ bool above(float mx, float m) { return mx > m + (far(m) ? -UP : LAZY); }
    static __device__ __forceinline__ float reference(float mx, float m) {
        return fmaxf(m, ceilf(mx) + (far(mx) ? UP : 0.f));
    }
    static __device__ __forceinline__ bool under(float mx, float m) {
        return !BF && mx - m + UP < LOW && mx != -INFINITY && !far(m) && !far(mx);
    }
    // By how much (log2) sums of up to `sum` may rise; with values below 2^16 and four lanes' sums of the weights, l.
    static __device__ __forceinline__ float room(float sum) { return MOST - __builtin_amdgcn_frexp_expf(sum); }
    static __device__ __forceinline__ float room_weights(float l) { return room(l) - 18.f; }
    // What they have to rise by for weights of z = -below (none past -126) to be in reach, whatever its rounding; whole
    // bands of that.
    static __device__ __forceinline__ float wanted(float below) {
        return BAND * ceilf((fminf(below, 126.f) + LEAST + 0.01f) / BAND);
    }
    static __device__ __forceinline__ float whole(float rise) { return BAND * floorf(rise / BAND); }
    // What z is for a score of 0.
    static __device__ __forceinline__ float offset(float m) { return UP - (m == -INFINITY ? 0.f : m); }
    // A tile whose sums rise by `most`, whole bands, in passes as `raise` goes up by BAND: the offset `up` of a pass is that
    // without a rise + raise.  Of the pass before (infinite: there is none; all is done):
    static __device__ __forceinline__ float before(float up, float raise, float most) {
        return raise == 0.f ? -INFINITY : raise <= most ? up - BAND : INFINITY;
    }
    // Whether a product x (score = x f) has a weight that is too small for the parts.
    static __device__ __forceinline__ bool tiny(float x, float f, float m) {
        return !BF && __builtin_fmaf(x, f, offset(m)) < LEAST;
    }
    // Whether `larger` of a tile's `seen` weights, those that are not too small, are few (and not all).
    static __device__ __forceinline__ bool few(float larger, float seen) {
        return larger < seen && larger <= fmaxf(1.f, fminf(FEW, 0.25f * seen));
    }
    // Whether a product x (score = x f) is none of the pass at offset up: too small for it, or done at the one before.
    static __device__ __forceinline__ bool other(float x, float f, float up, float before) {
        return __builtin_fmaf(x, f, up) < LEAST || __builtin_fmaf(x, f, before) >= LEAST;
    }
};

// The power of two by which sums that stand at reference `from` move to reference `to` (whole numbers; -inf: no sums).  For
// ldexp, not as a factor: sums of 2^100 may move by less than 2^-126 and be in range still.
__device__ __forceinline__ int sums_move(float from, float to) {
    return static_cast<int>(fminf(fmaxf(from - (to == -INFINITY ? 0.f : to), -1000.f), 1000.f));
}
__device__ __forceinline__ pg_f4 ldexp4(pg_f4 x, int by) {
    return pg_f4{ldexpf(x[0], by), ldexpf(x[1], by), ldexpf(x[2], by), ldexpf(x[3], by)};
}

// Joined parts are taken down by 2^kJoinDown: as many sums as high as they go stay finite.
constexpr int kJoinDown = 12;

// Scores are products times `f` >= 0: the query takes the scale's sign, and f stays above 0, so that a masked product
// of -inf is a score of -inf (of products up to 10^38, over bf16 pages, the least f makes 0).
__device__ __forceinline__ float score_factor(float f) { return fmaxf(fabsf(f), 1.4e-45f); }

// The power of two that brings a query row of largest magnitude m into f16's upper range
// ([2^13, 2^14)); 0 for zeros and non-finite values.
__device__ __forceinline__ int query_exponent(float m) {
    return m > 0.f && m <= 3.4e38f ? min(120, max(-120, 13 - ilogbf(m))) : 0;
}

}  // namespace larql
