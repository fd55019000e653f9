// delta_tiles.h — matrix-core tiles of the chunked gated delta rule.
//
// All products are 16 x 16 tiles.  A lane l has the row or column l % 16 of an
// operand and, of every 32 places of the summed axis, the eight places
//     4 (l / 16) + 0..3  and  16 + 4 (l / 16) + 0..3.
// That is where a 16 x 16 result keeps its rows (row 4 (l / 16) + r of column
// l % 16 in register r), so two results stacked to 32 rows are an operand of
// the next product as they stand, without a pass through LDS.
//
// Rounding.  The rows a caller passes in bfloat16 are operands as they are.
// What the chunk computes (states, solved rows, scores) is held in fp32 and
// enters a bfloat16 product as the sum of N bfloat16 values: two (16 to 17
// significand bits) where results are bfloat16 or gradients, three (all 24)
// where the fp32 state is a result; products of two such operands leave out
// the terms below the last kept one.  One rounding to bfloat16 (8 bits) per
// operand was not taken: it moves the fp32 results by 2e-3 of their norm, two
// terms by 4e-6, three by 1e-7, and the kernels are bound by memory, latency
// and vector instructions, not by the matrix cores.  fp32 rows use the fp32
// matrix cores with no rounding.
#ifndef MDNAV_DELTA_TILES_H
#define MDNAV_DELTA_TILES_H

#include "lane_sums.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace delta {

using namespace lanes;

typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// A lane's place in a tile.  Loops take a fresh() one in each pass: the LDS
// addresses made from it then stay inside the pass (as one register and
// immediate offsets), where the compiler would otherwise keep hundreds of
// them in registers across the loop, and spill.
struct Lane {
    int col, quad;  // l % 16, l / 16
    __device__ __forceinline__ static Lane mine() { return {int(threadIdx.x) & 15, (int(threadIdx.x) >> 4) & 3}; }
    __device__ __forceinline__ static Lane fresh() {
        int x = int(threadIdx.x) & 63;
        asm volatile("" : "+v"(x));
        return {x & 15, x >> 4};
    }
};

// ---- sums over lanes, without LDS (lane_sums.h), and running ones
// Inclusive sums over lanes 0..31, upwards (lane i: lanes 0..i) and downwards
// (lanes i..31): by DPP shifts inside each 16, then the other 16's total.
__device__ __forceinline__ double lane_value(double x, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), lane)), hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane));
    return __builtin_bit_cast(double, uint64_t(lo) | uint64_t(hi) << 32);
}
__device__ __forceinline__ double scan_up32(double x, int lane) {
    x += from_lane<0x111>(x);  // row_shr 1, 2, 4, 8: 0 where there is no such lane
    x += from_lane<0x112>(x);
    x += from_lane<0x114>(x);
    x += from_lane<0x118>(x);
    const double low = lane_value(x, 15);
    return (lane & 16) ? x + low : x;
}
__device__ __forceinline__ double scan_down32(double x, int lane) {
    x += from_lane<0x101>(x);  // row_shl
    x += from_lane<0x102>(x);
    x += from_lane<0x104>(x);
    x += from_lane<0x108>(x);
    const double high = lane_value(x, 16);
    return (lane & 16) ? x : x + high;
}
// Lanes 16 Q .. 16 Q + 15 to all four sixteens.
template <int Q> __device__ __forceinline__ float from_quad(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned half = Q & 2 ? r[1] : r[0];
    const auto t = __builtin_amdgcn_permlane16_swap(half, half, false, false);
    return __builtin_bit_cast(float, unsigned(Q & 1 ? t[1] : t[0]));
}

template <class E> struct Kind;
template <> struct Kind<bf16> {
    static constexpr int MID = 2;  // terms of a computed operand, if it is not three
    static constexpr int PAD = 8;  // elements past a row: 16 bytes
};
template <> struct Kind<float> {
    static constexpr int MID = 1;
    static constexpr int PAD = 4;
};

// An operand over 32 places of the summed axis, in N terms.
template <class E, int N> struct Frag;
template <int N> struct Frag<bf16, N> { bf16x8 t[N]; };
template <> struct Frag<float, 1> { f32x4 t[2]; };
// The same over 16 places.
template <class E, int N> struct Half;
template <int N> struct Half<bf16, N> { bf16x4 t[N]; };
template <> struct Half<float, 1> { f32x4 t[1]; };

template <int A, int B>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<bf16, A>& a, const Frag<bf16, B>& b) {
    constexpr int most = A > B ? A : B;
#pragma unroll
    for (int s = most - 1; s >= 0; s--)  // the small terms first
#pragma unroll
        for (int i = 0; i < A; i++)
            if (s - i >= 0 && s - i < B) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.t[i], b.t[s - i], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& acc, const Frag<float, 1>& a, const Frag<float, 1>& b) {
#pragma unroll
    for (int s = 0; s < 8; s++)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.t[s >> 2][s & 3], b.t[s >> 2][s & 3], acc, 0, 0, 0);
}
template <int A, int B>
__device__ __forceinline__ void mma(f32x4& acc, const Half<bf16, A>& a, const Half<bf16, B>& b) {
    constexpr int most = A > B ? A : B;
#pragma unroll
    for (int s = most - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < A; i++)
            if (s - i >= 0 && s - i < B)
                acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a.t[i]),
                                                                __builtin_bit_cast(s16x4, b.t[s - i]), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& acc, const Half<float, 1>& a, const Half<float, 1>& b) {
#pragma unroll
    for (int s = 0; s < 4; s++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.t[0][s], b.t[0][s], acc, 0, 0, 0);
}

__device__ __forceinline__ void settle_one(f32x4& a) { asm volatile("" : "+v"(a)); }
// Results that a loop with early ends may have written last: what reads them
// comes at least 16 wait states later.  The compiler sees to that itself, but
// where a loop over matrix products is unrolled and can end after each pass,
// it has been seen to count the way through all passes and not the short one
// (hipcc of ROCm 7.2: results of heads of at most 16 columns were read before
// they were there).  A matrix product here is done after at most 11; the code
// as built has no such read on any path (tests/test_matrix_waits.py).
template <class... X> __device__ __forceinline__ void settle(f32x4& a, X&... more) {
    asm volatile("s_nop 15" : "+v"(a));
    (settle_one(more), ...);
}

// ---- fp32 values to operands
template <int N> __device__ __forceinline__ void split4(f32x4 x, bf16x4 (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        t[i] = __builtin_convertvector(x, bf16x4);
        if (i + 1 < N) x -= __builtin_convertvector(t[i], f32x4);
    }
}
template <class E, int N> struct Make;
template <int N> struct Make<bf16, N> {
    __device__ __forceinline__ static Frag<bf16, N> frag(f32x4 x, f32x4 y) {
        bf16x4 xt[N], yt[N];
        split4(x, xt);
        split4(y, yt);
        Frag<bf16, N> f;
#pragma unroll
        for (int i = 0; i < N; i++) f.t[i] = __builtin_shufflevector(xt[i], yt[i], 0, 1, 2, 3, 4, 5, 6, 7);
        return f;
    }
    __device__ __forceinline__ static Half<bf16, N> half(f32x4 x) {
        Half<bf16, N> f;
        split4(x, f.t);
        return f;
    }
};
template <> struct Make<float, 1> {
    __device__ __forceinline__ static Frag<float, 1> frag(f32x4 x, f32x4 y) {
        Frag<float, 1> f;
        f.t[0] = x;
        f.t[1] = y;
        return f;
    }
    __device__ __forceinline__ static Half<float, 1> half(f32x4 x) {
        Half<float, 1> f;
        f.t[0] = x;
        return f;
    }
};
template <class E, int N = Kind<E>::MID> __device__ __forceinline__ Frag<E, N> frag_of(f32x4 x, f32x4 y) { return Make<E, N>::frag(x, y); }
template <class E, int N = Kind<E>::MID> __device__ __forceinline__ Half<E, N> half_of(f32x4 x) { return Make<E, N>::half(x); }

// Element e of an operand (of a computed one, its first term).
template <int N> __device__ __forceinline__ float first_term(const Frag<bf16, N>& f, int e) { return float(f.t[0][e]); }
__device__ __forceinline__ float first_term(const Frag<float, 1>& f, int e) { return f.t[e >> 2][e & 3]; }

// ---- LDS to operands.  `m` is a matrix with rows `stride` elements apart.
// Along a row: the lane's row or column of the operand is row `r0 + l % 16`,
// the summed axis runs along the row from `c0`.
__device__ __forceinline__ bf16x4 row4(Lane l, const bf16* m, int stride, int r0, int c0) {
    return *reinterpret_cast<const bf16x4*>(m + l.col * stride + 4 * l.quad + r0 * stride + c0);
}
__device__ __forceinline__ f32x4 row4(Lane l, const float* m, int stride, int r0, int c0) {
    return *reinterpret_cast<const f32x4*>(m + l.col * stride + 4 * l.quad + r0 * stride + c0);
}
// Across rows: the lane's row or column is column `c0 + l % 16`, the summed
// axis runs over the rows from `r0`.  For 16-bit elements the LDS read
// transposes: of each 16 lanes, lane i receives element i % 4 of what the
// addresses of lanes i / 4, 4 + i / 4, 8 + i / 4, 12 + i / 4 hold.
__device__ __forceinline__ bf16x4 transposed4(const bf16* p) {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p));
}
__device__ __forceinline__ bf16x4 col4(Lane l, const bf16* m, int stride, int r0, int c0) {
    return transposed4(m + (4 * l.quad + (l.col >> 2)) * stride + 4 * (l.col & 3) + r0 * stride + c0);
}
__device__ __forceinline__ f32x4 col4(Lane l, const float* m, int stride, int r0, int c0) {
    const float* p = m + 4 * l.quad * stride + l.col + r0 * stride + c0;
    return f32x4{p[0], p[stride], p[2 * stride], p[3 * stride]};
}

// Rows of q, k and the output's gradient are stored in the order in which
// a lane needs them, so that its eight places are one 16-byte read: of every
// 32 columns, column 16 h + 4 g + r is at place 8 g + 4 h + r.
__device__ __forceinline__ constexpr int place(int c) { return (c & ~31) + ((c >> 2) & 3) * 8 + ((c >> 4) & 1) * 4 + (c & 3); }
__device__ __forceinline__ Frag<bf16, 1> ordered_row(Lane l, const bf16* m, int stride, int r0, int c0) {
    Frag<bf16, 1> f;
    f.t[0] = *reinterpret_cast<const bf16x8*>(m + l.col * stride + 8 * l.quad + r0 * stride + c0);
    return f;
}
__device__ __forceinline__ Frag<float, 1> ordered_row(Lane l, const float* m, int stride, int r0, int c0) {
    Frag<float, 1> f;
    const float* p = m + l.col * stride + 8 * l.quad + r0 * stride + c0;
    f.t[0] = *reinterpret_cast<const f32x4*>(p);
    f.t[1] = *reinterpret_cast<const f32x4*>(p + 4);
    return f;
}
// Across such rows, 16 columns from c0 (a multiple of 16), 32 rows.
__device__ __forceinline__ Frag<bf16, 1> ordered_col(Lane l, const bf16* m, int stride, int c0) {
    const bf16* p = m + (4 * l.quad + (l.col >> 2)) * stride + 8 * (l.col & 3) + (c0 & ~31) + ((c0 >> 4) & 1) * 4;
    Frag<bf16, 1> f;
    f.t[0] = __builtin_shufflevector(transposed4(p), transposed4(p + 16 * stride), 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
__device__ __forceinline__ Frag<float, 1> ordered_col(Lane l, const float* m, int stride, int c0) {
    const float* p = m + 4 * l.quad * stride + 8 * (l.col >> 2) + (l.col & 3) + (c0 & ~31) + ((c0 >> 4) & 1) * 4;
    const float* q = p + 16 * stride;
    Frag<float, 1> f;
    f.t[0] = f32x4{p[0], p[stride], p[2 * stride], p[3 * stride]};
    f.t[1] = f32x4{q[0], q[stride], q[2 * stride], q[3 * stride]};
    return f;
}

// N planes of a matrix, `plane` elements apart: 32 places along a row, across
// rows, and 16 of them.
template <int N>
__device__ __forceinline__ Frag<bf16, N> row_frag(Lane l, const bf16* m, int stride, int plane, int r0, int c0) {
    Frag<bf16, N> f;
#pragma unroll
    for (int i = 0; i < N; i++)
        f.t[i] = __builtin_shufflevector(row4(l, m, stride, r0, c0 + i * plane), row4(l, m, stride, r0, c0 + 16 + i * plane),
                                         0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
template <int N>
__device__ __forceinline__ Frag<float, 1> row_frag(Lane l, const float* m, int stride, int, int r0, int c0) {
    Frag<float, 1> f;
    f.t[0] = row4(l, m, stride, r0, c0);
    f.t[1] = row4(l, m, stride, r0, c0 + 16);
    return f;
}
template <int N>
__device__ __forceinline__ Frag<bf16, N> col_frag(Lane l, const bf16* m, int stride, int plane, int r0, int c0) {
    Frag<bf16, N> f;
#pragma unroll
    for (int i = 0; i < N; i++)
        f.t[i] = __builtin_shufflevector(col4(l, m, stride, r0, c0 + i * plane), col4(l, m, stride, r0 + 16, c0 + i * plane),
                                         0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
template <int N>
__device__ __forceinline__ Frag<float, 1> col_frag(Lane l, const float* m, int stride, int, int r0, int c0) {
    Frag<float, 1> f;
    f.t[0] = col4(l, m, stride, r0, c0);
    f.t[1] = col4(l, m, stride, r0 + 16, c0);
    return f;
}
template <int N>
__device__ __forceinline__ Half<bf16, N> row_half(Lane l, const bf16* m, int stride, int plane, int r0, int c0) {
    Half<bf16, N> f;
#pragma unroll
    for (int i = 0; i < N; i++) f.t[i] = row4(l, m, stride, r0, c0 + i * plane);
    return f;
}
template <int N>
__device__ __forceinline__ Half<float, 1> row_half(Lane l, const float* m, int stride, int, int r0, int c0) {
    Half<float, 1> f;
    f.t[0] = row4(l, m, stride, r0, c0);
    return f;
}
template <int N>
__device__ __forceinline__ Half<bf16, N> col_half(Lane l, const bf16* m, int stride, int plane, int r0, int c0) {
    Half<bf16, N> f;
#pragma unroll
    for (int i = 0; i < N; i++) f.t[i] = col4(l, m, stride, r0, c0 + i * plane);
    return f;
}
template <int N>
__device__ __forceinline__ Half<float, 1> col_half(Lane l, const float* m, int stride, int, int r0, int c0) {
    Half<float, 1> f;
    f.t[0] = col4(l, m, stride, r0, c0);
    return f;
}

// A result tile to LDS, transposed: column c of the tile becomes row c0 + c of
// the matrix, whose places r0 + 4 (l / 16) .. + 3 the lane writes at once.
template <int N>
__device__ __forceinline__ void put_tile(Lane l, bf16* m, int stride, int plane, int c0, int r0, f32x4 x) {
    bf16x4 t[N];
    split4(x, t);
    bf16* p = m + l.col * stride + 4 * l.quad + c0 * stride + r0;
#pragma unroll
    for (int i = 0; i < N; i++) *reinterpret_cast<bf16x4*>(p + i * plane) = t[i];
}
template <int N>
__device__ __forceinline__ void put_tile(Lane l, float* m, int stride, int, int c0, int r0, f32x4 x) {
    *reinterpret_cast<f32x4*>(m + l.col * stride + 4 * l.quad + c0 * stride + r0) = x;
}
// Two result tiles that are an operand already (32 places from r0).
__device__ __forceinline__ void put_frag(Lane l, bf16* m, int stride, int plane, int c0, int r0, const Frag<bf16, 2>& f) {
    bf16* p = m + l.col * stride + 4 * l.quad + c0 * stride + r0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        *reinterpret_cast<bf16x4*>(p + i * plane) = __builtin_shufflevector(f.t[i], f.t[i], 0, 1, 2, 3);
        *reinterpret_cast<bf16x4*>(p + i * plane + 16) = __builtin_shufflevector(f.t[i], f.t[i], 4, 5, 6, 7);
    }
}
__device__ __forceinline__ void put_frag(Lane l, float* m, int stride, int, int c0, int r0, const Frag<float, 1>& f) {
    float* p = m + l.col * stride + 4 * l.quad + c0 * stride + r0;
    *reinterpret_cast<f32x4*>(p) = f.t[0];
    *reinterpret_cast<f32x4*>(p + 16) = f.t[1];
}

}  // namespace delta

#endif
