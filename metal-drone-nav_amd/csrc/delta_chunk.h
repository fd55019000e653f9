// delta_chunk.h — what the forward and the backward pass of a chunk share:
// its rows in LDS, its decays, and the triangular system of its ticks.
//
// With gamma_i = exp(g_1 + .. + g_i) inside the chunk, D_ij = gamma_i / gamma_j
// and S the state before the chunk, the rows u_i = beta_i (v_i - S_{i-1}^T k_i)
// that the ticks add to the state solve
//     (1 + A) U = beta (V - gamma (K S)),   A_ij = beta_i D_ij (k_i k_j), j < i
// and  O = scale (gamma (Q S) + (D Q K^T) U),  S' = gamma_C S + sum_j (gamma_C / gamma_j) k_j u_j^T.
// A tick flagged as an episode's first sees none of what is before it: D is 0
// between ticks of different episodes, gamma 0 after the first flag and
// gamma_C / gamma_j 0 before the last.
#ifndef MDNAV_DELTA_CHUNK_H
#define MDNAV_DELTA_CHUNK_H

#include "delta_rule.h"
#include "delta_tiles.h"

namespace delta {

constexpr int C = int(CHUNK);
constexpr int CP = C + 8;  // row of a chunk x chunk matrix in LDS

// A decay this low is exp(g) = 0 in fp32; taken as the flag is, so that sums
// of decays stay finite (-inf included).
constexpr float NO_DECAY = -104.0f;

// Wavefront `wave`'s tiles of the state before chunk `c` >= 1.
__device__ __forceinline__ f32x4* state_tiles(float* p, uint64_t seq, uint32_t chunks, uint32_t c, uint32_t kd, uint32_t vd, int wave) {
    const uint32_t kt = (kd + 15) / 16, vt = (vd + 15) / 16;
    return reinterpret_cast<f32x4*>(p) + ((seq * (chunks - 1) + c - 1) * (kt * vt) + wave * kt) * 64;
}

// A wavefront's 16 columns of a state [K][V] as result tiles; `col` is the lane's column.
template <int KT>
__device__ __forceinline__ void load_state(f32x4 (&x)[KT], const float* p, uint32_t kd, uint32_t vd, Lane l, uint32_t col) {
#pragma unroll
    for (int i = 0; i < KT; i++) x[i] = f32x4{0, 0, 0, 0};
    if (!p || col >= vd) return;
    if (kd == 16 * KT) {
#pragma unroll
        for (int i = 0; i < KT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) x[i][r] = p[uint32_t(16 * i + 4 * l.quad + r) * vd + col];
    } else {
#pragma unroll
        for (int i = 0; i < KT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint32_t kr = 16 * i + 4 * l.quad + r;
                const float y = p[(kr < kd ? kr : 0u) * vd + col];
                x[i][r] = kr < kd ? y : 0.0f;
            }
    }
}
template <int KT>
__device__ __forceinline__ void store_state(float* p, const f32x4 (&x)[KT], uint32_t kd, uint32_t vd, Lane l, uint32_t col) {
    if (col >= vd) return;
#pragma unroll
    for (int i = 0; i < KT; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t kr = 16 * i + 4 * l.quad + r;
            if (kr < kd) p[kr * vd + col] = x[i][r];
        }
}

// ---- a kernel's arguments, read from the kernel's argument memory where they
// are used.  A chunk kernel has more of them than scalar registers: kept
// across the loop they are spilled to lanes of vector registers, and each use
// costs vector instructions.
struct Call {
    Args a;
    GradArgs d;
};
typedef __attribute__((address_space(4))) const Call KernelCall;
typedef __attribute__((address_space(4))) const Rows KernelRows;
__device__ __forceinline__ KernelCall* fresh_call() {
    KernelCall* p = (KernelCall*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// ---- rows of one state's array: its env's and head's start, and the ticks' stride
template <class E> struct Track {
    E* p;
    int64_t tick;
    __device__ __forceinline__ Track(KernelRows* r, uint32_t n, uint32_t h)
        : p(reinterpret_cast<E*>(r->p) + int64_t(n) * r->env + int64_t(h) * r->head), tick(r->tick) {}
    __device__ __forceinline__ E* row(uint32_t t) const { return p + int64_t(t) * tick; }
};

// Whose rows a workgroup is at: a state (env and heads), a segment of its
// ticks and a chunk of that.  Workgroups stay for several segments and load
// the next chunk's rows, of this one or the next, while they compute.
struct Plan {
    uint32_t heads, shared, chunks, segments, segment, jobs, total;
    // `jobs` of a state: its segments, or what runs ahead of them
    __device__ __forceinline__ Plan(const Args& a, uint32_t j)
        : heads(a.heads), shared(a.heads / a.qk_heads), chunks((a.ticks + CHUNK - 1) / CHUNK), segments(a.segments),
          segment(a.segment), jobs(j), total(a.envs * a.heads * j) {}
};
struct At {
    uint32_t job, c, first, end;  // the chunk, its segment's first, and the first after it
    uint32_t state, seg, part, n, h, hq;
    // job -> state and job of the state; the caller's `seg`, `part` of those
    template <class F> __device__ __forceinline__ void split(const Plan& p, F which) {
        state = job / p.jobs;
        which(*this, job % p.jobs);
        n = state / p.heads;
        h = state % p.heads;
        hq = h / p.shared;
        first = seg * p.segment;
        end = first + p.segment < p.chunks ? first + p.segment : p.chunks;
    }
    template <class F> __device__ __forceinline__ void forth(const Plan& p, F which) {
        if (++c < end) return;
        job += gridDim.x;
        split(p, which);
        c = first;
    }
    template <class F> __device__ __forceinline__ void back(const Plan& p, F which) {
        if (c-- > first) return;
        job += gridDim.x;
        split(p, which);
        c = end - 1;
    }
};

// ---- eight elements of a row, in registers.  Whole pieces move in 16-byte
// words wherever the row starts (global memory takes them at any multiple of
// an element's size), the piece that a row ends in one element at a time.
typedef uint32_t Word __attribute__((ext_vector_type(4)));
template <class E> struct Words;
template <> struct Words<float> { typedef Word type __attribute__((aligned(4))); };
template <> struct Words<bf16> { typedef Word type __attribute__((aligned(2))); };
template <class E> struct Piece { Word w[sizeof(E) / 2]; };

template <class E>
__device__ __forceinline__ Piece<E> load_piece(const E* row, uint32_t dim, uint32_t col) {
    constexpr int W = sizeof(E) / 2, PER = 16 / sizeof(E);
    Piece<E> out;
    if (col + 8 <= dim) {
#pragma unroll
        for (int i = 0; i < W; i++) out.w[i] = *reinterpret_cast<const typename Words<E>::type*>(row + col + i * PER);
    } else {
#pragma unroll
        for (int i = 0; i < W; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t c = col + i * PER + e * (4 / sizeof(E));
                uint32_t bits = 0;
                if (sizeof(E) == 4) {
                    if (c < dim) bits = reinterpret_cast<const uint32_t*>(row)[c];
                } else {
                    if (c < dim) bits = reinterpret_cast<const uint16_t*>(row)[c];
                    if (c + 1 < dim) bits |= uint32_t(reinterpret_cast<const uint16_t*>(row)[c + 1]) << 16;
                }
                out.w[i][e] = bits;
            }
    }
    return out;
}
// Rows past the last tick: zeros, where the piece is used (where it is loaded
// the selection would wait for it).
template <class E>
__device__ __forceinline__ Piece<E> mask_piece(const Piece<E>& x, bool in) {
    Piece<E> out;
#pragma unroll
    for (int i = 0; i < int(sizeof(E) / 2); i++)
#pragma unroll
        for (int e = 0; e < 4; e++) out.w[i][e] = in ? x.w[i][e] : 0u;
    return out;
}
template <class E>
__device__ __forceinline__ void store_piece(E* row, uint32_t dim, uint32_t col, const Piece<E>& in) {
    constexpr int W = sizeof(E) / 2, PER = 16 / sizeof(E);
    if (col + 8 <= dim) {
#pragma unroll
        for (int i = 0; i < W; i++) *reinterpret_cast<typename Words<E>::type*>(row + col + i * PER) = in.w[i];
    } else {
#pragma unroll
        for (int i = 0; i < W; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t c = col + i * PER + e * (4 / sizeof(E)), bits = in.w[i][e];
                if (sizeof(E) == 4) {
                    if (c < dim) reinterpret_cast<uint32_t*>(row)[c] = bits;
                } else {
                    if (c < dim) reinterpret_cast<uint16_t*>(row)[c] = uint16_t(bits);
                    if (c + 1 < dim) reinterpret_cast<uint16_t*>(row)[c + 1] = uint16_t(bits >> 16);
                }
            }
    }
}
// A thread's piece of a chunk's rows: pieces of a row, then rows; there are
// at least as many threads as pieces.
struct Spot {
    uint32_t row, col;
    bool on;
    __device__ __forceinline__ explicit Spot(uint32_t dim) {
        const uint32_t per = (dim + 7) / 8;
        row = threadIdx.x / per;
        col = threadIdx.x % per * 8;
        on = row < uint32_t(CHUNK);
    }
};
// To a row in the order of place(); `m` is the row's start.
__device__ __forceinline__ void piece_to_ordered(bf16* m, uint32_t col, const Piece<bf16>& in) {
    *reinterpret_cast<uint2*>(m + place(int(col))) = uint2{in.w[0][0], in.w[0][1]};
    *reinterpret_cast<uint2*>(m + place(int(col)) + 8) = uint2{in.w[0][2], in.w[0][3]};
}
__device__ __forceinline__ void piece_to_ordered(float* m, uint32_t col, const Piece<float>& in) {
    *reinterpret_cast<Word*>(m + place(int(col))) = in.w[0];
    *reinterpret_cast<Word*>(m + place(int(col)) + 8) = in.w[1];
}
template <class E>
__device__ __forceinline__ void piece_to_lds(E* m, const Piece<E>& in) {
#pragma unroll
    for (int i = 0; i < int(sizeof(E) / 2); i++) reinterpret_cast<Word*>(m)[i] = in.w[i];
}
template <class E>
__device__ __forceinline__ Piece<E> piece_from_lds(const E* m) {
    Piece<E> out;
#pragma unroll
    for (int i = 0; i < int(sizeof(E) / 2); i++) out.w[i] = reinterpret_cast<const Word*>(m)[i];
    return out;
}

// ---- decays of a chunk, in LDS
struct __align__(16) Gates {
    double sum[C];     // g_1 + .. + g_i, in 64 bits: differences of nearby sums keep their digits
    float beta[C];
    float before[C];   // gamma_i, 0 after a flag
    float after[C];    // gamma_C / gamma_i, 0 before the last flag
    float decay[C];    // exp(g_i)
    int episode[C];    // flags up to and with tick i
};
// Four neighbouring values.
__device__ __forceinline__ f32x4 four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
// Whether tick i is an episode's first: nothing before it reaches it.
__device__ __forceinline__ bool gate_is_flag(const Gates& s, int i) {
    return s.episode[i] != (i ? s.episode[i - 1] : 0);
}

struct GateRegs { float g, beta; uint32_t flag; };

// LDS columns past a head's width stay 0: they are operands.
__device__ __forceinline__ void clear_lds(void* lds, uint32_t bytes) {
    for (uint32_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
        *reinterpret_cast<Word*>(static_cast<char*>(lds) + i) = Word{0, 0, 0, 0};
    __syncthreads();
}

__device__ __forceinline__ float one_gate(const char* p, int64_t i, bool f32) {
    return f32 ? reinterpret_cast<const float*>(p)[i] : float(reinterpret_cast<const bf16*>(p)[i]);
}
// One tick's; a tick past the end adds nothing and decays nothing.
template <class E, class A>
__device__ __forceinline__ GateRegs load_gates(const A* a, uint32_t n, uint32_t h, uint32_t t, bool in) {
    GateRegs r{0.0f, 0.0f, 0u};
    if (in) {
        const bool f32 = a->gate_f32 || sizeof(E) == 4;
        r.g = one_gate(a->g.p, int64_t(t) * a->g.tick + int64_t(n) * a->g.env + int64_t(h) * a->g.head, f32);
        r.beta = one_gate(a->beta.p, int64_t(t) * a->beta.tick + int64_t(n) * a->beta.env + int64_t(h) * a->beta.head, f32);
        if (a->reset) r.flag = a->reset[int64_t(t) * a->reset_tick + int64_t(n) * a->reset_env] != 0;
    }
    return r;
}
// By one wavefront, lanes 0..31 its ticks (the others are given zeros).
__device__ __forceinline__ void put_gates(Gates& s, const GateRegs& r) {
    const int l = int(threadIdx.x) & 63;
    const bool flag = r.flag != 0 || r.g < NO_DECAY;
    const uint32_t flags = uint32_t(__ballot(flag));
    const int i = l & 31;
    const int episode = __popc(flags & (0xffffffffu >> (31 - i)));
    const int last = __popc(flags);
    const double sum = scan_up32(flag ? 0.0 : double(r.g), l);
    const double total = lane_value(sum, C - 1);
    if (l < C) {
        s.sum[i] = sum;
        s.beta[i] = r.beta;
        s.decay[i] = __expf(r.g);
        s.episode[i] = episode;
        s.before[i] = episode == 0 ? __expf(float(sum)) : 0.0f;
        s.after[i] = episode == last ? __expf(float(total - sum)) : 0.0f;
    }
}

// D of a tile's entries: rows i0 + 4 (l / 16) + r, column j0 + l % 16; 0 above the diagonal.
__device__ __forceinline__ f32x4 decay_tile(Lane l, const Gates& s, int i0, int j0) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef double f64x2 __attribute__((ext_vector_type(2)));
    const int j = j0 + l.col, i = i0 + 4 * l.quad;
    const double sj = s.sum[j];
    const int ej = s.episode[j];
    const i32x4 ei = *reinterpret_cast<const i32x4*>(s.episode + i);
    const f64x2 lo = *reinterpret_cast<const f64x2*>(s.sum + i), hi = *reinterpret_cast<const f64x2*>(s.sum + i + 2);
    const double si[4] = {lo[0], lo[1], hi[0], hi[1]};
    f32x4 d;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float x = __expf(float(si[r] - sj));
        d[r] = int(i + r >= j) & int(ei[r] == ej) ? x : 0.0f;
    }
    return d;
}

// ---- the triangular system.  The inverse X of 1 + A for a diagonal block, by
// substitution, A and X as result tiles: lane l has rows 4 (l / 16) .. + 3 of
// column l % 16.  The rows of one quad of 16 lanes leave in order (A's entries
// come from the quad's lane of their column by DPP), then go to the quads
// below, which subtract them from their own rows.
template <int J> __device__ __forceinline__ float row_lane(float x) { return from_lane<0x150 + J>(x); }  // row_newbcast

template <int Q> __device__ __forceinline__ void invert_quad(f32x4 a, f32x4& x, int quad) {
    f32x4 y = x;
    y[1] = fmaf(-row_lane<4 * Q>(a[1]), y[0], y[1]);
    y[2] = fmaf(-row_lane<4 * Q>(a[2]), y[0], y[2]);
    y[3] = fmaf(-row_lane<4 * Q>(a[3]), y[0], y[3]);
    y[2] = fmaf(-row_lane<4 * Q + 1>(a[2]), y[1], y[2]);
    y[3] = fmaf(-row_lane<4 * Q + 1>(a[3]), y[1], y[3]);
    y[3] = fmaf(-row_lane<4 * Q + 2>(a[3]), y[2], y[3]);
    if (quad == Q) x = y;
    if (Q == 3) return;
    f32x4 done;
#pragma unroll
    for (int r = 0; r < 4; r++) done[r] = from_quad<Q>(x[r]);
    y = x;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        y[r] = fmaf(-row_lane<4 * Q>(a[r]), done[0], y[r]);
        y[r] = fmaf(-row_lane<4 * Q + 1>(a[r]), done[1], y[r]);
        y[r] = fmaf(-row_lane<4 * Q + 2>(a[r]), done[2], y[r]);
        y[r] = fmaf(-row_lane<4 * Q + 3>(a[r]), done[3], y[r]);
    }
    if (quad > Q) x = y;
}
__device__ __forceinline__ f32x4 invert_block(Lane l, f32x4 a) {
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = 4 * l.quad + r == l.col ? 1.0f : 0.0f;
    invert_quad<0>(a, x, l.quad);
    invert_quad<1>(a, x, l.quad);
    invert_quad<2>(a, x, l.quad);
    invert_quad<3>(a, x, l.quad);
    return x;
}

// The chunk's small matrices in LDS.  All are stored transposed, [j][i]:
// read across rows they are the operand with rows i, along a row the one with
// rows j.
template <class E, int TERMS = Kind<E>::MID> struct System {
    static constexpr int N = TERMS;
    static constexpr int PLANE = C * CP;
    E inv[N * PLANE];          // [j][i]: the diagonal blocks' inverses; A_10 at [j][16 + i]
    E scores[N * PLANE];       // scale D (q_i k_j)
};

// U = (1 + A)^-1 R for 16 columns of R, as two result tiles.
template <class E, int N>
__device__ __forceinline__ void solve(Lane l, const System<E, N>& s, const f32x4 r[2], f32x4 u[2]) {
    constexpr int P = System<E, N>::PLANE;
    const f32x4 zero{0, 0, 0, 0};
    u[0] = zero;
    mma(u[0], col_half<N>(l, s.inv, CP, P, 0, 0), half_of<E, N>(r[0]));
    f32x4 below = zero;
    mma(below, col_half<N>(l, s.inv, CP, P, 0, 16), half_of<E, N>(u[0]));
    u[1] = zero;
    mma(u[1], col_half<N>(l, s.inv, CP, P, 16, 16), half_of<E, N>(r[1] - below));
}
// R = (1 + A)^-T U.
template <class E, int N>
__device__ __forceinline__ void solve_transposed(Lane l, const System<E, N>& s, const f32x4 u[2], f32x4 r[2]) {
    constexpr int P = System<E, N>::PLANE;
    const f32x4 zero{0, 0, 0, 0};
    r[1] = zero;
    mma(r[1], row_half<N>(l, s.inv, CP, P, 16, 16), half_of<E, N>(u[1]));
    f32x4 above = zero;
    mma(above, row_half<N>(l, s.inv, CP, P, 0, 16), half_of<E, N>(r[1]));
    r[0] = zero;
    mma(r[0], row_half<N>(l, s.inv, CP, P, 0, 0), half_of<E, N>(u[0] - above));
}

// ---- chunks with infinities or NaN, passed in or made of numbers that grow
// past fp32 inside the chunk.  A matrix product spreads them: 0 times NaN is
// NaN, so what a tick may not see (a later tick, an episode before a flag)
// would reach it.  For the same reason none gets lost on the way: an operand
// that is not finite leaves a result that is not, in every column whose
// ticks could meet it, and a mask is a factor of 0.  So the results are looked
// at, before any is stored, and a chunk where one is not finite is taken tick
// by tick instead, by the definition.
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }
// Whether all are finite and of ordinary size (their sum is).
__device__ __forceinline__ bool finite(f32x4 x) { return finite((x[0] + x[1]) + (x[2] + x[3])); }

// Four neighbouring places of an ordered row, as fp32: rows 16 i + 4 quad .. + 3 of a state's column.
template <class E> __device__ __forceinline__ f32x4 ordered4(Lane l, const E* row, int i) {
    const E* p = row + (i >> 1) * 32 + 8 * l.quad + (i & 1) * 4;
    return f32x4{float(p[0]), float(p[1]), float(p[2]), float(p[3])};
}
// The decayed state of a tick, in place.
template <int KT> __device__ __forceinline__ void decay_state(f32x4 (&s)[KT], const Gates& gates, int t) {
    const bool flag = gate_is_flag(gates, t);
    const float decay = gates.decay[t];
#pragma unroll
    for (int i = 0; i < KT; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[i][r] = flag ? 0.0f : s[i][r] * decay;
}
// x^T S for the lane's column.
template <class E, int KT> __device__ __forceinline__ float column_dot(Lane l, const f32x4 (&s)[KT], const E* row) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < KT; i++) {
        const f32x4 k = ordered4(l, row, i);
#pragma unroll
        for (int r = 0; r < 4; r++) sum = fmaf(k[r], s[i][r], sum);
        asm volatile("" : "+v"(sum)::"memory");  // a row at a time: this is not to take registers from the products
    }
    return sum_rows32(sum_rows16(sum));
}
// S <- S + k u^T.
template <class E, int KT> __device__ __forceinline__ void add_outer(Lane l, f32x4 (&s)[KT], const E* row, float u) {
#pragma unroll
    for (int i = 0; i < KT; i++) {
        const f32x4 k = ordered4(l, row, i);
#pragma unroll
        for (int r = 0; r < 4; r++) s[i][r] = fmaf(k[r], u, s[i][r]);
        asm volatile("" : "+v"(s[i])::"memory");
    }
}

}  // namespace delta

#endif
