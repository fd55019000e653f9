// block_norm.hip — the norms around a block, fused with its gate and residual
// scale:  n = y / rms(y),  s = r x + gate n w_post,  h = (s / rms(s)) w_pre.
//
// A row belongs to `G` lanes (a part of a wavefront, one, or a workgroup); a
// lane has P pieces of W elements of it in registers from the loads to the
// stores, so a row is read once and written once.  All arithmetic is fp32;
// h is made from s before s is rounded to its type, in both directions.
//
// Backward, with dh and ds: z = dh w_pre,
//     t = ds + z / rms(s) - s mean(z s) / rms(s)^3      (the whole gradient of s)
//     dx = r t,   d_gate = t n w_post,   dn = t gate w_post,
//     dy = dn / rms(y) - y mean(dn y) / rms(y)^3
// with sum(dn y) = sum((ds + z / rms(s)) gate w_post y) - mean(z s) / rms(s)^3
// sum(s gate w_post y), so that a row's sums are made at once: a row of a
// workgroup has one barrier.  The column sums are those
// of dh s / rms(s), t gate n, t x (and t n w_post for a gate
// per channel).  A lane always has the same columns and adds up its rows' terms
// in registers; workgroups write one row of sums each and a second kernel adds
// those up in a fixed order: no atomics, the same bits every time.
#include "block_norm.h"

#include "lane_sums.h"

namespace blocknorm {
namespace {

typedef __bf16 bf16;

enum Gate { NONE = MDN_GATE_NONE, CHANNEL = MDN_GATE_CHANNEL, ROW = MDN_GATE_ROW, ELEMENT = MDN_GATE_ELEMENT };

__device__ __forceinline__ int64_t row_at(const Rows& r, const Args& a, uint64_t row) {
    if (r.outer == int64_t(a.inner_count) * r.inner) return int64_t(row) * r.inner;
    return int64_t(row / a.inner_count) * r.outer + int64_t(row % a.inner_count) * r.inner;
}

// A lane's elements: P pieces of W neighbours, a piece per lane and then the
// next ones.  A piece moves in 16-byte words at whatever address the row
// starts (global memory takes words at any multiple of the element's size);
// the piece that the row ends in moves one element at a time.
template <int W> __device__ __forceinline__ uint32_t place(uint32_t p, uint32_t lane, uint32_t group) { return (p * group + lane) * W; }

// Lanes of the widest workgroup: a lane of 8 elements needs up to 168 registers
// in the backward pass, of which 768 lanes (three wavefronts on each SIMD)
// have as many; one of 16 needs 256, which leaves 512 lanes.
constexpr uint32_t most_lanes(int p, int w) { return p * w <= 8 ? 768 : 512; }

typedef uint32_t Word __attribute__((ext_vector_type(4)));
template <class T> struct Words;
template <> struct Words<float> { typedef Word type __attribute__((aligned(4))); };
template <> struct Words<bf16> { typedef Word type __attribute__((aligned(2))); };

// A lane's part of a row as it is in memory: loaded a row ahead, and turned
// into fp32 where it is used (that costs an instruction each time and saves
// half of the registers).  Elements past the row's end are 0.
template <class T, int P, int W> struct Raw { Word w[P][W * sizeof(T) / 16]; };

template <class T, int P, int W>
__device__ __forceinline__ void fetch(Raw<T, P, W>& out, const T* row, uint32_t lane, uint32_t group, uint32_t width) {
    constexpr int N = W * sizeof(T) / 16, PER = 16 / sizeof(T);
#pragma unroll
    for (int p = 0; p < P; p++) {
        const uint32_t at = place<W>(p, lane, group);
        if (at + W <= width) {
#pragma unroll
            for (int w = 0; w < N; w++) out.w[p][w] = *reinterpret_cast<const typename Words<T>::type*>(row + at + w * PER);
        } else {
#pragma unroll
            for (int w = 0; w < N; w++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t c = at + w * PER + i * (4 / sizeof(T));
                    uint32_t bits = 0;
                    if (sizeof(T) == 4) {
                        if (c < width) bits = reinterpret_cast<const uint32_t*>(row)[c];
                    } else {
                        if (c < width) bits = reinterpret_cast<const uint16_t*>(row)[c];
                        if (c + 1 < width) bits |= uint32_t(reinterpret_cast<const uint16_t*>(row)[c + 1]) << 16;
                    }
                    out.w[p][w][i] = bits;
                }
        }
    }
}
// Element e of piece p in fp32.
template <class T, int P, int W>
__device__ __forceinline__ float value(const Raw<T, P, W>& in, int p, int e) {
    if (sizeof(T) == 2) {
        const uint32_t pair = in.w[p][e / 8][e / 2 % 4];
        return __builtin_bit_cast(float, e % 2 ? pair & 0xffff0000u : pair << 16);
    }
    return __builtin_bit_cast(float, uint32_t(in.w[p][e / 4][e % 4]));
}
template <class T, int P, int W>
__device__ __forceinline__ void load(float (&out)[P][W], const T* row, uint32_t lane, uint32_t group, uint32_t width) {
    Raw<T, P, W> raw;
    fetch<T, P, W>(raw, row, lane, group, width);
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
        for (int e = 0; e < W; e++) out[p][e] = value(raw, p, e);
}
// One piece.
template <class T, int W>
__device__ __forceinline__ void store(T* row, const float (&in)[W], uint32_t at, uint32_t width) {
    constexpr int N = W * sizeof(T) / 16, PER = 16 / sizeof(T);
    if (at + W <= width) {
#pragma unroll
        for (int w = 0; w < N; w++) {
            union { Word u; T t[PER]; } v;
#pragma unroll
            for (int e = 0; e < PER; e++) v.t[e] = T(in[w * PER + e]);
            *reinterpret_cast<typename Words<T>::type*>(row + at + w * PER) = v.u;
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < W; e++)
            if (at + e < width) row[at + e] = T(in[e]);
    }
}

// Sums over a row's lanes.  G 0: the whole workgroup, through LDS, where each
// sixteen lanes add up the wavefronts' sums; `lds` is another one than the last
// sum's, so that one barrier is enough, and 0 past the workgroup's wavefronts.
constexpr int WAVES = 16;
template <int G, int N, class A>
__device__ __forceinline__ void row_sum(A (&v)[N], A (*lds)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = lanes::sum16(v[i]);
        if constexpr (G == 0 || G >= 32) v[i] = lanes::sum_rows16(v[i]);
        if constexpr (G == 0 || G >= 64) v[i] = lanes::sum_rows32(v[i]);
    }
    if (G == 0) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) lds[threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = lanes::sum16(lds[threadIdx.x & 15][i]);
    }
}
template <int G, int N, class A> __device__ __forceinline__ void clear_sums(A (*lds)[WAVES][N]) {
    if (G != 0) return;
    if (threadIdx.x < 2 * WAVES)
#pragma unroll
        for (int i = 0; i < N; i++) lds[threadIdx.x / WAVES][threadIdx.x % WAVES][i] = 0;
    __syncthreads();
}

// The channels' vectors: in registers for the whole call where a row has at
// most a wavefront's lanes, else in LDS (a workgroup's rows share them, and
// the registers are needed for the row and for the next one).
template <int G, int P, int W> struct Channels {
    float v[P][W];
    __device__ __forceinline__ void init(const float* from, float*, uint32_t lane, uint32_t group, uint32_t width) {
        load<float, P, W>(v, from, lane, group, width);
    }
    __device__ __forceinline__ float at(int p, int e, const float*, uint32_t, uint32_t) const { return v[p][e]; }
};
template <int P, int W> struct Channels<0, P, W> {
    __device__ __forceinline__ void init(const float* from, float* lds, uint32_t lane, uint32_t group, uint32_t width) {
        float v[P][W];
        load<float, P, W>(v, from, lane, group, width);
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) lds[place<W>(p, lane, group) + e] = v[p][e];
    }
    __device__ __forceinline__ float at(int p, int e, const float* lds, uint32_t lane, uint32_t group) const {
        return lds[place<W>(p, lane, group) + e];
    }
};

template <class TY>
__device__ __forceinline__ float one_gate(const Args& a, int64_t at) {
    return a.gate_f32 ? reinterpret_cast<const float*>(a.gate.p)[at] : float(reinterpret_cast<const TY*>(a.gate.p)[at]);
}

// One row's inputs as loaded.
template <class TX, class TY, int P, int W, int GATE> struct Inputs {
    Raw<TX, P, W> x;
    Raw<TY, P, W> y, gate;
    float one;  // the row's gate
    __device__ __forceinline__ void fetch_row(const Args& a, uint64_t row, uint32_t lane, uint32_t group) {
        fetch<TY, P, W>(y, reinterpret_cast<const TY*>(a.y.p) + row_at(a.y, a, row), lane, group, a.width);
        fetch<TX, P, W>(x, reinterpret_cast<const TX*>(a.x.p) + row_at(a.x, a, row), lane, group, a.width);
        if (GATE == ELEMENT)
            fetch<TY, P, W>(gate, reinterpret_cast<const TY*>(a.gate.p) + row_at(a.gate, a, row), lane, group, a.width);
        one = GATE == ROW ? one_gate<TY>(a, row_at(a.gate, a, row)) : 1.0f;
    }
};
// The channels' vectors, with the gate's if it is one.
template <class TX, class TY, int G, int P, int W, int GATE> struct Weights {
    Channels<G, P, W> post, pre, residual;
    float gate[P][W];
    float* lds;
    uint32_t size, lane, group;
    bool scaled;
    __device__ __forceinline__ void init(const Args& a, float* shared, uint32_t l, uint32_t g) {
        lds = shared;
        lane = l;
        group = g;
        size = g * P * W;
        scaled = a.residual != nullptr;
        post.init(a.w_post, lds, l, g, a.width);
        pre.init(a.w_pre, lds + size, l, g, a.width);
        if (scaled) residual.init(a.residual, lds + 2 * size, l, g, a.width);
        if (GATE == CHANNEL) {
            if (a.gate_f32)
                load<float, P, W>(gate, reinterpret_cast<const float*>(a.gate.p), l, g, a.width);
            else
                load<TY, P, W>(gate, reinterpret_cast<const TY*>(a.gate.p), l, g, a.width);
        }
        // (a lane reads back only what it wrote: no barrier)
    }
    __device__ __forceinline__ float post_at(int p, int e) const { return post.at(p, e, lds, lane, group); }
    __device__ __forceinline__ float pre_at(int p, int e) const { return pre.at(p, e, lds + size, lane, group); }
    __device__ __forceinline__ float residual_at(int p, int e) const { return residual.at(p, e, lds + 2 * size, lane, group); }
    typedef Inputs<TX, TY, P, W, GATE> In;
    __device__ __forceinline__ float gate_at(const In& in, int p, int e) const {
        return GATE == NONE ? 1.0f : GATE == ROW ? in.one : GATE == ELEMENT ? value(in.gate, p, e) : gate[p][e];
    }
    // s from b = y / rms(y) w_post
    __device__ __forceinline__ float s(const In& in, int p, int e, float b) const {
        const float gb = GATE == NONE ? b : gate_at(in, p, e) * b, x = value(in.x, p, e);
        return scaled ? fmaf(residual_at(p, e), x, gb) : x + gb;
    }
};

// A wavefront whose lanes share rows has a row in scalar registers.
template <int G> __device__ __forceinline__ uint32_t row_in_group() {
    if (G == 0) return 0;
    const uint32_t r = threadIdx.x / G;
    return G == 64 ? __builtin_amdgcn_readfirstlane(r) : r;
}

// Bound by memory, under a profiler: 262,144 x 256 in bfloat16 (0.54 GB) takes 92
// us, 5.8 TB/s, with the stream in fp32 (0.81 GB) 147; 32,768 x 5,120 with a gate
// per element (1.68 GB) 317 us, 5.3 TB/s, with the stream in fp32 (2.35 GB) 462; 37,000 x
// 181 in fp32, rows of 724 bytes (0.11 GB), 30 us, 3.6 TB/s (24 us from the cache).
template <class TX, class TY, int G, int P, int W, int GATE>
__global__ void __launch_bounds__(G == 0 ? most_lanes(P, W) : 256) forward_kernel(Args a) {
    __shared__ float lds[2][WAVES][1];
    clear_sums<G>(lds);
    extern __shared__ __align__(16) float channels[];
    const uint32_t group = G == 0 ? blockDim.x : G, per = G == 0 ? 1 : 256 / G;
    const uint32_t lane = threadIdx.x % group, width = a.width;
    Weights<TX, TY, G, P, W, GATE> wt;
    wt.init(a, channels, lane, group);
    const uint64_t step = uint64_t(gridDim.x) * per;
    Inputs<TX, TY, P, W, GATE> now, next;
    const uint64_t mine0 = uint64_t(blockIdx.x) * per + row_in_group<G>();
    // lanes past the end repeat the last row's loads
    next.fetch_row(a, mine0 < a.rows ? mine0 : a.rows - 1, lane, group);
    for (uint64_t mine = mine0, first = uint64_t(blockIdx.x) * per; first < a.rows; first += step, mine += step) {
        const uint64_t row = mine < a.rows ? mine : a.rows - 1;
        now = next;
        if (first + step < a.rows) next.fetch_row(a, mine + step < a.rows ? mine + step : a.rows - 1, lane, group);
        float sum[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float y = value(now.y, p, e);
                sum[0] = fmaf(y, y, sum[0]);
            }
        row_sum<G>(sum, lds[0]);
        const float ry = 1.0f / sqrtf(sum[0] / float(width) + a.eps);
        sum[0] = 0.0f;
        float s[P][W];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                s[p][e] = wt.s(now, p, e, value(now.y, p, e) * ry * wt.post_at(p, e));
                sum[0] = fmaf(s[p][e], s[p][e], sum[0]);
            }
        row_sum<G>(sum, lds[1]);
        const float rs = 1.0f / sqrtf(sum[0] / float(width) + a.eps);
        if (mine < a.rows) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                const uint32_t at = place<W>(p, lane, group);
                store<TX, W>(reinterpret_cast<TX*>(a.s.p) + row_at(a.s, a, row), s[p], at, width);
#pragma unroll
                for (int e = 0; e < W; e++) s[p][e] = s[p][e] * rs * wt.pre_at(p, e);
                store<TY, W>(reinterpret_cast<TY*>(a.h.p) + row_at(a.h, a, row), s[p], at, width);
            }
            if (a.stats && lane == 0) {
                a.stats[2 * row] = ry;
                a.stats[2 * row + 1] = rs;
            }
        }
    }
}

// In rows of up to 16 pieces what the norms leave of a gradient can be a small
// difference of large parts (in a row of one element it is the share of
// epsilon): there the row's sums and differences are formed in 64 bits, and
// the norms again from the row.  Wider rows take them in 32 bits.
//
// Bound by memory, under a profiler: 262,144 x 256 in bfloat16 (0.81 GB) takes 160
// us, 5.0 TB/s, with the stream in fp32 (1.21 GB) 234; 32,768 x 5,120 with a gate per
// element (2.68 GB) 700 to 780 us, 3.6 TB/s, with the stream in fp32 (3.69 GB) 774: its
// column sums, the row and the next one fill the registers that one workgroup of
// ten wavefronts a compute unit has, so one row is on its way while one is worked
// on (vector units busy 37 % of the time, a wavefront waits 69 % of its).  Measured
// there beside 720 us: two rows ahead, which spills, 882; two sums a row one after
// the other through LDS 784 (and 209 beside 165 in the first case).
template <int G> struct Sum { typedef float type; };
template <> struct Sum<16> { typedef double type; };

template <class TX, class TY, int G, int P, int W, int GATE>
__global__ void __launch_bounds__(G == 0 ? most_lanes(P, W) : 256) backward_kernel(Args a, GradArgs d) {
    typedef typename Sum<G>::type A;
    constexpr bool AGAIN = G == 16;  // the norms are made again
    constexpr int SUMS = AGAIN ? 5 : 3;
    __shared__ A lds[2][WAVES][SUMS];
    clear_sums<G>(lds);
    extern __shared__ __align__(16) float channels[];
    const uint32_t group = G == 0 ? blockDim.x : G, per = G == 0 ? 1 : 256 / G;
    const uint32_t lane = threadIdx.x % group, width = a.width;
    // column sums of t gate n, dh s / rms(s), t x, t n w_post
    float c_post[P][W] = {}, c_pre[P][W] = {}, c_res[P][W] = {}, c_gate[P][W] = {};
    Weights<TX, TY, G, P, W, GATE> wt;
    wt.init(a, channels, lane, group);
    const uint64_t step = uint64_t(gridDim.x) * per;
    struct Row {
        Inputs<TX, TY, P, W, GATE> in;
        Raw<TX, P, W> ds;
        Raw<TY, P, W> dh;
        float ry, rs;
    } now = {}, next = {};
    const auto fetch_row = [&](Row& to, uint64_t mine) {
        const uint64_t row = mine < a.rows ? mine : a.rows - 1;  // lanes past the end repeat the last row's loads
        to.in.fetch_row(a, row, lane, group);
        if (d.d_h.p) fetch<TY, P, W>(to.dh, reinterpret_cast<const TY*>(d.d_h.p) + row_at(d.d_h, a, row), lane, group, width);
        if (d.d_s.p) fetch<TX, P, W>(to.ds, reinterpret_cast<const TX*>(d.d_s.p) + row_at(d.d_s, a, row), lane, group, width);
        to.ry = a.stats[2 * row];
        to.rs = a.stats[2 * row + 1];
    };
    const uint64_t mine0 = uint64_t(blockIdx.x) * per + row_in_group<G>();
    fetch_row(next, mine0);
    for (uint64_t mine = mine0, first = uint64_t(blockIdx.x) * per, turn = 0; first < a.rows; first += step, mine += step, turn ^= 1) {
        const bool in = mine < a.rows;
        const uint64_t row = in ? mine : a.rows - 1;
        now = next;
        if (first + step < a.rows) fetch_row(next, mine + step);
        A ry = now.ry, rs = now.rs;
        if (AGAIN) {
            A squares[1] = {0};
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++) squares[0] += A(value(now.in.y, p, e)) * A(value(now.in.y, p, e));
            row_sum<G, 1, A>(squares, nullptr);
            ry = A(1) / sqrt(squares[0] / A(width) + A(a.eps));
        }
        const float ryf = float(ry);
        // z s, what t is made of (z without rs where that is not known yet) times gate w_post y, s times that
        A sum[SUMS] = {};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float y = value(now.in.y, p, e), w = wt.post_at(p, e), s = wt.s(now.in, p, e, y * ryf * w);
                const A z = value(now.dh, p, e) * wt.pre_at(p, e), ds = value(now.ds, p, e);
                const A wy = (GATE == ROW ? A(w) : A(wt.gate_at(now.in, p, e)) * A(w)) * A(y);
                sum[0] += z * A(s);
                sum[1] += (AGAIN ? z : ds + rs * z) * wy;
                sum[2] += A(s) * wy;
                if (AGAIN) {
                    sum[SUMS - 2] += ds * wy;
                    sum[SUMS - 1] += A(s) * A(s);
                }
                if (P > 1 && e == W - 1) asm volatile("" : "+v"(sum[0])::"memory");  // the next piece's channels are read after this one's use
            }
        row_sum<G>(sum, lds[turn]);
        if (AGAIN) {
            rs = A(1) / sqrt(sum[SUMS - 1] / A(width) + A(a.eps));
            sum[1] = sum[SUMS - 2] + rs * sum[1];
        }
        if (!in) continue;
        const float rsf = float(rs);
        const A back = sum[0] / A(width) * rs * rs * rs;
        const A along = sum[1] - back * sum[2];  // t w_post y, times the gate if it is not the row's
        const A pull = along * (GATE == ROW ? A(now.in.one) : A(1)) / A(width) * ry * ry * ry;
#pragma unroll
        for (int p = 0; p < P; p++) {
            float out[W], dgate[W], dy[W];
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float y = value(now.in.y, p, e), x = value(now.in.x, p, e), dh = value(now.dh, p, e);
                const float n = y * ryf, w = wt.post_at(p, e), b = n * w, s = wt.s(now.in, p, e, b), gv = wt.gate_at(now.in, p, e);
                const A ta = A(value(now.ds, p, e)) + (rs * A(dh * wt.pre_at(p, e)) - back * A(s));
                const float t = float(ta);
                c_pre[p][e] = fmaf(dh, s * rsf, c_pre[p][e]);
                c_post[p][e] = fmaf(t, gv * n, c_post[p][e]);
                c_res[p][e] = fmaf(t, x, c_res[p][e]);
                if (GATE == CHANNEL) c_gate[p][e] = fmaf(t, b, c_gate[p][e]);
                if (GATE == ELEMENT) dgate[e] = t * b;
                out[e] = wt.scaled ? wt.residual_at(p, e) * t : t;
                dy[e] = float(ry * (ta * (A(gv) * A(w))) - pull * A(y));
            }
            const uint32_t at = place<W>(p, lane, group);
            store<TX, W>(reinterpret_cast<TX*>(d.d_x.p) + row_at(d.d_x, a, row), out, at, width);
            if (GATE == ELEMENT) store<TY, W>(reinterpret_cast<TY*>(d.d_gate.p) + row_at(d.d_gate, a, row), dgate, at, width);
            store<TY, W>(reinterpret_cast<TY*>(d.d_y.p) + row_at(d.d_y, a, row), dy, at, width);
            if (P > 1) asm volatile("" ::: "memory");
        }
        if (GATE == ROW && lane == 0) {
            const int64_t at = row_at(d.d_gate, a, row);
            const float value = float(ry * along);
            if (a.gate_f32)
                reinterpret_cast<float*>(d.d_gate.p)[at] = value;
            else
                reinterpret_cast<TY*>(d.d_gate.p)[at] = TY(value);
        }
    }
    // the workgroup's column sums: its groups of lanes add theirs up in order
    float* parts = d.parts + uint64_t(blockIdx.x) * 4 * width;
    const auto column_sum = [&](const float(&v)[P][W], float* out) {
        if (G != 0) {
            for (uint32_t r = 0; r < per; r++) {
                __syncthreads();
                if (threadIdx.x / group == r)
#pragma unroll
                    for (int p = 0; p < P; p++)
#pragma unroll
                        for (int e = 0; e < W; e++) {
                            float& to = channels[place<W>(p, lane, group) + e];
                            to = r ? to + v[p][e] : v[p][e];
                        }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < width; i += 256) out[i] = channels[i];
        } else {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++)
                    if (place<W>(p, lane, group) + e < width) out[place<W>(p, lane, group) + e] = v[p][e];
        }
    };
    column_sum(c_post, parts);
    column_sum(c_pre, parts + width);
    column_sum(c_res, parts + 2 * uint64_t(width));
    column_sum(c_gate, parts + 3 * uint64_t(width));
}

// Adds up the workgroups' rows of column sums: 64 columns per workgroup, a
// sixteenth of the rows per wavefront, eight loads in flight.  5 us for 256
// rows of 4 x 5,120 columns: a launch and three round trips to memory.
__global__ void __launch_bounds__(1024) columns_kernel(const float* parts, uint32_t count, uint32_t width, float* post, float* pre,
                                                       float* res, char* gate, uint32_t gate_f32) {
    __shared__ float lds[16][64];
    const uint32_t at = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    float part[8] = {};
    if (at < 4 * width) {
        uint32_t i = slice;
        for (; i + 7 * 16 < count; i += 8 * 16)
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) part[j] += parts[uint64_t(i + 16 * j) * 4 * width + at];
        for (uint32_t j = 0; i < count; i += 16, j++) part[j & 7] += parts[uint64_t(i) * 4 * width + at];
    }
    lds[slice][threadIdx.x & 63] = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
    __syncthreads();
    if (slice != 0 || at >= 4 * width) return;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) sum += lds[i][threadIdx.x];
    const uint32_t which = at / width, c = at % width;
    if (which == 0) post[c] = sum;
    if (which == 1) pre[c] = sum;
    if (which == 2 && res) res[c] = sum;
    if (which == 3 && gate) {
        if (gate_f32)
            reinterpret_cast<float*>(gate)[c] = sum;
        else
            reinterpret_cast<bf16*>(gate)[c] = bf16(sum);
    }
}

// The lanes of a row: one piece of W elements each on a part of a wavefront,
// one, or a workgroup of at most most_lanes(); up to 16 elements a lane in wider rows.
// 262,144 x 256 in bfloat16 on halves of wavefronts and on whole ones: 99 : 168 us
// forward, 265 : 686 with the backward pass; 1,048,576 x 64 in fp32 on quarters and on
// whole ones 214 : 468 and 589 : 1,334 (calls in a row, each with inputs of its own).
struct Shape { uint32_t lanes, pieces; };
inline Shape shape_of(uint32_t width, uint32_t w, uint32_t lanes_1, uint32_t lanes_2) {
    const uint32_t pieces = (width + w - 1) / w;
    if (pieces <= 16) return {16, 1};
    if (pieces <= 32) return {32, 1};
    if (pieces <= 64) return {64, 1};
    const uint32_t p = pieces <= lanes_1 ? 1 : pieces <= 2 * lanes_2 ? 2 : 4;
    return {((pieces + p - 1) / p + 63) / 64 * 64, p};
}
inline Shape backward_shape(uint32_t width, uint32_t w) { return shape_of(width, w, most_lanes(1, w), most_lanes(2, w)); }
// Forward, where a lane needs few registers, two workgroups of half the lanes
// are faster than one: 330 against 365 us at 32,768 x 5,120 bfloat16 (measured so too).
inline Shape forward_shape(uint32_t width, uint32_t w) { return shape_of(width, w, 512, 512); }
// Workgroups, each with several rows in turn: enough to fill the GPU's 256 compute units.
inline uint32_t blocks_of(const Args& a, const Shape& s) {
    const uint64_t per = s.lanes > 64 ? 1 : 256 / s.lanes;
    const uint64_t most = (a.rows + per - 1) / per;
    const uint64_t full = 256 * (s.lanes > 64 ? (s.lanes * s.pieces <= 256 ? 4 : s.lanes <= 384 ? 2 : 1) : 4);
    return uint32_t(most < full ? most : full);
}
// LDS for the channels' vectors of a row that takes a workgroup.
inline uint32_t channel_bytes(const Shape& s, uint32_t w) { return s.lanes > 64 ? 3 * s.lanes * s.pieces * w * 4 : 0; }

template <class K, class... X>
hipError_t launch(K kernel, uint32_t blocks, uint32_t threads, uint32_t bytes, hipStream_t st, X... args) {
    if (bytes > 64 * 1024)
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)))
            return e;
    kernel<<<dim3(blocks), dim3(threads), bytes, st>>>(args...);
    return hipGetLastError();
}

template <class TX, class TY, int W, int GATE>
hipError_t forward(const Args& a, hipStream_t st) {
    const Shape s = forward_shape(a.width, W);
    const uint64_t per = s.lanes > 64 ? 1 : 256 / s.lanes;
    const uint64_t rows = (a.rows + per - 1) / per;
    const uint32_t most = s.lanes > 64 ? 4 * blocks_of(a, s) : 4096, grid = uint32_t(rows < most ? rows : most), bytes = channel_bytes(s, W);
    if constexpr (W == 4)
        if (s.lanes > 64 && s.pieces == 4) return launch(forward_kernel<TX, TY, 0, 4, W, GATE>, grid, s.lanes, bytes, st, a);
    if (s.lanes > 64 && s.pieces == 2) return launch(forward_kernel<TX, TY, 0, 2, W, GATE>, grid, s.lanes, bytes, st, a);
    if (s.lanes > 64) return launch(forward_kernel<TX, TY, 0, 1, W, GATE>, grid, s.lanes, bytes, st, a);
    if (s.lanes == 16) return launch(forward_kernel<TX, TY, 16, 1, W, GATE>, grid, 256, 0, st, a);
    if (s.lanes == 32) return launch(forward_kernel<TX, TY, 32, 1, W, GATE>, grid, 256, 0, st, a);
    return launch(forward_kernel<TX, TY, 64, 1, W, GATE>, grid, 256, 0, st, a);
}
template <class TX, class TY, int W, int GATE>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t st) {
    const Shape s = backward_shape(a.width, W);
    const uint32_t grid = blocks_of(a, s), bytes = s.lanes > 64 ? channel_bytes(s, W) : s.lanes * W * 4;
    if constexpr (W == 4)
        if (s.lanes > 64 && s.pieces == 4) return launch(backward_kernel<TX, TY, 0, 4, W, GATE>, grid, s.lanes, bytes, st, a, d);
    if (s.lanes > 64 && s.pieces == 2) return launch(backward_kernel<TX, TY, 0, 2, W, GATE>, grid, s.lanes, bytes, st, a, d);
    if (s.lanes > 64) return launch(backward_kernel<TX, TY, 0, 1, W, GATE>, grid, s.lanes, bytes, st, a, d);
    if (s.lanes == 16) return launch(backward_kernel<TX, TY, 16, 1, W, GATE>, grid, 256, bytes, st, a, d);
    if (s.lanes == 32) return launch(backward_kernel<TX, TY, 32, 1, W, GATE>, grid, 256, bytes, st, a, d);
    return launch(backward_kernel<TX, TY, 64, 1, W, GATE>, grid, 256, bytes, st, a, d);
}

template <class TY> constexpr int words() { return 16 / int(sizeof(TY)); }

template <class TX, class TY, class F>
hipError_t by_gate(const Args& a, F f) {
    switch (a.gate_kind) {
        case CHANNEL: return f.template run<TX, TY, CHANNEL>();
        case ROW: return f.template run<TX, TY, ROW>();
        case ELEMENT: return f.template run<TX, TY, ELEMENT>();
        default: return f.template run<TX, TY, NONE>();
    }
}
template <class F>
hipError_t by_type(const Args& a, uint32_t x_type, uint32_t y_type, F f) {
    if (x_type == MDN_BF16) return by_gate<bf16, bf16>(a, f);
    return y_type == MDN_BF16 ? by_gate<float, bf16>(a, f) : by_gate<float, float>(a, f);
}
struct Forward {
    const Args& a;
    hipStream_t st;
    template <class TX, class TY, int GATE> hipError_t run() { return forward<TX, TY, words<TY>(), GATE>(a, st); }
};
struct Backward {
    const Args& a;
    const GradArgs& d;
    hipStream_t st;
    template <class TX, class TY, int GATE> hipError_t run() { return backward<TX, TY, words<TY>(), GATE>(a, d, st); }
};

}  // namespace

hipError_t launch_forward(const Args& a, uint32_t x_type, uint32_t y_type, hipStream_t stream) {
    return by_type(a, x_type, y_type, Forward{a, stream});
}

uint32_t parts(const Args& a, uint32_t y_type) {
    return a.rows ? blocks_of(a, backward_shape(a.width, y_type == MDN_BF16 ? 8 : 4)) : 0;
}

hipError_t launch_backward(const Args& a, const GradArgs& d, uint32_t x_type, uint32_t y_type, hipStream_t stream) {
    const uint32_t count = parts(a, y_type);
    if (count)
        if (hipError_t e = by_type(a, x_type, y_type, Backward{a, d, stream})) return e;
    columns_kernel<<<dim3((4 * a.width + 63) / 64), dim3(1024), 0, stream>>>(
        d.parts, count, a.width, d.d_w_post, d.d_w_pre, a.residual ? d.d_residual : nullptr,
        a.gate_kind == CHANNEL ? d.d_gate.p : nullptr, a.gate_f32);
    return hipGetLastError();
}

}  // namespace blocknorm
