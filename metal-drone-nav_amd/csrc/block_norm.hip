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
// and the column sums of dh s / rms(s), t gate n, t x (and t n w_post for a gate
// per channel).  A lane always has the same columns and adds up its rows' terms
// in registers; workgroups write one row of sums each and a second kernel adds
// those up in a fixed order: no atomics, the same bits every time.
#include "block_norm.h"

namespace blocknorm {
namespace {

typedef __bf16 bf16;

enum Gate { NONE = MDN_GATE_NONE, CHANNEL = MDN_GATE_CHANNEL, ROW = MDN_GATE_ROW, ELEMENT = MDN_GATE_ELEMENT };

__device__ __forceinline__ int64_t row_at(const Rows& r, const Args& a, uint64_t row) {
    if (r.outer == int64_t(a.inner_count) * r.inner) return int64_t(row) * r.inner;
    return int64_t(row / a.inner_count) * r.outer + int64_t(row % a.inner_count) * r.inner;
}

// Where a lane's elements are.  VEC (widths of whole pieces): pieces of W
// neighbours, moved in 16-byte words if all rows are aligned to them (`wide`)
// and one by one if not, so that alignment does not change the order of a sum;
// otherwise neighbouring lanes have neighbouring elements.
template <int W, bool VEC>
__device__ __forceinline__ uint32_t place(uint32_t p, uint32_t e, uint32_t lane, uint32_t group) {
    return VEC ? (p * group + lane) * W + e : (p * W + e) * group + lane;
}

template <class T, int P, int W, bool VEC>
__device__ __forceinline__ void load(float (&out)[P][W], const T* row, uint32_t lane, uint32_t group, uint32_t width, bool wide) {
#pragma unroll
    for (int p = 0; p < P; p++) {
        if (VEC && wide) {
            constexpr int PER = 16 / sizeof(T);
            const uint32_t at = place<W, true>(p, 0, lane, group);
            const bool in = at < width;
            const T* q = row + (in ? at : 0u);
#pragma unroll
            for (int w = 0; w < W; w += PER) {
                union { uint4 u; T t[PER]; } v;
                v.u = *reinterpret_cast<const uint4*>(q + w);
#pragma unroll
                for (int e = 0; e < PER; e++) out[p][w + e] = in ? float(v.t[e]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < W; e++) {
                const uint32_t at = place<W, VEC>(p, e, lane, group);
                const float v = float(row[at < width ? at : 0u]);
                out[p][e] = at < width ? v : 0.0f;
            }
        }
    }
}
template <class T, int P, int W, bool VEC>
__device__ __forceinline__ void store(T* row, const float (&in)[P][W], uint32_t lane, uint32_t group, uint32_t width, bool wide) {
#pragma unroll
    for (int p = 0; p < P; p++) {
        if (VEC && wide) {
            constexpr int PER = 16 / sizeof(T);
            const uint32_t at = place<W, true>(p, 0, lane, group);
            if (at >= width) continue;
#pragma unroll
            for (int w = 0; w < W; w += PER) {
                union { uint4 u; T t[PER]; } v;
#pragma unroll
                for (int e = 0; e < PER; e++) v.t[e] = T(in[p][w + e]);
                *reinterpret_cast<uint4*>(row + at + w) = v.u;
            }
        } else {
#pragma unroll
            for (int e = 0; e < W; e++) {
                const uint32_t at = place<W, VEC>(p, e, lane, group);
                if (at < width) row[at] = T(in[p][e]);
            }
        }
    }
}

// Sums over a row's lanes.  G 0: the whole workgroup, through LDS.
template <int G, int N, class A>
__device__ __forceinline__ void row_sum(A (&v)[N], A (*lds)[N]) {
    constexpr int IN_WAVE = G == 0 ? 64 : G;
#pragma unroll
    for (int d = 1; d < IN_WAVE; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor(v[i], d);
    if (G == 0) {
        const uint32_t waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
        __syncthreads();  // the last sum's readers are done
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; i++) lds[wave][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 0;
        for (uint32_t w = 0; w < waves; w++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += lds[w][i];
    }
}

template <class TY>
__device__ __forceinline__ float one_gate(const Args& a, int64_t at) {
    return a.gate_f32 ? reinterpret_cast<const float*>(a.gate.p)[at] : float(reinterpret_cast<const TY*>(a.gate.p)[at]);
}

template <class TX, class TY, int G, int P, int W, bool VEC, int GATE>
__global__ void __launch_bounds__(G == 0 ? 1024 : 256) forward_kernel(Args a) {
    __shared__ float lds[16][1];
    const uint32_t group = G == 0 ? blockDim.x : G, per = G == 0 ? 1 : 256 / G;
    const uint32_t lane = threadIdx.x % group, width = a.width;
    float wp[P][W], wq[P][W], res[P][W], gate[P][W];
    load<float, P, W, VEC>(wp, a.w_post, lane, group, width, a.wide);
    load<float, P, W, VEC>(wq, a.w_pre, lane, group, width, a.wide);
    if (a.residual) load<float, P, W, VEC>(res, a.residual, lane, group, width, a.wide);
    if (GATE == CHANNEL) {
        if (a.gate_f32)
            load<float, P, W, VEC>(gate, reinterpret_cast<const float*>(a.gate.p), lane, group, width, a.wide);
        else
            load<TY, P, W, VEC>(gate, reinterpret_cast<const TY*>(a.gate.p), lane, group, width, a.wide);
    }
    const uint64_t step = uint64_t(gridDim.x) * per;
    for (uint64_t first = uint64_t(blockIdx.x) * per; first < a.rows; first += step) {
        const uint64_t mine = first + (G == 0 ? 0 : threadIdx.x / group);
        const uint64_t row = mine < a.rows ? mine : a.rows - 1;  // lanes past the end repeat the last row's loads
        float x[P][W], y[P][W];
        load<TY, P, W, VEC>(y, reinterpret_cast<const TY*>(a.y.p) + row_at(a.y, a, row), lane, group, width, a.wide);
        load<TX, P, W, VEC>(x, reinterpret_cast<const TX*>(a.x.p) + row_at(a.x, a, row), lane, group, width, a.wide);
        if (GATE == ELEMENT) load<TY, P, W, VEC>(gate, reinterpret_cast<const TY*>(a.gate.p) + row_at(a.gate, a, row), lane, group, width, a.wide);
        const float gr = GATE == ROW ? one_gate<TY>(a, row_at(a.gate, a, row)) : 1.0f;
        float sum[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) sum[0] = fmaf(y[p][e], y[p][e], sum[0]);
        row_sum<G>(sum, lds);
        const float ry = 1.0f / sqrtf(sum[0] / float(width) + a.eps);
        sum[0] = 0.0f;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float b = y[p][e] * ry * wp[p][e];
                const float gb = GATE == NONE ? b : (GATE == ROW ? gr : gate[p][e]) * b;
                x[p][e] = a.residual ? fmaf(res[p][e], x[p][e], gb) : x[p][e] + gb;
                sum[0] = fmaf(x[p][e], x[p][e], sum[0]);
            }
        row_sum<G>(sum, lds);
        const float rs = 1.0f / sqrtf(sum[0] / float(width) + a.eps);
        if (mine < a.rows) {
            store<TX, P, W, VEC>(reinterpret_cast<TX*>(a.s.p) + row_at(a.s, a, row), x, lane, group, width, a.wide);
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++) x[p][e] = x[p][e] * rs * wq[p][e];
            store<TY, P, W, VEC>(reinterpret_cast<TY*>(a.h.p) + row_at(a.h, a, row), x, lane, group, width, a.wide);
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
template <int G> struct Sum { typedef float type; };
template <> struct Sum<16> { typedef double type; };

template <class TX, class TY, int G, int P, int W, bool VEC, int GATE>
__global__ void __launch_bounds__(G == 0 ? 1024 : 256) backward_kernel(Args a, GradArgs d) {
    typedef typename Sum<G>::type A;
    constexpr int SUMS = GATE == ROW ? 2 : 1;
    __shared__ A lds[16][2];
    extern __shared__ float columns[];
    const uint32_t group = G == 0 ? blockDim.x : G, per = G == 0 ? 1 : 256 / G;
    const uint32_t lane = threadIdx.x % group, width = a.width;
    float wp[P][W], wq[P][W], res[P][W], gate[P][W];
    float c_post[P][W] = {}, c_pre[P][W] = {}, c_res[P][W] = {}, c_gate[P][W] = {};
    load<float, P, W, VEC>(wp, a.w_post, lane, group, width, a.wide);
    load<float, P, W, VEC>(wq, a.w_pre, lane, group, width, a.wide);
    if (a.residual) load<float, P, W, VEC>(res, a.residual, lane, group, width, a.wide);
    if (GATE == CHANNEL) {
        if (a.gate_f32)
            load<float, P, W, VEC>(gate, reinterpret_cast<const float*>(a.gate.p), lane, group, width, a.wide);
        else
            load<TY, P, W, VEC>(gate, reinterpret_cast<const TY*>(a.gate.p), lane, group, width, a.wide);
    }
    const uint64_t step = uint64_t(gridDim.x) * per;
    for (uint64_t first = uint64_t(blockIdx.x) * per; first < a.rows; first += step) {
        const uint64_t mine = first + (G == 0 ? 0 : threadIdx.x / group);
        const bool in = mine < a.rows;
        const uint64_t row = in ? mine : a.rows - 1;
        float x[P][W], y[P][W], dh[P][W], t[P][W];
        load<TY, P, W, VEC>(y, reinterpret_cast<const TY*>(a.y.p) + row_at(a.y, a, row), lane, group, width, a.wide);
        load<TX, P, W, VEC>(x, reinterpret_cast<const TX*>(a.x.p) + row_at(a.x, a, row), lane, group, width, a.wide);
        if (GATE == ELEMENT) load<TY, P, W, VEC>(gate, reinterpret_cast<const TY*>(a.gate.p) + row_at(a.gate, a, row), lane, group, width, a.wide);
        if (d.d_h.p)
            load<TY, P, W, VEC>(dh, reinterpret_cast<const TY*>(d.d_h.p) + row_at(d.d_h, a, row), lane, group, width, a.wide);
        if (d.d_s.p)
            load<TX, P, W, VEC>(t, reinterpret_cast<const TX*>(d.d_s.p) + row_at(d.d_s, a, row), lane, group, width, a.wide);
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                if (!d.d_h.p) dh[p][e] = 0.0f;
                if (!d.d_s.p) t[p][e] = 0.0f;
            }
        const float gr = GATE == ROW ? one_gate<TY>(a, row_at(a.gate, a, row)) : 1.0f;
        A ry = a.stats[2 * row], rs = a.stats[2 * row + 1];
        const float keep = in ? 1.0f : 0.0f;
        if (G == 16) {
            A squares[1] = {0};
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++) squares[0] += A(y[p][e]) * A(y[p][e]);
            row_sum<G>(squares, reinterpret_cast<A(*)[1]>(lds));
            ry = A(1) / sqrt(squares[0] / A(width) + A(a.eps));
        }
        const float ryf = float(ry);
        A sum[G == 16 ? 2 : 1] = {};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float b = y[p][e] * ryf * wp[p][e];
                const float gb = GATE == NONE ? b : (GATE == ROW ? gr : gate[p][e]) * b;
                const float s = a.residual ? fmaf(res[p][e], x[p][e], gb) : x[p][e] + gb;
                sum[0] += A(dh[p][e] * wq[p][e]) * A(s);
                if (G == 16) sum[G == 16 ? 1 : 0] += A(s) * A(s);
            }
        row_sum<G>(sum, reinterpret_cast<A(*)[G == 16 ? 2 : 1]>(lds));
        if (G == 16) rs = A(1) / sqrt(sum[G == 16 ? 1 : 0] / A(width) + A(a.eps));
        const float rsf = float(rs);
        const A back = sum[0] / A(width) * rs * rs * rs;
        A sums[SUMS] = {};
        float dgate[P][W];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < W; e++) {
                const float nn = y[p][e] * ryf, b = nn * wp[p][e];
                const float gv = GATE == NONE ? 1.0f : GATE == ROW ? gr : gate[p][e];
                const float gb = GATE == NONE ? b : gv * b;
                const float s = a.residual ? fmaf(res[p][e], x[p][e], gb) : x[p][e] + gb;
                const float all = float(A(t[p][e]) + (rs * A(dh[p][e] * wq[p][e]) - back * A(s)));
                c_pre[p][e] = fmaf(keep * dh[p][e], s * rsf, c_pre[p][e]);
                c_post[p][e] = fmaf(keep * all, gv * nn, c_post[p][e]);
                c_res[p][e] = fmaf(keep * all, x[p][e], c_res[p][e]);
                if (GATE == CHANNEL) c_gate[p][e] = fmaf(keep * all, b, c_gate[p][e]);
                if (GATE == ELEMENT) dgate[p][e] = all * b;
                if (GATE == ROW) sums[SUMS - 1] += A(all) * A(b);
                x[p][e] = a.residual ? res[p][e] * all : all;
                const float dn = all * gv * wp[p][e];
                t[p][e] = dn;
                sums[0] += A(dn) * A(y[p][e]);
            }
        row_sum<G>(sums, reinterpret_cast<A(*)[SUMS]>(lds));
        const A pull = sums[0] / A(width) * ry * ry * ry;
        if (in) {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++) y[p][e] = float(ry * A(t[p][e]) - pull * A(y[p][e]));
            store<TX, P, W, VEC>(reinterpret_cast<TX*>(d.d_x.p) + row_at(d.d_x, a, row), x, lane, group, width, a.wide);
            store<TY, P, W, VEC>(reinterpret_cast<TY*>(d.d_y.p) + row_at(d.d_y, a, row), y, lane, group, width, a.wide);
            if (GATE == ELEMENT) store<TY, P, W, VEC>(reinterpret_cast<TY*>(d.d_gate.p) + row_at(d.d_gate, a, row), dgate, lane, group, width, a.wide);
            if (GATE == ROW && lane == 0) {
                const int64_t at = row_at(d.d_gate, a, row);
                if (a.gate_f32)
                    reinterpret_cast<float*>(d.d_gate.p)[at] = float(sums[SUMS - 1]);
                else
                    reinterpret_cast<TY*>(d.d_gate.p)[at] = TY(float(sums[SUMS - 1]));
            }
        }
    }
    // the workgroup's column sums: its groups of lanes add theirs up in order
    float* out = d.parts + uint64_t(blockIdx.x) * 4 * width;
    for (int c = 0; c < 4; c++) {
        float(&v)[P][W] = c == 0 ? c_post : c == 1 ? c_pre : c == 2 ? c_res : c_gate;
        if (G != 0) {
            for (uint32_t r = 0; r < per; r++) {
                __syncthreads();
                if (threadIdx.x / group == r)
#pragma unroll
                    for (int p = 0; p < P; p++)
#pragma unroll
                        for (int e = 0; e < W; e++) {
                            float& to = columns[place<W, VEC>(p, e, lane, group)];
                            to = r ? to + v[p][e] : v[p][e];
                        }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < width; i += 256) out[uint64_t(c) * width + i] = columns[i];
        } else {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < W; e++) {
                    const uint32_t at = place<W, VEC>(p, e, lane, group);
                    if (at < width) out[uint64_t(c) * width + at] = v[p][e];
                }
        }
    }
}

// Adds up the workgroups' rows of column sums: 64 columns and 4 quarters of the rows per workgroup.
__global__ void __launch_bounds__(256) columns_kernel(const float* parts, uint32_t count, uint32_t width, float* post, float* pre,
                                                      float* res, char* gate, uint32_t gate_f32) {
    __shared__ float lds[4][64];
    const uint32_t at = blockIdx.x * 64 + (threadIdx.x & 63), quarter = threadIdx.x >> 6;
    float sum = 0.0f;
    if (at < 4 * width)
        for (uint32_t i = quarter; i < count; i += 4) sum += parts[uint64_t(i) * 4 * width + at];
    lds[quarter][threadIdx.x & 63] = sum;
    __syncthreads();
    if (quarter != 0 || at >= 4 * width) return;
    sum = (lds[0][threadIdx.x] + lds[1][threadIdx.x]) + (lds[2][threadIdx.x] + lds[3][threadIdx.x]);
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

// The lanes of a row: pieces of W elements over G lanes, P each.
struct Shape { uint32_t lanes, pieces; };  // lanes 16, 32, 64, or a workgroup's threads
inline Shape shape_of(uint32_t width, uint32_t w) {
    const uint32_t pieces = (width + w - 1) / w;
    if (pieces <= 16) return {16, 1};
    if (pieces <= 32) return {32, 1};
    if (pieces <= 64) return {64, 1};
    if (pieces <= 128) return {64, 2};
    const uint32_t p = pieces <= 512 ? 1 : 2;
    return {((pieces + p - 1) / p + 63) / 64 * 64, p};
}
inline uint32_t blocks_of(const Args& a, const Shape& s) {
    const uint64_t per = s.lanes > 64 ? 1 : 256 / s.lanes;
    const uint64_t most = (a.rows + per - 1) / per;
    const uint64_t full = s.lanes > 64 ? 256 * (s.lanes <= 512 ? 3 : 2) : 1024;
    return uint32_t(most < full ? most : full);
}

template <class TX, class TY, int W, bool VEC, int GATE>
hipError_t forward(const Args& a, hipStream_t st) {
    const Shape s = shape_of(a.width, W);
    const bool block = s.lanes > 64;
    const uint64_t per = block ? 1 : 256 / s.lanes;
    const uint64_t rows = (a.rows + per - 1) / per;
    const dim3 grid(uint32_t(rows < 4096 ? rows : 4096)), wg(256);
    if (block && s.pieces == 1) forward_kernel<TX, TY, 0, 1, W, VEC, GATE><<<grid, dim3(s.lanes), 0, st>>>(a);
    else if (block) forward_kernel<TX, TY, 0, 2, W, VEC, GATE><<<grid, dim3(s.lanes), 0, st>>>(a);
    else if (s.lanes == 16) forward_kernel<TX, TY, 16, 1, W, VEC, GATE><<<grid, wg, 0, st>>>(a);
    else if (s.lanes == 32) forward_kernel<TX, TY, 32, 1, W, VEC, GATE><<<grid, wg, 0, st>>>(a);
    else if (s.pieces == 1) forward_kernel<TX, TY, 64, 1, W, VEC, GATE><<<grid, wg, 0, st>>>(a);
    else forward_kernel<TX, TY, 64, 2, W, VEC, GATE><<<grid, wg, 0, st>>>(a);
    return hipGetLastError();
}
template <class TX, class TY, int W, bool VEC, int GATE>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t st) {
    const Shape s = shape_of(a.width, W);
    const dim3 grid(blocks_of(a, s)), wg(256);
    const uint32_t columns = s.lanes > 64 ? 0 : s.lanes * s.pieces * W * 4;
    if (s.lanes > 64 && s.pieces == 1) backward_kernel<TX, TY, 0, 1, W, VEC, GATE><<<grid, dim3(s.lanes), 0, st>>>(a, d);
    else if (s.lanes > 64) backward_kernel<TX, TY, 0, 2, W, VEC, GATE><<<grid, dim3(s.lanes), 0, st>>>(a, d);
    else if (s.lanes == 16) backward_kernel<TX, TY, 16, 1, W, VEC, GATE><<<grid, wg, columns, st>>>(a, d);
    else if (s.lanes == 32) backward_kernel<TX, TY, 32, 1, W, VEC, GATE><<<grid, wg, columns, st>>>(a, d);
    else if (s.pieces == 1) backward_kernel<TX, TY, 64, 1, W, VEC, GATE><<<grid, wg, columns, st>>>(a, d);
    else backward_kernel<TX, TY, 64, 2, W, VEC, GATE><<<grid, wg, columns, st>>>(a, d);
    return hipGetLastError();
}

template <class TY> constexpr int words() { return 16 / int(sizeof(TY)); }

template <class TX, class TY, bool VEC, class F>
hipError_t by_gate(const Args& a, F f) {
    switch (a.gate_kind) {
        case CHANNEL: return f.template run<TX, TY, VEC, CHANNEL>();
        case ROW: return f.template run<TX, TY, VEC, ROW>();
        case ELEMENT: return f.template run<TX, TY, VEC, ELEMENT>();
        default: return f.template run<TX, TY, VEC, NONE>();
    }
}
template <class F>
hipError_t by_type(const Args& a, uint32_t x_type, uint32_t y_type, F f) {
    const bool vec = a.width % (y_type == MDN_BF16 ? 8 : 4) == 0;
    if (x_type == MDN_BF16) return vec ? by_gate<bf16, bf16, true>(a, f) : by_gate<bf16, bf16, false>(a, f);
    if (y_type == MDN_BF16) return vec ? by_gate<float, bf16, true>(a, f) : by_gate<float, bf16, false>(a, f);
    return vec ? by_gate<float, float, true>(a, f) : by_gate<float, float, false>(a, f);
}
struct Forward {
    const Args& a;
    hipStream_t st;
    template <class TX, class TY, bool VEC, int GATE> hipError_t run() { return forward<TX, TY, words<TY>(), VEC, GATE>(a, st); }
};
struct Backward {
    const Args& a;
    const GradArgs& d;
    hipStream_t st;
    template <class TX, class TY, bool VEC, int GATE> hipError_t run() { return backward<TX, TY, words<TY>(), VEC, GATE>(a, d, st); }
};

}  // namespace

hipError_t launch_forward(const Args& a, uint32_t x_type, uint32_t y_type, hipStream_t stream) {
    return by_type(a, x_type, y_type, Forward{a, stream});
}

uint32_t parts(const Args& a, uint32_t y_type) {
    return a.rows ? blocks_of(a, shape_of(a.width, y_type == MDN_BF16 ? 8 : 4)) : 0;
}

hipError_t launch_backward(const Args& a, const GradArgs& d, uint32_t x_type, uint32_t y_type, hipStream_t stream) {
    const uint32_t count = parts(a, y_type);
    if (count)
        if (hipError_t e = by_type(a, x_type, y_type, Backward{a, d, stream})) return e;
    columns_kernel<<<dim3((4 * a.width + 63) / 64), dim3(256), 0, stream>>>(
        d.parts, count, a.width, d.d_w_post, d.d_w_pre, a.residual ? d.d_residual : nullptr,
        a.gate_kind == CHANNEL ? d.d_gate.p : nullptr, a.gate_f32);
    return hipGetLastError();
}

}  // namespace blocknorm
