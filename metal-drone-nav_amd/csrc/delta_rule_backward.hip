// delta_rule_backward.hip — gradients of the gated delta rule, chunk by chunk
// from the last to the first.
//
// With the symbols of delta_chunk.h, X = V - gamma (K S), U = (1 + A)^-1 beta X,
// P = scale D Q K^T, G the gradient of the state after the chunk, and dO:
//     dU = P^T dO + (gamma_C / gamma) K G          R = (1 + A)^-T dU
//     dP = dO U^T   dA = -R U^T                    dV = beta R
//     dQ = scale gamma dO S^T + (scale D dP) K
//     dK = -beta gamma R S^T + (gamma_C / gamma) U G^T + (scale D dP)^T Q + (E + E^T) K,   E = beta D dA
//     d_beta_i = R_i X_i + sum_j dA_ij A_ij / beta_i
//     G <- gamma_C G + Q^T (scale gamma dO) - K^T (gamma beta R)
// The gradient of g_t collects what every factor exp(g_s + .. + g_i) that
// spans tick t multiplies: with M = dP P + dA A (element by element), a_i the
// part of q_i dq_i + k_i dk_i that goes through S, and b_j the part of k_j dk_j that
// goes through G,
//     d_g_t = sum_{i >= t} a_i + sum_{j < t} b_j + sum_{i >= t > j} M_ij + gamma_C <S, G>,
// sums of terms that do not cancel, but for the one over M, which is formed
// from row and column sums of M in 64 bits.
#include "delta_rule.h"

#include "delta_chunk.h"
#include "delta_tiles.h"

namespace delta {
namespace {

template <class E, int D> struct BackwardShared {
    static constexpr int STRIDE = D + Kind<E>::PAD;
    static constexpr int N = Kind<E>::MID;
    // S and G pass through LDS, transposed, in fp32; both 128-wide operands
    // and the fp32 rows do not fit beside each other, and take halves of V
    static constexpr int HALVES = sizeof(E) == 4 && D == 128 ? 2 : 1;
    static constexpr int TS = D + 4;
    static constexpr int PLANE = D * CP;
    static constexpr int W = D / 16;
    E k[C * STRIDE], q[C * STRIDE], d_o[C * STRIDE];  // ordered rows
    E u[N * PLANE], r[N * PLANE];                     // U and R transposed, [v][tick]
    float through[D / HALVES * TS];                   // S, then G, transposed: [v][k]
    System<E> sys;
    E d_scores[N * System<E>::PLANE], d_a[N * System<E>::PLANE];  // scale D dP and E, [j][i]
    Gates gates[2];  // of this chunk and the next
    float beta_v[W][C], a[W][C], b[W][C], dot[W];
    double m_row[3][16], m_col[3][16];
    float beta_a[3][16];
};

template <class E>
__device__ __forceinline__ void put_grad(const Rows& r, int64_t at, float x, bool partial) {
    if (partial)
        reinterpret_cast<float*>(r.p)[at] = x;
    else
        reinterpret_cast<E*>(r.p)[at] = E(x);
}
__device__ __forceinline__ void put_gate(const Args& a, const Rows& r, int64_t at, float x, bool bf) {
    if (a.gate_f32 || !bf)
        reinterpret_cast<float*>(r.p)[at] = x;
    else
        reinterpret_cast<bf16*>(r.p)[at] = bf16(x);
}

// One workgroup per state, D / 16 wavefronts.  A wavefront has 16 columns of V
// (its slices of S, G, U and R) and, for the gradients of q and k, 16 columns
// of K; U, R, S and G change hands through LDS.
template <class E, int D, bool WIDE>
__global__ void __launch_bounds__(D * 4, 2) backward_kernel(Args a, GradArgs d) {
    typedef BackwardShared<E, D> Shared;
    constexpr int ST = Shared::STRIDE, N = Kind<E>::MID, KT = D / 16, SP = System<E>::PLANE, PL = Shared::PLANE;
    constexpr int HALVES = Shared::HALVES, TS = Shared::TS, VH = D / HALVES;
    constexpr bool bf = sizeof(E) == 2;
    extern __shared__ __align__(16) char lds[];
    Shared& s = *reinterpret_cast<Shared*>(lds);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const uint64_t seq = blockIdx.x;
    const uint32_t n = uint32_t(seq / a.heads), h = uint32_t(seq % a.heads);
    const uint32_t hq = h / (a.heads / a.qk_heads), hg = d.partial ? h : hq;
    const uint32_t kd = a.k_dim, vd = a.v_dim;
    const uint32_t row = uint32_t(tid) / (D / 8), col = uint32_t(tid) % (D / 8) * 8;
    const uint32_t chunks = (a.ticks + CHUNK - 1) / CHUNK;
    const f32x4 zero{0, 0, 0, 0};

    f32x4 g[KT];  // G, K x 16
    {
        const Lane l = Lane::fresh();
        load_state(g, d.d_state_out ? d.d_state_out + seq * kd * vd : nullptr, kd, vd, l, 16 * wave + l.col);
        // the matrices' upper right blocks stay 0
        if (wave < N) {
            E* m[4] = {s.sys.scores, s.sys.inv, s.d_scores, s.d_a};
#pragma unroll
            for (int x = 0; x < 4; x++)
#pragma unroll
                for (int i = 0; i < 4; i++) m[x][wave * SP + (16 + l.col) * CP + 4 * l.quad + i] = E(0.0f);
        }
    }
    Piece<E> pk, pq, po;
    GateRegs gate{0.0f, 0.0f, 0u};
    const auto fetch = [&](uint32_t c) {
        const uint32_t at = c * C + row;
        const int64_t t = at < a.ticks ? at : 0;
        pk = load_piece<E, WIDE>(a.k, t * a.k.tick + n * a.k.env + hq * a.k.head, kd, col);
        pq = load_piece<E, WIDE>(a.q, t * a.q.tick + n * a.q.env + hq * a.q.head, kd, col);
        po = load_piece<E, WIDE>(d.d_o, t * d.d_o.tick + n * d.d_o.env + h * d.d_o.head, vd, col);
    };
    // the last wavefront has no tile of A: it makes the next chunk's decays meanwhile
    const auto fetch_gates = [&](uint32_t c) {
        const int64_t t = int64_t(c) * C + lane;
        gate = load_gates(a, bf, n, h, t, lane < C && t < a.ticks);
    };
    if (wave == Shared::W - 1) {
        fetch_gates(chunks - 1);
        put_gates(s.gates[(chunks - 1) & 1], gate);
        if (chunks > 1) fetch_gates(chunks - 2);
    }
    fetch(chunks - 1);
    for (uint32_t c = chunks; c-- > 0;) {
        const Lane l = Lane::fresh();
        const uint32_t vc = 16 * wave + l.col;  // the lane's column of V, and of K
        const Gates& gates = s.gates[c & 1];
        const uint32_t left = a.ticks - c * C;  // ticks from the chunk's first
        const bool in = c * C + row < a.ticks;
        piece_to_ordered(s.k + row * ST, col, mask_piece<E, WIDE>(pk, kd, col, in));
        piece_to_ordered(s.q + row * ST, col, mask_piece<E, WIDE>(pq, kd, col, in));
        piece_to_ordered(s.d_o + row * ST, col, mask_piece<E, WIDE>(po, vd, col, in));
        // S and V, in result layout
        f32x4 st[KT], x[2];
        if (c > 0) {
            const f32x4* p = state_tiles(a, seq, c, wave);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                st[i] = zero;
                if (16 * i < int(kd) && 16 * wave < int(vd)) st[i] = p[64 * i + lane];
            }
        } else {
            load_state(st, a.state ? a.state + seq * kd * vd : nullptr, kd, vd, l, vc);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t t = 16 * i + 4 * l.quad + e;
                const bool in = t < left && vc < vd;
                const float y = load_one<E>(a.v.p, (in ? int64_t(c * C + t) * a.v.tick : 0) + n * a.v.env + h * a.v.head + (in ? vc : 0u));
                x[i][e] = in ? y : 0.0f;
            }
        __syncthreads();
        if (c > 0) fetch(c - 1);

        // the chunk's scores and A: tiles (0,0), (1,1), (1,0), kept by their wavefronts
        f32x4 dec = zero, kk = zero, pm = zero, am = zero;
        const int i0 = wave ? 16 : 0, j0 = wave == 1 ? 16 : 0;
        if (wave < 3) {
            f32x4 qk = zero;
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                const auto kj = ordered_row(l, s.k, ST, j0, y);
                mma(kk, ordered_row(l, s.k, ST, i0, y), kj);
                mma(qk, ordered_row(l, s.q, ST, i0, y), kj);
            }
            dec = decay_tile(l, gates, i0, j0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = i0 + 4 * l.quad + r;
                if (i <= j0 + l.col) kk[r] = 0.0f;
                kk[r] *= dec[r];
                am[r] = gates.beta[i] * kk[r];
                pm[r] = a.scale * dec[r] * qk[r];
            }
            put_tile(l, s.sys.scores, CP, SP, j0, i0, pm);
            if (wave < 2)
                solve_diagonal(l, s.sys, wave, am);
            else
                put_tile(l, s.sys.inv, CP, SP, 0, 16, am);
        }
        if (wave == Shared::W - 1 && c > 0) {
            put_gates(s.gates[(c - 1) & 1], gate);
            if (c > 1) fetch_gates(c - 2);
        }
        // X, and the part of dU through G
        f32x4 dr[2] = {zero, zero}, du[2] = {zero, zero};
        {
            f32x4 ks[2] = {zero, zero};
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                const auto sf = frag_of<E>(st[y / 16], st[y / 16 + 1]);
                const auto gf = frag_of<E>(g[y / 16], g[y / 16 + 1]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const auto kf = ordered_row(l, s.k, ST, 16 * i, y);
                    mma(ks[i], kf, sf);
                    mma(du[i], kf, gf);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int t = 16 * i + 4 * l.quad + e;
                    x[i][e] -= gates.before[t] * ks[i][e];
                    dr[i][e] = gates.beta[t] * x[i][e];
                    du[i][e] *= gates.after[t];
                }
        }
        if (HALVES == 1 || 16 * wave < VH)
#pragma unroll
            for (int i = 0; i < KT; i++) put_tile(l, s.through, TS, 0, 16 * wave, 16 * i, st[i]);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < KT; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) dot = fmaf(st[i][r], g[i][r], dot);
        dot = sum_rows32(sum_rows16(sum16(dot)));
        if (lane == 0) s.dot[wave] = dot;
        __syncthreads();

        // U and R
        {
            f32x4 u[2];
            solve(l, s.sys, dr, u);
#pragma unroll
            for (int i = 0; i < 2; i++) put_tile(l, s.u, CP, PL, 16 * wave, 16 * i, u[i]);
            const auto of = ordered_col(l, s.d_o, ST, 16 * wave);
#pragma unroll
            for (int i = 0; i < 2; i++) mma(du[i], row_frag<N>(l, s.sys.scores, CP, SP, 16 * i, 0), of);
            solve_transposed(l, s.sys, du, dr);
#pragma unroll
            for (int i = 0; i < 2; i++) put_tile(l, s.r, CP, PL, 16 * wave, 16 * i, dr[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t t = 16 * i + 4 * l.quad + e;
                const float sum = sum16(dr[i][e] * x[i][e]);
                if (l.col == 0) s.beta_v[wave][t] = sum;
                const float beta = gates.beta[t];
                if (t < left && vc < vd)
                    reinterpret_cast<E*>(d.d_v.p)[int64_t(c * C + t) * d.d_v.tick + n * d.d_v.env + h * d.d_v.head + vc] =
                        E(beta * dr[i][e]);
                dr[i][e] *= beta * gates.before[t];  // from here on gamma beta R
            }
        __syncthreads();

        // dP and dA, by the wavefronts that hold P and A
        f32x4 dp = zero, da = zero;
        if (wave < 3) {
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                const auto uj = col_frag<N>(l, s.u, CP, PL, y, j0);
                mma(dp, ordered_row(l, s.d_o, ST, i0, y), uj);
                mma(da, col_frag<N>(l, s.r, CP, PL, y, i0), uj);
            }
            double m_row[4], m_col = 0.0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = i0 + 4 * l.quad + r;
                da[r] = i > j0 + l.col ? -da[r] : 0.0f;
                const float m = dp[r] * pm[r] + da[r] * am[r];
                m_row[r] = double(m);
                m_col += double(m);
                m_row[r] = sum16(m_row[r]);
                const float b = sum16(da[r] * kk[r]);
                if (l.col == 0) {
                    s.m_row[wave][4 * l.quad + r] = m_row[r];
                    s.beta_a[wave][4 * l.quad + r] = b;
                }
                dp[r] *= a.scale * dec[r];
                da[r] *= gates.beta[i] * dec[r];
            }
            m_col += __shfl_xor(m_col, 16);
            m_col += __shfl_xor(m_col, 32);
            if (l.quad == 0) s.m_col[wave][l.col] = m_col;
            put_tile(l, s.d_scores, CP, SP, j0, i0, dp);
            put_tile(l, s.d_a, CP, SP, j0, i0, da);
        }
        // through S
        f32x4 dq[2] = {zero, zero}, dk[2] = {zero, zero}, dkg[2] = {zero, zero};
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            if (half > 0) {
                __syncthreads();
                if (16 * wave >= VH)
#pragma unroll
                    for (int i = 0; i < KT; i++) put_tile(l, s.through, TS, 0, 16 * wave - VH, 16 * i, st[i]);
                __syncthreads();
            }
#pragma unroll
            for (int y = 0; y < VH; y += 32) {
                const auto sf = frag_of<E>(col4(l, s.through, TS, y, 16 * wave), col4(l, s.through, TS, y + 16, 16 * wave));
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mma(dq[i], ordered_row(l, s.d_o, ST, 16 * i, half * VH + y), sf);
                    mma(dk[i], col_frag<N>(l, s.r, CP, PL, half * VH + y, 16 * i), sf);
                }
            }
        }
        // through G
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            __syncthreads();
            if (HALVES == 1 || (16 * wave >= VH) == (half == 1))
#pragma unroll
                for (int i = 0; i < KT; i++) put_tile(l, s.through, TS, 0, 16 * wave - half * VH, 16 * i, g[i]);
            __syncthreads();
#pragma unroll
            for (int y = 0; y < VH; y += 32) {
                const auto gf = frag_of<E>(col4(l, s.through, TS, y, 16 * wave), col4(l, s.through, TS, y + 16, 16 * wave));
#pragma unroll
                for (int i = 0; i < 2; i++) mma(dkg[i], col_frag<N>(l, s.u, CP, PL, half * VH + y, 16 * i), gf);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int t = 16 * i + 4 * l.quad + e;
                const int at = t * ST + place(16 * wave) + 8 * (l.col >> 2) + (l.col & 3);
                const float qv = float(s.q[at]), kv = float(s.k[at]);
                const float before = gates.before[t];
                dq[i][e] *= a.scale * before;
                dk[i][e] *= -gates.beta[t] * before;
                dkg[i][e] *= gates.after[t];
                const float pa = sum16(fmaf(qv, dq[i][e], kv * dk[i][e])), pb = sum16(kv * dkg[i][e]);
                if (l.col == 0) {
                    s.a[wave][t] = pa;
                    s.b[wave][t] = pb;
                }
                dk[i][e] += dkg[i][e];
            }
        // inside the chunk
        {
            const auto kf = ordered_col(l, s.k, ST, 16 * wave);
            const auto qf = ordered_col(l, s.q, ST, 16 * wave);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mma(dq[i], col_frag<N>(l, s.d_scores, CP, SP, 0, 16 * i), kf);
                mma(dk[i], row_frag<N>(l, s.d_scores, CP, SP, 16 * i, 0), qf);
                mma(dk[i], row_frag<N>(l, s.d_a, CP, SP, 16 * i, 0), kf);
                mma(dk[i], col_frag<N>(l, s.d_a, CP, SP, 0, 16 * i), kf);
            }
        }
        if (vc < kd)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t t = 16 * i + 4 * l.quad + e;
                    if (t >= left) continue;
                    const int64_t at = int64_t(c * C + t);
                    put_grad<E>(d.d_q, at * d.d_q.tick + n * d.d_q.env + hg * d.d_q.head + vc, dq[i][e], d.partial);
                    put_grad<E>(d.d_k, at * d.d_k.tick + n * d.d_k.env + hg * d.d_k.head + vc, dk[i][e], d.partial);
                }
        // G before the chunk
        {
            const float total = gates.before[C - 1];
            const auto of = ordered_col(l, s.d_o, ST, 16 * wave);
            f32x4 lo, hi;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo[e] = a.scale * gates.before[4 * l.quad + e] * first_term(of, e);
                hi[e] = a.scale * gates.before[16 + 4 * l.quad + e] * first_term(of, 4 + e);
            }
            const auto of2 = frag_of<E>(lo, hi);
            const auto rf = frag_of<E>(-dr[0], -dr[1]);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                g[i] *= total;
                mma(g[i], ordered_col(l, s.q, ST, 16 * i), of2);
                mma(g[i], ordered_col(l, s.k, ST, 16 * i), rf);
            }
        }
        __syncthreads();
        if (wave == 0) {
            const int t = lane & 31;
            float pa = 0.0f, pb = 0.0f, beta = 0.0f, all = 0.0f;
#pragma unroll
            for (int w = 0; w < Shared::W; w++) {
                pa += s.a[w][t];
                pb += s.b[w][t];
                beta += s.beta_v[w][t];
                all += s.dot[w];
            }
            // tiles (0,0), (1,1), (1,0)
            const double mr = t < 16 ? s.m_row[0][t] : s.m_row[1][t - 16] + s.m_row[2][t - 16];
            const double mc = t < 16 ? s.m_col[0][t] + s.m_col[2][t] : s.m_col[1][t - 16];
            beta += t < 16 ? s.beta_a[0][t] : s.beta_a[1][t - 16] + s.beta_a[2][t - 16];
            double after = double(pa) + mr - mc;  // summed over the ticks from t on
            double before = double(pb);           // summed over the ticks before t
#pragma unroll
            for (int y = 1; y < C; y <<= 1) {
                const double down = __shfl_down(after, y, C), up = __shfl_up(before, y, C);
                if (t + y < C) after += down;
                if (t >= y) before += up;
            }
            before -= double(pb);
            const float dg = gate_is_flag(gates, t) ? 0.0f : float(after + before + double(gates.before[C - 1]) * double(all));
            if (lane < C && uint32_t(t) < left) {
                const int64_t at = int64_t(c * C + t);
                put_gate(a, d.d_g, at * d.d_g.tick + n * d.d_g.env + h * d.d_g.head, dg, bf);
                put_gate(a, d.d_beta, at * d.d_beta.tick + n * d.d_beta.env + h * d.d_beta.head, beta, bf);
            }
        }
    }
    if (d.d_state) {
        const Lane l = Lane::fresh();
        store_state(d.d_state + seq * kd * vd, g, kd, vd, l, 16 * wave + l.col);
    }
}

template <class E>
__global__ void sum_heads_kernel(const float* in, E* out, uint64_t count, uint32_t shared, uint32_t width) {
    for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += uint64_t(gridDim.x) * blockDim.x) {
        const uint64_t head = i / width;
        const float* p = in + head * shared * width + i % width;
        float sum = 0.0f;
        for (uint32_t j = 0; j < shared; j++) sum += p[uint64_t(j) * width];
        out[i] = E(sum);
    }
}

template <class E, int D, bool WIDE>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t stream) {
    constexpr uint32_t bytes = sizeof(BackwardShared<E, D>);
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    const void* f = reinterpret_cast<const void*>(&backward_kernel<E, D, WIDE>);
    if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes))) return e;
    backward_kernel<E, D, WIDE><<<dim3(a.envs * a.heads), dim3(D * 4), bytes, stream>>>(a, d);
    return hipGetLastError();
}
template <class E>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t stream) {
    const bool narrow = a.k_dim <= 64 && a.v_dim <= 64;
    const bool wide = (a.q.wide & a.k.wide & d.d_o.wide) && a.k_dim % 8 == 0 && a.v_dim % 8 == 0;
    if (wide) return narrow ? backward<E, 64, true>(a, d, stream) : backward<E, 128, true>(a, d, stream);
    return narrow ? backward<E, 64, false>(a, d, stream) : backward<E, 128, false>(a, d, stream);
}

}  // namespace

hipError_t launch_backward(const Args& a, const GradArgs& d, bool bf, hipStream_t stream) {
    return bf ? backward<bf16>(a, d, stream) : backward<float>(a, d, stream);
}

hipError_t launch_sum_heads(const float* in, void* out, uint64_t rows, uint32_t qk_heads, uint32_t shared, uint32_t width,
                            bool bf, hipStream_t stream) {
    const uint64_t count = rows * qk_heads * width;
    if (count == 0) return hipSuccess;
    const uint64_t blocks = (count + 255) / 256;
    const dim3 grid(uint32_t(blocks < 8192 ? blocks : 8192));
    if (bf)
        sum_heads_kernel<bf16><<<grid, dim3(256), 0, stream>>>(in, static_cast<bf16*>(out), count, shared, width);
    else
        sum_heads_kernel<float><<<grid, dim3(256), 0, stream>>>(in, static_cast<float*>(out), count, shared, width);
    return hipGetLastError();
}

}  // namespace delta
