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
    // S and G pass through LDS, transposed, as operands; in fp32 in halves of V:
    // of 128 columns they would not fit beside the rows, of 64 a compute unit
    // would have room for one workgroup and not two (4,096 states 48 x 48, 64
    // ticks, forward and backward: 698 us whole, 516 in halves)
    static constexpr int HALVES = sizeof(E) == 4 ? 2 : 1;
    static constexpr int TP = D / HALVES * STRIDE;
    static constexpr int PLANE = D * CP;
    static constexpr int W = D / 16;
    E k[C * STRIDE], q[C * STRIDE], d_o[C * STRIDE];  // ordered rows
    E v[C * STRIDE];
    // from here on the gradients' rows take the place of what is done with
    E u[N * PLANE], r[N * PLANE];                     // U and R transposed, [v][tick]
    E through[N * TP];                                // S, then G, transposed: [v][k]
    // inv and scores give their places to E = beta D dA and to scale D dP
    System<E> sys;
    Gates gates[2];  // of this chunk and the next
    int odd;         // whether the chunk has results that are not finite
    float odd_sums[2][W];
    __align__(16) float beta_v[W][C], a[W][C], b[W][C], dot[W];
    double m_row[3][16], m_col[3][16];
    __align__(16) float beta_a[3][16];
};

template <class E> __device__ __forceinline__ void put_gate(KernelCall* k, const At& now, uint32_t tick, float dg, float db) {
    if (k->a.gate_f32 || sizeof(E) == 4) {
        *Track<float>(&k->d.d_g, now.n, now.h).row(tick) = dg;
        *Track<float>(&k->d.d_beta, now.n, now.h).row(tick) = db;
    } else {
        *Track<bf16>(&k->d.d_g, now.n, now.h).row(tick) = bf16(dg);
        *Track<bf16>(&k->d.d_beta, now.n, now.h).row(tick) = bf16(db);
    }
}

// One workgroup per state, a wavefront for each 16 columns (at least four).  A
// wavefront has 16 columns of V (its slices of S, G, U and R) and, for the
// gradients of q and k, 16 columns of K; U, R, S and G change hands through
// LDS.  F is the type of the rows of d_q and d_k.
//
// AHEAD: what the segments of a cut state need before they run, the gradient
// that each would pass to the one before it if it received none itself (the
// last one receives the final state's).
//
// Bound by vector instructions and the waits between the chunk's products, each
// of which needs the last one's result: two wavefronts on a SIMD hold S, G and a
// chunk's rows.  32,768 states 64 x 64 of 32 ticks in bfloat16 (1.3 GB) take 752 to
// 773 us under a profiler, vector units 43 % and matrix cores 13 % busy, in fp32
// 1,356; 5,120 states 128 x 128 of 64 ticks 615 us, in fp32 1,161; 6,000 of 40 x 72, 37
// ticks, in fp32, 1,160 us: there 155 KB of LDS leave one workgroup of five wavefronts
// a compute unit, which wait 61 % of the time.  The states before the chunks come
// from the forward pass, one K x V for 32 ticks of rows.
template <class E, class F, int D, bool FULL, bool AHEAD>
__global__ void __launch_bounds__(D * 4, 2) backward_kernel(Call call) {
    typedef BackwardShared<E, D> Shared;
    constexpr int ST = Shared::STRIDE, N = Kind<E>::MID, KT = D / 16, SP = System<E>::PLANE, PL = Shared::PLANE;
    constexpr int HALVES = Shared::HALVES, TP = Shared::TP, VH = D / HALVES;
    constexpr int FT = D + Kind<F>::PAD;  // row of d_q and d_k in LDS
    static_assert(sizeof(F) * 2 * C * FT + sizeof(E) * C * ST <= sizeof(Shared::u) + sizeof(Shared::r) + sizeof(Shared::through), "");
    extern __shared__ __align__(16) char lds[];
    Shared& s = *reinterpret_cast<Shared*>(lds);
    F* const dq_rows = reinterpret_cast<F*>(s.u);
    F* const dk_rows = dq_rows + C * FT;
    E* const dv_rows = reinterpret_cast<E*>(dk_rows + C * FT);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int waves = FULL ? D / 16 : blockDim.x >> 6;
    const int kd = FULL ? D : int(call.a.k_dim), vd = FULL ? D : int(call.a.v_dim);
    const bool v_wave = FULL || 16 * wave < vd, k_wave = FULL || 16 * wave < kd;
    const uint32_t ticks = call.a.ticks;
    const Plan plan(call.a, AHEAD ? call.a.segments - 1 : call.a.segments);
    const auto which = [&](At& at, uint32_t j) {
        at.part = 0;
        at.seg = AHEAD ? j + 1 : j;
    };
    const float scale = call.a.scale;
    const Spot on_k(kd), on_v(vd);
    const f32x4 zero{0, 0, 0, 0};
    if (!FULL) clear_lds(lds, sizeof(Shared));
    // the matrices' upper right blocks stay 0
    for (int p = wave; p < 2 * N; p += waves) {
        const Lane l = Lane::mine();
        E* m = (p & 1 ? s.sys.scores : s.sys.inv) + (p >> 1) * SP;
#pragma unroll
        for (int i = 0; i < 4; i++) m[(16 + l.col) * CP + 4 * l.quad + i] = E(0.0f);
    }
    f32x4 g[KT], st[KT];  // G and S, K x 16, in result layout
    Piece<E> pk, pq, pv, po;
    const auto fetch = [&](const At& at) {
        KernelCall* k = fresh_call();
        if (on_k.on) {
            const uint32_t x = at.c * C + on_k.row, t = x < ticks ? x : 0u;
            pk = load_piece<E>(Track<const E>(&k->a.k, at.n, at.hq).row(t), kd, on_k.col);
            pq = load_piece<E>(Track<const E>(&k->a.q, at.n, at.hq).row(t), kd, on_k.col);
        }
        if (on_v.on) {
            const uint32_t x = at.c * C + on_v.row, t = x < ticks ? x : 0u;
            if (!AHEAD) pv = load_piece<E>(Track<const E>(&k->a.v, at.n, at.h).row(t), vd, on_v.col);
            po = load_piece<E>(Track<const E>(&k->d.d_o, at.n, at.h).row(t), vd, on_v.col);
        }
    };
    const auto put_rows = [&](const At& at) {
        const uint32_t left = ticks - at.c * C;
        if (on_k.on) {
            piece_to_ordered(s.k + on_k.row * ST, on_k.col, mask_piece<E>(pk, on_k.row < left));
            piece_to_ordered(s.q + on_k.row * ST, on_k.col, mask_piece<E>(pq, on_k.row < left));
        }
        if (on_v.on) {
            if (!AHEAD) piece_to_lds(s.v + on_v.row * ST + on_v.col, mask_piece<E>(pv, on_v.row < left));
            piece_to_ordered(s.d_o + on_v.row * ST, on_v.col, mask_piece<E>(po, on_v.row < left));
        }
    };
    const auto fetch_state = [&](const At& at) {
        const Lane l = Lane::fresh();
        KernelCall* k = fresh_call();
        if (at.c > 0) {
            const f32x4* p = state_tiles(k->a.chunk_states, at.state, plan.chunks, at.c, kd, vd, wave);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                st[i] = zero;
                if (16 * i < kd && v_wave) st[i] = p[64 * i + lane];
            }
        } else {
            const float* p = k->a.state;
            load_state(st, p ? p + uint64_t(at.state) * kd * vd : nullptr, kd, vd, l, 16 * wave + l.col);
        }
    };
    // the last wavefront has no tile of A: it makes the next chunk's decays
    // meanwhile, from what it loaded a chunk before that
    GateRegs gate{0.0f, 0.0f, 0u};
    const auto fetch_gates = [&](const At& at) {
        const uint32_t t = at.c * C + lane;
        gate = load_gates<E>(&fresh_call()->a, at.n, at.h, t, lane < C && t < ticks);
    };
    // G before a segment: for the one before it, or the state's gradient
    const auto leave = [&](const At& at, const f32x4(&x)[KT]) {
        KernelCall* k = fresh_call();
        float* p = at.seg == 0 ? k->d.d_state : nullptr;
        if (p) p += uint64_t(at.state) * kd * vd;
        if (AHEAD) p = k->a.seg_grads + (uint64_t(at.state) * plan.segments + at.seg - 1) * kd * vd;
        const Lane l = Lane::fresh();
        if (p) store_state(p, x, kd, vd, l, 16 * wave + l.col);
    };
    At now, next, later;
    now.job = blockIdx.x;
    now.split(plan, which);
    now.c = now.end - 1;
    next = now;
    next.back(plan, which);
    later = next;
    later.back(plan, which);
    fetch(now);
    if (!AHEAD) fetch_state(now);
    if (wave == waves - 1) {
        fetch_gates(now);
        put_gates(s.gates[0], gate);
        if (next.job < plan.total) fetch_gates(next);
    }
    put_rows(now);
    __syncthreads();
    for (uint32_t turn = 0; now.job < plan.total; turn ^= 1) {
        const Lane l = Lane::fresh();
        const Gates& gates = s.gates[turn];
        const uint32_t left = ticks - now.c * C;  // ticks from the chunk's first
        if (now.c == now.end - 1) {
            KernelCall* k = fresh_call();
            const float* p = k->d.d_state_out;
            if (p) p += uint64_t(now.state) * kd * vd;
            if (now.seg + 1 < plan.segments)
                p = AHEAD ? nullptr : k->a.seg_grads + (uint64_t(now.state) * plan.segments + now.seg) * kd * vd;
            load_state(g, p, kd, vd, l, 16 * wave + l.col);
        }
        if (next.job < plan.total) fetch(next);

        // the chunk's scores and A: tiles (0,0), (1,1), (1,0), kept by their wavefronts
        f32x4 dec = zero, kk = zero, pm = zero, am = zero;
        const int i0 = wave ? 16 : 0, j0 = wave == 1 ? 16 : 0;
        if (wave < 3) {
            f32x4 qk = zero;
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                if (y >= kd) continue;
                const auto kj = ordered_row(l, s.k, ST, j0, y);
                mma(kk, ordered_row(l, s.k, ST, i0, y), kj);
                mma(qk, ordered_row(l, s.q, ST, i0, y), kj);
            }
            if (!FULL) settle(kk, qk);
            dec = decay_tile(l, gates, i0, j0);
            kk *= dec;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (i0 + 4 * l.quad + r <= j0 + l.col) kk[r] = 0.0f;
            am = four(gates.beta + i0 + 4 * l.quad) * kk;
            pm = scale * dec * qk;
            put_tile<N>(l, s.sys.scores, CP, SP, j0, i0, pm);
            if (wave < 2)
                put_tile<N>(l, s.sys.inv, CP, System<E>::PLANE, 16 * wave, 16 * wave, invert_block(l, am));
            else
                put_tile<N>(l, s.sys.inv, CP, SP, 0, 16, am);
        }
        if (wave == waves - 1 && next.job < plan.total) {
            put_gates(s.gates[turn ^ 1], gate);
            if (later.job < plan.total) fetch_gates(later);
        }
        // X, and the part of dU through G
        f32x4 x[2], dr[2] = {zero, zero}, du[2] = {zero, zero};
        if (v_wave) {
            f32x4 ks[2] = {zero, zero};
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                if (y >= kd) continue;
                const auto gf = frag_of<E>(g[y / 16], g[y / 16 + 1]);
                if (AHEAD) {
#pragma unroll
                    for (int i = 0; i < 2; i++) mma(du[i], ordered_row(l, s.k, ST, 16 * i, y), gf);
                    continue;
                }
                const auto sf = frag_of<E>(st[y / 16], st[y / 16 + 1]);
                if (HALVES == 1 || 16 * wave < VH) put_frag(l, s.through, ST, TP, 16 * wave, y, sf);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const auto kf = ordered_row(l, s.k, ST, 16 * i, y);
                    mma(ks[i], kf, sf);
                    mma(du[i], kf, gf);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int t = 16 * i + 4 * l.quad;
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][e] = AHEAD ? 0.0f : float(s.v[(t + e) * ST + 16 * wave + l.col]);
                if (!FULL) settle(ks[i], du[i]);
                du[i] *= four(gates.after + t);
                if (AHEAD) continue;
                x[i] -= four(gates.before + t) * ks[i];
                dr[i] = four(gates.beta + t) * x[i];
            }
        }
        bool odd = false;  // a result is not finite
        if (!AHEAD) {
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < KT; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) dot = fmaf(st[i][r], g[i][r], dot);
            dot = sum_rows32(sum_rows16(sum16(dot)));
            if (lane == 0) s.dot[wave] = dot;
            odd = !finite(dot);
        }
        __syncthreads();
        if (!AHEAD && tid == 0) s.odd = 0;

        // The chunk by the definition, from its last tick to its first; G in a
        // copy, or the products' registers would follow this loop's order.
        const auto by_definition = [&] {
            f32x4 gx[KT];
#pragma unroll
            for (int i = 0; i < KT; i++) {
                gx[i] = g[i];
                asm volatile("" : "+v"(gx[i]));
            }
            KernelCall* call_now = fresh_call();
            float* const parts = reinterpret_cast<float*>(s.u);  // [wavefront][d_q, d_k][K]
#pragma unroll 1
            for (int t = int(left < uint32_t(C) ? left : uint32_t(C)) - 1; t >= 0; t--) {
                const E *k = s.k + t * ST, *q = s.q + t * ST;
                const float beta = gates.beta[t], decay = gates.decay[t];
                const bool flag = gate_is_flag(gates, t);
                const uint32_t at = now.c * C + t;
                if (v_wave) {
                    const float o = float(s.d_o[t * ST + place(16 * wave) + 8 * (l.col >> 2) + (l.col & 3)]);
                    float error = 0.0f;
                    if (!AHEAD) {
                        fetch_state(now);  // S before the chunk, which becomes S before the tick's update
#pragma unroll 1
                        for (int j = 0; j < t; j++) {
                            const E* kj = s.k + j * ST;
                            decay_state(st, gates, j);
                            add_outer(l, st, kj,
                                      gates.beta[j] * (float(s.v[j * ST + 16 * wave + l.col]) - column_dot(l, st, kj)));
                        }
                        decay_state(st, gates, t);
                        error = float(s.v[t * ST + 16 * wave + l.col]) - column_dot(l, st, k);
                    }
                    const float u = beta * error;
                    add_outer(l, gx, q, scale * o);
                    const float du = column_dot(l, gx, k), dv = beta * du;
                    float dg = 0.0f;
#pragma unroll
                    for (int i = 0; i < KT && !AHEAD; i++) {
                        const f32x4 kr = ordered4(l, k, i);
                        f32x4 pq, pk;
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            pq[r] = sum16(scale * fmaf(kr[r], u, st[i][r]) * o);
                            pk[r] = sum16(gx[i][r] * u - st[i][r] * dv);
                            dg = fmaf(fmaf(-kr[r], dv, gx[i][r]), st[i][r], dg);
                        }
                        if (l.col == 0) {
                            *reinterpret_cast<f32x4*>(parts + (2 * wave) * D + 16 * i + 4 * l.quad) = pq;
                            *reinterpret_cast<f32x4*>(parts + (2 * wave + 1) * D + 16 * i + 4 * l.quad) = pk;
                        }
                        asm volatile("" : "+v"(dg)::"memory");
                    }
                    add_outer(l, gx, k, -dv);
#pragma unroll
                    for (int i = 0; i < KT; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) gx[i][r] = flag ? 0.0f : gx[i][r] * decay;
                    if (!AHEAD) {
                        dg = sum_rows32(sum_rows16(sum16(dg)));
                        const float db = sum16(16 * wave + l.col < vd ? du * error : 0.0f);
                        if (lane == 0) {
                            s.odd_sums[0][wave] = dg;
                            s.odd_sums[1][wave] = db;
                        }
                        if (l.quad == 0 && 16 * wave + l.col < vd)
                            Track<E>(&call_now->d.d_v, now.n, now.h).row(at)[16 * wave + l.col] = E(dv);
                    }
                }
                if (AHEAD) continue;
                __syncthreads();
                const int v_waves = (vd + 15) / 16;
                const uint32_t hg = call_now->d.partial ? now.h : now.hq;
                if (tid < kd) {
                    float dq = 0.0f, dk = 0.0f;
                    for (int w = 0; w < v_waves; w++) {
                        dq += parts[2 * w * D + tid];
                        dk += parts[(2 * w + 1) * D + tid];
                    }
                    Track<F>(&call_now->d.d_q, now.n, hg).row(at)[tid] = F(dq);
                    Track<F>(&call_now->d.d_k, now.n, hg).row(at)[tid] = F(dk);
                }
                if (tid == 0) {
                    float dg = 0.0f, db = 0.0f;
                    for (int w = 0; w < v_waves; w++) {
                        dg += s.odd_sums[0][w];
                        db += s.odd_sums[1][w];
                    }
                    put_gate<E>(call_now, now, at, flag ? 0.0f : dg, db);
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < KT; i++) g[i] = gx[i];
        };

        // U and R
        f32x4 dv[2];
        if (v_wave) {
            if (!AHEAD) {
                f32x4 u[2];
                solve(l, s.sys, dr, u);
#pragma unroll
                for (int i = 0; i < 2; i++) put_tile<N>(l, s.u, CP, PL, 16 * wave, 16 * i, u[i]);
            }
            const auto of = ordered_col(l, s.d_o, ST, 16 * wave);
#pragma unroll
            for (int i = 0; i < 2; i++) mma(du[i], row_frag<N>(l, s.sys.scores, CP, SP, 16 * i, 0), of);
            solve_transposed(l, s.sys, du, dr);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (!AHEAD) put_tile<N>(l, s.r, CP, PL, 16 * wave, 16 * i, dr[i]);
                f32x4 sum = dr[i] * x[i];
#pragma unroll
                for (int e = 0; e < 4 && !AHEAD; e++) sum[e] = sum16(sum[e]);
                dv[i] = four(gates.beta + 16 * i + 4 * l.quad) * dr[i];
                dr[i] = dv[i] * four(gates.before + 16 * i + 4 * l.quad);  // from here on gamma beta R
                if (!AHEAD && l.col == 0) *reinterpret_cast<f32x4*>(&s.beta_v[wave][16 * i + 4 * l.quad]) = sum;
                odd |= !finite(dr[i] + sum);
            }
        }
        __syncthreads();

        // G before the chunk
        const auto step_back = [&] {
            if (!v_wave) return;
            const float total = gates.before[C - 1];
            const auto of = ordered_col(l, s.d_o, ST, 16 * wave);
            f32x4 lo, hi;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo[e] = first_term(of, e);
                hi[e] = first_term(of, 4 + e);
            }
            lo *= scale * four(gates.before + 4 * l.quad);
            hi *= scale * four(gates.before + 16 + 4 * l.quad);
            const auto of2 = frag_of<E>(lo, hi);
            const auto rf = frag_of<E>(-dr[0], -dr[1]);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                if (16 * i >= kd) continue;
                g[i] *= total;
                mma(g[i], ordered_col(l, s.q, ST, 16 * i), of2);
                mma(g[i], ordered_col(l, s.k, ST, 16 * i), rf);
            }
#pragma unroll
            for (int i = 0; i < KT && !FULL; i++) settle(g[i]);
        };
        if constexpr (AHEAD) {
            if (__builtin_expect(__any(odd), 0))
                by_definition();
            else
                step_back();
            // all have read k, q and d_o, and the matrices
            __syncthreads();
            if (next.job < plan.total) put_rows(next);
            if (now.c == now.first) leave(now, g);
            __syncthreads();
            now = next;
            next = later;
            later.back(plan, which);
            continue;
        }

        // dP and dA, by the wavefronts that hold P and A
        if (wave < 3) {
            f32x4 dp = zero, da = zero;
#pragma unroll
            for (int y = 0; y < D; y += 32) {
                if (y >= vd) continue;
                const auto uj = col_frag<N>(l, s.u, CP, PL, y, j0);
                mma(dp, ordered_row(l, s.d_o, ST, i0, y), uj);
                mma(da, col_frag<N>(l, s.r, CP, PL, y, i0), uj);
            }
            if (!FULL) settle(dp, da);
            double m_row[4], m_col = 0.0;
            f32x4 b;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                da[r] = i0 + 4 * l.quad + r > j0 + l.col ? -da[r] : 0.0f;
                const double m = double(dp[r] * pm[r] + da[r] * am[r]);
                m_row[r] = sum16(m);
                m_col += m;
                b[r] = sum16(da[r] * kk[r]);
            }
            dp *= scale * dec;
            da *= four(gates.beta + i0 + 4 * l.quad) * dec;
            odd |= !finite(float(m_col)) | !finite(b);
            if (l.col == 0) {
#pragma unroll
                for (int r = 0; r < 4; r++) s.m_row[wave][4 * l.quad + r] = m_row[r];
                *reinterpret_cast<f32x4*>(&s.beta_a[wave][4 * l.quad]) = b;
            }
            m_col += __shfl_xor(m_col, 16);
            m_col += __shfl_xor(m_col, 32);
            if (l.quad == 0) s.m_col[wave][l.col] = m_col;
            put_tile<N>(l, s.sys.scores, CP, SP, j0, i0, dp);  // scale D dP, and E
            put_tile<N>(l, s.sys.inv, CP, SP, j0, i0, da);
        }
        // through S
        f32x4 dq[2] = {zero, zero}, dk[2] = {zero, zero}, dkg[2] = {zero, zero};
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            if (half > 0) {
                __syncthreads();
                if (16 * wave >= VH && v_wave)
#pragma unroll
                    for (int y = 0; y < D; y += 32)
                        if (y < kd) put_frag(l, s.through, ST, TP, 16 * wave - VH, y, frag_of<E>(st[y / 16], st[y / 16 + 1]));
                __syncthreads();
            }
            if (k_wave)
#pragma unroll
                for (int y = 0; y < VH; y += 32) {
                    if (half * VH + y >= vd) continue;
                    const auto sf = col_frag<N>(l, s.through, ST, TP, y, 16 * wave);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        mma(dq[i], ordered_row(l, s.d_o, ST, 16 * i, half * VH + y), sf);
                        mma(dk[i], col_frag<N>(l, s.r, CP, PL, half * VH + y, 16 * i), sf);
                    }
                }
        }
        if (next.job < plan.total) fetch_state(next);  // S is done with
        // through G
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
            __syncthreads();
            if (v_wave && (HALVES == 1 || (16 * wave >= VH) == (half == 1)))
#pragma unroll
                for (int y = 0; y < D; y += 32) {
                    if (y >= kd) continue;
                    // 64 wide, the operand is kept from above; 128 wide the registers do not reach
                    if (FULL && D > 64 && sizeof(E) == 2) asm volatile("" : "+v"(g[y / 16]), "+v"(g[y / 16 + 1]));
                    put_frag(l, s.through, ST, TP, 16 * wave - half * VH, y, frag_of<E>(g[y / 16], g[y / 16 + 1]));
                }
            __syncthreads();
            if (k_wave)
#pragma unroll
                for (int y = 0; y < VH; y += 32) {
                    if (half * VH + y >= vd) continue;
                    const auto gf = col_frag<N>(l, s.through, ST, TP, y, 16 * wave);
#pragma unroll
                    for (int i = 0; i < 2; i++) mma(dkg[i], col_frag<N>(l, s.u, CP, PL, half * VH + y, 16 * i), gf);
                }
        }
        if (k_wave) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (!FULL) settle(dq[i], dk[i], dkg[i]);
                const int t = 16 * i + 4 * l.quad;
                const f32x4 before = four(gates.before + t);
                dq[i] *= scale * before;
                dk[i] *= -four(gates.beta + t) * before;
                dkg[i] *= four(gates.after + t);
                f32x4 pa, pb;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int at = (t + e) * ST + place(16 * wave) + 8 * (l.col >> 2) + (l.col & 3);
                    const float qv = float(s.q[at]), kv = float(s.k[at]);
                    pa[e] = sum16(fmaf(qv, dq[i][e], kv * dk[i][e]));
                    pb[e] = sum16(kv * dkg[i][e]);
                }
                odd |= !finite(pa + pb);
                dk[i] += dkg[i];
                if (l.col == 0) {
                    *reinterpret_cast<f32x4*>(&s.a[wave][16 * i + 4 * l.quad]) = pa;
                    *reinterpret_cast<f32x4*>(&s.b[wave][16 * i + 4 * l.quad]) = pb;
                }
            }
            // inside the chunk
            const auto kf = ordered_col(l, s.k, ST, 16 * wave);
            const auto qf = ordered_col(l, s.q, ST, 16 * wave);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const auto pc = col_frag<N>(l, s.sys.scores, CP, SP, 0, 16 * i);
                const auto pr = row_frag<N>(l, s.sys.scores, CP, SP, 16 * i, 0);
                mma(dq[i], pc, kf);
                mma(dk[i], pr, qf);
                const auto ec = col_frag<N>(l, s.sys.inv, CP, SP, 0, 16 * i);
                const auto er = row_frag<N>(l, s.sys.inv, CP, SP, 16 * i, 0);
                mma(dk[i], er, kf);
                mma(dk[i], ec, kf);
            }
            odd |= !finite((dq[0] + dq[1]) + (dk[0] + dk[1]));
        }
        if (__any(odd)) s.odd = 1;
        __syncthreads();
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(s.odd), 0)) {
            by_definition();
            __syncthreads();
            if (next.job < plan.total) {
                put_rows(next);
                fetch_state(next);
            }
            if (now.c == now.first) leave(now, g);
            if (!FULL) clear_lds(s.u, sizeof(s.u) + sizeof(s.r) + sizeof(s.through));
            __syncthreads();
            now = next;
            next = later;
            later.back(plan, which);
            continue;
        }
        step_back();
        // the rows' gradients, through LDS to whole rows
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int t = 16 * i + 4 * l.quad + e;
                if (k_wave) {
                    dq_rows[t * FT + 16 * wave + l.col] = F(dq[i][e]);
                    dk_rows[t * FT + 16 * wave + l.col] = F(dk[i][e]);
                }
                if (v_wave) dv_rows[t * ST + 16 * wave + l.col] = E(dv[i][e]);
            }
        if (wave == 0) {
            const int t = lane & 31;
            float pa = 0.0f, pb = 0.0f, beta = 0.0f, all = 0.0f;
#pragma unroll
            for (int w = 0; w < Shared::W; w++) {
                // (what no wavefront writes in a narrow head stays 0)
                pa += s.a[w][t];
                pb += s.b[w][t];
                beta += s.beta_v[w][t];
                all += s.dot[w];
            }
            // tiles (0,0), (1,1), (1,0)
            const int hi = t >> 4, in = t & 15;
            const double mr = s.m_row[hi][in] + (hi ? s.m_row[2][in] : 0.0), mc = s.m_col[hi][in] + (hi ? 0.0 : s.m_col[2][in]);
            beta += s.beta_a[hi][in] + (hi ? s.beta_a[2][in] : 0.0f);
            const double after = scan_down32(double(pa) + mr - mc, lane);      // over the ticks from t on
            const double before = scan_up32(double(pb), lane) - double(pb);   // over the ticks before t
            const float dg = gate_is_flag(gates, t) ? 0.0f : float(after + before + double(gates.before[C - 1]) * double(all));
            if (lane < C && uint32_t(t) < left) {
                put_gate<E>(fresh_call(), now, now.c * C + t, dg, beta);
            }
        }
        __syncthreads();
        // all have read k, q and d_o.  The next chunk's rows and S are waited for
        // before this one's gradients leave: loads and stores are counted in
        // order, and the loads would wait for the stores
        if (next.job < plan.total) put_rows(next);
#pragma unroll
        for (int i = 0; i < KT; i++) asm volatile("" : "+v"(st[i]));
        asm volatile("" : "+v"(gate.g), "+v"(gate.beta), "+v"(gate.flag));
        KernelCall* k = fresh_call();
        const uint32_t hg = k->d.partial ? now.h : now.hq;
        if (on_k.on && on_k.row < left) {
            const uint32_t t = now.c * C + on_k.row;
            store_piece<F>(Track<F>(&k->d.d_q, now.n, hg).row(t), kd, on_k.col, piece_from_lds(dq_rows + on_k.row * FT + on_k.col));
            store_piece<F>(Track<F>(&k->d.d_k, now.n, hg).row(t), kd, on_k.col, piece_from_lds(dk_rows + on_k.row * FT + on_k.col));
        }
        if (on_v.on && on_v.row < left)
            store_piece<E>(Track<E>(&k->d.d_v, now.n, now.h).row(now.c * C + on_v.row), vd, on_v.col,
                           piece_from_lds(dv_rows + on_v.row * ST + on_v.col));
        if (now.c == now.first) leave(now, g);
        // u, r and `through` take the next chunk's operands.  `through` is the
        // first, before the next barrier: all have to have read their gradients'
        // rows.  In narrow heads the columns past the width are operands too
        // and have to be 0 again.
        __syncthreads();
        if (!FULL) clear_lds(s.u, sizeof(s.u) + sizeof(s.r) + sizeof(s.through));
        now = next;
        next = later;
        later.back(plan, which);
    }
}

// Gradients of shared query heads: each value head's fp32 rows, added up in
// order.  37,000 rows of six heads of 40 (two query heads) take 15 us, 3.2 TB/s.
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

template <class E, class F, int D, bool FULL, bool AHEAD>
hipError_t chunks(const Args& a, const GradArgs& d, hipStream_t stream) {
    constexpr uint32_t bytes = sizeof(BackwardShared<E, D>);
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    const void* f = reinterpret_cast<const void*>(&backward_kernel<E, F, D, FULL, AHEAD>);
    if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes))) return e;
    const uint32_t jobs = a.envs * a.heads * (AHEAD ? a.segments - 1 : a.segments);
    backward_kernel<E, F, D, FULL, AHEAD><<<dim3(resident_blocks(f, a, jobs, bytes)), dim3(64 * waves_of(a)), bytes, stream>>>(Call{a, d});
    return hipGetLastError();
}
template <class E, class F, int D, bool FULL>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t stream) {
    if (a.segments > 1) {
        if (hipError_t e = chunks<E, E, D, FULL, true>(a, d, stream)) return e;
        if (hipError_t e = launch_join_grads(a, sizeof(E) == 2, stream)) return e;
    }
    return chunks<E, F, D, FULL, false>(a, d, stream);
}
template <class E, class F, int D>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t stream) {
    return a.k_dim == D && a.v_dim == D ? backward<E, F, D, true>(a, d, stream) : backward<E, F, D, false>(a, d, stream);
}
template <class E, class F>
hipError_t backward(const Args& a, const GradArgs& d, hipStream_t stream) {
    return a.k_dim <= 64 && a.v_dim <= 64 ? backward<E, F, 64>(a, d, stream) : backward<E, F, 128>(a, d, stream);
}

}  // namespace

hipError_t launch_backward(const Args& a, const GradArgs& d, bool bf, hipStream_t stream) {
    if (!bf) return backward<float, float>(a, d, stream);
    return d.partial ? backward<bf16, float>(a, d, stream) : backward<bf16, bf16>(a, d, stream);
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
