// delta_rule.hip — the gated delta rule forward: single ticks and chunks.
#include "delta_rule.h"

#include "delta_chunk.h"
#include "delta_tiles.h"

namespace delta {
namespace {

// ---------------------------------------------------------------- recurrent
// The sum over the lanes that share l % CG.
template <int CG> __device__ __forceinline__ float sum_columns(float x) {
    if (CG <= 8) x += from_lane<0x128>(x);  // row_ror by 8
    return sum_rows32(sum_rows16(x));
}

// Four neighbours of a row of `dim` from `col` on, those past its end 0.
struct __attribute__((aligned(4))) Four32 { float x[4]; };
struct __attribute__((aligned(2))) Four16 { bf16 x[4]; };
template <class E> struct FourOf;
template <> struct FourOf<float> { typedef Four32 type; };
template <> struct FourOf<bf16> { typedef Four16 type; };
template <class E> __device__ __forceinline__ typename FourOf<E>::type load_four(const E* row, uint32_t dim, uint32_t col) {
    typename FourOf<E>::type r;
    if (col + 4 <= dim) {
        r = *reinterpret_cast<const typename FourOf<E>::type*>(row + col);
    } else {
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) r.x[c] = col + c < dim ? row[col + c] : E(0.0f);
    }
    return r;
}
template <class E> __device__ __forceinline__ void store_four(E* row, uint32_t dim, uint32_t col, f32x4 x) {
    typename FourOf<E>::type r;
#pragma unroll
    for (int c = 0; c < 4; c++) r.x[c] = E(x[c]);
    if (col + 4 <= dim) {
        *reinterpret_cast<typename FourOf<E>::type*>(row + col) = r;
    } else {
#pragma unroll
        for (uint32_t c = 0; c < 4; c++)
            if (col + c < dim) row[col + c] = r.x[c];
    }
}

// One wavefront has all K rows of 4 CG columns of a state in registers for
// the whole call: lane l the four columns 4 (l % CG) of rows l / CG, + 64 / CG,
// ..  (a load of the wavefront then covers neighbouring rows).  Columns of a
// state do not meet in a tick (u_c needs column c of S only), so wavefronts
// need no exchange; a tick's two sums over K are made in the lane, then over
// the 64 / CG lanes of a column.  k and q are loaded an element a lane and
// handed round through LDS, where a lane's rows are neighbours.
//
// Bound by memory: a tick in place of 32,768 states 64 x 64 in bf16 (1.09 GB with
// the rows) takes 200 us, 5.5 TB/s; of 18,006 states 40 x 72, rows of 288 bytes,
// 118 to 125 us for 0.42 GB.  Lanes with 16 neighbouring rows each, whose k and q
// are plain wide loads, were as fast in the first and took 1.6 times as long in
// the second: their loads touch more cache lines in rows that do not fill them.
// Each further tick of 16,384 states 64 x 64 adds 10 to 13 us, vector work.
template <class E, int CG>
__global__ void __launch_bounds__(256, CG == 8 ? 3 : 4) recurrent_kernel(Args a) {
    constexpr int RG = 64 / CG, ROWS = 16;  // rows of a step, most steps
    __shared__ __align__(16) float rows_of[4][2][RG][ROWS];
    const int lane = int(threadIdx.x) & 63, wave_here = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slices = (a.v_dim + 4 * CG - 1) / (4 * CG);
    const uint64_t wave = uint64_t(blockIdx.x) * 4 + wave_here;
    if (wave >= uint64_t(a.envs) * a.heads * slices) return;
    const uint32_t slice = uint32_t(wave % slices);
    const uint64_t seq = wave / slices;
    const uint32_t n = uint32_t(seq / a.heads), h = uint32_t(seq % a.heads);
    const uint32_t hq = h / (a.heads / a.qk_heads);
    const uint32_t kd = a.k_dim, vd = a.v_dim;
    const int steps = int((kd + RG - 1) / RG);
    const uint32_t col = slice * 4 * CG + 4 * (lane % CG), row0 = lane / CG;
    const uint64_t base = seq * kd * vd;
    // a tick's inputs, loaded a tick ahead
    constexpr int EACH = RG * ROWS / 64;
    GateRegs gate;
    float ke[EACH], qe[EACH];
    typename FourOf<E>::type vp;
    const auto fetch = [&](uint32_t t) {
        const E* k = reinterpret_cast<const E*>(a.k.p) + (t * a.k.tick + n * a.k.env + hq * a.k.head);
        const E* q = reinterpret_cast<const E*>(a.q.p) + (t * a.q.tick + n * a.q.env + hq * a.q.head);
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const uint32_t row = lane + 64 * i;
            ke[i] = row < kd ? float(k[row]) : 0.0f;
            qe[i] = row < kd ? float(q[row]) : 0.0f;
        }
        vp = load_four(reinterpret_cast<const E*>(a.v.p) + (t * a.v.tick + n * a.v.env + h * a.v.head), vd, col);
        gate = load_gates<E>(&a, n, h, t, true);
    };
    // over the lane's rows, four at a time
    const auto each_row = [&](auto&& f) {
#pragma unroll
        for (int i0 = 0; i0 < ROWS; i0 += 4)
            if (i0 < steps) {
#pragma unroll
                for (int i = i0; i < i0 + 4; i++) f(i);
            }
    };
    if (a.ticks) fetch(0);
    f32x4 s[ROWS];
    const bool cleared = a.reset && a.ticks && a.reset[n * a.reset_env] != 0;  // the first tick reads no state
    each_row([&](int i) {
        s[i] = f32x4{0, 0, 0, 0};
        const uint32_t row = row0 + i * RG;
        if (a.state && !cleared && row < kd) {
            const Four32 x = load_four(a.state + base + row * vd, vd, col);
            s[i] = f32x4{x.x[0], x.x[1], x.x[2], x.x[3]};
        }
    });
    for (uint32_t t = 0; t < a.ticks; t++) {
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int row = lane + 64 * i;
            rows_of[wave_here][0][row % RG][row / RG] = ke[i];
            rows_of[wave_here][1][row % RG][row / RG] = qe[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f32x4 kr[ROWS / 4], qr[ROWS / 4];
#pragma unroll
        for (int i = 0; i < ROWS / 4; i++) {
            kr[i] = *reinterpret_cast<const f32x4*>(&rows_of[wave_here][0][row0][4 * i]);
            qr[i] = *reinterpret_cast<const f32x4*>(&rows_of[wave_here][1][row0][4 * i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const f32x4 v{float(vp.x[0]), float(vp.x[1]), float(vp.x[2]), float(vp.x[3])};
        const float beta = gate.beta, g = gate.g;
        const bool flag = gate.flag || g < NO_DECAY;
        if (t + 1 < a.ticks) fetch(t + 1);
        if (flag) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) s[i] = f32x4{0, 0, 0, 0};
        }
        const float decay = flag ? 1.0f : __expf(g);
        f32x4 ks{0, 0, 0, 0}, qs{0, 0, 0, 0};
        float kq = 0.0f;
        each_row([&](int i) {
            s[i] *= decay;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                ks[c] = fmaf(kr[i / 4][i % 4], s[i][c], ks[c]);
                qs[c] = fmaf(qr[i / 4][i % 4], s[i][c], qs[c]);
            }
            kq = fmaf(kr[i / 4][i % 4], qr[i / 4][i % 4], kq);
        });
#pragma unroll
        for (int c = 0; c < 4; c++) {
            ks[c] = sum_columns<CG>(ks[c]);
            qs[c] = sum_columns<CG>(qs[c]);
        }
        kq = sum_columns<CG>(kq);
        f32x4 u, o;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            u[c] = beta * (v[c] - ks[c]);
            o[c] = a.scale * fmaf(kq, u[c], qs[c]);
        }
        each_row([&](int i) {
#pragma unroll
            for (int c = 0; c < 4; c++) s[i][c] = fmaf(kr[i / 4][i % 4], u[c], s[i][c]);
        });
        if (row0 == 0) store_four(reinterpret_cast<E*>(a.o.p) + (t * a.o.tick + n * a.o.env + h * a.o.head), vd, col, o);
    }
    if (!a.state_out) return;
    each_row([&](int i) {
        const uint32_t row = row0 + i * RG;
        if (row < kd) store_four(a.state_out + base + row * vd, vd, col, s[i]);
    });
}

// ---------------------------------------------------------------- chunks
template <class E, int D, int N> struct ForwardShared {
    static constexpr int STRIDE = D + Kind<E>::PAD;
    E k[C * STRIDE], q[C * STRIDE], v[C * STRIDE], o[C * STRIDE];
    System<E, N> sys;
    Gates gates[2];  // of this chunk and the next
};

// One workgroup per state, a wavefront for each 16 columns of V (at least
// four): a wavefront has its K x 16 slice of the state in result tiles, which
// are operands as they are (delta_tiles.h).  D, 64 or 128, is what registers
// and LDS rows are sized for; narrower heads leave out whole steps of 32.
//
// AHEAD: what the segments of a cut state need before they run.  Part 0 of a
// segment starts from zeros (the first from the state) and leaves B, part 1
// starts from the identity with no v and leaves M; neither has outputs.
//
// Bound by the issue of vector instructions (the products' operands are split
// and scaled between the matrix cores) and the waits between them: 32,768 states
// 64 x 64 of 128 ticks in bfloat16 (2.7 GB) take 852 to 882 us, 3.1 TB/s, with the
// vector units issuing 60 % and the matrix cores busy 16 % of the time and a
// wavefront waiting 53 % of its; with a final state, in three terms, 1,100 to 1,140;
// of 32 ticks 262 to 269 us.  5,120 states 128 x 128 of 64 ticks 189 us, with a
// final state 278; 6,000 of 40 x 72, 37 ticks, in fp32, 313 us, where the fp32 matrix
// cores (four places of the summed axis each) and waits between them count.
// Chunks of 32 ticks: of 16 there would be twice the passes over the state, of
// 64 a triangle that takes four times the work.
template <class E, int N, int D, bool FULL, bool AHEAD>
__global__ void __launch_bounds__(D * 4, 4) forward_kernel(Call call) {
    typedef ForwardShared<E, D, N> Shared;
    constexpr int ST = Shared::STRIDE, KT = D / 16;
    extern __shared__ __align__(16) char lds[];
    Shared& s = *reinterpret_cast<Shared*>(lds);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int waves = FULL ? D / 16 : blockDim.x >> 6;
    const uint32_t kd = FULL ? D : call.a.k_dim, vd = FULL ? D : call.a.v_dim;
    const uint32_t ticks = call.a.ticks;
    const Plan plan(call.a, AHEAD ? 2 * call.a.segments - 3 : call.a.segments);
    const auto which = [&](At& at, uint32_t j) {
        // AHEAD: part 0 of all segments but the last, then part 1 of all but the first and the last
        at.part = AHEAD && j >= plan.segments - 1 ? 1 : 0;
        at.seg = at.part ? j - (plan.segments - 1) + 1 : j;
    };
    const float scale = call.a.scale;
    const Spot on_k(kd), on_v(vd);  // the thread's piece of k and q, and of v and o
    if (!FULL) clear_lds(lds, sizeof(Shared));
    // the matrices' upper right block stays 0
    for (int p = wave; p < 2 * N; p += waves) {
        const Lane l = Lane::mine();
        E* m = (p & 1 ? s.sys.scores : s.sys.inv) + (p >> 1) * System<E, N>::PLANE;
#pragma unroll
        for (int i = 0; i < 4; i++) m[(16 + l.col) * CP + 4 * l.quad + i] = E(0.0f);
    }
    f32x4 state[KT];
    bool flagged = false;  // AHEAD: an episode has begun in the segment, nothing of the state before it is left
    Piece<E> pk, pq, pv;
    const auto fetch = [&](const At& at) {
        KernelCall* k = fresh_call();
        if (on_k.on) {
            const uint32_t x = at.c * C + on_k.row, t = x < ticks ? x : 0u;
            pk = load_piece<E>(Track<const E>(&k->a.k, at.n, at.hq).row(t), kd, on_k.col);
            if (!AHEAD) pq = load_piece<E>(Track<const E>(&k->a.q, at.n, at.hq).row(t), kd, on_k.col);
        }
        if (on_v.on) {
            const uint32_t x = at.c * C + on_v.row, t = x < ticks ? x : 0u;
            pv = load_piece<E>(Track<const E>(&k->a.v, at.n, at.h).row(t), vd, on_v.col);
        }
    };
    const auto put_rows = [&](const At& at) {
        const uint32_t left = ticks - at.c * C;
        if (on_k.on) {
            piece_to_ordered(s.k + on_k.row * ST, on_k.col, mask_piece<E>(pk, on_k.row < left));
            if (!AHEAD) piece_to_ordered(s.q + on_k.row * ST, on_k.col, mask_piece<E>(pq, on_k.row < left));
        }
        if (on_v.on) piece_to_lds(s.v + on_v.row * ST + on_v.col, mask_piece<E>(pv, on_v.row < left && (!AHEAD || at.part == 0)));
    };
    const auto fetch_state = [&](const At& at) {
        const Lane l = Lane::fresh();
        KernelCall* k = fresh_call();
        const uint64_t words = kd * vd;
        const float* p = k->a.state;
        if (p) p += at.state * words;
        if (AHEAD && at.seg > 0) p = nullptr;
        if (!AHEAD && plan.segments > 1) p = k->a.seg_states + (uint64_t(at.state) * plan.segments + at.seg) * words;
        load_state(state, p, kd, vd, l, 16 * wave + l.col);
        if (AHEAD && at.part)
#pragma unroll
            for (int i = 0; i < KT; i++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    state[i][r] = 16 * i + 4 * l.quad + r == 16 * wave + l.col && uint32_t(16 * wave + l.col) < kd ? 1.0f : 0.0f;
    };
    // the last wavefront has no tile of A: it makes the next chunk's decays
    // meanwhile, from what it loaded a chunk before that
    GateRegs gate{0.0f, 0.0f, 0u};
    const auto fetch_gates = [&](const At& at) {
        const uint32_t t = at.c * C + lane;
        gate = load_gates<E>(&fresh_call()->a, at.n, at.h, t, lane < C && t < ticks);
    };
    At now, next, later;
    now.job = blockIdx.x;
    now.split(plan, which);
    now.c = now.first;
    next = now;
    next.forth(plan, which);
    later = next;
    later.forth(plan, which);
    fetch(now);
    if (wave == waves - 1) {
        fetch_gates(now);
        put_gates(s.gates[0], gate);
        if (next.job < plan.total) fetch_gates(next);
    }
    fetch_state(now);
    put_rows(now);
    __syncthreads();
    for (uint32_t turn = 0; now.job < plan.total; turn ^= 1) {
        const Lane l = Lane::fresh();
        const Gates& gates = s.gates[turn];
        const uint32_t left = ticks - now.c * C;  // ticks from the chunk's first
        if (next.job < plan.total) fetch(next);
        const uint32_t cols = AHEAD && now.part ? kd : vd;  // of the state
        // the main pass takes the first segment's state from here: the caller's
        // may be state_out too, which the last segment writes when it likes
        if (AHEAD && now.c == 0) store_state(fresh_call()->a.seg_states + uint64_t(now.state) * plan.segments * kd * vd, state, kd, vd, l, 16 * wave + l.col);
        if (!AHEAD && now.c > 0 && 16 * wave < int(vd)) {
            if (float* keep = fresh_call()->a.chunk_states) {
                f32x4* p = state_tiles(keep, now.state, plan.chunks, now.c, kd, vd, wave);
#pragma unroll
                for (int i = 0; i < KT; i++)
                    if (16 * i < int(kd)) p[64 * i + lane] = state[i];
            }
        }
        // the chunk's scores and A: tiles (0,0), (1,1), (1,0)
        if (wave < 3) {
            const int i0 = wave ? 16 : 0, j0 = wave == 1 ? 16 : 0;
            f32x4 kk{0, 0, 0, 0}, qk{0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < D; x += 32) {
                if (x >= int(kd)) continue;
                const auto kj = ordered_row(l, s.k, ST, j0, x);
                mma(kk, ordered_row(l, s.k, ST, i0, x), kj);
                if (!AHEAD) mma(qk, ordered_row(l, s.q, ST, i0, x), kj);
            }
            if (!FULL) settle(kk, qk);
            const f32x4 d = decay_tile(l, gates, i0, j0);
            f32x4 am = four(gates.beta + i0 + 4 * l.quad) * d * kk;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (i0 + 4 * l.quad + r <= j0 + l.col) am[r] = 0.0f;
            const f32x4 pm = scale * d * qk;
            if (!AHEAD) put_tile<N>(l, s.sys.scores, CP, System<E, N>::PLANE, j0, i0, pm);
            if (wave < 2)
                put_tile<N>(l, s.sys.inv, CP, System<E, N>::PLANE, 16 * wave, 16 * wave, invert_block(l, am));
            else
                put_tile<N>(l, s.sys.inv, CP, System<E, N>::PLANE, 0, 16, am);
        }
        if (wave == waves - 1 && next.job < plan.total) {
            put_gates(s.gates[turn ^ 1], gate);
            if (later.job < plan.total) fetch_gates(later);
        }
        // the state's part of the ticks
        f32x4 ks[2] = {}, qs[2] = {}, r[2], u[2];
        if (16 * wave < int(cols)) {
#pragma unroll
            for (int x = 0; x < D; x += 32) {
                if (x >= int(kd)) continue;
                const auto st = frag_of<E, N>(state[x / 16], state[x / 16 + 1]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mma(ks[i], ordered_row(l, s.k, ST, 16 * i, x), st);
                    if (!AHEAD) mma(qs[i], ordered_row(l, s.q, ST, 16 * i, x), st);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (!FULL) settle(ks[i], qs[i]);
                const int t = 16 * i + 4 * l.quad;
                const f32x4 g = four(gates.before + t);
#pragma unroll
                for (int e = 0; e < 4; e++) r[i][e] = float(s.v[(t + e) * ST + 16 * wave + l.col]);
                r[i] = four(gates.beta + t) * (r[i] - g * ks[i]);
                qs[i] *= scale * g;
            }
        }
        __syncthreads();
        // the columns' outputs and what they add to the state; where one of
        // these is not finite, the chunk by the definition
        bool odd = false;
        if (16 * wave < int(cols)) {
            solve(l, s.sys, r, u);
            // o = scale gamma (q S) + scores u
            if (!AHEAD) {
                const auto uf = frag_of<E, N>(u[0], u[1]);
#pragma unroll
                for (int i = 0; i < 2; i++) mma(qs[i], col_frag<N>(l, s.sys.scores, CP, System<E, N>::PLANE, 0, 16 * i), uf);
            }
            f32x4 sum = qs[0] + qs[1];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int t = 16 * i + 4 * l.quad;
#pragma unroll
                for (int e = 0; e < 4 && !AHEAD; e++) s.o[(t + e) * ST + 16 * wave + l.col] = E(qs[i][e]);
                u[i] *= four(gates.after + t);
                sum += u[i];
            }
            odd = __any(!finite(sum));
            asm volatile("" : "+v"(u[0]), "+v"(u[1]));  // (kept as they are, or three-term instances spill)
        }
        if (__builtin_expect(odd, 0)) {
            // (copied, or the products' registers would follow this loop's order)
            f32x4 sx[KT];
#pragma unroll
            for (int i = 0; i < KT; i++) {
                sx[i] = state[i];
                asm volatile("" : "+v"(sx[i]));
            }
            const uint32_t ticks_here = left < uint32_t(C) ? left : uint32_t(C);
#pragma unroll 1
            for (uint32_t t = 0; t < ticks_here; t++) {
                const E* k = s.k + t * ST;
                decay_state(sx, gates, t);
                const float v = float(s.v[t * ST + 16 * wave + l.col]);
                add_outer(l, sx, k, gates.beta[t] * (v - column_dot(l, sx, k)));
                if (!AHEAD) {
                    const float o = scale * column_dot(l, sx, s.q + t * ST);
                    if (l.quad == 0) s.o[t * ST + 16 * wave + l.col] = E(o);
                }
            }
#pragma unroll
            for (int i = 0; i < KT; i++) state[i] = sx[i];
        } else if (16 * wave < int(cols)) {
            // S <- gamma_C S + K^T u
            const float total = gates.before[C - 1];
            const auto uf = frag_of<E, N>(u[0], u[1]);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                if (16 * i >= int(kd)) continue;
                state[i] *= total;
                mma(state[i], ordered_col(l, s.k, ST, 16 * i), uf);
            }
#pragma unroll
            for (int i = 0; i < KT && !FULL; i++) settle(state[i]);
        }
        __syncthreads();
        // the next chunk's rows go to LDS before this one's leave: loads and
        // stores are counted in order, and the loads would wait for the stores
        if (next.job < plan.total) put_rows(next);
        if (!AHEAD && on_v.on && on_v.row < left)
            store_piece<E>(Track<E>(&fresh_call()->a.o, now.n, now.h).row(now.c * C + on_v.row), vd, on_v.col,
                           piece_from_lds(s.o + on_v.row * ST + on_v.col));
        if (AHEAD) flagged = (now.c > now.first && flagged) | (__builtin_amdgcn_readfirstlane(gates.episode[C - 1]) != 0);
        if (now.c + 1 == now.end) {
            KernelCall* k = fresh_call();
            float* p = now.seg + 1 == plan.segments ? k->a.state_out : nullptr;
            if (p) p += uint64_t(now.state) * kd * vd;
            const uint64_t slot = uint64_t(now.state) * plan.segments + now.seg;
            if (AHEAD) p = now.part ? k->a.seg_moves + slot * kd * kd : k->a.seg_states + (slot + 1) * kd * vd;
            if (p) store_state(p, state, kd, cols, l, 16 * wave + l.col);
            if (AHEAD && now.part && tid == 0) seg_flags(k->a.seg_moves, k->a.envs * k->a.heads, plan.segments, kd)[slot] = flagged;
            if (next.job < plan.total) fetch_state(next);
        }
        now = next;
        next = later;
        later.forth(plan, which);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- joining segments
// A workgroup per 16 columns of a state, a wavefront for each 16 rows: it has
// its rows of M ahead of the product, and the columns' last values come from
// LDS.  Bound by the latency of its steps, one after the other: 30 segments
// of 16 states 128 x 128 take 82 us under a profiler, 3 us each.
template <class E, int N, bool TRANSPOSED>
__global__ void __launch_bounds__(512) join_kernel(Args a, float* seg) {
    constexpr int D = int(MAX_DIM), ST = D + Kind<E>::PAD, PL = 16 * ST;
    __shared__ __align__(16) E last[2][N * PL];  // [column][row]
    const Lane l = Lane::mine();
    const int kd = a.k_dim, vd = a.v_dim, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slices = (vd + 15) / 16, state = blockIdx.x / slices, col = blockIdx.x % slices * 16 + l.col;
    float* const own = seg + uint64_t(state) * a.segments * kd * vd;
    const float* const moves = a.seg_moves + uint64_t(state) * a.segments * kd * kd;
    // the wavefront's tile of the value before or after segment s
    const auto tile_at = [&](uint32_t s, int r) { return own + uint64_t(s) * kd * vd + uint32_t(16 * wave + 4 * l.quad + r) * vd + col; };
    const auto load_tile = [&](uint32_t s) {
        f32x4 x{0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (16 * wave + 4 * l.quad + r < kd && int(col) < vd) x[r] = *tile_at(s, r);
        return x;
    };
    f32x4 m[D / 16];
    uint32_t flagged = 0;  // M is not looked at: what is before the flag is gone, NaN too, which M = 0 would not end
    const auto fetch = [&](uint32_t s) {
        flagged = seg_flags(a.seg_moves, a.envs * a.heads, a.segments, kd)[uint64_t(state) * a.segments + s];
        const float* p = moves + uint64_t(s) * kd * kd;
        const int r = 16 * wave + l.col;
        if (!TRANSPOSED && kd % 4 == 0) {  // four neighbours in one word: a call of 16 states 128 x 128 of 30,011 ticks 785 us and not 986
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                const int c = 16 * k + 4 * l.quad;
                const bool in = r < kd && c < kd;
                const f32x4 v = *reinterpret_cast<const f32x4*>(p + (in ? r * kd + c : 0));
#pragma unroll
                for (int e = 0; e < 4; e++) m[k][e] = in ? v[e] : 0.0f;
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < D / 16; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = 16 * k + 4 * l.quad + e;
                const bool in = r < kd && c < kd;
                const float v = p[in ? (TRANSPOSED ? c * kd + r : r * kd + c) : 0];
                m[k][e] = in ? v : 0.0f;
            }
    };
    uint32_t s = TRANSPOSED ? a.segments - 2 : 1;
    fetch(s);
    put_tile<N>(l, last[0], ST, PL, 0, 16 * wave, load_tile(s));
    f32x4 next = load_tile(TRANSPOSED ? s - 1 : s + 1);
    __syncthreads();
    for (uint32_t left = a.segments - 2, turn = 0; left > 0; left--, turn ^= 1) {
        Frag<E, N> mf[D / 32];
        const bool moved = __builtin_amdgcn_readfirstlane(flagged) == 0;
#pragma unroll
        for (int k = 0; k < D / 32; k++) mf[k] = frag_of<E, N>(m[2 * k], m[2 * k + 1]);
        s = TRANSPOSED ? s - 1 : s + 1;
        f32x4 y = next;
        if (left > 1) {
            fetch(s);
            next = load_tile(TRANSPOSED ? s - 1 : s + 1);
        }
        if (moved) {
            // a column of zeros stays one, also where M has outgrown fp32
            const f32x4 own = y;
            bool some = false;
#pragma unroll
            for (int k = 0; k < D / 32; k++) {
                const Frag<E, N> x = row_frag<N>(l, last[turn], ST, PL, 0, 32 * k);
#pragma unroll
                for (int e = 0; e < 8; e++) some |= first_term(x, e) != 0.0f;
                mma(y, mf[k], x);
            }
            const float any = sum_rows32(sum_rows16(some ? 1.0f : 0.0f));
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = any != 0.0f ? y[r] : own[r];
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (16 * wave + 4 * l.quad + r < kd && int(col) < vd) *tile_at(s, r) = y[r];
        put_tile<N>(l, last[turn ^ 1], ST, PL, 0, 16 * wave, y);
        __syncthreads();
    }
}

template <class E, int N, int D, bool FULL, bool AHEAD>
hipError_t chunks(const Args& a, hipStream_t stream) {
    constexpr uint32_t bytes = sizeof(ForwardShared<E, D, N>);
    const void* f = reinterpret_cast<const void*>(&forward_kernel<E, N, D, FULL, AHEAD>);
    if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes))) return e;
    const uint32_t jobs = a.envs * a.heads * (AHEAD ? 2 * a.segments - 3 : a.segments);
    forward_kernel<E, N, D, FULL, AHEAD><<<dim3(resident_blocks(f, a, jobs, bytes)), dim3(64 * waves_of(a)), bytes, stream>>>(Call{a, GradArgs{}});
    return hipGetLastError();
}
template <class E, int N, bool TRANSPOSED>
hipError_t join(const Args& a, float* seg, hipStream_t stream) {
    if (a.segments < 3) return hipSuccess;
    join_kernel<E, N, TRANSPOSED><<<dim3(a.envs * a.heads * ((a.v_dim + 15) / 16)), dim3(512), 0, stream>>>(a, seg);
    return hipGetLastError();
}
template <class E, int N, int D, bool FULL>
hipError_t forward(const Args& a, hipStream_t stream) {
    if (a.segments > 1) {
        if (hipError_t e = chunks<E, N, D, FULL, true>(a, stream)) return e;
        if (hipError_t e = join<E, N, false>(a, a.seg_states, stream)) return e;
    }
    return chunks<E, N, D, FULL, false>(a, stream);
}
// FULL: heads as wide as the kernel's tiles, without the branches for narrower
// ones.  With it and without, in us, forward and forward with backward: 32,768
// states 64 x 64 of 32 ticks in bfloat16 269 : 270 and 1,000 : 1,113, in fp32 473 : 500
// and 1,792 : 1,974; 5,120 states 128 x 128 of 64 ticks in bfloat16 190 : 196 and 806 :
// 904, in fp32 405 : 421 and 1,545 : 1,835.
template <class E, int N, int D>
hipError_t forward(const Args& a, hipStream_t stream) {
    return a.k_dim == D && a.v_dim == D ? forward<E, N, D, true>(a, stream) : forward<E, N, D, false>(a, stream);
}
template <class E, int N>
hipError_t forward(const Args& a, hipStream_t stream) {
    return a.k_dim <= 64 && a.v_dim <= 64 ? forward<E, N, 64>(a, stream) : forward<E, N, 128>(a, stream);
}

// Wavefronts of 32 columns have room for 128 rows, those of 64 for 64; in heads
// of at most 32 columns half the lanes of the wider ones would idle.  A tick in
// place in narrow : wide ones, in us: 16,384 states 32 x 32 in bf16 36 : 62,
// in fp32 37 : 56; 64 x 64 in bf16 105 : 118, in fp32 111 : 110; 18,006 states 48 x 48
// in bf16 90 : 103, in fp32 99 : 96; of 40 x 72 128 : 125 and 144 : 107; 12,000 of 64 x 96
// 113 : 165 and 122 : 137.  Each further tick costs narrow ones more (twice as many
// hand k and q round): 4 ticks of 16,384 states 64 x 64 in bf16 156 : 137; and so do
// few rows: a tick of 16 x 64, 47 : 34.  So narrow ones for at most 32 columns, and
// in bf16 for one tick of more rows, where they leave at most 16 columns idle.
template <class E>
hipError_t recurrent(const Args& a, hipStream_t stream) {
    const bool one = sizeof(E) == 2 && a.ticks == 1 && a.state_out && a.k_dim > 32 && (0u - a.v_dim) % 32 <= 16;
    const uint32_t cols = a.k_dim > 64 || a.v_dim <= 32 || one ? 32 : 64;
    const uint64_t waves = uint64_t(a.envs) * a.heads * ((a.v_dim + cols - 1) / cols);
    const dim3 grid(uint32_t((waves + 3) / 4));
    if (cols == 64)
        recurrent_kernel<E, 16><<<grid, dim3(256), 0, stream>>>(a);
    else
        recurrent_kernel<E, 8><<<grid, dim3(256), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_recurrent(const Args& a, bool bf, hipStream_t stream) {
    return bf ? recurrent<bf16>(a, stream) : recurrent<float>(a, stream);
}

hipError_t launch_join_grads(const Args& a, bool bf, hipStream_t stream) {
    return bf ? join<bf16, Kind<bf16>::MID, true>(a, a.seg_grads, stream) : join<float, 1, true>(a, a.seg_grads, stream);
}

hipError_t launch_forward(const Args& a, bool bf, hipStream_t stream) {
    if (!bf) return forward<float, 1>(a, stream);
    return a.state_out ? forward<bf16, 3>(a, stream) : forward<bf16, 2>(a, stream);
}

}  // namespace delta
