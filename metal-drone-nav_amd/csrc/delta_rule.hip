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

// One wavefront has all K rows of 4 CG columns of a state in registers for
// the whole call: lane l the four columns 4 (l % CG) of rows l / CG, + 64 / CG, ..
// Columns of a state do not meet in a tick (u_c needs column c of S only), so
// wavefronts need no exchange; a tick's two sums over K are made in the lane,
// then over the 64 / CG lanes of a column.
template <class E, int CG, int ROWS>
__global__ void __launch_bounds__(256, 3) recurrent_kernel(Args a) {
    constexpr int RG = 64 / CG;  // rows of a step of the loop over K
    const int lane = int(threadIdx.x) & 63;
    const uint32_t slices = (a.v_dim + 4 * CG - 1) / (4 * CG);
    const uint64_t wave = uint64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave >= uint64_t(a.envs) * a.heads * slices) return;
    const uint32_t slice = uint32_t(wave % slices);
    const uint64_t seq = wave / slices;
    const uint32_t n = uint32_t(seq / a.heads), h = uint32_t(seq % a.heads);
    const uint32_t hq = h / (a.heads / a.qk_heads);
    const uint32_t col = slice * 4 * CG + 4 * (lane % CG), row0 = lane / CG;
    const uint32_t kd = a.k_dim, vd = a.v_dim;
    const bool wide = (vd & 3u) == 0 && col < vd;
    const uint64_t base = seq * kd * vd;
    f32x4 s[ROWS];
    const bool cleared = a.reset && a.ticks && a.reset[n * a.reset_env] != 0;  // the first tick reads no state
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint32_t row = row0 + i * RG;
        s[i] = f32x4{0, 0, 0, 0};
        if (a.state && !cleared && row < kd) {
            const float* p = a.state + base + (row * vd + col);
            if (wide) {
                s[i] = *reinterpret_cast<const f32x4*>(p);
            } else {
#pragma unroll
                for (uint32_t c = 0; c < 4; c++)
                    if (col + c < vd) s[i][c] = p[c];
            }
        }
    }
    for (uint32_t t = 0; t < a.ticks; t++) {
        const int64_t qo = t * a.q.tick + n * a.q.env + hq * a.q.head;
        const int64_t ko = t * a.k.tick + n * a.k.env + hq * a.k.head;
        GateRegs gate = load_gates<E>(&a, n, h, t, true);
        gate.flag |= gate.g < NO_DECAY;
        f32x4 v{0, 0, 0, 0};
        const int64_t vo = t * a.v.tick + n * a.v.env + h * a.v.head + col;
#pragma unroll
        for (uint32_t c = 0; c < 4; c++)
            if (col + c < vd) v[c] = load_one<E>(a.v.p, vo + c);
        float kr[ROWS], qr[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const uint32_t row = row0 + i * RG;
            kr[i] = row < kd ? load_one<E>(a.k.p, ko + row) : 0.0f;
            qr[i] = row < kd ? load_one<E>(a.q.p, qo + row) : 0.0f;
        }
        if (gate.flag) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) s[i] = f32x4{0, 0, 0, 0};
        }
        const float decay = gate.flag ? 1.0f : __expf(gate.g);
        f32x4 ks{0, 0, 0, 0}, qs{0, 0, 0, 0};
        float kq = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            s[i] *= decay;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                ks[c] = fmaf(kr[i], s[i][c], ks[c]);
                qs[c] = fmaf(qr[i], s[i][c], qs[c]);
            }
            kq = fmaf(kr[i], qr[i], kq);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            ks[c] = sum_columns<CG>(ks[c]);
            qs[c] = sum_columns<CG>(qs[c]);
        }
        kq = sum_columns<CG>(kq);
        f32x4 u, o;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            u[c] = gate.beta * (v[c] - ks[c]);
            o[c] = a.scale * fmaf(kq, u[c], qs[c]);
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) s[i][c] = fmaf(kr[i], u[c], s[i][c]);
        if (row0 == 0) {
            const int64_t oo = t * a.o.tick + n * a.o.env + h * a.o.head + col;
#pragma unroll
            for (uint32_t c = 0; c < 4; c++)
                if (col + c < vd) reinterpret_cast<E*>(a.o.p)[oo + c] = E(o[c]);
        }
    }
    if (!a.state_out) return;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint32_t row = row0 + i * RG;
        if (row >= kd) continue;
        float* p = a.state_out + base + (row * vd + col);
        if (wide) {
            *reinterpret_cast<f32x4*>(p) = s[i];
        } else {
#pragma unroll
            for (uint32_t c = 0; c < 4; c++)
                if (col + c < vd) p[c] = s[i][c];
        }
    }
}

// ---------------------------------------------------------------- chunks
template <class E, int D> struct ForwardShared {
    static constexpr int STRIDE = D + Kind<E>::PAD;
    E k[C * STRIDE], q[C * STRIDE], v[C * STRIDE], o[C * STRIDE];
    System<E> sys;
    Gates gates[2];  // of this chunk and the next
};

// One workgroup per state, a wavefront for each 16 columns of V (at least
// four): a wavefront has its K x 16 slice of the state in result tiles, which
// are operands as they are (delta_tiles.h).  D, 64 or 128, is what registers
// and LDS rows are sized for; narrower heads leave out whole steps of 32.
template <class E, int D, bool FULL>
__global__ void __launch_bounds__(D * 4, 4) forward_kernel(Call call) {
    typedef ForwardShared<E, D> Shared;
    constexpr int ST = Shared::STRIDE, N = Kind<E>::MID, KT = D / 16;
    extern __shared__ __align__(16) char lds[];
    Shared& s = *reinterpret_cast<Shared*>(lds);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int waves = FULL ? D / 16 : blockDim.x >> 6;
    const uint32_t kd = FULL ? D : call.a.k_dim, vd = FULL ? D : call.a.v_dim;
    const uint32_t ticks = call.a.ticks, chunks = (ticks + CHUNK - 1) / CHUNK;
    const uint32_t heads = call.a.heads, shared = heads / call.a.qk_heads, states = call.a.envs * heads;
    const float scale = call.a.scale;
    const Spot on_k(kd), on_v(vd);  // the thread's piece of k and q, and of v and o
    if (!FULL) clear_lds(lds, sizeof(Shared));
    // the matrices' upper right block stays 0
    if (wave < 2 * N) {
        const Lane l = Lane::mine();
        E* m = (wave & 1 ? s.sys.scores : s.sys.inv) + (wave >> 1) * System<E>::PLANE;
#pragma unroll
        for (int i = 0; i < 4; i++) m[(16 + l.col) * CP + 4 * l.quad + i] = E(0.0f);
    }
    f32x4 state[KT];
    Piece<E> pk, pq, pv;
    const auto fetch = [&](const At& at) {
        KernelCall* k = fresh_call();
        if (on_k.on) {
            const uint32_t x = at.c * C + on_k.row, t = x < ticks ? x : 0u;
            pk = load_piece<E>(Track<const E>(&k->a.k, at.n, at.hq).row(t), kd, on_k.col);
            pq = load_piece<E>(Track<const E>(&k->a.q, at.n, at.hq).row(t), kd, on_k.col);
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
            piece_to_ordered(s.q + on_k.row * ST, on_k.col, mask_piece<E>(pq, on_k.row < left));
        }
        if (on_v.on) piece_to_lds(s.v + on_v.row * ST + on_v.col, mask_piece<E>(pv, on_v.row < left));
    };
    const auto fetch_state = [&](const At& at) {
        const Lane l = Lane::fresh();
        const float* p = fresh_call()->a.state;
        load_state(state, p ? p + uint64_t(at.seq) * kd * vd : nullptr, kd, vd, l, 16 * wave + l.col);
    };
    // the last wavefront has no tile of A: it makes the next chunk's decays
    // meanwhile, from what it loaded a chunk before that
    GateRegs gate{0.0f, 0.0f, 0u};
    const auto fetch_gates = [&](const At& at) {
        const uint32_t t = at.c * C + lane;
        gate = load_gates<E>(&fresh_call()->a, at.n, at.h, t, lane < C && t < ticks);
    };
    At now{blockIdx.x, 0, 0, 0, 0};
    now.split(heads, shared);
    At next = now, later;
    next.forth(chunks, heads, shared);
    later = next;
    later.forth(chunks, heads, shared);
    fetch(now);
    if (wave == waves - 1) {
        fetch_gates(now);
        put_gates(s.gates[0], gate);
        if (next.seq < states) fetch_gates(next);
    }
    fetch_state(now);
    put_rows(now);
    __syncthreads();
    for (uint32_t turn = 0; now.seq < states; turn ^= 1) {
        const Lane l = Lane::fresh();
        const Gates& gates = s.gates[turn];
        const uint32_t left = ticks - now.c * C;  // ticks from the chunk's first
        if (next.seq < states) fetch(next);
        if (now.c > 0 && 16 * wave < int(vd)) {
            if (float* keep = fresh_call()->a.chunk_states) {
                f32x4* p = state_tiles(keep, now.seq, chunks, now.c, kd, vd, wave);
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
                mma(qk, ordered_row(l, s.q, ST, i0, x), kj);
            }
            const f32x4 d = decay_tile(l, gates, i0, j0);
            f32x4 am = four(gates.beta + i0 + 4 * l.quad) * d * kk;
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (i0 + 4 * l.quad + r <= j0 + l.col) am[r] = 0.0f;
            const f32x4 pm = scale * d * qk;
            put_tile(l, s.sys.scores, CP, System<E>::PLANE, j0, i0, pm);
            if (wave < 2)
                put_tile(l, s.sys.inv, CP, System<E>::PLANE, 16 * wave, 16 * wave, invert_block(l, am));
            else
                put_tile(l, s.sys.inv, CP, System<E>::PLANE, 0, 16, am);
        }
        if (wave == waves - 1 && next.seq < states) {
            put_gates(s.gates[turn ^ 1], gate);
            if (later.seq < states) fetch_gates(later);
        }
        // the state's part of the ticks
        f32x4 ks[2] = {}, qs[2] = {}, r[2], u[2];
        if (16 * wave < int(vd)) {
#pragma unroll
            for (int x = 0; x < D; x += 32) {
                if (x >= int(kd)) continue;
                const auto st = frag_of<E>(state[x / 16], state[x / 16 + 1]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mma(ks[i], ordered_row(l, s.k, ST, 16 * i, x), st);
                    mma(qs[i], ordered_row(l, s.q, ST, 16 * i, x), st);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int t = 16 * i + 4 * l.quad;
                const f32x4 g = four(gates.before + t);
#pragma unroll
                for (int e = 0; e < 4; e++) r[i][e] = float(s.v[(t + e) * ST + 16 * wave + l.col]);
                r[i] = four(gates.beta + t) * (r[i] - g * ks[i]);
                qs[i] *= scale * g;
            }
        }
        __syncthreads();
        if (16 * wave < int(vd)) {
            solve(l, s.sys, r, u);
            // o = scale gamma (q S) + scores u
            {
                const auto uf = frag_of<E>(u[0], u[1]);
#pragma unroll
                for (int i = 0; i < 2; i++) mma(qs[i], col_frag<N>(l, s.sys.scores, CP, System<E>::PLANE, 0, 16 * i), uf);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int t = 16 * i + 4 * l.quad;
#pragma unroll
                for (int e = 0; e < 4; e++) s.o[(t + e) * ST + 16 * wave + l.col] = E(qs[i][e]);
                u[i] *= four(gates.after + t);
            }
            // S <- gamma_C S + K^T u
            const float total = gates.before[C - 1];
            const auto uf = frag_of<E>(u[0], u[1]);
#pragma unroll
            for (int i = 0; i < KT; i++) {
                if (16 * i >= int(kd)) continue;
                state[i] *= total;
                mma(state[i], ordered_col(l, s.k, ST, 16 * i), uf);
            }
        }
        __syncthreads();
        // the next chunk's rows go to LDS before this one's leave: loads and
        // stores are counted in order, and the loads would wait for the stores
        if (next.seq < states) put_rows(next);
        if (on_v.on && on_v.row < left)
            store_piece<E>(Track<E>(&fresh_call()->a.o, now.n, now.h).row(now.c * C + on_v.row), vd, on_v.col,
                           piece_from_lds(s.o + on_v.row * ST + on_v.col));
        if (now.c + 1 == chunks) {
            if (float* p = fresh_call()->a.state_out)
                store_state(p + uint64_t(now.seq) * kd * vd, state, kd, vd, l, 16 * wave + l.col);
            if (next.seq < states) fetch_state(next);
        }
        now = next;
        next = later;
        later.forth(chunks, heads, shared);
        __syncthreads();
    }
}

template <class E, int D, bool FULL>
hipError_t forward(const Args& a, hipStream_t stream) {
    constexpr uint32_t bytes = sizeof(ForwardShared<E, D>);
    const void* f = reinterpret_cast<const void*>(&forward_kernel<E, D, FULL>);
    if (hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes))) return e;
    forward_kernel<E, D, FULL><<<dim3(resident_blocks(f, a, bytes)), dim3(64 * waves_of(a)), bytes, stream>>>(Call{a, GradArgs{}});
    return hipGetLastError();
}
// FULL: heads as wide as the kernel's tiles, without the branches for narrower ones.
template <class E, int D>
hipError_t forward(const Args& a, hipStream_t stream) {
    return a.k_dim == D && a.v_dim == D ? forward<E, D, true>(a, stream) : forward<E, D, false>(a, stream);
}
template <class E>
hipError_t forward(const Args& a, hipStream_t stream) {
    return a.k_dim <= 64 && a.v_dim <= 64 ? forward<E, 64>(a, stream) : forward<E, 128>(a, stream);
}

template <class E>
hipError_t recurrent(const Args& a, hipStream_t stream) {
    const uint64_t seqs = uint64_t(a.envs) * a.heads;
    if (a.k_dim <= 64) {
        const uint64_t waves = seqs * ((a.v_dim + 63) / 64);
        recurrent_kernel<E, 16, 16><<<dim3(uint32_t((waves + 3) / 4)), dim3(256), 0, stream>>>(a);
    } else {
        const uint64_t waves = seqs * ((a.v_dim + 31) / 32);
        recurrent_kernel<E, 8, 16><<<dim3(uint32_t((waves + 3) / 4)), dim3(256), 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_recurrent(const Args& a, bool bf, hipStream_t stream) {
    return bf ? recurrent<bf16>(a, stream) : recurrent<float>(a, stream);
}

hipError_t launch_forward(const Args& a, bool bf, hipStream_t stream) {
    return bf ? forward<bf16>(a, stream) : forward<float>(a, stream);
}

}  // namespace delta
