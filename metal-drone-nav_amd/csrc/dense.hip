// dense.hip — the linear layer y = residual + act(x W^T + b) and the gated
// feed-forward block y = act(x Wg^T + bg) * (x Wu^T + bu), with gradients.
//
// Forward: one product (dense_tiles.h) whose tile holds, for the gated block,
// the same columns of both projections, so that a lane has z of the gate and of
// the other at the same place; bias, activation and product or residual are
// made from the fp32 sums, which are rounded once.
//
// Backward: z is made again by the same product with
//     dz = dy act'(z)        or  dzg = dy zu act'(zg),  dzu = dy act(zg)
// in its epilogue, rounded once to the rows' type (the matrix cores' operand),
// and the column sums that are the biases' gradients, from the unrounded
// values.  Then dx = dz W (of the gated block, both terms in one sum) and
// dW = dz^T x, the latter's long sum over rows cut into parts that a second
// kernel adds up in order: no atomics, the same bits every time.
//
// Bound: long sums by the matrix cores and the power that they may draw (8,192^3 in
// bfloat16 runs at 1,180 to 1,370 TFLOP/s on the cards seen, 0.92 of a plain
// library product beside it; 4,096^3 in fp32 at 128 to 144, 0.96 of it). Short ones
// by what a tile does besides its products: 262,144 rows of 256 to 1,024, gated, take
// 400 us, and 215 with 64 in place of 256, whose results a copy writes in 105. (Results
// straight from registers, twice as long pieces of rows and four workgroups a compute
// unit in place of three each took at most 4 % off, or added as much.)
#include "dense.h"

#include "dense_act.h"
#include "dense_tiles.h"

#include <type_traits>

namespace dense {
namespace {

enum Result { LINEAR, GATED, SLOPE, GATED_SLOPE, STORE, PART };
constexpr bool two_weights(int r) { return r == GATED || r == GATED_SLOPE; }

struct Job {
    Side m, n;
    uint32_t k, segments;                // of the sum; segments: 2 adds a second product of m.p2 and n.p2
    uint32_t m_tiles, n_tiles;
    uint32_t splits, split_k;            // PART, STORE: pieces of k; blockIdx.y = batch splits + piece
    uint32_t act;
    Matrix y, y2, residual, dy, dz;      // y2: of a second batch (m.p2, n.p)
    const char* bias[2];
    uint32_t dz_half;                    // columns from dzg to dzu
    float* sums;                         // [m_tiles WM][2][n] or null
};

__device__ __forceinline__ f32x4 four(const f32x16& v, int g) { return f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]}; }

// ---------------------------------------------------------------- results through LDS
// A lane has four neighbours of one row of a tile, and 32 rows are 32 lines of
// memory. So a wavefront turns PW columns of 32 rows at a time, in fp32 in LDS
// of its own, and then has whole pieces of rows: a lane the word of the
// result's type (N columns) that it moves.
template <class T, int PW> struct Piece {
    static constexpr uint32_t N = per_word<T>(), LANES = PW / N, ROWS = 64 / LANES, TURNS = 32 / ROWS, BYTES = 32 * PW * 4;
    typedef T Word __attribute__((ext_vector_type(N), aligned(sizeof(T))));  // in memory: at any multiple of an element
    typedef T LdsWord __attribute__((ext_vector_type(N)));

    // Orders LDS accesses of one wavefront; it serves them in order itself.
    static __device__ __forceinline__ void order() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
    // Words of four columns change places by the row, so that no two lanes that LDS serves together meet in a bank.
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t word) { return row * (PW * 4) + ((word ^ (row & (PW / 4 - 1))) << 4); }
    static __device__ __forceinline__ void put(char* lds, const f32x16& tile, int i, uint32_t lane) {
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<f32x4*>(lds + at(lane & 31, 8 * i + 2 * g + (lane >> 5))) = four(tile, g);
    }
    static __device__ __forceinline__ uint32_t row(uint32_t lane, uint32_t turn) { return lane / LANES + turn * ROWS; }
    static __device__ __forceinline__ uint32_t column(uint32_t lane) { return lane % LANES * N; }
    static __device__ __forceinline__ void get(const char* lds, uint32_t row, uint32_t lane, float (&z)[N]) {
#pragma unroll
        for (uint32_t w = 0; w < N / 4; w++) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(lds + at(row, lane % LANES * (N / 4) + w));
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) z[4 * w + e] = v[e];
        }
    }
    // One word of a row, columns c .. c + N - 1 of `count`; 0 outside.
    // ONCE: past the caches, which large tiles fill with operands.
    template <bool ONCE> static __device__ __forceinline__ LdsWord load(const Matrix& from, uint32_t m, uint32_t c, uint32_t count) {
        const T* p = reinterpret_cast<const T*>(from.p) + int64_t(m) * from.ld + c;
        LdsWord v;
        if (c + N <= count) {
            v = ONCE ? __builtin_nontemporal_load(reinterpret_cast<const Word*>(p)) : *reinterpret_cast<const Word*>(p);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < N; e++) v[e] = c + e < count ? p[e] : T(0.0f);
        }
        return v;
    }
    template <bool ONCE> static __device__ __forceinline__ void store(const Matrix& to, uint32_t m, uint32_t c, uint32_t count, const float (&z)[N]) {
        T* p = reinterpret_cast<T*>(to.p) + int64_t(m) * to.ld + c;
        if (c + N <= count) {
            Word v;
#pragma unroll
            for (uint32_t e = 0; e < N; e++) v[e] = T(z[e]);
            if (ONCE)
                __builtin_nontemporal_store(v, reinterpret_cast<Word*>(p));
            else
                *reinterpret_cast<Word*>(p) = v;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < N; e++)
                if (c + e < count) p[e] = T(z[e]);
        }
    }
};

// A wavefront's LDS for pieces of 32 or 64 columns, of both projections and of what is beside them; which fits into `room`.
template <class T, bool N2> constexpr uint32_t piece_bytes(int tiles) {
    return tiles == 2 ? (N2 ? 2 : 1) * Piece<T, 64>::BYTES + Piece<T, 64>::TURNS * 1024 : (N2 ? 2 : 1) * Piece<T, 32>::BYTES + Piece<T, 32>::TURNS * 1024;
}
template <class T, bool N2> constexpr int piece_tiles(int tiles, uint32_t room) { return tiles >= 2 && piece_bytes<T, N2>(2) <= room ? 2 : 1; }

// ---------------------------------------------------------------- the product
// BN counts the rows of LDS: of the gated block's projections, half each.
// PIPED: one wavefront on each SIMD, whose loads and LDS reads go out between
// its own products (there is no other to fill the gaps).
template <class T, int BM, int BN, int WM, int WN, int KB, int STAGES, bool PIPED, bool MC, bool NC, int RESULT>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(BM == 256 ? 1 : KB == 64 ? 3 : 2))) product_kernel(Job a) {
    constexpr int W = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr bool N2 = two_weights(RESULT);
    constexpr int OUT = N2 ? BN / 2 : BN, TO = N2 ? TN / 2 : TN;  // columns of the result, and a wavefront's tiles of them
    static_assert(TM >= 1 && TN >= (N2 ? 2 : 1), "");
    typedef Staged<T, BM, W, KB, MC, false> SideM;
    typedef Staged<T, BN, W, KB, NC, N2> SideN;
    constexpr uint32_t STAGE = SideM::BYTES + SideN::BYTES, STEP = KB / sizeof(T);
    constexpr int KK = KB / 32;
    constexpr int LOADS = SideM::LOADS + SideN::LOADS;
    extern __shared__ __align__(16) char shared[];
    const uint32_t lds = uint32_t(uintptr_t((__attribute__((address_space(3))) char*)shared));

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN;
    // Workgroups go to the 8 XCDs in turn: each gets a run of tiles, n first
    // inside a band of 8 tiles, so that what its L2 holds is used again.
    uint32_t mt, nt;
    {
        const uint32_t tiles = a.m_tiles * a.n_tiles, xcd = blockIdx.x & 7, per = tiles / 8, rest = tiles % 8;
        const uint32_t t = xcd * per + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3);
        const uint32_t band = t / (8 * a.m_tiles), in = t - band * 8 * a.m_tiles;
        const uint32_t wide = a.n_tiles - band * 8 < 8 ? a.n_tiles - band * 8 : 8;
        mt = in / wide;
        nt = band * 8 + in % wide;
    }
    uint32_t k_first = 0, k_end = a.k;
    const uint32_t batch = blockIdx.y / a.splits, piece = blockIdx.y % a.splits;
    if (RESULT == PART || RESULT == STORE) {
        k_first = piece * a.split_k;
        k_end = k_first + a.split_k < a.k ? k_first + a.split_k : a.k;
    }
    SideM sm;
    SideN sn;
    {
        Side m = a.m;
        if ((RESULT == PART || RESULT == STORE) && batch) m.p = a.m.p2;
        sm.init(m, mt * BM, wave, lane);
        sn.init(a.n, nt * OUT, wave, lane);
    }
    const uint32_t steps = (k_end - k_first + STEP - 1) / STEP, total = steps * a.segments;
    uint32_t next = 0, next_k = k_first, into = 0;  // the step to load, its k, its stage
    bool second = false;
    const auto load = [&](int i) {
        const uint32_t to = lds + into * STAGE;
        i < SideM::LOADS ? sm.load(i, to, next_k, wave, second) : sn.load(i - SideM::LOADS, to + SideM::BYTES, next_k, wave, second);
    };
    const auto load_end = [&](int i) {
        const uint32_t to = lds + into * STAGE;
        i < SideM::LOADS ? sm.load_end(i, to, next_k, k_end, wave, second)
                         : sn.load_end(i - SideM::LOADS, to + SideM::BYTES, next_k, k_end, wave, second);
    };
    const auto whole = [&]() { return next_k + STEP <= k_end; };
    const auto loaded = [&]() {
        next++;
        next_k += STEP;
        if (next == steps) {
            next_k = k_first;
            second = true;
        }
        into = into + 1 == STAGES ? 0 : into + 1;
    };
    const auto fetch = [&]() {
        if (whole()) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load(i);
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_end(i);
        }
        loaded();
    };
    const auto past_end = [&]() {
        if (next >= total) next_k = k_end;
    };
    if constexpr (PIPED) {
#pragma unroll
        for (int s = 0; s < STAGES - 1; s++) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load_end(i);
            loaded();
            past_end();
        }
    } else {
        for (int s = 0; s < STAGES - 1; s++)
            if (uint32_t(s) < total) fetch();
    }

    typename SideM::Reader rm;
    typename SideN::Reader rn;
    rm.init(lane);
    rn.init(lane);
    const uint32_t m0 = mt * BM + wm * (BM / WM), n0 = nt * OUT + wn * (OUT / WN);
    const uint32_t mc = a.m.count, nc = a.n.count;
    // sums begin with the bias
    f32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++) {
        f32x16 b;
#pragma unroll
        for (int e = 0; e < 16; e++) b[e] = 0.0f;
        if constexpr (RESULT != STORE && RESULT != PART) {
            const char* from = a.bias[N2 && i >= TO ? 1 : 0];
            if (from)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const f32x4 v = load4<T>(from, n0 + 32 * (i % TO) + 8 * g + 4 * (lane >> 5), nc);
#pragma unroll
                    for (int e = 0; e < 4; e++) b[4 * g + e] = v[e];
                }
        }
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = b;
    }

    constexpr int AHEAD = PIPED ? 2 : 1, READS = TM + TN, MULS = TM * TN;
    Frag<T> fm[AHEAD][TM], fn[AHEAD][TN];
    // Operand i of a quarter of the step in stage `from`.
    const auto read = [&](uint32_t from, int kk, int i) {
        const uint32_t at_m = lds + from * STAGE, at_n = at_m + SideM::BYTES;
        if (i < TN)
            fn[kk % AHEAD][i] = rn.get(at_n, (N2 && i >= TO ? BN / 2 : 0) + wn * (OUT / WN) + 32 * (i % TO), kk);
        else
            fm[kk % AHEAD][i - TN] = rm.get(at_m, wm * (BM / WM) + 32 * (i - TN), kk);
    };
    const auto multiply = [&](int kk, int i) { mma(acc[i / TM][i % TM], fn[kk % AHEAD][i / TM], fm[kk % AHEAD][i % TM]); };
    uint32_t from = 0;
    if constexpr (PIPED) {
        // A step's last place is read while the one before is multiplied, so its
        // stage is free from the barrier before the last place's products on, where
        // the next step has landed too. The step STAGES later is loaded behind the
        // products of half a step from there, where its loads keep the memory pipe
        // busy, and has the other half to arrive in. (8,192 x 4,096 x 8,192 of zeros, which
        // draw little power: a step takes 0.98 us of which the products are 0.85; with
        // loads over a quarter of it 1.14, over three quarters 1.06.) Past the sum's end
        // these are loads of zeros that no one reads, as the last step's reads of a
        // next one are of what was there.
        landed<LOADS*(STAGES - 2)>();
        constexpr int SLOTS = KK / 2 * MULS;  // products that loads go out behind
        const auto load_at = [&](auto whole_steps, int slot) {
#pragma unroll
            for (int l = slot * LOADS / SLOTS; l < (slot + 1) * LOADS / SLOTS; l++) whole_steps() ? load(l) : load_end(l);
        };
#pragma unroll
        for (int i = 0; i < MULS; i++) load_at(std::false_type(), i);
#pragma unroll
        for (int i = 0; i < READS; i++) read(from, 0, i);
        const auto step = [&](auto whole_steps) {
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                if (kk == KK - 1) {
                    loaded();
                    past_end();
                    landed<LOADS*(STAGES - 2)>();
                    from = from + 1 == STAGES ? 0 : from + 1;
                }
#pragma unroll
                for (int i = 0; i < MULS; i++) {
                    multiply(kk, i);
                    if (i < READS) read(from, (kk + 1) % KK, i);
                    if ((kk + 1) % KK * MULS < SLOTS) load_at(whole_steps, (kk + 1) % KK * MULS + i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        // the steps whose loads, of the two steps after them, are whole
        static_assert(STAGES == 2, "");
        const uint32_t full = (k_end - k_first) / STEP, ahead = full == steps ? total : full;
        const uint32_t fast = ahead > 2 ? ahead - 2 : 0;
        uint32_t s = 0;
        for (; s < fast; s++) step(std::true_type());
        for (; s < total; s++) step(std::false_type());
        landed<0>();
    } else {
        for (uint32_t s = 0; s < total; s++) {
            // this step's words are there for all, and all have read the step before it
            if (STAGES > 2 && s + STAGES - 2 < total)
                landed<LOADS*(STAGES - 2)>();
            else
                landed<0>();
            if (next < total) fetch();
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
#pragma unroll
                for (int i = 0; i < READS; i++) read(from, kk, i);
#pragma unroll
                for (int i = 0; i < MULS; i++) multiply(kk, i);
            }
            from = from + 1 == STAGES ? 0 : from + 1;
        }
        landed<0>();
    }

    // ---- the result, PW columns of 32 rows at a time
    typedef typename std::conditional<RESULT == PART, float, T>::type TR;
    constexpr int PT = piece_tiles<TR, N2>(TO, STAGES * STAGE / W), PW = 32 * PT;
    constexpr uint32_t REGION = piece_bytes<TR, N2>(PT);
    typedef Piece<TR, PW> Out;
    constexpr uint32_t N = Out::N;
    constexpr bool SLOPES = RESULT == SLOPE || RESULT == GATED_SLOPE;
    // (With gelu 32,768 x 2,560 to 5,120, gated: 1,387 us, and 1,458 with y by way of the caches; its slopes 1,512, and
    // 1,635 with dy and dz by way of them.  With silu 1,345 and 1,442; a quarter of the rows 346 and 355, with all
    // gradients 1,564 and 1,547; 14,374 x 203 to 3,935 123 and 127; 49,596 x 304 to 66 22 either way.)
    constexpr bool ONCE = BM == 256 && RESULT != STORE && RESULT != PART;
    constexpr uint32_t BESIDE = (N2 ? 2 : 1) * Out::BYTES;
    char* own = shared + wave * REGION;
    Matrix y = (RESULT == STORE || RESULT == PART) && batch ? a.y2 : a.y;
    if (RESULT == PART) y.p += uint64_t(piece) * mc * y.ld * 4;
    Matrix dz2 = a.dz;
    dz2.p += uint64_t(a.dz_half) * sizeof(T);
    // What is beside a piece, the residual or the gradient of y, is loaded while
    // the piece before it is worked on, and waits in LDS.
    const bool beside = SLOPES || (RESULT == LINEAR && a.residual.p);
    const bool as_is = RESULT == STORE || RESULT == PART || (RESULT == LINEAR && a.act == MDN_ACT_NONE && !beside);
    const Matrix side = RESULT == LINEAR ? a.residual : a.dy;
    typename Out::LdsWord words[Out::TURNS];
    const auto load_beside = [&](int i0, int j) {
        const uint32_t n = n0 + 32 * i0 + Out::column(lane);
#pragma unroll
        for (uint32_t t = 0; t < Out::TURNS; t++) {
            const uint32_t m = m0 + 32 * j + Out::row(lane, t);
            if (m < mc) words[t] = Out::template load<BM == 256>(side, m, n, nc);
        }
    };
    if (beside) load_beside(0, 0);
#pragma unroll
    for (int i0 = 0; i0 < TO; i0 += PT) {
        const uint32_t n = n0 + 32 * i0 + Out::column(lane);
        float sum[SLOPES ? 2 : 1][N] = {};
        const bool whole = n0 + 32 * i0 + PW <= nc;
#pragma unroll
        for (int j = 0; j < TM; j++) {
            Out::order();
#pragma unroll
            for (int i = 0; i < PT; i++) {
                Out::put(own, acc[i0 + i][j], i, lane);
                if constexpr (N2) Out::put(own + Out::BYTES, acc[TO + i0 + i][j], i, lane);
            }
            if (beside) {
#pragma unroll
                for (uint32_t t = 0; t < Out::TURNS; t++)
                    *reinterpret_cast<typename Out::LdsWord*>(own + BESIDE + t * 1024 + lane * 16) = words[t];
                if (j + 1 < TM)
                    load_beside(i0, j + 1);
                else if (i0 + PT < TO)
                    load_beside(i0 + PT, 0);
            }
            Out::order();
            if (as_is) {
                float z[Out::TURNS][N];
#pragma unroll
                for (uint32_t t = 0; t < Out::TURNS; t++) Out::get(own, Out::row(lane, t), lane, z[t]);
#pragma unroll
                for (uint32_t t = 0; t < Out::TURNS; t++)
                    if (m0 + 32 * j + Out::row(lane, t) < mc) Out::template store<ONCE>(y, m0 + 32 * j + Out::row(lane, t), n, nc, z[t]);
                continue;
            }
            // (not unrolled, the activations would fill the instruction cache; the next turn's values are read ahead)
            float z_next[N], up_next[N];
            Out::get(own, Out::row(lane, 0), lane, z_next);
            if constexpr (N2) Out::get(own + Out::BYTES, Out::row(lane, 0), lane, up_next);
#pragma unroll 1
            for (uint32_t t = 0; t < Out::TURNS; t++) {
                const uint32_t m = m0 + 32 * j + Out::row(lane, t);
                float z[N], up[N], with[N];
#pragma unroll
                for (uint32_t e = 0; e < N; e++) {
                    z[e] = z_next[e];
                    if constexpr (N2) up[e] = up_next[e];
                }
                const uint32_t ahead = t + 1 < Out::TURNS ? t + 1 : t;
                Out::get(own, Out::row(lane, ahead), lane, z_next);
                if constexpr (N2) Out::get(own + Out::BYTES, Out::row(lane, ahead), lane, up_next);
                if (beside) {
                    const auto word = *reinterpret_cast<const typename Out::LdsWord*>(own + BESIDE + t * 1024 + lane * 16);
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) with[e] = float(word[e]);
                }
                if (m >= mc) continue;
                if constexpr (RESULT == LINEAR) {
                    act_of<T>(a.act, z);
                    if (beside)
#pragma unroll
                        for (uint32_t e = 0; e < N; e++) z[e] += with[e];
                }
                if constexpr (RESULT == GATED) {
                    act_of<T>(a.act, z);
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) z[e] *= up[e];
                }
                if constexpr (SLOPES) {
                    float slope[N];
                    act_of<T>(a.act, z, slope);
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) {
                        if constexpr (N2) {
                            slope[e] *= up[e];
                            up[e] = with[e] * z[e];
                        }
                        z[e] = with[e] * slope[e];
                    }
                    if (!whole) {  // zeros past the last column, also where z is none: the next products read whole words
#pragma unroll
                        for (uint32_t e = 0; e < N; e++) {
                            z[e] = n + e < nc ? z[e] : 0.0f;
                            if constexpr (N2) up[e] = n + e < nc ? up[e] : 0.0f;
                        }
                    }
                    if (a.sums) {
#pragma unroll
                        for (uint32_t e = 0; e < N; e++) {
                            sum[0][e] += z[e];
                            if constexpr (N2) sum[1][e] += up[e];
                        }
                    }
                    Out::template store<ONCE>(a.dz, m, n, a.dz_half, z);
                    if constexpr (N2) Out::template store<ONCE>(dz2, m, n, a.dz_half, up);
                } else
                    Out::template store<ONCE>(y, m, n, nc, z);
            }
        }
        if constexpr (SLOPES) {
            if (a.sums) {
                float* to = a.sums + uint64_t(mt * WM + wm) * 2 * nc + n;
#pragma unroll
                for (int half = 0; half < (N2 ? 2 : 1); half++)
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) {
                        float v = sum[half][e];
#pragma unroll
                        for (uint32_t l = Out::LANES; l < 64; l *= 2) v += __shfl_xor(v, l);
                        if (lane < Out::LANES && n + e < nc) to[uint64_t(half) * nc + e] = v;
                    }
            }
        }
    }
}

// ---------------------------------------------------------------- what is left
// Rows with words of their own: row r of `to` (ld elements, a multiple of a
// word's) is row r of `from`, zeros behind it.  I: an index that all words fit.
template <class T, class I>
__global__ void __launch_bounds__(256) lay_out_kernel(Matrix from, Matrix to, I all, uint32_t width) {
    constexpr uint32_t N = per_word<T>();
    typedef T Word __attribute__((ext_vector_type(N)));
    typedef T AnyWord __attribute__((ext_vector_type(N), aligned(sizeof(T))));  // at any multiple of an element
    const I words = I(to.ld) / N, step = I(gridDim.x) * 256;
    for (I i = I(blockIdx.x) * 256 + threadIdx.x; i < all; i += step) {
        const I row = i / words;
        const uint32_t c = uint32_t(i - row * words) * N;
        const T* src = reinterpret_cast<const T*>(from.p) + int64_t(row) * from.ld + c;
        Word v;
        if (c + N <= width) {
            v = *reinterpret_cast<const AnyWord*>(src);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < N; e++) v[e] = c + e < width ? src[e] : T(0.0f);
        }
        *reinterpret_cast<Word*>(reinterpret_cast<T*>(to.p) + int64_t(row) * to.ld + c) = v;
    }
}

// Zeros in a matrix of `width` columns.
template <class T>
__global__ void __launch_bounds__(256) clear_kernel(Matrix to, uint64_t rows, uint32_t width) {
    const uint64_t all = rows * width;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += uint64_t(gridDim.x) * 256)
        reinterpret_cast<T*>(to.p)[int64_t(i / width) * to.ld + int64_t(i % width)] = T(0.0f);
}

// Adds up the parts of a product, in order: to[r][c] = sum of from[s][r][c]; blockIdx.y: of which of two products.
template <class T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* from, uint32_t parts, Matrix to0, Matrix to1, uint32_t rows, uint32_t width) {
    const Matrix to = blockIdx.y ? to1 : to0;
    const uint64_t all = uint64_t(rows) * width;
    from += blockIdx.y * parts * all;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < all; i += uint64_t(gridDim.x) * 256) {
        float v = 0.0f;
        for (uint32_t s = 0; s < parts; s++) v += from[s * all + i];
        const uint64_t row = i / width;
        reinterpret_cast<T*>(to.p)[int64_t(row) * to.ld + int64_t(i - row * width)] = T(v);
    }
}

// Column sums of rows, in two steps: blockIdx.y's share of the rows to a row
// of sums, 64 columns a workgroup, a quarter of the share a wavefront.
template <class T>
__global__ void __launch_bounds__(256) column_sums_kernel(Matrix from, uint64_t rows, uint32_t width, uint64_t share, float* sums) {
    __shared__ float part[4][64];
    const uint32_t c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    const uint64_t first = blockIdx.y * share, end = first + share < rows ? first + share : rows;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < width) {
        const T* p = reinterpret_cast<const T*>(from.p) + c;
        uint64_t r = first + slice;
        for (; r + 12 < end; r += 16)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += float(p[int64_t(r + 4 * i) * from.ld]);
        for (; r < end; r += 4) v[0] += float(p[int64_t(r) * from.ld]);
    }
    part[slice][threadIdx.x & 63] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (slice == 0 && c < width)
        sums[uint64_t(blockIdx.y) * width + c] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
}
// Rows of sums, `pitch` apart, to one vector or two (blockIdx.y; null: none): 64 columns a workgroup, a sixteenth of the
// rows a wavefront.
template <class T>
__global__ void __launch_bounds__(1024) add_sums_kernel(const float* sums, uint32_t count, uint64_t pitch, uint32_t width, char* to0, char* to1) {
    __shared__ float part[16][64];
    char* to = blockIdx.y ? to1 : to0;
    if (!to) return;
    sums += blockIdx.y * width;
    const uint32_t c = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < width) {
        uint32_t i = slice;
        for (; i + 48 < count; i += 64)
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += sums[uint64_t(i + 16 * j) * pitch + c];
        for (; i < count; i += 16) v[0] += sums[uint64_t(i) * pitch + c];
    }
    part[slice][threadIdx.x & 63] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (slice != 0 || c >= width) return;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += part[i][threadIdx.x];
    reinterpret_cast<T*>(to)[c] = T(s);
}

// ---------------------------------------------------------------- launches
uint32_t blocks_for(uint64_t items, uint32_t per, uint32_t most) {
    const uint64_t n = (items + per - 1) / per;
    return uint32_t(n < most ? (n ? n : 1) : most);
}

constexpr uint64_t MOST_TILES = 0xffffffffull / 256;  // a launch has below 2^32 threads

template <class T, int BM, int BN, int WM, int WN, int KB, int STAGES, bool PIPED, bool MC, bool NC, int RESULT>
hipError_t launch(Job a, uint32_t batches, hipStream_t st) {
    constexpr bool N2 = two_weights(RESULT);
    typedef typename std::conditional<RESULT == PART, float, T>::type TR;
    constexpr uint32_t OUT = N2 ? BN / 2 : BN, stages = STAGES * (BM + BN) * KB, room = stages / (WM * WN);
    constexpr uint32_t pieces = WM * WN * piece_bytes<TR, N2>(piece_tiles<TR, N2>(OUT / WN / 32, room)), bytes = pieces > stages ? pieces : stages;
    static_assert(bytes <= 160 * 1024, "");
    a.m_tiles = (a.m.count + BM - 1) / BM;
    a.n_tiles = (a.n.count + OUT - 1) / OUT;
    if (uint64_t(a.m_tiles) * a.n_tiles > MOST_TILES) return hipErrorInvalidConfiguration;
    const auto kernel = product_kernel<T, BM, BN, WM, WN, KB, STAGES, PIPED, MC, NC, RESULT>;
    if (bytes > 64 * 1024)
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)))
            return e;
    kernel<<<dim3(a.m_tiles * a.n_tiles, batches * a.splits), dim3(64 * WM * WN), bytes, st>>>(a);
    return hipGetLastError();
}

// The tile of a product: the one of the least estimated time.  A compute unit
// takes one large tile at a time and two of the others; measured, in us: a step
// of 128 bytes of k alone on a compute unit and beside another tile, and what a
// tile takes besides (1,024 x 2,048 x 2,048 in bfloat16: 18, 27 and 51 us on small,
// middle and large tiles; 4,096 x 2,048 x 2,048: 58, 42 and 53; 32,768 x 5,120 to 1,280:
// 775, 506 and 404; 262,144 x 256 to 1,024 with silu: 511, 316 and 360).  Large ones are
// for bfloat16: in fp32 a step took 8.2 us, as the four middle tiles in its place do, and
// the rest 20 where theirs is 12, so by this no size gains by them.  Middle ones have one
// set of numbers for both of their kernels (short_sum).
enum Tile { SMALL, MIDDLE, LARGE };
constexpr uint32_t UNITS = 256;
struct Cost { uint32_t m, n; float alone, beside, rest; };
enum Kind { PLAIN, SHAPED, TWO };  // sums alone, with an epilogue, of both projections of a gated block
Cost cost_of(Tile t, bool bf, Kind kind) {
    const bool two = kind == TWO, plain = kind == PLAIN;
    switch (t) {
        case SMALL: return {64, 64, (bf ? 0.40f : 0.55f) * (two ? 1.6f : 1.0f), (bf ? 0.48f : 1.02f) * (two ? 1.8f : 1.0f), bf ? (two ? 2.2f : 1.8f) : 5.0f};
        case MIDDLE: return {128, two ? 64u : 128u, bf ? 0.72f : 2.1f, bf ? (two ? 1.05f : 1.15f) : 4.1f, bf ? (two ? 3.4f : plain ? 3.0f : 4.4f) : (two ? 2.0f : 6.0f)};
        default: return {256, two ? 128u : 256u, 1.55f, 3.1f, plain || two ? 9.0f : 15.0f};
    }
}
float time_of(Tile t, bool bf, Kind kind, uint64_t m, uint64_t n, uint64_t k, uint64_t times) {
    const Cost c = cost_of(t, bf, kind);
    const uint64_t tiles = (m + c.m - 1) / c.m * ((n + c.n - 1) / c.n) * times, each = (tiles + UNITS - 1) / UNITS;
    if (tiles > MOST_TILES || (t == LARGE && !bf)) return 1e30f;
    const float steps = float((k * (bf ? 2 : 4) + 127) / 128), rest = t == LARGE ? 2.0f * c.rest : c.rest;
    return float(each / 2) * (steps * c.beside + rest) + (each & 1 ? steps * c.alone + c.rest : 0.0f);
}
Tile tile_of(bool bf, Kind kind, uint64_t m, uint64_t n, uint64_t k) {
    Tile best = SMALL;
    for (Tile t : {MIDDLE, LARGE})
        if (time_of(t, bf, kind, m, n, k, 1) < time_of(best, bf, kind, m, n, k, 1)) best = t;
    return best;
}

// Of products of rows by rows. Where there are more than two middle tiles a compute unit and few
// steps, three tiles at once with half the LDS. In bfloat16, 131,072 rows to 1,024, gated: of 64
// 109 us, and 130 with two; of 256 211 and 245; of 512 334 and 333; not gated: 114 and 100, 166 and 168,
// 221 and 236. In fp32, 65,536 rows to 512: of 64 66 and 72, of 256 153 and 161, of 512, past the limit, 271
// and 281. Long sums are slower: 32,768 of 2,560 to 5,120, gated, in bfloat16: 2,207 and 1,743.
bool short_sum(uint64_t m, uint64_t n, uint64_t bytes, bool two) {
    const uint64_t out = two ? 64 : 128;
    return bytes <= 1024 && (m + 127) / 128 * ((n + out - 1) / out) > 2 * UNITS;
}

template <class T, bool MC, bool NC, int RESULT>
hipError_t product(const Job& a, Tile tile, uint32_t batches, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (tile == LARGE) return launch<T, 256, 256, 2, 2, 128, 2, true, MC, NC, RESULT>(a, batches, st);
    if constexpr (!MC && !NC)
        if (tile == MIDDLE && short_sum(a.m.count, a.n.count, a.k * sizeof(T), two_weights(RESULT)))
            return launch<T, 128, 128, 2, 2, 64, 2, false, MC, NC, RESULT>(a, batches, st);
    if (tile == MIDDLE) return launch<T, 128, 128, 2, 2, 128, 2, false, MC, NC, RESULT>(a, batches, st);
    if constexpr (two_weights(RESULT))
        return launch<T, 64, 128, 2, 2, 128, 3, false, MC, NC, RESULT>(a, batches, st);
    else
        return launch<T, 64, 64, 2, 2, 128, 4, false, MC, NC, RESULT>(a, batches, st);
}

// ---- memory
constexpr uint64_t ALIGN = 256;
uint64_t aligned(uint64_t bytes) { return (bytes + ALIGN - 1) / ALIGN * ALIGN; }

// A matrix whose rows move in 16-byte words as they are.
bool in_words(const Matrix& m, uint32_t width, uint32_t size) {
    return width % (16 / size) == 0 && m.ld >= 0 && m.ld <= int64_t((1u << 22) / size) && (m.ld * size) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(m.p) % 16 == 0;
}
uint32_t pieces_of(const Args& a) { return a.gated ? 2 : 1; }
uint32_t words_of(uint32_t width, uint32_t size) { return (width + 16 / size - 1) / (16 / size) * (16 / size); }

// Where the operands of a call's products lie: as they are, or copied.
struct Plan {
    uint32_t size, in_ld, out_ld;  // widths in whole words
    bool x_copy, w_copy;
    uint64_t x_bytes, w_bytes;     // w_bytes: of one of the weights
    Tile forward_tile;
};
Plan plan_of(const Args& a) {
    Plan p{};
    p.size = a.bf ? 2 : 4;
    p.in_ld = words_of(a.in, p.size);
    p.out_ld = words_of(a.out, p.size);
    p.x_copy = !in_words(a.x, a.in, p.size);
    p.w_copy = !in_words(a.w[0], a.in, p.size) || (a.gated && (!in_words(a.w[1], a.in, p.size) || a.w[1].ld != a.w[0].ld));
    p.x_bytes = p.x_copy ? aligned(a.rows * p.in_ld * p.size) : 0;
    p.w_bytes = p.w_copy ? aligned(uint64_t(a.out) * p.in_ld * p.size) : 0;
    p.forward_tile = tile_of(a.bf, a.gated ? TWO : SHAPED, a.rows, a.out, a.in);
    return p;
}
// Of the backward pass.
constexpr uint32_t SHARES = 256;  // of rows, in column sums
struct BackPlan : Plan {
    bool slope, dz_copy, w_needed, x_needed;
    uint64_t dz_bytes, sums_bytes, parts_bytes;
    uint32_t sum_rows, splits, split_k;
    Tile dx_tile, dw_tile;
};
BackPlan back_plan_of(const Args& a, const GradArgs& d) {
    BackPlan p{};
    static_cast<Plan&>(p) = plan_of(a);
    const uint32_t pieces = pieces_of(a);
    p.slope = a.gated || a.activation != MDN_ACT_NONE;
    const bool dw = d.d_w[0].p || d.d_w[1].p, dx = d.d_x.p, db = d.d_b[0] || d.d_b[1];
    p.x_needed = p.slope || dw;
    p.w_needed = p.slope || dx;
    if (!p.x_needed) p.x_copy = false, p.x_bytes = 0;
    if (!p.w_needed) p.w_copy = false, p.w_bytes = 0;
    p.dz_copy = !p.slope && (dx || dw) && !in_words(d.d_y, a.out, p.size);
    p.dz_bytes = p.slope || p.dz_copy ? aligned(a.rows * pieces * p.out_ld * p.size) : 0;
    if (p.slope) {
        const uint32_t bm = p.forward_tile == LARGE ? 256 : p.forward_tile == MIDDLE ? 128 : 64;
        p.sum_rows = uint32_t((a.rows + bm - 1) / bm) * 2;
    } else
        p.sum_rows = uint32_t(a.rows < 16 * SHARES ? (a.rows + 15) / 16 : SHARES);
    p.sums_bytes = db ? aligned(uint64_t(p.sum_rows) * 2 * a.out * 4) : 0;
    p.dx_tile = tile_of(a.bf, PLAIN, a.rows, a.in, uint64_t(a.out) * pieces);
    // dW has few results and a long sum, which is cut into pieces of at least 256
    // rows: as many as are worth the 4.5 TB/s at which their fp32 results are
    // written and added up.
    float least = 0.0f;
    uint32_t rows = 0;
    const uint64_t most = (a.rows + 255) / 256;
    for (uint32_t splits = 1; splits <= (most < 64 ? most : 64); splits++) {
        const uint32_t k = uint32_t((a.rows + splits - 1) / splits + 63) / 64 * 64;
        const float parts = splits == 1 ? 0.0f : 5.0f + float(splits) * float(a.out) * float(a.in) * float(pieces) * 8.0f / 4.5e6f;
        for (Tile t : {SMALL, MIDDLE, LARGE}) {
            const float time = time_of(t, a.bf, PLAIN, a.out, a.in, k, uint64_t(pieces) * splits) + parts;
            if (rows == 0 || time < least) least = time, rows = k, p.dw_tile = t;
        }
    }
    p.split_k = rows;
    p.splits = uint32_t((a.rows + rows - 1) / rows);
    p.parts_bytes = dw && p.splits > 1 ? aligned(uint64_t(pieces) * p.splits * a.out * a.in * 4) : 0;
    return p;
}

template <class T> hipError_t lay_out(const Matrix& from, const Matrix& to, uint64_t rows, uint32_t width, hipStream_t st) {
    const uint64_t words = rows * (to.ld / per_word<T>());
    const dim3 grid(blocks_for(words, 256, 16384));
    if (words < (1ull << 31))
        lay_out_kernel<T, uint32_t><<<grid, dim3(256), 0, st>>>(from, to, uint32_t(words), width);
    else
        lay_out_kernel<T, uint64_t><<<grid, dim3(256), 0, st>>>(from, to, words, width);
    return hipGetLastError();
}
// x and the weights in words; copies go to `work`, which is advanced.
template <class T> hipError_t operands(Args& a, const Plan& p, char*& work, hipStream_t st) {
    if (p.x_copy) {
        const Matrix to{work, p.in_ld};
        if (hipError_t e = lay_out<T>(a.x, to, a.rows, a.in, st)) return e;
        a.x = to;
        work += p.x_bytes;
    }
    if (p.w_copy)
        for (uint32_t i = 0; i < pieces_of(a); i++) {
            const Matrix to{work, p.in_ld};
            if (hipError_t e = lay_out<T>(a.w[i], to, a.out, a.in, st)) return e;
            a.w[i] = to;
            work += p.w_bytes;
        }
    return hipSuccess;
}
Side side(const Matrix& m, const char* second, uint64_t count, uint32_t size) {
    return {m.p, second, m.ld * int64_t(size), uint32_t(count)};
}
Job forward_job(const Args& a, const Plan& p) {
    Job j{};
    j.m = side(a.x, nullptr, a.rows, p.size);
    j.n = side(a.w[0], a.w[1].p, a.out, p.size);
    j.k = p.in_ld;
    j.segments = j.splits = 1;
    j.split_k = j.k;
    j.act = a.activation;
    j.y = a.y;
    j.residual = a.residual;
    j.bias[0] = a.b[0];
    j.bias[1] = a.b[1];
    return j;
}

template <class T> hipError_t forward_of(Args a, char* work, hipStream_t st) {
    const Plan p = plan_of(a);
    if (hipError_t e = operands<T>(a, p, work, st)) return e;
    const Job j = forward_job(a, p);
    return a.gated ? product<T, false, false, GATED>(j, p.forward_tile, 1, st) : product<T, false, false, LINEAR>(j, p.forward_tile, 1, st);
}

template <class T> hipError_t add_sums(const float* sums, uint32_t count, uint64_t pitch, uint32_t width, char* const (&to)[2], hipStream_t st) {
    add_sums_kernel<T><<<dim3((width + 63) / 64, to[1] ? 2 : 1), dim3(1024), 0, st>>>(sums, count, pitch, width, to[0], to[1]);
    return hipGetLastError();
}

// The gradients of no rows.
template <class T> hipError_t clear(const Args& a, const GradArgs& d, hipStream_t st) {
    for (uint32_t i = 0; i < pieces_of(a); i++) {
        if (d.d_w[i].p)
            clear_kernel<T><<<dim3(blocks_for(uint64_t(a.out) * a.in, 256, 4096)), dim3(256), 0, st>>>(d.d_w[i], a.out, a.in);
        if (d.d_b[i]) clear_kernel<T><<<dim3(blocks_for(a.out, 256, 4096)), dim3(256), 0, st>>>(Matrix{d.d_b[i], a.out}, 1, a.out);
    }
    return hipGetLastError();
}

template <class T> hipError_t backward_of(Args a, const GradArgs& d, char* work, hipStream_t st) {
    if (a.rows == 0) return clear<T>(a, d, st);
    const BackPlan p = back_plan_of(a, d);
    const uint32_t pieces = pieces_of(a);
    if (hipError_t e = operands<T>(a, p, work, st)) return e;
    Matrix dz = d.d_y;
    if (p.dz_bytes) {
        dz = Matrix{work, int64_t(pieces) * p.out_ld};
        work += p.dz_bytes;
    }
    float* sums = p.sums_bytes ? reinterpret_cast<float*>(work) : nullptr;
    work += p.sums_bytes;
    if (p.slope) {
        Job j = forward_job(a, p);
        j.dy = d.d_y;
        j.dz = dz;
        j.dz_half = p.out_ld;
        j.sums = sums;
        if (hipError_t e = a.gated ? product<T, false, false, GATED_SLOPE>(j, p.forward_tile, 1, st)
                                   : product<T, false, false, SLOPE>(j, p.forward_tile, 1, st))
            return e;
        if (sums)
            if (hipError_t e = add_sums<T>(sums, p.sum_rows, 2 * uint64_t(a.out), a.out, d.d_b, st)) return e;
    } else {
        if (p.dz_copy)
            if (hipError_t e = lay_out<T>(d.d_y, dz, a.rows, a.out, st)) return e;
        if (d.d_b[0]) {
            const uint64_t share = (a.rows + p.sum_rows - 1) / p.sum_rows;
            column_sums_kernel<T><<<dim3((a.out + 63) / 64, p.sum_rows), dim3(256), 0, st>>>(d.d_y, a.rows, a.out, share, sums);
            if (hipError_t e = hipGetLastError()) return e;
            if (hipError_t e = add_sums<T>(sums, p.sum_rows, a.out, a.out, d.d_b, st)) return e;
        }
    }
    const char* dz2 = dz.p + uint64_t(p.out_ld) * p.size;
    if (d.d_x.p) {
        Job j{};
        j.m = side(dz, dz2, a.rows, p.size);
        j.n = side(a.w[0], a.w[1].p, a.in, p.size);
        j.k = j.split_k = a.out;
        j.segments = pieces;
        j.splits = 1;
        j.y = d.d_x;
        if (hipError_t e = product<T, false, true, STORE>(j, p.dx_tile, 1, st)) return e;
    }
    if (d.d_w[0].p || d.d_w[1].p) {
        Job j{};
        const bool both = d.d_w[0].p && d.d_w[1].p;
        const uint32_t first = d.d_w[0].p ? 0 : 1;
        j.m = side(dz, dz2, a.out, p.size);
        if (first) j.m.p = dz2;
        j.n = side(a.x, nullptr, a.in, p.size);
        j.k = uint32_t(a.rows);
        j.segments = 1;
        j.splits = p.splits;
        j.split_k = p.split_k;
        j.y = d.d_w[first];
        j.y2 = d.d_w[1];
        if (p.splits == 1) return product<T, true, true, STORE>(j, p.dw_tile, both ? 2 : 1, st);
        float* parts = reinterpret_cast<float*>(work);
        const uint64_t all = uint64_t(a.out) * a.in;
        j.y = Matrix{reinterpret_cast<char*>(parts), a.in};
        j.y2 = Matrix{reinterpret_cast<char*>(parts + p.splits * all), a.in};
        if (hipError_t e = product<T, true, true, PART>(j, p.dw_tile, both ? 2 : 1, st)) return e;
        add_parts_kernel<T><<<dim3(blocks_for(all, 256, 4096), both ? 2 : 1), dim3(256), 0, st>>>(parts, p.splits, d.d_w[first], d.d_w[1],
                                                                                                  a.out, a.in);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

uint64_t forward_bytes(const Args& a) {
    if (few_rows(a)) return 0;
    const Plan p = plan_of(a);
    return p.x_bytes + pieces_of(a) * p.w_bytes;
}
uint64_t backward_bytes(const Args& a, const GradArgs& d) {
    const BackPlan p = back_plan_of(a, d);
    return p.x_bytes + pieces_of(a) * p.w_bytes + p.dz_bytes + p.sums_bytes + p.parts_bytes;
}
void choices(const Args& a, const GradArgs* d, Choice (&to)[4]) {
    for (Choice& c : to) c = Choice{0, 0, 0};
    if (a.rows == 0) return;
    const auto choice = [](Tile t, uint32_t parts) { return Choice{t == LARGE ? 256u : t == MIDDLE ? 128u : 64u, 128, parts}; };
    const auto forward = [&](const Plan& p) {
        Choice c = choice(p.forward_tile, 1);
        if (p.forward_tile == MIDDLE && short_sum(a.rows, a.out, uint64_t(p.in_ld) * p.size, a.gated)) c.step = 64;
        return c;
    };
    if (!few_rows(a)) to[0] = forward(plan_of(a));
    if (!d) return;
    const BackPlan p = back_plan_of(a, *d);
    if (p.slope) to[1] = forward(p);
    if (d->d_x.p) to[2] = choice(p.dx_tile, 1);
    if (d->d_w[0].p || d->d_w[1].p) to[3] = choice(p.dw_tile, p.splits);
}
hipError_t forward(const Args& a, char* work, hipStream_t st) {
    if (few_rows(a)) return forward_few(a, st);
    return a.bf ? forward_of<bf16>(a, work, st) : forward_of<float>(a, work, st);
}
hipError_t backward(const Args& a, const GradArgs& d, char* work, hipStream_t st) {
    return a.bf ? backward_of<bf16>(a, d, work, st) : backward_of<float>(a, d, work, st);
}

}  // namespace dense
