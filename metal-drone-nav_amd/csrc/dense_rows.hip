// dense_rows.hip — the forward call of few rows: a tick of a few vehicles, whose
// cost is reading the weights.
//
// A workgroup makes up to 16 columns of the result for up to 16 MT rows.  Its W
// wavefronts take turns along k, 128 bytes of each of the weight rows at a time
// (whole lines, straight to registers, UNROLL of them on their way), as operands
// of 16 x 16 tiles; their sums meet in LDS.  The weights are read once for every 32
// rows.  Bound by memory: one row of 5,120 to 65,536 in bfloat16 reads its weights at
// 5.4 TB/s.
#include "dense.h"

#include "dense_tiles.h"
#include "dense_act.h"

namespace dense {
namespace {

template <class T> constexpr uint32_t step_of() { return 128 / sizeof(T); }  // k of a turn
template <class T> struct Word;
template <> struct Word<bf16> { typedef bf16x8 type; };
template <> struct Word<float> { typedef f32x4 type; };

__device__ __forceinline__ void mma16(f32x4& acc, const bf16x8& a, const bf16x8& b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4& acc, const f32x4& a, const f32x4& b) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
}

// One word of a row; places past its end are 0.
template <class T, bool WORDS> __device__ __forceinline__ typename Word<T>::type word_at(const T* row, uint32_t k, uint32_t width) {
    typedef typename Word<T>::type V;
    V v;
#pragma unroll
    for (uint32_t i = 0; i < per_word<T>(); i++) v[i] = T(0.0f);
    if (WORDS) {
        if (k < width) v = *reinterpret_cast<const V*>(row + k);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < per_word<T>(); i++)
            if (k + i < width) v[i] = row[k + i];
    }
    return v;
}

template <class T, int MT, int W, bool G, bool WORDS>
__global__ void __launch_bounds__(64 * W) rows_kernel(Args a, uint32_t columns) {
    constexpr int N = G ? 2 : 1, UNROLL = WORDS ? (MT * N <= 2 ? 4 : 2) : 1;
    __shared__ f32x4 part[W][N * MT][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * columns, m0 = blockIdx.y * 16 * MT, rows = uint32_t(a.rows);
    const uint32_t n_end = n0 + columns < a.out ? n0 + columns : a.out;
    const T *w[N], *x[MT];
    const uint32_t n = n0 + (lane & 15) < n_end ? n0 + (lane & 15) : n_end - 1;
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = reinterpret_cast<const T*>(a.w[i].p) + int64_t(n) * a.w[i].ld;
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const uint32_t m = m0 + 16 * j + (lane & 15);
        x[j] = reinterpret_cast<const T*>(a.x.p) + int64_t(m < rows ? m : rows - 1) * a.x.ld;
    }
    f32x4 acc[N][MT];
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t step = step_of<T>(), at = (lane >> 4) * per_word<T>();
    for (uint32_t k = wave * step; k < a.in; k += W * step * UNROLL) {
        typename Word<T>::type fw[UNROLL][2][N], fx[UNROLL][2][MT];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t c = k + u * W * step + h * (step / 2) + at;
#pragma unroll
                for (int i = 0; i < N; i++) fw[u][h][i] = word_at<T, WORDS>(w[i], c, a.in);
#pragma unroll
                for (int j = 0; j < MT; j++) fx[u][h][j] = word_at<T, WORDS>(x[j], c, a.in);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < MT; j++) mma16(acc[i][j], fw[u][h][i], fx[u][h][j]);
    }
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    // a wavefront sums up and finishes every W-th tile of 16 rows
    for (int j = wave; j < MT; j += W) {
        f32x4 z[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            z[i] = part[0][i * MT + j][lane];
#pragma unroll
            for (int s = 1; s < W; s++) z[i] += part[s][i * MT + j][lane];
        }
        const uint32_t m = m0 + 16 * j + (lane & 15), c = n0 + 4 * (lane >> 4);
        if (m >= rows || c >= n_end) continue;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (a.b[i]) z[i] += load4<T>(a.b[i], c, n_end);
        float act[4] = {z[0][0], z[0][1], z[0][2], z[0][3]};
        act_of<T>(a.activation, act);
        f32x4 v = {act[0], act[1], act[2], act[3]};
        if constexpr (G) v = v * z[1];
        if (!G && a.residual.p) v = load4<T>(row_of<T>(a.residual, m), c, n_end) + v;
        store4<T>(row_of<T>(a.y, m), c, n_end, v);
    }
}

// Columns of a workgroup, so that the compute units have the same to read: a
// weight's row each, and the rows of x, which come from the L2, at a third.  (1 row of
// 5,120 to 5,120 in bfloat16: 13.6 us with 10, and 17 with 16, which is 320
// workgroups on 256 units; 24 rows of 5,120 to 1,280: 13.3 with 5 and 17.5 with 16.)
uint32_t columns_of(const Args& a) {
    uint32_t best = 16;
    const auto cost = [&](uint32_t c) { return ((a.out + c - 1) / c + 255) / 256 * (float(c) + 0.33f * float(a.rows)); };
    for (uint32_t c = 15; c >= 1; c--)
        if (cost(c) < 0.95f * cost(best)) best = c;
    return best;
}
template <class T, int MT, int W, bool G> hipError_t launch(const Args& a, bool words, hipStream_t st) {
    const uint32_t columns = columns_of(a);
    const dim3 grid((a.out + columns - 1) / columns, uint32_t((a.rows + 16 * MT - 1) / (16 * MT)));
    if (words)
        rows_kernel<T, MT, W, G, true><<<grid, dim3(64 * W), 0, st>>>(a, columns);
    else
        rows_kernel<T, MT, W, G, false><<<grid, dim3(64 * W), 0, st>>>(a, columns);
    return hipGetLastError();
}
template <class T, int MT, bool G> hipError_t by_waves(const Args& a, bool words, hipStream_t st) {
    const uint32_t steps = (a.in + step_of<T>() - 1) / step_of<T>();
    if (steps <= 4) return launch<T, MT, 2, G>(a, words, st);
    if (steps <= 16) return launch<T, MT, 4, G>(a, words, st);
    return launch<T, MT, 8, G>(a, words, st);
}
template <class T, bool G> hipError_t by_rows(const Args& a, bool words, hipStream_t st) {
    if (a.rows <= 16) return by_waves<T, 1, G>(a, words, st);
    return by_waves<T, 2, G>(a, words, st);
}

}  // namespace

// Up to about where this is faster than tiles: 64 rows in bfloat16 and 128 in fp32, more
// where the weights are small. In bfloat16, 64 rows of 1,024 to 1,024: 7.1 us here and 7.5
// on tiles, 96: 9.5 and 7.5; of 256 to 1,024: 3.7 and 4.0, 4.4 and 4.1; of 5,120 to 1,280, 48 rows: 22.2 and
// 25.0, 64: 25.5 and 25.0; of 184 to 256, 256 rows: 3.0 and 3.5, 512: 3.7 and 3.6. In fp32, 128 rows of
// 1,024 to 1,024: 25 and 34, 192: 36 and 34; of 2,048 to 2,048, 128 rows: 51 and 65, 192: 78 and 65; of 181 to
// 333, 512 rows: 12.3 and 12.9.  Where there are as many columns as tiles need, in bfloat16, tiles are faster
// from fewer rows on, and the rule does not know it: of 5,120 to 5,120, 32 rows: 34 and 27, 64: 58 and 30.
bool few_rows(const Args& a) {
    const bool small = uint64_t(a.in) * a.out * (a.gated ? 2 : 1) <= 1u << 16;
    return a.rows <= (a.bf ? (small ? 256u : 64u) : (small ? 512u : 128u));
}

hipError_t forward_few(const Args& a, hipStream_t st) {
    const uint32_t size = a.bf ? 2 : 4, per = 16 / size;
    const auto words = [&](const Matrix& m) { return m.ld % per == 0 && reinterpret_cast<uintptr_t>(m.p) % 16 == 0; };
    const bool all = a.in % per == 0 && words(a.x) && words(a.w[0]) && (!a.gated || words(a.w[1]));
    if (a.bf) return a.gated ? by_rows<bf16, true>(a, all, st) : by_rows<bf16, false>(a, all, st);
    return a.gated ? by_rows<float, true>(a, all, st) : by_rows<float, false>(a, all, st);
}

}  // namespace dense
