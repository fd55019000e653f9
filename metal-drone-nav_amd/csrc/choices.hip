// choices.hip — the clipped loss of a policy over discrete choices, and the
// log-probabilities that acting stores for it.
//
// Per step, over its heads: l = sum log softmax(z)[action], H = sum of the
// heads' entropies, r = exp(l - l_old), and
//     L = -min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(l_ref - l) - (l_ref - l) - 1) - entropy H
// averaged over the steps that count.  Backward, per choice,
//     dz = dL/dl (1[action] - p) + entropy p (log p + H)
// over the number of those steps.
//
// Forward reads the logits once. A lane keeps the largest logit m that it has
// seen, s = sum 2^y and t = sum y 2^y with y = (z - m) log2 e, in fp32, a few
// 16-byte words at a time; a row's lanes join theirs at the end, so log-sum-exp
// is m + log s and the entropy log s - t log 2 / s. m, s and the entropy of every
// row are kept. What a step makes of its rows is 64 bits, as are the sums over
// steps, since the means are small differences of many terms; that takes some
// hundreds of instructions and registers that the rows need, so a second kernel
// does it, a step to a lane, and a third adds up the workgroups' sums.
//
// Whether r is past the clip's border decides over a step's whole gradient.
// Where r of 32-bit sums is so near that their error could decide, the step's
// exponentials are summed again in 64 bits.
//
// Backward reads the logits once more and writes their gradient: a step's
// statistics are four floats a head and the slope.
#include "choices.h"

#include "lane_sums.h"

namespace choices {
namespace {

typedef __bf16 bf16;
typedef uint32_t Word __attribute__((ext_vector_type(4)));
template <class T> struct Words;
template <> struct Words<float> { typedef Word type __attribute__((aligned(4))); };
template <> struct Words<bf16> { typedef Word type __attribute__((aligned(2))); };
template <class T> constexpr uint32_t per_word() { return 16 / sizeof(T); }

// Elements at .. at + per_word - 1 of a row as they are; past its end, -inf (a choice that has no share).
template <class T> __device__ __forceinline__ Word fetch(const T* row, uint32_t at, uint32_t count) {
    constexpr uint32_t N = per_word<T>();
    if (at + N <= count) return *reinterpret_cast<const typename Words<T>::type*>(row + at);
    union { Word u; T t[N]; } v;
#pragma unroll
    for (uint32_t e = 0; e < N; e++) v.t[e] = at + e < count ? row[at + e] : T(-__builtin_inff());
    return v.u;
}
// The same in fp32.
template <class T> __device__ __forceinline__ void spread(float (&z)[per_word<T>()], const Word& w) {
#pragma unroll
    for (uint32_t e = 0; e < per_word<T>(); e++)
        z[e] = sizeof(T) == 4 ? __builtin_bit_cast(float, uint32_t(w[e]))
                              : __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}

constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f, LOWEST = -3.402823466e38f;

// A row's or a lane's largest logit and sums (2^y in hardware: 1 unit in the last place).
struct Sums {
    float m, s, t;
    static __device__ __forceinline__ Sums none() { return {LOWEST, 0.0f, 0.0f}; }
    __device__ __forceinline__ void rescale(float to) {
        const float y = (m - to) * LOG2E, by = __builtin_amdgcn_exp2f(y);
        t = by * fmaf(s, fmaxf(y, -1000.0f), t);  // (y may be -inf where there is nothing yet)
        s *= by;
        m = to;
    }
    template <int W, int N> __device__ __forceinline__ void add(const float (&z)[W][N]) {
        float top = m;
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int e = 0; e < N; e++) top = fmaxf(top, z[w][e]);
        if (top > m) rescale(top);
        float s_of = 0.0f, t_of = 0.0f;  // these logits' own: a long row's are added up in two levels
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float y = (z[w][e] - m) * LOG2E, p = __builtin_amdgcn_exp2f(y);
                s_of += p;
                t_of = fmaf(p, fmaxf(y, -1000.0f), t_of);  // a choice ruled out: 0, and not 0 times -inf
            }
        s += s_of;
        t += t_of;
    }
};
// Over the G lanes that have a row: neighbours, pairs, mirrored eights and sixteens, then other rows of sixteen.
template <int G, class F> __device__ __forceinline__ float over_lanes(float x, F f) {
    x = f(x, lanes::from_lane<0xB1>(x));
    x = f(x, lanes::from_lane<0x4E>(x));
    if (G >= 8) x = f(x, lanes::from_lane<0x141>(x));
    if (G >= 16) x = f(x, lanes::from_lane<0x140>(x));
    if (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
        x = f(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
    }
    if (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
        x = f(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
    }
    return x;
}
template <int G> __device__ __forceinline__ float lanes_max(float x) {
    return over_lanes<G>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int G> __device__ __forceinline__ float lanes_sum(float x) {
    return over_lanes<G>(x, [](float a, float b) { return a + b; });
}
template <int G> __device__ __forceinline__ double lanes_sum(double x) {
#pragma unroll
    for (int i = 1; i < G; i *= 2) x += __shfl_xor(x, i);
    return x;
}
template <int G> __device__ __forceinline__ Sums join(Sums a) {
    const float top = lanes_max<G>(a.m);
    a.rescale(top);
    return {top, lanes_sum<G>(a.s), lanes_sum<G>(a.t)};
}

__device__ __forceinline__ int64_t action_of(const Args& a, uint64_t row) {
    return a.index64 ? reinterpret_cast<const int64_t*>(a.actions)[row] : reinterpret_cast<const int32_t*>(a.actions)[row];
}
template <class T> __device__ __forceinline__ const T* row_of(const Args& a, uint64_t step, uint32_t head) {
    return reinterpret_cast<const T*>(a.logits) + int64_t(step) * a.step + int64_t(head) * a.head;
}
// The chosen logit; an action that is none has no log-probability.
template <class T> __device__ __forceinline__ float chosen(const T* row, int64_t action, uint32_t count) {
    return action >= 0 && action < int64_t(count) ? float(row[action]) : __builtin_nanf("");
}

// Lanes of a row: G of a wavefront, or (0) a workgroup of WIDE.
constexpr uint32_t WIDE = 512;
template <int G> constexpr uint32_t lanes_of() { return G ? G : WIDE; }
template <int G> constexpr uint32_t threads_of() { return G ? 256 : WIDE; }

// A row's sums, of which this lane has the words first, first + lanes, ..
template <class T, int G, int W> __device__ __forceinline__ Sums sum_row(const T* row, uint32_t lane, uint32_t count, uint32_t words) {
    Sums r = Sums::none();
    for (uint32_t first = lane; first < words; first += W * lanes_of<G>()) {
        Word got[W];
        float z[W][per_word<T>()];
#pragma unroll
        for (uint32_t w = 0; w < W; w++) got[w] = fetch<T>(row, (first + w * lanes_of<G>()) * per_word<T>(), count);
#pragma unroll
        for (uint32_t w = 0; w < W; w++) spread<T>(z[w], got[w]);
        r.add(z);
    }
    if constexpr (G != 0) return join<G>(r);
    __shared__ float lds[3][16];
    r = join<64>(r);
    __syncthreads();
    if (threadIdx.x < 16 * 3) lds[threadIdx.x / 16][threadIdx.x % 16] = threadIdx.x < 16 ? LOWEST : 0.0f;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        lds[0][threadIdx.x >> 6] = r.m;
        lds[1][threadIdx.x >> 6] = r.s;
        lds[2][threadIdx.x >> 6] = r.t;
    }
    __syncthreads();
    return join<16>(Sums{lds[0][threadIdx.x & 15], lds[1][threadIdx.x & 15], lds[2][threadIdx.x & 15]});
}
__device__ __forceinline__ float entropy_of(const Sums& r) {
    return LN2 * __builtin_amdgcn_logf(r.s) - LN2 * r.t * __builtin_amdgcn_rcpf(r.s);
}

// The statistics of rows, R of them at once in a group of lanes, W words each, so
// that 64 bytes a lane are on their way. Bound by memory where rows are wide
// (8,192 x 65,003 in bfloat16: 247 us, 4.3 TB/s); of short ones a third of the time is
// the joining of lanes and the round from the action to its logit (262,144 x 4 x 64: 43 us, 3.1 TB/s).
template <class T, int G, int R, int W>
__global__ void __launch_bounds__(threads_of<G>()) rows_kernel(Args a) {
    constexpr uint32_t LANES = lanes_of<G>(), GROUPS = threads_of<G>() / LANES, N = per_word<T>();
    const uint32_t lane = threadIdx.x % LANES, words = (a.choices + N - 1) / N;
    const uint64_t rows = a.steps * a.heads, per = uint64_t(GROUPS) * R;
    const bool even = a.step == int64_t(a.heads) * a.head;  // rows are all `head` apart
    for (uint64_t first = blockIdx.x * per; first < rows; first += gridDim.x * per) {
        Sums r[R];
        const T* at[R];
        int64_t action[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t row = first + i * GROUPS + threadIdx.x / LANES, in = row < rows ? row : rows - 1;
            action[i] = action_of(a, in);
            at[i] = even ? reinterpret_cast<const T*>(a.logits) + int64_t(in) * a.head : row_of<T>(a, in / a.heads, uint32_t(in % a.heads));
        }
        if constexpr (R > 1) {
            Word got[R];
            float z[R][1][N];
#pragma unroll
            for (int i = 0; i < R; i++) got[i] = fetch<T>(at[i], lane * N, a.choices);
#pragma unroll
            for (int i = 0; i < R; i++) {
                spread<T>(z[i][0], got[i]);
                r[i] = Sums::none();
                r[i].add(z[i]);
            }
#pragma unroll
            for (int i = 0; i < R; i++) r[i] = join<G>(r[i]);
        } else
            r[0] = sum_row<T, G, W>(at[0], lane, a.choices, words);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint64_t row = first + i * GROUPS + threadIdx.x / LANES;
            if (lane == 0 && row < rows) a.stats[row] = Stat{r[i].m, r[i].s, entropy_of(r[i]), chosen(at[i], action[i], a.choices)};
        }
    }
}

// The error of r, relative: a row's sum is off by 2^-23 for an exponential, by
// as much times the mean |y| (at most the logarithm of the choices, 24, and a
// little) for its argument, and by 2^-24 for each addition that a term passes:
// a lane adds up to 32 and then, of the widest rows, a sum and a factor for every
// 8,192 choices, and the lanes join in 10 more.
__device__ __forceinline__ bool near_border(const Args& a, double r) {
    const double room = double(a.heads) * 1.2e-7 * (30.0 + 0.5 * (42.0 + 4.0 * double(1 + a.choices / 8192))) * r;
    return fabs(r - (1.0 - a.low)) < room || fabs(r - (1.0 + a.high)) < room;
}
// 2^y in 64 bits, y <= 0: the series of 2^f, |f| <= 1/2, whose next term is below 2^-52.
__device__ __forceinline__ double exp2_of(double y) {
    if (!(y > -1000.0)) return y == y ? 0.0 : y;
    const double n = rint(y), x = (y - n) * 0.693147180559945309417;
    double p = 1.0 / 6227020800.0;
    p = fma(p, x, 1.0 / 479001600.0);
    p = fma(p, x, 1.0 / 39916800.0);
    p = fma(p, x, 1.0 / 3628800.0);
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return ldexp(p, int(n));
}
// l with sums in 64 bits, by a workgroup of 256 that is all here.
template <class T> __device__ __forceinline__ double exact_log_prob(const Args& a, uint64_t step) {
    __shared__ double lds[4];
    constexpr uint32_t N = per_word<T>();
    double l = 0.0;
    for (uint32_t h = 0; h < a.heads; h++) {
        const T* row = row_of<T>(a, step, h);
        const Stat stat = a.stats[step * a.heads + h];
        double s = 0.0;
        for (uint32_t at = threadIdx.x * N; at < a.choices; at += 256 * N) {
            float z[N];
            spread<T>(z, fetch<T>(row, at, a.choices));
#pragma unroll
            for (uint32_t e = 0; e < N; e++) s += exp2_of((double(z[e]) - double(stat.m)) * 1.44269504088896340736);
        }
        s = lanes_sum<64>(s);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
        __syncthreads();
        l += double(stat.chosen) - double(stat.m) - log((lds[0] + lds[1]) + (lds[2] + lds[3]));
    }
    return l;
}

// Every step's loss and slope, a step to a lane, and the workgroup's sums over steps.
// Bound by 64-bit logarithms and exponentials and their latency (262,144 steps: 22 us; 8,192 of
// 65,003 choices: 7, and 33 with a border's room of four times the width).  Where 64 bits decide every step, as with a clip of
// 0 in a first update, the steps' rows are read once more, one step a workgroup at a time.
template <class T>
__global__ void __launch_bounds__(256) steps_kernel(Args a) {
    double total[6] = {};
    for (uint64_t first = uint64_t(blockIdx.x) * 256; first < a.steps; first += uint64_t(gridDim.x) * 256) {
        const uint64_t step = first + threadIdx.x;
        const bool have = step < a.steps, counts = have && (!a.mask || a.mask[step]);
        double l = 0.0, r = 0.0, entropy = 0.0;
        if (counts) {
            double product = 1.0;  // of the sums: one logarithm for many
            for (uint32_t h = 0; h < a.heads; h++) {
                const Stat stat = a.stats[step * a.heads + h];
                l += double(stat.chosen) - double(stat.m);
                product *= double(stat.s);
                entropy += double(stat.entropy);
                if ((h & 31) == 31) {  // a sum is below 2^25
                    l -= log(product);
                    product = 1.0;
                }
            }
            l -= log(product);
            r = exp(l - double(a.old_log_prob[step]));
        }
        // steps that 64 bits decide, one after the other by the workgroup
        const bool near = counts && near_border(a, r);
        if (__syncthreads_or(near)) {
            __shared__ uint64_t open[4];
            const uint64_t mine = __ballot(near);
            if ((threadIdx.x & 63) == 0) open[threadIdx.x >> 6] = mine;
            __syncthreads();
            for (uint32_t wave = 0; wave < 4; wave++)
                for (uint64_t left = open[wave]; left; left &= left - 1) {
                    const uint32_t who = wave * 64 + uint32_t(__builtin_ctzll(left));
                    const double exact = exact_log_prob<T>(a, first + who);
                    if (threadIdx.x == who) {
                        l = exact;
                        r = exp(l - double(a.old_log_prob[step]));
                    }
                }
            __syncthreads();  // before the next steps' flags
        }
        double slope = 0.0;
        if (counts) {
            const double adv = a.advantages[step], inside = fmin(fmax(r, 1.0 - a.low), 1.0 + a.high);
            const bool cut = inside * adv < r * adv;
            slope = cut ? 0.0 : -adv * r;
            total[0] -= cut ? inside * adv : r * adv;
            if (a.ref_log_prob) {
                const double far = double(a.ref_log_prob[step]) - l, e = expm1(far);
                total[1] += e - far;
                if (a.kl_coef != 0.0) slope -= a.kl_coef * e;  // (0 leaves the term out, infinite or not)
            }
            total[2] += entropy;
            total[3] += r;
            total[4] += inside == r ? 0.0 : 1.0;
            total[5] += 1.0;
        }
        if (have) a.slopes[step] = float(slope);
    }
    // in the order of the lanes: the same bits every time
    __shared__ double waves[6][4];
#pragma unroll
    for (int i = 0; i < 6; i++) {
        const double v = lanes_sum<64>(total[i]);
        if ((threadIdx.x & 63) == 0) waves[i][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (threadIdx.x < 6)
        a.parts[uint64_t(blockIdx.x) * 6 + threadIdx.x] =
            (waves[threadIdx.x][0] + waves[threadIdx.x][1]) + (waves[threadIdx.x][2] + waves[threadIdx.x][3]);
}

// Acting: log-probabilities and entropies in one launch, G lanes to a step, whose
// heads follow each other. Bound by the launch and that chain (8,192 x 4 x 33 in fp32: 6.7 us).
template <class T, int G, int W>
__global__ void __launch_bounds__(threads_of<G>()) act_kernel(Args a) {
    constexpr uint32_t LANES = lanes_of<G>(), PER = threads_of<G>() / LANES, N = per_word<T>();
    const uint32_t lane = threadIdx.x % LANES, words = (a.choices + N - 1) / N;
    for (uint64_t first = uint64_t(blockIdx.x) * PER; first < a.steps; first += uint64_t(gridDim.x) * PER) {
        const uint64_t at = first + threadIdx.x / LANES, step = at < a.steps ? at : a.steps - 1;
        double l = 0.0, product = 1.0, entropy = 0.0;
        for (uint32_t h = 0; h < a.heads; h++) {
            const T* row = row_of<T>(a, step, h);
            const double logit = chosen(row, action_of(a, step * a.heads + h), a.choices);
            const Sums r = sum_row<T, G, W>(row, lane, a.choices, words);
            l += logit - double(r.m);
            product *= double(r.s);
            entropy += double(entropy_of(r));
            if ((h & 31) == 31) {
                l -= log(product);
                product = 1.0;
            }
        }
        if (lane == 0 && at < a.steps) {
            a.log_prob[step] = float(l - log(product));
            a.entropy[step] = float(entropy);
        }
    }
}

// The workgroups' sums to means.
__global__ void __launch_bounds__(384) finish_kernel(Args a, uint32_t count) {
    __shared__ double sums[6];
    const uint32_t which = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double v = 0.0;
    for (uint32_t i = lane; i < count; i += 64) v += a.parts[uint64_t(i) * 6 + which];
    v = lanes_sum<64>(v);
    if (lane == 0) sums[which] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double by = sums[5] > 0.0 ? 1.0 / sums[5] : 0.0;  // no step counts: all is 0
        a.loss[0] = float((sums[0] + (a.kl_coef != 0.0 ? a.kl_coef * sums[1] : 0.0) - a.entropy_coef * sums[2]) * by);
#pragma unroll
        for (int i = 0; i < 5; i++) a.metrics[i] = float(sums[i] * by);
        a.one_over[0] = float(by);
    }
}

// G lanes have a row, or (0) a workgroup.  Bound by memory (8,192 x 65,003 in
// bfloat16: 418 us, 5.1 TB/s; 262,144 x 4 x 64: 52 us, 5.2 TB/s).
template <class T, int G>
__global__ void __launch_bounds__(threads_of<G>()) backward_kernel(Args a, GradArgs d) {
    constexpr uint32_t N = per_word<T>(), LANES = lanes_of<G>(), PER = threads_of<G>() / LANES;
    const uint32_t lane = threadIdx.x % LANES, words = (a.choices + N - 1) / N;
    const float by = a.one_over[0] * d.d_loss[0], pull = float(a.entropy_coef) * by;
    for (uint64_t step = uint64_t(blockIdx.x) * PER + threadIdx.x / LANES; step < a.steps; step += uint64_t(gridDim.x) * PER) {
        const bool counts = !a.mask || a.mask[step];
        const float slope = a.slopes[step] * by;
        for (uint32_t h = 0; h < a.heads; h++) {
            const T* in = row_of<T>(a, step, h);
            const uint64_t row = step * a.heads + h;
            T* out = reinterpret_cast<T*>(d.d_logits) + row * a.choices;
            const Stat stat = a.stats[row];
            const float m = stat.m, log_sum = LN2 * __builtin_amdgcn_logf(stat.s), entropy = stat.entropy;
            const int64_t at = action_of(a, row);
            for (uint32_t w = lane; w < words; w += LANES) {
                float z[N];
                if (counts) {
                    spread<T>(z, fetch<T>(in, w * N, a.choices));
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) {
                        const float lp = (z[e] - m) - log_sum, p = __builtin_amdgcn_exp2f(lp * LOG2E);
                        const float free = p > 0.0f ? p * (lp + entropy) : p;
                        z[e] = fmaf(slope, (int64_t(w * N + e) == at ? 1.0f : 0.0f) - p, pull * free);
                    }
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) z[e] = 0.0f;
                }
                if (w * N + N <= a.choices) {
                    union { Word u; T t[N]; } v;
#pragma unroll
                    for (uint32_t e = 0; e < N; e++) v.t[e] = T(z[e]);
                    *reinterpret_cast<typename Words<T>::type*>(out + w * N) = v.u;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < N; e++)
                        if (w * N + e < a.choices) out[w * N + e] = T(z[e]);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- launches
// Lanes of a row, and words of each: a word a lane up to a wavefront, then up
// to four; a workgroup for wider rows.
struct Shape { uint32_t lanes, words; };
Shape shape_of(const Args& a) {
    const uint32_t n = a.bf ? 8 : 4, words = (a.choices + n - 1) / n;
    if (words <= 4) return {4, 1};
    if (words <= 8) return {8, 1};
    if (words <= 16) return {16, 1};
    if (words <= 32) return {32, 1};
    if (words <= 64) return {64, 1};
    return words <= 256 ? Shape{64, 4} : Shape{0, 0};
}
constexpr uint32_t UNITS = 256;
uint32_t blocks_of(uint64_t items, uint64_t per, uint64_t most) {
    const uint64_t n = (items + per - 1) / per;
    return uint32_t(n < most ? n : most);
}
uint32_t step_blocks(const Args& a) { return blocks_of(a.steps, 256, 4 * UNITS); }

template <class T> void rows(const Args& a, hipStream_t st) {
    const Shape s = shape_of(a);
    const uint64_t n = a.steps * a.heads;
    const auto grid = [&](uint64_t per) { return dim3(blocks_of(n, per, 64 * UNITS)); };
    if (!s.lanes) return rows_kernel<T, 0, 1, 4><<<grid(1), dim3(WIDE), 0, st>>>(a);
    if (s.words == 4) return rows_kernel<T, 64, 1, 4><<<grid(4), dim3(256), 0, st>>>(a);
    switch (s.lanes) {
        case 4: return rows_kernel<T, 4, 4, 1><<<grid(256), dim3(256), 0, st>>>(a);
        case 8: return rows_kernel<T, 8, 4, 1><<<grid(128), dim3(256), 0, st>>>(a);
        case 16: return rows_kernel<T, 16, 4, 1><<<grid(64), dim3(256), 0, st>>>(a);
        case 32: return rows_kernel<T, 32, 4, 1><<<grid(32), dim3(256), 0, st>>>(a);
        default: return rows_kernel<T, 64, 4, 1><<<grid(16), dim3(256), 0, st>>>(a);
    }
}
template <class T> void act(const Args& a, hipStream_t st) {
    const Shape s = shape_of(a);
    const auto grid = [&](uint64_t per) { return dim3(blocks_of(a.steps, per, 64 * UNITS)); };
    if (!s.lanes) return act_kernel<T, 0, 4><<<grid(1), dim3(WIDE), 0, st>>>(a);
    if (s.words == 4) return act_kernel<T, 64, 4><<<grid(4), dim3(256), 0, st>>>(a);
    switch (s.lanes) {
        case 4: return act_kernel<T, 4, 1><<<grid(64), dim3(256), 0, st>>>(a);
        case 8: return act_kernel<T, 8, 1><<<grid(32), dim3(256), 0, st>>>(a);
        case 16: return act_kernel<T, 16, 1><<<grid(16), dim3(256), 0, st>>>(a);
        case 32: return act_kernel<T, 32, 1><<<grid(8), dim3(256), 0, st>>>(a);
        default: return act_kernel<T, 64, 1><<<grid(4), dim3(256), 0, st>>>(a);
    }
}
template <class T> void backward(const Args& a, const GradArgs& d, hipStream_t st) {
    const Shape s = shape_of(a);
    const uint64_t per = s.lanes ? 256 / s.lanes : 1, n = (a.steps + per - 1) / per;
    const dim3 grid(uint32_t(n < (1u << 16) ? n : (1u << 16))), block(s.lanes ? 256 : WIDE);
    switch (s.lanes) {
        case 4: return backward_kernel<T, 4><<<grid, block, 0, st>>>(a, d);
        case 8: return backward_kernel<T, 8><<<grid, block, 0, st>>>(a, d);
        case 16: return backward_kernel<T, 16><<<grid, block, 0, st>>>(a, d);
        case 32: return backward_kernel<T, 32><<<grid, block, 0, st>>>(a, d);
        case 64: return backward_kernel<T, 64><<<grid, block, 0, st>>>(a, d);
        default: return backward_kernel<T, 0><<<grid, block, 0, st>>>(a, d);
    }
}

}  // namespace

uint64_t keep_floats(const Args& a) { return a.steps * a.heads * 4 + a.steps + 1; }
uint32_t parts_of(const Args& a) { return step_blocks(a); }

hipError_t launch_log_prob(const Args& a, hipStream_t st) {
    a.bf ? act<bf16>(a, st) : act<float>(a, st);
    return hipGetLastError();
}
hipError_t launch_loss(const Args& a, hipStream_t st) {
    const uint32_t count = parts_of(a);
    if (count) {
        a.bf ? rows<bf16>(a, st) : rows<float>(a, st);
        if (hipError_t e = hipGetLastError()) return e;
        if (a.bf)
            steps_kernel<bf16><<<dim3(count), dim3(256), 0, st>>>(a);
        else
            steps_kernel<float><<<dim3(count), dim3(256), 0, st>>>(a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    finish_kernel<<<dim3(1), dim3(384), 0, st>>>(a, count);
    return hipGetLastError();
}
hipError_t launch_loss_backward(const Args& a, const GradArgs& d, hipStream_t st) {
    a.bf ? backward<bf16>(a, d, st) : backward<float>(a, d, st);
    return hipGetLastError();
}

}  // namespace choices
