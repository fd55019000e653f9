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
// Forward reads the logits once: G lanes have a step and go through its heads,
// each lane with a running maximum m, s = sum exp(z - m) and t = sum exp(z - m)
// (z - m), so that log-sum-exp is m + log s and the entropy log s - t / s.
// Words of 16 bytes in fp32; what a step makes of them, and the sums over
// steps, in 64 bits, since the means are small differences of many terms.
//
// Whether r is past the clip's border decides over a step's whole gradient.
// Where r in 32-bit sums is so near that their error could decide, the
// step's exponentials are summed again in 64 bits.
//
// Backward reads the logits once more and writes their gradient: a step's
// statistics are three floats a head and the slope.
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

// Elements at .. at + per_word - 1 of a row in fp32; past its end, -inf (a choice that has no share).
template <class T> __device__ __forceinline__ void load(float (&z)[per_word<T>()], const T* row, uint32_t at, uint32_t count) {
    constexpr uint32_t N = per_word<T>();
    if (at + N <= count) {
        const Word w = *reinterpret_cast<const typename Words<T>::type*>(row + at);
#pragma unroll
        for (uint32_t e = 0; e < N; e++)
            z[e] = sizeof(T) == 4 ? __builtin_bit_cast(float, uint32_t(w[e]))
                                  : __builtin_bit_cast(float, e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < N; e++) z[e] = at + e < count ? float(row[at + e]) : -__builtin_inff();
    }
}

// A running maximum and sums.
struct Sums {
    float m, s, t;
    static __device__ __forceinline__ Sums none() { return {-__builtin_inff(), 0.0f, 0.0f}; }
    __device__ __forceinline__ void rescale(float to) {  // to >= m, above -inf
        const float by = m == to ? 1.0f : expf(m - to), gap = m - to;
        t = s > 0.0f ? by * fmaf(s, gap, t) : by * t;    // (no sum yet: m may be -inf)
        s *= by;
        m = to;
    }
    template <int N> __device__ __forceinline__ void add(const float (&z)[N]) {
        float top = z[0];
#pragma unroll
        for (int e = 1; e < N; e++) top = fmaxf(top, z[e]);
        if (!(top > -__builtin_inff())) {  // nothing to add, or NaN alone
#pragma unroll
            for (int e = 0; e < N; e++)
                if (z[e] != z[e]) s = z[e];
            return;
        }
        if (top > m) rescale(top);
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float x = z[e] - m, p = expf(x);
            s += p;
            t += p > 0.0f ? p * x : 0.0f;
        }
    }
    __device__ __forceinline__ void join(const Sums& o) {
        const float top = fmaxf(m, o.m);
        if (top > -__builtin_inff()) {
            Sums b = o;
            rescale(top);
            b.rescale(top);
            s += b.s;
            t += b.t;
        } else
            s += o.s;
    }
};
__device__ __forceinline__ Sums from_lane(const Sums& a, int mask) {
    return {__shfl_xor(a.m, mask), __shfl_xor(a.s, mask), __shfl_xor(a.t, mask)};
}

// What a group of lanes has a row with: a part of a wavefront, or (0) a workgroup of 1,024.
template <int G> struct Group {
    static constexpr uint32_t LANES = G ? G : 1024, PER = G ? 256 / G : 1, THREADS = G ? 256 : 1024;
    static __device__ __forceinline__ Sums join(Sums a) {
#pragma unroll
        for (int i = 1; i < (G ? G : 64); i *= 2) a.join(from_lane(a, i));
        if constexpr (G == 0) {
            __shared__ Sums lds[16];
            __syncthreads();
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
            __syncthreads();
            a = lds[threadIdx.x & 15];
#pragma unroll
            for (int i = 1; i < 16; i *= 2) a.join(from_lane(a, i));
        }
        return a;
    }
    static __device__ __forceinline__ double sum(double a) {
#pragma unroll
        for (int i = 1; i < (G ? G : 64); i *= 2) a += __shfl_xor(a, i);
        if constexpr (G == 0) {
            __shared__ double lds[16];
            __syncthreads();
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
            __syncthreads();
            a = lds[threadIdx.x & 15];
#pragma unroll
            for (int i = 1; i < 16; i *= 2) a += __shfl_xor(a, i);
        }
        return a;
    }
};

__device__ __forceinline__ int64_t action_of(const Args& a, uint64_t step, uint32_t head) {
    const uint64_t at = step * a.heads + head;
    return a.index64 ? reinterpret_cast<const int64_t*>(a.actions)[at] : reinterpret_cast<const int32_t*>(a.actions)[at];
}

template <class T, int G> __device__ __forceinline__ double exact_log_sum(const T* row, uint32_t lane, uint32_t count, float m) {
    double s = 0.0;
    for (uint32_t i = lane; i < count; i += Group<G>::LANES) s += exp(double(float(row[i])) - double(m));
    return log(Group<G>::sum(s));
}

// LOSS false: log-probabilities and entropies alone.
template <class T, int G, bool LOSS>
__global__ void __launch_bounds__(Group<G>::THREADS) forward_kernel(Args a) {
    constexpr uint32_t N = per_word<T>(), LANES = Group<G>::LANES, PER = Group<G>::PER;
    const uint32_t lane = threadIdx.x % LANES, words = (a.choices + N - 1) / N;
    double total[6] = {};
    for (uint64_t first = uint64_t(blockIdx.x) * PER; first < a.steps; first += uint64_t(gridDim.x) * PER) {
        const uint64_t step = first + threadIdx.x / LANES;
        if (step >= a.steps) continue;
        if (LOSS && a.mask && !a.mask[step]) {
            if (lane == 0) a.slopes[step] = 0.0f;
            continue;
        }
        double l = 0.0, entropy = 0.0;
        const auto each_head = [&](bool again) {
            l = entropy = 0.0;
            for (uint32_t h = 0; h < a.heads; h++) {
                const T* row = reinterpret_cast<const T*>(a.logits) + int64_t(step) * a.step + int64_t(h) * a.head;
                Sums sums = Sums::none();
                for (uint32_t w = lane; w < words; w += LANES) {
                    float z[N];
                    load<T>(z, row, w * N, a.choices);
                    sums.add(z);
                }
                sums = Group<G>::join(sums);
                const double log_sum = again ? exact_log_sum<T, G>(row, lane, a.choices, sums.m) : log(double(sums.s));
                const int64_t at = action_of(a, step, h);
                // an action that is none has no log-probability
                const double z = at >= 0 && at < int64_t(a.choices) ? double(float(row[at])) : __builtin_nan("");
                const double own = log_sum - double(sums.t) / double(sums.s);
                l += (z - double(sums.m)) - log_sum;
                entropy += own;
                if (LOSS && lane == 0) {
                    float* to = a.stats + (step * a.heads + h) * 3;
                    to[0] = sums.m;
                    to[1] = float(log_sum);
                    to[2] = float(own);
                }
            }
        };
        each_head(false);
        if constexpr (!LOSS) {
            if (lane == 0) {
                a.log_prob[step] = float(l);
                a.entropy[step] = float(entropy);
            }
        } else {
            const double old = a.old_log_prob[step], adv = a.advantages[step];
            double r = exp(l - old);
            // The 32-bit sums' error: 2^-23 an exponential, and 2^-24 for each of the additions that a term passes.
            const double room = double(a.heads) * 6e-8 * (12.0 + double(words / LANES + 1) * N);
            if (fabs(r - (1.0 - a.low)) < room * r || fabs(r - (1.0 + a.high)) < room * r) {
                each_head(true);
                r = exp(l - old);
            }
            const double inside = fmin(fmax(r, 1.0 - a.low), 1.0 + a.high);
            const bool cut = inside * adv < r * adv;
            double slope = cut ? 0.0 : -adv * r, kl = 0.0;
            if (a.ref_log_prob) {
                const double far = double(a.ref_log_prob[step]) - l, e = expm1(far);
                kl = e - far;
                slope -= a.kl_coef * e;
            }
            if (lane == 0) {
                a.slopes[step] = float(slope);
                total[0] -= cut ? inside * adv : r * adv;
                total[1] += kl;
                total[2] += entropy;
                total[3] += r;
                total[4] += inside == r ? 0.0 : 1.0;
                total[5] += 1.0;
            }
        }
    }
    if constexpr (LOSS) {
        __shared__ double lds[6];
        // in the order of the workgroup's lanes: the same bits every time
#pragma unroll
        for (int i = 0; i < 6; i++) {
            const double v = Group<G ? 64 : 0>::sum(total[i]);
            if (G == 0) {
                if (threadIdx.x == 0) lds[i] = v;
            } else {
                __shared__ double waves[4];
                if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
                __syncthreads();
                if (threadIdx.x == 0) lds[i] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
                __syncthreads();
            }
        }
        if (threadIdx.x == 0)
#pragma unroll
            for (int i = 0; i < 6; i++) a.parts[uint64_t(blockIdx.x) * 6 + i] = lds[i];
    }
}

// The workgroups' sums to means.
__global__ void __launch_bounds__(384) finish_kernel(Args a, uint32_t count) {
    __shared__ double sums[6];
    const uint32_t which = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double v = 0.0;
    for (uint32_t i = lane; i < count; i += 64) v += a.parts[uint64_t(i) * 6 + which];
    v = Group<64>::sum(v);
    if (lane == 0) sums[which] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double by = sums[5] > 0.0 ? 1.0 / sums[5] : 0.0;  // no step counts: all is 0
        a.loss[0] = float((sums[0] + a.kl_coef * sums[1] - a.entropy_coef * sums[2]) * by);
#pragma unroll
        for (int i = 0; i < 5; i++) a.loss[1 + i] = float(sums[i] * by);
        a.one_over[0] = float(by);
    }
}

template <class T, int G>
__global__ void __launch_bounds__(Group<G>::THREADS) backward_kernel(Args a, GradArgs d) {
    constexpr uint32_t N = per_word<T>(), LANES = Group<G>::LANES, PER = Group<G>::PER;
    const uint32_t lane = threadIdx.x % LANES, words = (a.choices + N - 1) / N;
    const float by = a.one_over[0] * d.d_loss[0], pull = float(a.entropy_coef) * by;
    const uint64_t rows = a.steps * a.heads;
    for (uint64_t row = uint64_t(blockIdx.x) * PER + threadIdx.x / LANES; row < rows; row += uint64_t(gridDim.x) * PER) {
        const uint64_t step = row / a.heads;
        const uint32_t head = uint32_t(row - step * a.heads);
        T* out = reinterpret_cast<T*>(d.d_logits) + row * a.choices;
        const bool counts = !a.mask || a.mask[step];
        const T* in = reinterpret_cast<const T*>(a.logits) + int64_t(step) * a.step + int64_t(head) * a.head;
        const float *stat = a.stats + row * 3, slope = a.slopes[step] * by;
        const float m = stat[0], log_sum = stat[1], entropy = stat[2];
        const int64_t chosen = action_of(a, step, head);
        for (uint32_t w = lane; w < words; w += LANES) {
            float z[N];
            if (counts) {
                load<T>(z, in, w * N, a.choices);
#pragma unroll
                for (uint32_t e = 0; e < N; e++) {
                    const float lp = (z[e] - m) - log_sum, p = expf(lp);
                    const float free = p > 0.0f ? p * (lp + entropy) : p;
                    z[e] = fmaf(slope, (int64_t(w) * N + e == chosen ? 1.0f : 0.0f) - p, pull * free);
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

// ---------------------------------------------------------------- launches
// Lanes of a row: as many as it has words, up to a wavefront; a workgroup where
// a lane would have more than 16 words.
int lanes_of(const Args& a) {
    const uint32_t n = a.bf ? 8 : 4, words = (a.choices + n - 1) / n;
    return words <= 4 ? 4 : words <= 8 ? 8 : words <= 16 ? 16 : words <= 32 ? 32 : words <= 1024 ? 64 : 0;
}
uint32_t blocks_of(uint64_t rows, int lanes, uint32_t most) {
    const uint64_t per = lanes ? 256 / lanes : 1, n = (rows + per - 1) / per;
    return uint32_t(n < most ? n : most);
}
constexpr uint32_t MOST_BLOCKS = 2048;

struct Forward {
    const Args& a;
    hipStream_t st;
    uint32_t blocks;
    bool loss;
    template <class T, int G> void run() const {
        if (loss)
            forward_kernel<T, G, true><<<dim3(blocks), dim3(Group<G>::THREADS), 0, st>>>(a);
        else
            forward_kernel<T, G, false><<<dim3(blocks), dim3(Group<G>::THREADS), 0, st>>>(a);
    }
};
struct Backward {
    const Args& a;
    const GradArgs& d;
    hipStream_t st;
    uint32_t blocks;
    template <class T, int G> void run() const { backward_kernel<T, G><<<dim3(blocks), dim3(Group<G>::THREADS), 0, st>>>(a, d); }
};
template <class T, class F> void by_lanes(int lanes, const F& f) {
    switch (lanes) {
        case 4: return f.template run<T, 4>();
        case 8: return f.template run<T, 8>();
        case 16: return f.template run<T, 16>();
        case 32: return f.template run<T, 32>();
        case 64: return f.template run<T, 64>();
        default: return f.template run<T, 0>();
    }
}
template <class F> hipError_t by_type(const Args& a, const F& f) {
    a.bf ? by_lanes<bf16>(lanes_of(a), f) : by_lanes<float>(lanes_of(a), f);
    return hipGetLastError();
}

}  // namespace

uint64_t keep_floats(const Args& a) { return a.steps * a.heads * 3 + a.steps + 1; }
uint32_t parts_of(const Args& a) { return blocks_of(a.steps, lanes_of(a), MOST_BLOCKS); }

hipError_t launch_log_prob(const Args& a, hipStream_t st) { return by_type(a, Forward{a, st, parts_of(a), false}); }

hipError_t launch_loss(const Args& a, hipStream_t st) {
    const uint32_t count = parts_of(a);
    if (count)
        if (hipError_t e = by_type(a, Forward{a, st, count, true})) return e;
    finish_kernel<<<dim3(1), dim3(384), 0, st>>>(a, count);
    return hipGetLastError();
}

hipError_t launch_loss_backward(const Args& a, const GradArgs& d, hipStream_t st) {
    return by_type(a, Backward{a, d, st, blocks_of(a.steps * a.heads, lanes_of(a), 1u << 16)});
}

}  // namespace choices
