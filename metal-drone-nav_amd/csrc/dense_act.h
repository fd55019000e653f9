// dense_act.h — activations with their slopes, and four neighbours of a row.
#ifndef MDNAV_DENSE_ACT_H
#define MDNAV_DENSE_ACT_H

#include "dense.h"
#include "dense_tiles.h"

#include <type_traits>

namespace dense {

// ---------------------------------------------------------------- activations
// T: the type that the value is rounded to. bfloat16 leaves room for the
// faster exponential, whose relative error is |z| 2^-24.
template <class T> __device__ __forceinline__ float exp_of(float x) { return sizeof(T) == 2 ? __expf(x) : expf(x); }
template <class T> __device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_of<T>(-z)); }
// sigmoid(z) and sigmoid(-z), neither by a difference from 1.
template <class T> __device__ __forceinline__ float sigmoids(float z, float& other) {
    const float e = exp_of<T>(-fabsf(z)), big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
    other = z < 0.0f ? big : small;
    return z < 0.0f ? small : big;
}
template <class T> __device__ __forceinline__ float tanh_of(float z) {
    if (sizeof(T) == 4) return tanhf(z);
    // 1 - 2 / (e^2z + 1) cancels near 0, where the series' next term is below 2^-17 of the value
    const float e = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__expf(2.0f * z) + 1.0f), q = z * z;
    return q < 0.0025f ? z * (1.0f - q * 0.33333333f) : e;
}
constexpr float C_TANH = 1.5957691216f;  // 2 sqrt(2 / pi)

// Phi(z) of the normal distribution, and exp(-z^2 / 2).  For bfloat16 exp(z^2 / 2) Phi(-|z|) is a polynomial in
// t = 1 / (1 + 0.29 |z|), fitted for the least error that is at most 2^-13 of its value to z = -13, where the numbers end,
// and of Phi 2e-7, in place of erfc: 262,144 x 1,024 to 1,024 takes 688 us, and 1,029 with erfc (gated: 1,132 and 1,356);
// silu takes 11 % less (8).
template <class T> __device__ __forceinline__ float normal(float z, float& e) {
    e = exp_of<T>(-0.5f * z * z);
    if (sizeof(T) == 4) return 0.5f * erfcf(-0.70710678f * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.28991377f, fabsf(z), 1.0f));
    float q = fmaf(-0.08933758f, t, 0.28708297f);
    q = fmaf(q, t, -0.09619254f);
    q = fmaf(q, t, 0.1814572f);
    q = fmaf(q, t, 0.10008496f);
    q = fmaf(q, t, 0.116905004f);
    q *= t * e;
    return z < 0.0f ? q : 1.0f - q;
}

template <class T, uint32_t ACT> __device__ __forceinline__ float act_of(float z) {
    if (ACT == MDN_ACT_RELU) return z > 0.0f ? z : z == z ? 0.0f : z;
    if (ACT == MDN_ACT_TANH) return tanh_of<T>(z);
    if (ACT == MDN_ACT_SIGMOID) return sigmoid<T>(z);
    if (ACT == MDN_ACT_SILU) return z * sigmoid<T>(z);
    if (ACT == MDN_ACT_GELU) {
        float e;
        return z * normal<T>(z, e);
    }
    if (ACT == MDN_ACT_GELU_TANH) return z * sigmoid<T>(C_TANH * z * fmaf(0.044715f * z, z, 1.0f));
    return z;
}
// act(z) and act'(z)
template <class T, uint32_t ACT> __device__ __forceinline__ float act_of(float z, float& slope) {
    if (ACT == MDN_ACT_RELU) {
        slope = z > 0.0f ? 1.0f : z == z ? 0.0f : z;
        return act_of<T, ACT>(z);
    }
    if (ACT == MDN_ACT_TANH) {
        const float t = tanh_of<T>(z);
        slope = fmaf(-t, t, 1.0f);
        if (fabsf(z) > 4.0f) {  // 1 - t^2 cancels
            const float e = exp_of<T>(-2.0f * fabsf(z)), q = 1.0f + e;
            slope = 4.0f * e / (q * q);
        }
        return t;
    }
    if (ACT == MDN_ACT_SIGMOID) {
        float other;
        const float s = sigmoids<T>(z, other);
        slope = s * other;
        return s;
    }
    if (ACT == MDN_ACT_SILU) {
        // e s must not be inf times 0: below -87, where 1 / e^87 is still a normal number, value and slope stay those of
        // -87, under 1.5e-36 and next to the 0 that they go to (the comparison lets a NaN through)
        const float c = z < -87.0f ? -87.0f : z, e = exp_of<T>(-c), s = __builtin_amdgcn_rcpf(1.0f + e);
        slope = s * fmaf(c, e * s, 1.0f);
        return c * s;
    }
    if (ACT == MDN_ACT_GELU) {
        float e;
        const float s = normal<T>(z, e);
        slope = fmaf(z * 0.39894228f, e, s);
        return z * s;
    }
    if (ACT == MDN_ACT_GELU_TANH) {
        // beyond 30 the slope is 0 or 1; the polynomial would overflow
        const float c = fminf(fmaxf(z, -30.0f), 30.0f), u = C_TANH * c * fmaf(0.044715f * c, c, 1.0f);
        float other;
        const float s = sigmoids<T>(u, other);
        slope = fmaf(c * s * other, C_TANH * fmaf(0.134145f * c, c, 1.0f), s) + 0.0f * z;
        return z * s;
    }
    slope = 1.0f;
    return z;
}
// The activation of a call, chosen once for N values.
template <class F> __device__ __forceinline__ void by_act(uint32_t act, F f) {
    switch (act) {
        case MDN_ACT_RELU: return f(std::integral_constant<uint32_t, MDN_ACT_RELU>());
        case MDN_ACT_TANH: return f(std::integral_constant<uint32_t, MDN_ACT_TANH>());
        case MDN_ACT_SIGMOID: return f(std::integral_constant<uint32_t, MDN_ACT_SIGMOID>());
        case MDN_ACT_SILU: return f(std::integral_constant<uint32_t, MDN_ACT_SILU>());
        case MDN_ACT_GELU: return f(std::integral_constant<uint32_t, MDN_ACT_GELU>());
        case MDN_ACT_GELU_TANH: return f(std::integral_constant<uint32_t, MDN_ACT_GELU_TANH>());
        default: return f(std::integral_constant<uint32_t, MDN_ACT_NONE>());
    }
}
template <class T, int N> __device__ __forceinline__ void act_of(uint32_t act, float (&z)[N]) {
    by_act(act, [&](auto kind) {
#pragma unroll
        for (int e = 0; e < N; e++) z[e] = act_of<T, kind()>(z[e]);
    });
}
// z to act(z), and act'(z)
template <class T, int N> __device__ __forceinline__ void act_of(uint32_t act, float (&z)[N], float (&slope)[N]) {
    by_act(act, [&](auto kind) {
#pragma unroll
        for (int e = 0; e < N; e++) z[e] = act_of<T, kind()>(z[e], slope[e]);
    });
}

// ---------------------------------------------------------------- four neighbours of a row
template <class T> struct Four;
template <> struct Four<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Four<bf16> { typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2))); };

template <class T> __device__ __forceinline__ f32x4 load4(const char* row, uint32_t n, uint32_t count) {
    const T* p = reinterpret_cast<const T*>(row) + n;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n + 4 <= count) {
        const typename Four<T>::type t = *reinterpret_cast<const typename Four<T>::type*>(p);
        v = f32x4{float(t[0]), float(t[1]), float(t[2]), float(t[3])};
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            if (n + i < count) v[i] = float(p[i]);
    }
    return v;
}
template <class T> __device__ __forceinline__ void store4(char* row, uint32_t n, uint32_t count, f32x4 v) {
    T* p = reinterpret_cast<T*>(row) + n;
    if (n + 4 <= count) {
        *reinterpret_cast<typename Four<T>::type*>(p) = typename Four<T>::type{T(v[0]), T(v[1]), T(v[2]), T(v[3])};
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
            if (n + i < count) p[i] = T(v[i]);
    }
}
template <class T> __device__ __forceinline__ char* row_of(const Matrix& m, uint32_t row) { return m.p + int64_t(row) * m.ld * int64_t(sizeof(T)); }

}  // namespace dense

#endif
