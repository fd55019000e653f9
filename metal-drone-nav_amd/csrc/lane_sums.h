// lane_sums.h — sums over lanes of a wavefront without LDS: by the lane order
// that vector instructions can read their operand in, and by swapped rows.
#ifndef MDNAV_LANE_SUMS_H
#define MDNAV_LANE_SUMS_H
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lanes {

template <int CTRL> __device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ double from_lane(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, 0xf, 0xf, true));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, 0xf, 0xf, true));
    return __builtin_bit_cast(double, uint64_t(lo) | uint64_t(hi) << 32);
}
// Over the 16 lanes with the same l / 16: neighbours, pairs, then mirrored eights and sixteens.
template <class T> __device__ __forceinline__ T sum16(T x) {
    x += from_lane<0xB1>(x);
    x += from_lane<0x4E>(x);
    x += from_lane<0x141>(x);
    return x + from_lane<0x140>(x);
}
// Over lanes l, l ^ 16, and over l, l ^ 32.
__device__ __forceinline__ float sum_rows16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
}
__device__ __forceinline__ float sum_rows32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
}

}  // namespace lanes

#endif
