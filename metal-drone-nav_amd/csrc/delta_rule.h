// delta_rule.h — arguments and launchers of the gated delta rule kernels
// (delta_rule.hip, delta_rule_backward.hip).
#ifndef MDNAV_DELTA_RULE_H
#define MDNAV_DELTA_RULE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mdnav.h"

namespace delta {

constexpr uint32_t CHUNK = 32;    // ticks of a chunk
constexpr uint32_t MAX_DIM = 128; // widest head

// One strided [ticks][envs][heads][width] array; the width is contiguous.
struct Rows {
    char* p;
    int64_t tick, env, head;  // strides in elements
};

struct Args {
    uint32_t ticks, envs, qk_heads, heads, k_dim, v_dim;
    uint32_t gate_f32;        // g and beta are fp32 (else the type of q)
    float scale;
    Rows q, k, v, o, g, beta; // g and beta have width 1
    const uint8_t* reset;     // [ticks][envs] with the strides below, or null
    int64_t reset_tick, reset_env;
    const float* state;       // [envs][heads][k][v] or null (zeros)
    float* state_out;         // the same, or null
    float* chunk_states;      // the states before chunks 1.. for the backward pass, or null
    // Few states of many ticks are cut into segments of `segment` chunks that
    // run side by side (cut()): a state that a segment begins with is a linear
    // function of the one the last segment began with, S' = M S + B.
    uint32_t segments, segment;
    float* seg_states;        // [state][segments][k][v]: B of the segment before (the first has the state), then the state before the segment
    float* seg_moves;         // [state][segments][k][k]: M; then [state][segments] words, 1 where an episode's first tick is in the segment
    float* seg_grads;         // [state][segments][k][v]: the same for the state's gradient after the segment
};

// The segments.  Each costs its chunks three times (B, M and the outputs) but
// for the first, and the join: that pays while most compute units would idle.
// In one piece against cut, in us, bf16, forward and forward with backward:
//   2 states 128 x 128:   512 ticks 75 : 54 and 301 : 231, 4,096 ticks 553 : 136 and 2,215 : 284
//   64 states 128 x 128:  512 ticks 79 : 81 and 307 : 234, 4,096 ticks 585 : 351 and 2,340 : 1,121
//   128 states 128 x 128: 512 ticks 80 : 120 and 316 : 360, 1,024 ticks 151 : 176 and 610 : 591,
//                         4,096 ticks 615 : 527 and 2,437 : 1,943
//   128 states 64 x 64:   512 ticks 62 : 64 and 226 : 231, 1,024 ticks 114 : 96 and 391 : 253
//   170 states 128 x 128: 4,096 ticks 631 : 576 and 2,532 : 2,439, 1,024 ticks 152 : 191 and 631 : 714
// So: up to 128 states, at least four segments of at least four chunks each, and
// of sixteen where there are more than 64 states of wide heads.
inline void cut(Args& a) {
    const uint32_t states = a.envs * a.heads, chunks = (a.ticks + CHUNK - 1) / CHUNK;
    const uint32_t least = states > 64 && (a.k_dim > 64 || a.v_dim > 64) ? 16 : 4;  // chunks of a segment
    uint32_t segments = states && states <= 128 ? 512 / states : 1;
    if (segments > chunks / least) segments = chunks / least;
    if (segments < 4) segments = 1;
    a.segment = (chunks + segments - 1) / (segments ? segments : 1);
    a.segments = a.segment ? (chunks + a.segment - 1) / a.segment : 1;
}
inline uint64_t seg_state_words(const Args& a) {
    return a.segments > 1 ? uint64_t(a.envs) * a.heads * a.segments * a.k_dim * a.v_dim : 0;
}
inline uint64_t seg_move_words(const Args& a) {
    return a.segments > 1 ? uint64_t(a.envs) * a.heads * a.segments * (uint64_t(a.k_dim) * a.k_dim + 1) : 0;
}
inline __host__ __device__ uint32_t* seg_flags(float* moves, uint32_t states, uint32_t segments, uint32_t k_dim) {
    return reinterpret_cast<uint32_t*>(moves + uint64_t(states) * segments * k_dim * k_dim);
}

// chunk_states keeps result tiles as they are in registers: of each state and
// chunk, [v / 16][k / 16] tiles of 64 lanes x 4 values.
inline __host__ __device__ uint64_t state_tile_words(const Args& a) {
    return uint64_t((a.k_dim + 15) / 16) * ((a.v_dim + 15) / 16) * 256;
}

// Wavefronts of a chunk's workgroup: one for each 16 columns of a head, and at
// least four (three hold the chunk's tiles of A, the last makes decays).
inline __host__ uint32_t waves_of(const Args& a) {
    const uint32_t dim = a.k_dim > a.v_dim ? a.k_dim : a.v_dim, waves = (dim + 15) / 16;
    return waves < 4 ? 4 : waves;
}

// Workgroups of a chunk kernel: as many as the GPU holds at once, which then
// go through the states in turn, or one for each state.
inline __host__ uint32_t resident_blocks(const void* kernel, const Args& a, uint32_t states, uint32_t bytes) {
    int device = 0, units = 0, per = 0;
    if (hipGetDevice(&device) != hipSuccess || hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, int(64 * waves_of(a)), bytes) != hipSuccess || units * per < 1)
        return states;
    const uint32_t most = uint32_t(units) * uint32_t(per);
    return states < most ? states : most;
}

// The backward pass: gradients of o and of the final state in, of the inputs
// out.  Where several value heads share a query head, d_q and d_k are fp32
// rows of every value head (`partial`) and sum_heads adds them up.
struct GradArgs {
    Rows d_o;
    const float* d_state_out;  // [envs][heads][k][v] or null (zeros)
    Rows d_q, d_k, d_v, d_g, d_beta;
    uint32_t partial;
    float* d_state;            // or null
};

hipError_t launch_backward(const Args& a, const GradArgs& d, bool bf16, hipStream_t stream);
// out[row][qk head][width] = sum of the `shared` heads of in[row][head][width]
hipError_t launch_sum_heads(const float* in, void* out, uint64_t rows, uint32_t qk_heads, uint32_t shared, uint32_t width,
                            bool bf16, hipStream_t stream);
// seg_grads[s - 1] += M_s^T seg_grads[s], from the last segment but one downwards.
hipError_t launch_join_grads(const Args& a, bool bf16, hipStream_t stream);
// The ticks up to which the recurrent kernel is taken.  It reads and writes a
// state as fast as a copy does but works its ticks off on the vector units; the
// chunk kernel costs much the same for 1 tick and 16, more in fp32 and where
// heads do not fill its tiles.  Recurrent against chunks, in us:
//   bf16, 16,384 states 64 x 64:  1 tick 106 : 173, 4 ticks 131 : 160, 6 ticks 153 : 161, 8 ticks 173 : 162
//   bf16, 8,192 states 128 x 128: 1 tick 204 : 259, 4 ticks 231 : 243, 6 ticks 266 : 246
//   bf16, 4,096 states 91 x 87:   1 tick 74 : 160, 8 ticks 127 : 188, 12 ticks 163 : 200
//   bf16, 16,384 states 32 x 32:  1 tick 30 : 153, 12 ticks 99 : 155
//   fp32, 16,384 states 64 x 64:  1 tick 104 : 248, 8 ticks 164 : 252, 12 ticks 203 : 257
//   fp32, 8,192 states 128 x 128: 1 tick 202 : 397, 8 ticks 310 : 400, 12 ticks 394 : 406
inline uint32_t recurrent_ticks(const Args& a, bool bf16) {
    const bool full = a.k_dim == a.v_dim && (a.k_dim == 64 || a.k_dim == 128);
    return bf16 && full ? 4 : 12;
}
hipError_t launch_recurrent(const Args& a, bool bf16, hipStream_t stream);
hipError_t launch_forward(const Args& a, bool bf16, hipStream_t stream);

}  // namespace delta

#endif
