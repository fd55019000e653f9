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
    float* seg_states;        // [state][segments][k][v]: B of the segment before, then the state before the segment
    float* seg_moves;         // [state][segments][k][k]: M
    float* seg_grads;         // [state][segments][k][v]: the same for the state's gradient after the segment
};

// The segments.  Each costs its chunks three times (B, M and the outputs) but
// for the first; 30,011 ticks of two envs and eight 128-wide heads went from 4,140 us
// in one piece to 660 us (332 ahead, 92 joining, 228).  A workgroup for each of the 256 compute units or
// more needs no cut: with 128 states and fewer there are at least four
// segments to a state.
inline void cut(Args& a) {
    const uint32_t states = a.envs * a.heads, chunks = (a.ticks + CHUNK - 1) / CHUNK;
    uint32_t segments = states && states <= 128 ? 512 / states : 1;
    if (segments > chunks / 4) segments = chunks / 4;
    if (segments < 4) segments = 1;
    a.segment = (chunks + segments - 1) / (segments ? segments : 1);
    a.segments = a.segment ? (chunks + a.segment - 1) / a.segment : 1;
}
inline uint64_t seg_state_words(const Args& a) {
    return a.segments > 1 ? uint64_t(a.envs) * a.heads * a.segments * a.k_dim * a.v_dim : 0;
}
inline uint64_t seg_move_words(const Args& a) {
    return a.segments > 1 ? uint64_t(a.envs) * a.heads * a.segments * a.k_dim * a.k_dim : 0;
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
hipError_t launch_recurrent(const Args& a, bool bf16, hipStream_t stream);
hipError_t launch_forward(const Args& a, bool bf16, hipStream_t stream);

}  // namespace delta

#endif
