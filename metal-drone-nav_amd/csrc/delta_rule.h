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
//   2 states 128 x 128:   512 ticks 77 : 51 and 280 : 184, 4,096 ticks 607 : 130 and 2,222 : 270
//   64 states 128 x 128:  512 ticks 81 : 79 and 312 : 209, 4,096 ticks 705 : 378 and 2,530 : 1,177
//   128 states 128 x 128: 512 ticks 96 : 130 and 332 : 363, 1,024 ticks 187 : 196 and 666 : 610,
//                         4,096 ticks 725 : 592 and 2,680 : 2,033
//   128 states 64 x 64:   512 ticks 58 : 60 and 213 : 182, 1,024 ticks 142 : 100 and 423 : 262
//   170 states 128 x 128: 1,024 ticks 191 : 260 and 689 : 814, 4,096 ticks 756 : 839 and 2,803 : 2,853
// So: up to 128 states, at least four segments of at least four chunks each, and
// of sixteen where there are more than 64 states of wide heads.  (170 states 64 x
// 64, of which a compute unit holds several, would gain too: 1,024 ticks 145 :
// 116 and 441 : 344.)
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
// heads do not fill its tiles.  Recurrent against chunks, in us, with a final
// state : without one:
//   bf16, 16,384 states 64 x 64:   1 tick 108 : 161 and 51 : 108, 4 ticks 137 : 165 and 93 : 109, 8 ticks 187 : 168 and 141 : 111
//   bf16, 8,192 states 128 x 128:  1 tick 207 : 251 and 97 : 147, 4 ticks 254 : 255 and 174 : 153, 6 ticks 297 : 257 and 219 : 157
//   bf16, 8,192 states 128 x 64:   4 ticks 140 : 171 and 95 : 120, 8 ticks 185 : 173 and 144 : 120, 12 ticks 236 : 175 and 195 : 121
//   bf16, 16,384 states 64 x 32:   4 ticks 84 : 132 and 65 : 90, 6 ticks 105 : 133 and 86 : 90
//   bf16, 8,192 states 128 x 32:   8 ticks 104 : 154 and 79 : 111, 12 ticks 132 : 156 and 107 : 113
//   bf16, 8,192 states 64 x 128:   8 ticks 182 : 326 and 138 : 250, 12 ticks 231 : 329 and 186 : 251
//   bf16, 8,192 states 96 x 96:    8 ticks 221 : 399 and 179 : 305, 12 ticks 289 : 400 and 248 : 307
//   bf16, 4,096 states 91 x 87:    8 ticks 141 : 205 and 111 : 167, 12 ticks 181 : 208 and 150 : 168
//   bf16, 16,384 states 48 x 48:   8 ticks 175 : 233 and 142 : 140, 12 ticks 224 : 237 and 191 : 143
//   bf16, 16,384 states 32 x 32:   8 ticks 98 : 177 and 91 : 122, 12 ticks 136 : 179 and 128 : 123
//   fp32, 16,384 states 64 x 64:   8 ticks 169 : 255 and 125 : 223, 12 ticks 206 : 259 and 166 : 226
//   fp32, 8,192 states 128 x 128:  8 ticks 324 : 400 and 231 : 323, 12 ticks 407 : 405 and 313 : 327
// (calls in a row, each with inputs of its own, as all sides of choices here).
// So in bfloat16, where a state's rows fill the tiles and its columns half of
// them, 4; in other heads of up to 64 without a final state 8; else 12.
inline uint32_t recurrent_ticks(const Args& a, bool bf16) {
    if (!bf16) return 12;
    if ((a.k_dim == 64 || a.k_dim == 128) && a.v_dim <= a.k_dim && 2 * a.v_dim >= a.k_dim) return 4;
    return a.k_dim <= 64 && a.v_dim <= 64 && !a.state_out ? 8 : 12;
}
hipError_t launch_recurrent(const Args& a, bool bf16, hipStream_t stream);
hipError_t launch_forward(const Args& a, bool bf16, hipStream_t stream);

}  // namespace delta

#endif
