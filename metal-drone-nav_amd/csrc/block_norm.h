// block_norm.h — arguments and launchers of the norm block kernels (block_norm.hip).
#ifndef MDNAV_BLOCK_NORM_H
#define MDNAV_BLOCK_NORM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mdnav.h"

namespace blocknorm {

constexpr uint32_t MAX_WIDTH = 8192;

struct Rows { char* p; int64_t outer, inner; };  // row r at (r / inner_count) outer + (r % inner_count) inner elements

struct Args {
    uint64_t rows;
    uint32_t inner_count, width;
    uint32_t gate_kind, gate_f32;
    float eps;
    Rows x, y, gate, s, h;
    const float *w_post, *w_pre, *residual;  // residual may be null (ones)
    float* stats;                            // [rows][2]: 1 / rms of y and of s; null in a forward call without gradients
};

struct GradArgs {
    Rows d_s, d_h, d_x, d_y, d_gate;  // d_s or d_h may be null (zeros)
    float *d_w_post, *d_w_pre, *d_residual;
    float* parts;                     // [workgroups][4][width]
};

// Workgroups of a backward call, each with a row of column sums.
uint32_t parts(const Args& a, uint32_t y_type);
hipError_t launch_forward(const Args& a, uint32_t x_type, uint32_t y_type, hipStream_t stream);
hipError_t launch_backward(const Args& a, const GradArgs& d, uint32_t x_type, uint32_t y_type, hipStream_t stream);

}  // namespace blocknorm

#endif
