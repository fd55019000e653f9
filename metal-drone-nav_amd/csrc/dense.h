// dense.h — arguments and launchers of the linear layer and the gated feed-forward block (dense.hip, dense_rows.hip).
#ifndef MDNAV_DENSE_H
#define MDNAV_DENSE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mdnav.h"

namespace dense {

constexpr uint32_t MAX_WIDTH = 1u << 16;

struct Matrix { char* p; int64_t ld; };  // rows ld elements apart, columns contiguous

struct Args {
    uint64_t rows;
    uint32_t in, out, activation, gated, bf;
    Matrix x, w[2], residual, y;
    const char* b[2];
};
struct GradArgs {
    Matrix d_y, d_x, d_w[2];
    char* d_b[2];
};

// Bytes of workspace, by sizes, strides and addresses.
uint64_t forward_bytes(const Args& a);
uint64_t backward_bytes(const Args& a, const GradArgs& d);  // (which gradients are wanted, and d_y)
// The tiles of the forward product, the arguments' gradients, d_x and the weights' gradients: their rows (0: no such
// product, or the kernel of few rows), bytes of a step, pieces of the sum.
struct Choice { uint32_t rows, step, parts; };
void choices(const Args& a, const GradArgs* d, Choice (&to)[4]);
hipError_t forward(const Args& a, char* work, hipStream_t st);
hipError_t backward(const Args& a, const GradArgs& d, char* work, hipStream_t st);

// Few rows (dense_rows.hip).
bool few_rows(const Args& a);
hipError_t forward_few(const Args& a, hipStream_t st);

}  // namespace dense

#endif
