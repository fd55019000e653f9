// choices.h — arguments and launchers of the clipped loss over discrete choices (choices.hip).
#ifndef MDNAV_CHOICES_H
#define MDNAV_CHOICES_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mdnav.h"

namespace choices {

// Of a row: the largest logit, the sum of exponentials below it, the entropy and the chosen logit.
struct __align__(16) Stat { float m, s, entropy, chosen; };

struct Args {
    uint64_t steps;
    uint32_t heads, choices, bf, index64;
    const char* logits;
    int64_t step, head;    // elements
    const char* actions;   // [steps][heads]
    // acting
    float *log_prob, *entropy;
    // the loss
    const float *old_log_prob, *advantages, *ref_log_prob;
    const uint8_t* mask;
    double low, high, kl_coef, entropy_coef;
    float* loss;
    float* metrics;        // the means of its five terms
    Stat* stats;           // [steps][heads]
    float* slopes;         // [steps]: of the loss (not yet a mean) by the log-probability; NaN-free 0 where masked
    double* parts;         // [workgroups][6]
    float* one_over;       // 1 / the steps that count
};
struct GradArgs {
    const float* d_loss;
    char* d_logits;        // contiguous
};

// Floats of stats, slopes and one_over, in this order.
uint64_t keep_floats(const Args& a);
uint32_t parts_of(const Args& a);
hipError_t launch_log_prob(const Args& a, hipStream_t st);
hipError_t launch_loss(const Args& a, hipStream_t st);
hipError_t launch_loss_backward(const Args& a, const GradArgs& d, hipStream_t st);

}  // namespace choices

#endif
