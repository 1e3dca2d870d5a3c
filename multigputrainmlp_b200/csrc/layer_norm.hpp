// Layer normalisation over the columns of a row: what the engine and the C entry points share. Kernels: layer_norm_forward.cu,
// layer_norm_backward.cu.
#pragma once

#include "../../include/mgt_b200.h"
#include "launch.cuh"

#include <cuda_runtime.h>
#include <stdint.h>

namespace mgt {
namespace ln {

struct Forward {
    const void* x;
    void* y;
    const float* gamma;  // nullptr: ones
    const float* beta;   // nullptr: zeros
    float* mean;         // nullptr: not wanted
    float* rstd;
    float* state;        // tower form: the fp32 residual stream, x_pitch apart; else nullptr
    uint64_t x_pitch, y_pitch;
    uint32_t rows, cols;
    float eps;
    uint32_t lanes;      // threads that share a row (set by the launch)
    bool add;            // tower form: the row is added to the stream (else it begins it)
};

struct Backward {
    const void* dy;
    const void* x;
    void* dx;
    const float* gamma;
    const float* mean;
    const float* rstd;
    float* sums[3];      // dgamma, dbeta, dbias; nullptr: not wanted
    float* partial;      // [CTAs][3][cols], then two values a row for the widest rows
    uint64_t dy_pitch, x_pitch, dx_pitch;
    uint32_t rows, cols;
    uint32_t lanes;
};

// y = gamma * (x - mean) * rstd + beta
mgt_status_t LaunchForward(Forward a, int32_t x_type, int32_t y_type, LaunchOn on);
// state = relu((add ? state : 0) + gamma * (x - mean) * rstd + beta) in fp32 and as 16-bit operand y; x fp32, pitches of whole vectors
mgt_status_t LaunchTowerForward(Forward a, bool bf16, LaunchOn on);
// dx, and the column sums of dy * xhat, dy and dx. *launches: kernels enqueued.
mgt_status_t LaunchBackward(Backward a, int32_t dy_type, int32_t x_type, int32_t dx_type, LaunchOn on, uint32_t* launches);
uint64_t BackwardFloats(uint32_t rows, uint32_t cols);

}  // namespace ln
}  // namespace mgt
