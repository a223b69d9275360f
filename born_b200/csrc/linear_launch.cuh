// Host-side entry points of the output head's kernel (linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/born_sampler.h"

namespace born {

constexpr int kLinMost = 0x7fffffff - 1024;  // rows, hidden, features: a tile further is still an int

constexpr int kLinMaxCluster = 8;  // larger clusters are not portable
struct LinearLimits {
    int clusters[kLinMaxCluster + 1];  // so many of 2, 3, ... CTAs run at once
};

struct LinearArgs {
    int M, K, V;
    int activation;
    float scale;
    const void* x;
    const void* weight;
    const float* bias;
    const void* residual;
    void* out;
    int64_t x_stride, weight_stride, residual_stride, out_stride;  // elements
    int* dev_error;
    unsigned long long timeout_ns;
};
cudaError_t linear_attrs(LinearLimits& limits);
// dtype: of out and residual
cudaError_t linear_launch(const LinearArgs& A, int dtype, int num_sms, const LinearLimits& limits, cudaStream_t st);

}  // namespace born
