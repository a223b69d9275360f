// Host-side entry points of the output head's kernel (linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/born_sampler.h"

namespace born {

constexpr int kLinMost = 0x7fffffff - 1024;  // rows, hidden, features: a tile further is still an int

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
    // scratch for tiles whose K several CTAs share: their sums, and tickets that are 0 between launches
    float* partial;
    uint32_t* tickets;
    int* dev_error;
    unsigned long long timeout_ns;
};
int64_t linear_scratch_bytes(int num_sms);
int linear_tickets(int num_sms);
cudaError_t linear_attrs();
// dtype: of out and residual
cudaError_t linear_launch(const LinearArgs& A, int dtype, int num_sms, cudaStream_t st);

}  // namespace born
