// Host-side entry points of the output head's kernel (linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/born_sampler.h"

namespace born {

constexpr int kLinMost = 0x7fffffff - 1024;  // rows, hidden, features: a tile further is still an int

// Tiles of `most` columns at most for a batch of `rows`: as few as hold it, of equal widths (`unit`: a multiple of 16 for either half
// of the epilogue).
inline void linear_columns(int rows, int most, int& cols, int& tiles) {
    const int64_t r = rows, n = (r + most - 1) / most;
    const int unit = rows <= 16 ? 16 : 32;
    cols = (int)(((r + n - 1) / n + unit - 1) / unit * unit);
    tiles = (int)((r + cols - 1) / cols);
}

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
