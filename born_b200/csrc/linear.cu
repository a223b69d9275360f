// The output head: tensor maps, tile shape and launch.
#include <string.h>
#include "linear_kernel.cuh"

namespace born {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// (the library does not link the driver: its one entry point is looked up)
static EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// [rows, K] bf16 with `stride` elements between rows, in boxes of `box` rows by 64 elements
static bool make_map(CUtensorMap* map, const void* p, int rows, int K, int64_t stride, int box) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t boxes[2] = {(cuuint32_t)kLinK, (cuuint32_t)box};
    const cuuint32_t steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t linear_attrs() {
    cudaError_t e = cudaFuncSetAttribute(linear_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmem);
    return e;
}

cudaError_t linear_launch(const LinearArgs& A, int dtype, int num_sms, cudaStream_t st) {
    LinearParams P;
    memset(&P, 0, sizeof P);
    P.M = A.M; P.K = A.K; P.V = A.V;
    // as few column tiles as hold the rows, of equal widths
    P.m_tiles = (A.M + kLinMaxCols - 1) / kLinMaxCols;
    P.cols = ((A.M + P.m_tiles - 1) / P.m_tiles + 15) / 16 * 16;
    P.m_tiles = (A.M + P.cols - 1) / P.cols;
    P.v_tiles = (A.V + kLinRows - 1) / kLinRows;
    P.stage_bytes = (kLinRows + P.cols) * kLinK * 2;  // (16 rows of a slice are 2 KB: atoms stay on 1024 bytes)
    P.stages = (kLinSmem - 1024) / P.stage_bytes;
    if (P.stages > kLinMaxStages) P.stages = kLinMaxStages;
    P.tmem_cols = 32;
    while (P.tmem_cols < 2 * P.cols) P.tmem_cols *= 2;
    P.activation = A.activation; P.scale = A.scale;
    P.bias = A.bias; P.residual = A.residual; P.out = A.out;
    P.residual_stride = A.residual_stride; P.out_stride = A.out_stride;
    P.dev_error = A.dev_error; P.timeout_ns = A.timeout_ns;
    CUtensorMap w, x;
    if (!make_map(&w, A.weight, A.V, A.K, A.weight_stride, kLinRows) || !make_map(&x, A.x, A.M, A.K, A.x_stride, P.cols)) return cudaErrorInvalidValue;
    const int64_t tiles = (int64_t)P.v_tiles * P.m_tiles;
    const unsigned grid = (unsigned)(tiles < num_sms ? tiles : num_sms);
    const size_t smem = (size_t)P.stages * P.stage_bytes + 1024;
    if (dtype == BORN_DTYPE_F32) linear_kernel<float><<<grid, kLinThreads, smem, st>>>(w, x, P);
    else linear_kernel<__nv_bfloat16><<<grid, kLinThreads, smem, st>>>(w, x, P);
    return cudaGetLastError();
}

}  // namespace born
