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

template <typename O, int kCols, bool kPair>
static cudaError_t raise_limit() {
    return cudaFuncSetAttribute(linear_kernel<O, kCols, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmem);
}
template <typename O>
static cudaError_t raise_limits() {
    const cudaError_t e[] = {raise_limit<O, 16, false>(), raise_limit<O, 32, false>(), raise_limit<O, 64, false>(),
                             raise_limit<O, 128, false>(), raise_limit<O, 64, true>(), raise_limit<O, 128, true>()};
    for (const cudaError_t x : e)
        if (x != cudaSuccess) return x;
    return cudaSuccess;
}
cudaError_t linear_attrs(LinearLimits& limits) {
    cudaError_t e = raise_limits<float>();
    if (e == cudaSuccess) e = raise_limits<__nv_bfloat16>();
    for (int n = 2; n <= kLinMaxCluster && e == cudaSuccess; ++n) {
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)n;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof cfg);
        cfg.gridDim = dim3((unsigned)n, 1, 1);
        cfg.blockDim = dim3(kLinThreads, 1, 1);
        cfg.dynamicSmemBytes = kLinSmem;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&limits.clusters[n], linear_kernel<float, 64, false>, &cfg);
    }
    return e;
}

template <typename O, int kCols, bool kPair>
static cudaError_t launch(const CUtensorMap& w, const CUtensorMap& x, const LinearParams& P, unsigned grid, cudaStream_t st) {
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)(P.splits * (kPair ? 2 : 1));
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(kLinThreads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)P.stages * kLinDeep * P.slice_bytes + 1024;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = kPair || P.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, linear_kernel<O, kCols, kPair>, w, x, P);
}
template <typename O>
static cudaError_t launch_as(const CUtensorMap& w, const CUtensorMap& x, const LinearParams& P, bool pair, unsigned grid, cudaStream_t st) {
    const int cols = P.cols > 16 ? P.cols / 2 : 16;  // of a thread of the epilogue
    if (pair) return cols <= 64 ? launch<O, 64, true>(w, x, P, grid, st) : launch<O, 128, true>(w, x, P, grid, st);
    if (cols <= 16) return launch<O, 16, false>(w, x, P, grid, st);
    if (cols <= 32) return launch<O, 32, false>(w, x, P, grid, st);
    return cols <= 64 ? launch<O, 64, false>(w, x, P, grid, st) : launch<O, 128, false>(w, x, P, grid, st);
}

// How a product is cut: the tiles, who shares what, and what that costs.
struct LinearShape {
    int cols, m_tiles, v_tiles, splits, part;
    bool pair;
    int64_t cost;  // nanoseconds, about: see below
};
// ... with tiles of `most` columns at most
static LinearShape shape_of(const LinearArgs& A, int most, int num_sms, const LinearLimits& limits) {
    LinearShape S;
    linear_columns(A.M, most, S.cols, S.m_tiles);
    // A pair from 65 columns on: below that the batch's slices are a third of the bytes at most
    S.pair = S.cols > 64 && A.V > kLinRows;
    const int ctas = S.pair ? 2 : 1, unit_rows = ctas * kLinRows, room = num_sms / ctas, x_rows = S.cols / ctas;
    S.v_tiles = (A.V + unit_rows - 1) / unit_rows;
    const int64_t tiles = (int64_t)S.v_tiles * S.m_tiles, each = (tiles + room - 1) / room;
    // K is shared out while CTAs are left, in parts of four slices at least, over the CTAs of a cluster, and so that all
    // clusters run at once (16 of 8 CTAs do not: 1 x 2048 x 2048 11.3 us with those, 6.8 with 16 of 7).
    const int slices = (A.K + kLinK - 1) / kLinK;
    int64_t splits = room / tiles;
    if (splits > slices / 4) splits = slices / 4;
    if (splits > kLinMaxCluster / ctas) splits = kLinMaxCluster / ctas;
    while (splits > 1 && limits.clusters[splits * ctas] < tiles) --splits;
    if (splits < 1) splits = 1;
    S.part = (int)((slices + splits - 1) / splits);
    S.splits = (slices + S.part - 1) / S.part;
    // The busiest CTA: 1.1 ns for 64 elements of a row, of weights or batch; per tile 22 ns a column for the epilogue's end; the
    // joining of parts 2 us and 25 ns a column.  (Fitted to 16 shapes of 80 to 512 rows, most within 2 us.)
    S.cost = 11 * S.part * each * (kLinRows + x_rows) / 10 + 22 * each * S.cols + (S.splits > 1 ? 2000 + 25 * S.cols : 0);
    return S;
}

cudaError_t linear_launch(const LinearArgs& A, int dtype, int num_sms, const LinearLimits& limits, cudaStream_t st) {
    // Wide tiles read the weights once, narrow ones fill the GPU and have less of an end.  Rows x hidden x features with
    // 256, 128, 64 columns: 256 x 512 x 4096 12.9, 9.2, 4.8 us; 512 x 4096 x 4096 23.7, 18.6, 26.9; 512 x 2048 x 32000 59, 63, 86.
    LinearShape S = shape_of(A, kLinMaxCols, num_sms, limits);
    for (int most = kLinMaxCols / 2; most >= 64 && A.M > 64; most /= 2) {
        const LinearShape o = shape_of(A, most, num_sms, limits);
        if (o.cost < S.cost) S = o;
    }
    LinearParams P;
    memset(&P, 0, sizeof P);
    P.M = A.M; P.K = A.K; P.V = A.V;
    P.cols = S.cols; P.m_tiles = S.m_tiles; P.v_tiles = S.v_tiles;
    P.splits = S.splits; P.part = S.part;
    const int x_rows = S.pair ? S.cols / 2 : S.cols;
    P.slice_bytes = (kLinRows + x_rows) * kLinK * 2;  // (8 rows of a slice are 1 KB: atoms stay on 1024 bytes)
    P.stages = (kLinSmem - 1024) / (kLinDeep * P.slice_bytes);
    if (P.stages > kLinMaxStages) P.stages = kLinMaxStages;
    P.tmem_cols = 32;
    while (P.tmem_cols < 2 * P.cols) P.tmem_cols *= 2;
    P.activation = A.activation; P.scale = A.scale; P.inv_scale = 1.0f / A.scale;
    P.bias = A.bias; P.residual = A.residual; P.out = A.out;
    P.residual_stride = A.residual_stride; P.out_stride = A.out_stride;
    P.dev_error = A.dev_error; P.timeout_ns = A.timeout_ns;
    CUtensorMap w, x;
    if (!make_map(&w, A.weight, A.V, A.K, A.weight_stride, kLinRows) || !make_map(&x, A.x, A.M, A.K, A.x_stride, x_rows)) return cudaErrorInvalidValue;
    const int64_t units = (int64_t)P.v_tiles * P.m_tiles * P.splits, room = S.pair ? num_sms / 2 : num_sms;
    const unsigned grid = (unsigned)(units < room ? units : room) * (S.pair ? 2u : 1u);
    if (dtype == BORN_DTYPE_F32) return launch_as<float>(w, x, P, S.pair, grid, st);
    return launch_as<__nv_bfloat16>(w, x, P, S.pair, grid, st);
}

}  // namespace born
