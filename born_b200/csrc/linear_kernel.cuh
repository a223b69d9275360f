// out[m][v] = act(sum_k x[m][k] weight[v][k] + bias[v]) + residual[m][v] on the tensor cores.
//
// A decode batch has few rows and a vocabulary many, so the weights take the tile's 128 rows and the
// batch its columns (16 to 256): D[128 v][n m] = W[128][K] X[n][K]^T, both operands K-major as they lie in
// memory.  One CTA per SM walks over tiles; a warp fills a ring of 64-element slices of both operands by
// TMA (128-byte swizzle), a thread issues the tcgen05 products into one of two accumulators in tensor
// memory, four warps empty the other one: a lane holds one v, so that a column of 32 lanes is a
// contiguous piece of an output row.
//
// What bounds it: up to some 200 rows the bytes of the weights, beyond that the tensor pipe.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include "linear_launch.cuh"
#include "spec.cuh"
#include "warp_ring.cuh"

namespace born {

constexpr int kLinRows = 128;      // v of a tile
constexpr int kLinK = 64;          // elements of a slice: 128 bytes, one swizzle atom
constexpr int kLinMaxCols = 256;   // m of a tile
constexpr int kLinMaxStages = 12;
constexpr int kLinThreads = 256;   // warps: 0 TMA, 1 products, 2 tensor memory, 3 idle, 4..7 epilogue
constexpr int kLinSmem = 220 * 1024;

struct LinearParams {
    int M, K, V;
    int cols;          // m of a tile, a multiple of 16
    int v_tiles, m_tiles;
    int stages, stage_bytes, tmem_cols;
    int activation;
    float scale;
    const float* bias;
    const void* residual;
    void* out;
    int64_t residual_stride, out_stride;
    int* dev_error;
    unsigned long long timeout_ns;
};

struct LinearShared {
    uint64_t full[kLinMaxStages], empty[kLinMaxStages];
    uint64_t acc_full[2], acc_empty[2], drained;
    uint32_t tmem;
    volatile int failed;
};

// Bounded wait of one thread; false once the limit has run out here or elsewhere in the CTA.
__device__ __forceinline__ bool lin_wait(LinearShared& sh, uint64_t* bar, uint32_t parity, unsigned long long limit_ns) {
    const uint32_t b = smem_u32(bar);
    if (ring_try(b, parity)) return true;
    unsigned long long t0 = 0;
    for (uint32_t it = 0; it < kMbarSpinLimit; ++it) {
        if (ring_try(b, parity)) return true;
        if ((it & 15u) == 15u) {
            if (sh.failed) return false;
            const unsigned long long now = global_timer_ns();
            if (t0 == 0) t0 = now;
            else if (now - t0 > limit_ns) break;
        }
    }
    sh.failed = 1;
    return false;
}

// Bounded wait whatever happened elsewhere.
__device__ __forceinline__ void lin_settle(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t it = 0; it < kMbarSpinLimit && !ring_try(bar, parity); ++it)
        if ((it & 15u) == 15u && global_timer_ns() - t0 > limit_ns) break;
}

// K-major operand with the 128-byte swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void activate(int activation, float scale, float (&v)[16]) {
    switch (activation) {
        case BORN_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
            break;
        case BORN_ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 1.0f / (1.0f + expf(-v[i]));
            break;
        case BORN_ACT_TANH:
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = scale * tanhf(v[i] / scale);
            break;
        case BORN_ACT_GELU:
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * (float)M_SQRT1_2));
            break;
        case BORN_ACT_SILU:
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = v[i] / (1.0f + expf(-v[i]));
            break;
        default: break;
    }
}

__device__ __forceinline__ float load_out(const float* p) { return *p; }
__device__ __forceinline__ float load_out(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename O>
__global__ void __launch_bounds__(kLinThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const LinearParams P) {
    extern __shared__ uint8_t raw[];
    __shared__ LinearShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;  // swizzle atoms start on 1024 bytes
    const int tiles = P.v_tiles * P.m_tiles;
    const int slices = (P.K + kLinK - 1) / kLinK;
    if (tid == 0) {
        for (int i = 0; i < P.stages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.acc_full[i], 1);
            mbar_init(&sh.acc_empty[i], 4);
        }
        mbar_init(&sh.drained, 1);
        sh.failed = 0;
        mbar_fence_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(P.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    const uint32_t x_at = kLinRows * kLinK * 2;  // the batch's slice behind the weights' one

    if (warp == 0 && lane == 0) {
        // ---- producer
        int stage = 0;
        uint32_t phase = 0;
        long long issued = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const int v0 = t / P.m_tiles * kLinRows, m0 = t % P.m_tiles * P.cols;
            for (int k = 0; k < slices; ++k) {
                if (!lin_wait(sh, &sh.empty[stage], phase ^ 1u, P.timeout_ns)) {
                    ok = false;
                    break;
                }
                const uint32_t bar = smem_u32(&sh.full[stage]), at = ring + (uint32_t)(stage * P.stage_bytes);
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(P.stage_bytes) : "memory");
                tma_load_2d(at, &wmap, k * kLinK, v0, bar);
                tma_load_2d(at + x_at, &xmap, k * kLinK, m0, bar);
                ++issued;
                if (++stage == P.stages) { stage = 0; phase ^= 1u; }
            }
        }
        // the copies in flight land before the CTA ends (bounded, whatever happened to the others)
        const int last = issued < P.stages ? (int)issued : P.stages;
        for (int i = 0; i < last; ++i) {
            if (--stage < 0) { stage = P.stages - 1; phase ^= 1u; }
            lin_settle(smem_u32(&sh.full[stage]), phase, P.timeout_ns);
        }
    } else if (warp == 1 && lane == 0) {
        // ---- products: D fp32, A and B bf16, both K-major, N = cols, M = 128
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(P.cols >> 3) << 17) | ((uint32_t)(kLinRows >> 4) << 24);
        int stage = 0, n = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++n) {
            const int acc = n & 1;
            if (!lin_wait(sh, &sh.acc_empty[acc], ((uint32_t)(n >> 1) & 1u) ^ 1u, P.timeout_ns)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + (uint32_t)(acc * P.cols);
            for (int k = 0; k < slices; ++k) {
                if (!lin_wait(sh, &sh.full[stage], phase, P.timeout_ns)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = ring + (uint32_t)(stage * P.stage_bytes);
                const uint64_t a = smem_desc(at), b = smem_desc(at + x_at);
#pragma unroll
                for (int i = 0; i < kLinK / 16; ++i) mma_bf16(d, a + 2 * i, b + 2 * i, idesc, (uint32_t)(k | i));
                mma_commit(&sh.empty[stage]);
                if (++stage == P.stages) { stage = 0; phase ^= 1u; }
            }
            if (ok) mma_commit(&sh.acc_full[acc]);
        }
        // tensor memory is given back only after the last product (bounded, like the copies)
        mma_commit(&sh.drained);
        lin_settle(smem_u32(&sh.drained), 0, P.timeout_ns);
    } else if (warp >= 4) {
        // ---- epilogue
        int n = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            const int acc = n & 1;
            int ok = 1;
            if (lane == 0) ok = lin_wait(sh, &sh.acc_full[acc], (uint32_t)(n >> 1) & 1u, P.timeout_ns);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            // (every lane observes the phase itself before it reads what the products wrote)
            ring_try(smem_u32(&sh.acc_full[acc]), (uint32_t)(n >> 1) & 1u);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int v = t / P.m_tiles * kLinRows + (warp - 4) * 32 + lane, m0 = t % P.m_tiles * P.cols;
            const int count = min(P.cols, P.M - m0);
            const uint32_t d = tmem + ((uint32_t)(warp - 4) << 21) + (uint32_t)(acc * P.cols);
            const bool in = v < P.V;
            const float bias = P.bias && in ? P.bias[v] : 0.0f;
            O* out = reinterpret_cast<O*>(P.out) + (int64_t)m0 * P.out_stride + v;
            const O* res = reinterpret_cast<const O*>(P.residual) + (int64_t)m0 * P.residual_stride + v;
            for (int c = 0; c < count; c += 16) {
                float y[16], r[16];
                tmem_load16(d + (uint32_t)c, y);
                if (P.residual) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) r[i] = in && c + i < count ? load_out(res + (int64_t)(c + i) * P.residual_stride) : 0.0f;
                }
                if (P.bias) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] += bias;
                }
                activate(P.activation, P.scale, y);
                if (P.residual) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] += r[i];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (in && c + i < count) store_out(out + (int64_t)(c + i) * P.out_stride, y[i]);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.acc_empty[acc]);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (tid == 0 && sh.failed) atomicExch(P.dev_error, BORN_ERR_DEVICE_TIMEOUT);
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols) : "memory");
}

}  // namespace born
