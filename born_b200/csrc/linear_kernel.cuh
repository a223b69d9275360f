// out[m][v] = act(sum_k x[m][k] weight[v][k] + bias[v]) + residual[m][v] on the tensor cores.
//
// A decode batch has few rows and a vocabulary many, so the weights take the tile's 128 rows and the
// batch its columns (16 to 256): D[128 v][n m] = W[128][K] X[n][K]^T, both operands K-major as they lie in
// memory.  A CTA per SM walks over tiles; a warp fills a ring of 64-element slices of both operands by
// TMA (128-byte swizzle), a warp issues the tcgen05 products into one of two accumulators in tensor
// memory, eight warps empty the other one: a lane holds one v, so that a column of 32 lanes is a
// contiguous piece of an output row.
//
// Two CTAs share a tile of 256 v from 65 columns on (kPair): each holds its own 128 rows of weights and half
// of the batch's rows, which the other one's tensor core reads too.  One CTA alone reads the batch's slice
// for every 128 rows of weights, and 256 columns of it twice the weights' bytes: out of L2, 256 rows of hidden
// 4096 over 128256 features took 330 us with that.
//
// The tensor core cuts partial sums off rather than rounding them, once per 16 products, which adds up: 4.3e-6 of
// the result at K = 4096.  So it sums 512 products at most; those sums are added in registers, rounded: 3.9e-7 there (products and
// sums in fp32 have 5.9e-7), 4.1e-7 at K = 1000 (2.2e-7).  Shorter sums would keep more and empty the accumulators more often.
//
// Where the tiles are too few for the GPU, the CTAs (or pairs) of a cluster share one, each with a part of K (splits).  They
// leave their sums in the place of their rings; every CTA adds up a share of the columns out of all of them, in the
// order of the parts, and finishes those.  8192 x 1024 weights for one row: 45 us on the eight SMs that have a tile, 15
// with the sums in scratch and the last CTA adding them up, 6.8 so.
//
// One thread's instructions set the pace wherever the slices are small: wait, fence, four products, arrival took 600 cycles
// a slice, whatever its bytes.  So a ring stage has two slices (256 x 8192 x 2000 24 -> 20.5 us), and the warps that load and that
// issue products stay together with one elected lane (-> 17.8): their loops run on the uniform side.
//
// What bounds it, hidden 4096, 128256 features: the bytes of the weights for few rows (1 row 158 us, 64 rows 167, of 161 and
// 166), then what L2 hands out of weights and batch together (128 rows 180, of 171); 256 rows 224 to 229 us after a pause, 181 of
// bytes and 160 of products.  In a loop of seconds the GPU is at its power limit: 256 rows with tanh 288 to 297 us, 235 to 241 after a
// pause.
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

constexpr int kLinRows = 128;      // v of a CTA's tile
constexpr int kLinK = 64;          // elements of a slice: 128 bytes, one swizzle atom
constexpr int kLinChunk = 8;       // slices that the tensor core sums
constexpr int kLinMaxCols = 256;   // m of a tile
constexpr int kLinMaxStages = 12;
constexpr int kLinDeep = 2;        // slices of a ring stage
constexpr int kLinThreads = 384;   // warps: 0 TMA, 1 products, 2 tensor memory, 3 idle, 4..11 epilogue
constexpr int kLinSmem = 220 * 1024;

struct LinearParams {
    int M, K, V;
    int cols;          // m of a tile
    int v_tiles, m_tiles;
    int splits, part;  // CTAs (pairs) of a tile; slices of each
    int stages, slice_bytes, tmem_cols;  // of a CTA
    int activation;
    float scale, inv_scale;
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
// Waits for a phase until `until` (a time) at most, whatever happened elsewhere.
__device__ __forceinline__ void lin_settle(uint32_t bar, uint32_t parity, unsigned long long until) {
    for (uint32_t it = 0; it < kMbarSpinLimit && !ring_try(bar, parity); ++it)
        if ((it & 15u) == 15u && global_timer_ns() > until) break;
}

__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}
// K-major operand with the 128-byte swizzle: groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// bar: address in the cluster; in kPair of the pair's first CTA, whose bytes both CTAs' copies count towards
template <bool kPair>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (kPair)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                     "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
}
template <bool kPair>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Shared memory of the cluster's CTA `rank`, at the place that `at` is in this one.
__device__ __forceinline__ uint32_t remote_smem(uint32_t at, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at), "r"(rank));
    return a;
}
__device__ __forceinline__ float load_remote(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
// pair: rank of the pair's first CTA in the cluster.  An arrival, once the products issued so far are done, at the barrier (of both CTAs in kPair).
template <bool kPair>
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t pair) {
    if constexpr (kPair)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"((uint16_t)(3u << pair))
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// An arrival at the barrier of the pair's first CTA.  What it orders are reads of tensor memory that tcgen05.wait::ld has
// seen done; a release to the whole cluster would wait for the output's stores as well (128 rows of hidden 1024, 151936
// features 73.6 -> 70.1 us without, 256 rows of hidden 4096, 128256 features with tanh 265 -> 257.5).
__device__ __forceinline__ void arrive_first(uint64_t* bar, uint32_t pair) {
    const uint32_t a = remote_smem(smem_u32(bar), (int)pair);
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 16 columns of the accumulator.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}

// y (1 + erf(y/sqrt 2)) / 2 as max(y, 0) - |y| erfc(|y|/sqrt 2) / 2: 1 + erf has no digits left below -5, this one all of them.
// erfc(x) = exp(-x^2) erfcx(x), and half of erfcx(|y|/sqrt 2) is a polynomial in 1/(1 + 0.3 |y|), fitted at Chebyshev nodes (least
// squares, reweighted towards the largest relative error, 2^-24) up to |y| = 14.5; exp(-y^2/2) is 0 behind that.  (256 rows of hidden
// 4096, 128256 features: 240 us; with erfcf 269, with the cancelling 1 + erff 244.)
__device__ __forceinline__ float gelu(float y) {
    const float a = fabsf(y);
    float s;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(__fmaf_rn(a, 0.3f, 1.0f)));
    float p = 3.8407404e-2f;
    p = __fmaf_rn(p, s, -1.6930752e-1f);
    p = __fmaf_rn(p, s, 2.2895190e-1f);
    p = __fmaf_rn(p, s, -7.6839767e-2f);
    p = __fmaf_rn(p, s, 1.4276534e-1f);
    p = __fmaf_rn(p, s, 9.4585836e-2f);
    p = __fmaf_rn(p, s, 1.2194527e-1f);
    p = __fmaf_rn(p, s, 1.1948421e-1f);
    p = __fmaf_rn(p, s, 7.3724286e-6f);
    const float e = exp2f(y * y * -0.72134752f);
    const float q = (y < 32.0f ? a : 32.0f) * p * e;  // (inf - 0; NaN comes in by the other part)
    return (y < 0.0f ? 0.0f : y) - q;
}

template <int N>
__device__ __forceinline__ void activate(const LinearParams& P, float (&v)[N]) {
    switch (P.activation) {
        case BORN_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // (NaN stays)
            break;
        case BORN_ACT_SIGMOID:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 1.0f / (1.0f + expf(-v[i]));
            break;
        case BORN_ACT_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = P.scale * tanhf(v[i] * P.inv_scale);
            break;
        case BORN_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = gelu(v[i]);
            break;
        case BORN_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] / (1.0f + expf(-v[i]));
            break;
        default: break;
    }
}

__device__ __forceinline__ float load_out(const float* p) { return *p; }
__device__ __forceinline__ float load_out(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// kCols: columns of the tile that a thread of the epilogue holds at most (the two groups of four warps take half
// of the tile's columns each, or the first one all 16).
template <typename O, int kCols, bool kPair>
__global__ void __launch_bounds__(kLinThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ LinearParams P) {
    extern __shared__ uint8_t raw[];
    __shared__ LinearShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // (known to be uniform)
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;  // swizzle atoms start on 1024 bytes
    const int rank = kPair ? (int)(blockIdx.x & 1u) : 0;     // in the pair
    const uint32_t pair = kPair ? (blockIdx.x & ~1u) % (2u * (uint32_t)P.splits) : 0;  // its first CTA's rank in the cluster
    float* sums = reinterpret_cast<float*>(raw + (ring - smem_u32(raw)));
    const int first = kPair ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, step = kPair ? (int)(gridDim.x >> 1) : (int)gridDim.x;
    const int units = P.v_tiles * P.m_tiles * P.splits;      // tiles, times the parts of K
    const int all_slices = (P.K + kLinK - 1) / kLinK;
    const int groups = P.cols > 16 ? 2 : 1;          // of warps that take part in the epilogue
    constexpr int kTileRows = kPair ? 2 * kLinRows : kLinRows;  // v of a unit
    const int stage_bytes = kLinDeep * P.slice_bytes;
    const auto first_v = [&](int t) { return t / P.m_tiles * kTileRows + rank * kLinRows; };  // of a tile in this CTA
    if (tid == 0) {
        for (int i = 0; i < P.stages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.acc_full[i], 1);
            mbar_init(&sh.acc_empty[i], (uint32_t)(4 * groups * (kPair ? 2 : 1)));
        }
        mbar_init(&sh.drained, 1);
        sh.failed = 0;
        mbar_fence_init();
    }
    if (warp == 2) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(P.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(P.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    const uint32_t x_at = kLinRows * kLinK * 2;  // the batch's slice behind the weights' one
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        // ---- producer: this CTA's rows of weights, its share of the batch's.  (The whole warp, like the products'.)
        const bool issues = elected();
        const uint32_t counts = kPair ? remote_smem(smem_u32(&sh.full[0]), (int)pair) : smem_u32(&sh.full[0]);
        int stage = 0;
        uint32_t phase = 0;
        long long issued = 0;
        bool ok = true;
        for (int u = first; u < units && ok; u += step) {
            const int t = u / P.splits, s0 = (u - t * P.splits) * P.part, slices = min(P.part, all_slices - s0);
            const int v0 = first_v(t);
            const int m0 = t % P.m_tiles * P.cols + (kPair ? rank * (P.cols / 2) : 0);
            for (int k = 0; k < slices; k += kLinDeep) {
                if (!__all_sync(0xffffffffu, lin_wait(sh, &sh.empty[stage], phase ^ 1u, P.timeout_ns))) {
                    ok = false;
                    break;
                }
                const uint32_t bar = counts + (uint32_t)stage * 8u, at = ring + (uint32_t)(stage * stage_bytes);
                const int n = min(kLinDeep, slices - k);
                if (issues) {
                    if (rank == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&sh.full[stage])), "r"(n * P.slice_bytes * (kPair ? 2 : 1)) : "memory");
#pragma unroll
                    for (int j = 0; j < kLinDeep; ++j) {
                        if (j >= n) break;
                        const uint32_t to = at + (uint32_t)(j * P.slice_bytes);
                        tma_load_2d<kPair>(to, &wmap, (s0 + k + j) * kLinK, v0, bar);
                        tma_load_2d<kPair>(to + x_at, &xmap, (s0 + k + j) * kLinK, m0, bar);
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == P.stages) { stage = 0; phase ^= 1u; }
            }
        }
        // What is on its way into this CTA arrives before the CTA ends (bounded, whatever happened to the others): the
        // copies, and the products' arrivals, which in a pair come from the other CTA.  The first CTA's barriers count the second
        // one's copies too, and neither ends before the other; a copy that the second one alone has issued, where the
        // first one gave up, gets the time of a wait.
        const unsigned long long until = global_timer_ns() + P.timeout_ns;
        if (kPair && rank == 0 && !ok) lin_settle(smem_u32(&sh.full[stage]), phase, until);
        for (int i = issued < P.stages ? (int)issued : P.stages; i > 0; --i) {
            if (--stage < 0) { stage = P.stages - 1; phase ^= 1u; }
            if (rank == 0) lin_settle(smem_u32(&sh.full[stage]), phase, until);
            lin_settle(smem_u32(&sh.empty[stage]), phase, until);
        }
        if (rank != 0) lin_settle(smem_u32(&sh.drained), 0, until);
    } else if (warp == 1 && rank == 0) {
        // ---- products: D fp32, A and B bf16, both K-major.  The whole warp goes along, one lane issues.
        const bool issues = elected();
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(P.cols >> 3) << 17) | ((uint32_t)((kPair ? 2 * kLinRows : kLinRows) >> 4) << 24);
        int stage = 0, n = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = first; u < units && ok; u += step) {
            const int t = u / P.splits, s0 = (u - t * P.splits) * P.part, slices = min(P.part, all_slices - s0);
            for (int k0 = 0; k0 < slices && ok; k0 += kLinChunk, ++n) {
                const int acc = n & 1;
                if (!__all_sync(0xffffffffu, lin_wait(sh, &sh.acc_empty[acc], ((uint32_t)(n >> 1) & 1u) ^ 1u, P.timeout_ns))) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + (uint32_t)(acc * P.cols);
                const int k1 = min(slices, k0 + kLinChunk);
                for (int k = k0; k < k1; k += kLinDeep) {
                    if (!__all_sync(0xffffffffu, lin_wait(sh, &sh.full[stage], phase, P.timeout_ns))) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (issues) {
#pragma unroll
                        for (int j = 0; j < kLinDeep; ++j) {
                            if (k + j >= k1) break;
                            const uint32_t at = ring + (uint32_t)(stage * stage_bytes + j * P.slice_bytes);
                            const uint64_t a = smem_desc(at), b = smem_desc(at + x_at);
#pragma unroll
                            for (int i = 0; i < kLinK / 16; ++i) mma_bf16<kPair>(d, a + 2 * i, b + 2 * i, idesc, (uint32_t)((k + j - k0) | i));
                        }
                        mma_commit<kPair>(&sh.empty[stage], pair);
                    }
                    __syncwarp();
                    if (++stage == P.stages) { stage = 0; phase ^= 1u; }
                }
                if (ok && issues) mma_commit<kPair>(&sh.acc_full[acc], pair);
                __syncwarp();
            }
        }
        // tensor memory is given back only after the last product (bounded, like the copies; in a pair either CTA
        // waits for its own arrival: the second one's load warp does)
        if (issues) mma_commit<kPair>(&sh.drained, pair);
        lin_settle(smem_u32(&sh.drained), 0, global_timer_ns() + P.timeout_ns);
    } else if (warp >= 4 && (warp - 4) >> 2 < groups) {
        // ---- epilogue
        const int group = (warp - 4) >> 2, quad = warp & 3;
        const int half = P.cols / groups, c0 = group * half;  // its columns
        const int r0 = quad * 32 + lane;  // its v
        const uint32_t d0 = tmem + ((uint32_t)quad << 21) + (uint32_t)c0;
        int n = 0;
        bool ok = true;
        for (int u = first; u < units && ok; u += step) {
            const int t = u / P.splits, s0 = (u - t * P.splits) * P.part, slices = min(P.part, all_slices - s0);
            const int v = first_v(t) + r0, m0 = t % P.m_tiles * P.cols + c0;
            const int count = min(half, P.M - m0);  // (none for a group whose columns lie behind the batch)
            const bool in = v < P.V;
            const float bias = P.bias && in ? P.bias[v] : 0.0f;
            float y[kCols];
            for (int k0 = 0; k0 < slices; k0 += kLinChunk, ++n) {
                const int acc = n & 1;
                int got = 1;
                if (lane == 0) got = lin_wait(sh, &sh.acc_full[acc], (uint32_t)(n >> 1) & 1u, P.timeout_ns);
                ok = __shfl_sync(0xffffffffu, got, 0) != 0;
                if (!ok) break;
                // (every lane observes the phase itself before it reads what the products wrote)
                ring_try(smem_u32(&sh.acc_full[acc]), (uint32_t)(n >> 1) & 1u);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = d0 + (uint32_t)(acc * P.cols);
#pragma unroll
                for (int c = 0; c < kCols; c += 16) {
                    if (c >= half) break;
                    uint32_t r[16];
                    tmem_load16(d + (uint32_t)c, r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (k0 == 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[c + i] = __uint_as_float(r[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[c + i] += __uint_as_float(r[i]);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if constexpr (kPair) arrive_first(&sh.acc_empty[acc], pair);
                    else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sh.acc_empty[acc])) : "memory");
                }
            }
            if (P.splits > 1) {  // (every slice has been used up: the sums take the ring's place)
                float* to = sums + c0 * kLinRows + r0;
#pragma unroll
                for (int c = 0; c < kCols; ++c)
                    if (c < half) to[c * kLinRows] = y[c];
                continue;
            }
            if (!ok) break;
            O* out = reinterpret_cast<O*>(P.out) + (int64_t)m0 * P.out_stride + v;
            const O* res = reinterpret_cast<const O*>(P.residual) + (int64_t)m0 * P.residual_stride + v;
            if (P.bias) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) y[c] += bias;
            }
            if (P.activation == BORN_ACT_NONE && !P.residual) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    if (in && c < count) store_out(out, y[c]);
                    out += P.out_stride;
                }
                continue;
            }
            // (16 columns at a time, those behind them moved up: with all 128 unrolled the code does not stay in the
            // instruction cache: of 256 rows of 128256 features gelu took 110 us and tanh 26, now 16 and 12)
#pragma unroll 1
            for (int c = 0; c < count; c += 16) {
                activate(P, reinterpret_cast<float(&)[16]>(y));
                if (P.residual) {
                    float r[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        r[i] = in && c + i < count ? load_out(res) : 0.0f;
                        res += P.residual_stride;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] += r[i];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (in && c + i < count) store_out(out, y[i]);
                    out += P.out_stride;
                }
#pragma unroll
                for (int i = 0; i + 16 < kCols; ++i) y[i] = y[i + 16];
            }
        }
    }
    __syncwarp();
    if (P.splits > 1) {
        // ---- the parts of K: a CTA of the cluster adds up its share of the columns and finishes them
        cluster_sync();
        const int S = P.splits, t = first / S, row = tid % kLinRows, v = first_v(t) + row, m0 = t % P.m_tiles * P.cols;
        const int cols = min(P.cols, P.M - m0), stride = kLinThreads / kLinRows * S;
        const float bias = P.bias && v < P.V ? P.bias[v] : 0.0f;
        for (int c = first % S + tid / kLinRows * S; c < cols; c += 4 * stride) {
            float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int s = 0; s < S; ++s) {
                const uint32_t from = remote_smem(ring + (uint32_t)((c * kLinRows + row) * 4), kPair ? 2 * s + rank : s);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j * stride < cols) z[j] += load_remote(from + (uint32_t)(j * stride * kLinRows * 4));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] += bias;
            activate(P, z);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + c + j * stride;
                if (c + j * stride >= cols || v >= P.V) break;
                if (P.residual) z[j] += load_out(reinterpret_cast<const O*>(P.residual) + (int64_t)m * P.residual_stride + v);
                store_out(reinterpret_cast<O*>(P.out) + (int64_t)m * P.out_stride + v, z[j]);
            }
        }
        __syncwarp();
        if constexpr (!kPair) cluster_sync();  // (the others have read this CTA's sums)
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kPair) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (tid == 0 && sh.failed) atomicExch(P.dev_error, BORN_ERR_DEVICE_TIMEOUT);
    if (warp == 2) {
        if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols) : "memory");
    }
}

}  // namespace born
