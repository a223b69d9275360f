// Rows of the caller's per-beam states follow the beams: new row b = old row parent[b], in place.
//
// A CTA owns one range of bytes of one piece of all rows of a group, so that no two CTAs touch the
// same bytes: a thread reads its vector of every row that is moved from, then writes those that are
// moved to, and no order of permutations or cycles matters.  Rows whose parent is themselves cost
// nothing.  Bound by the bytes that move: 128 rows of four buffers of 2 MB, 1.4 GB read and written, take 212 us, 6.5
// TB/s; 345 MB in pieces of 64 KB 57 us, their bytes 53.  Up to four beams have a kernel of their own, which fits four
// CTAs to an SM (216 us with the registers that sixteen need, 16 groups of 2 beams 88 instead of 83).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "beam_launch.cuh"

namespace born {

constexpr int kReorderThreads = 256;

// kM: moves that the registers hold at once (moves.n <= kM); vectors of W per thread and turn: 8 / kM
template <typename W, int kM>
__device__ __forceinline__ void move_bytes(uint8_t* base, int64_t row_stride, const int* dst, const int* src, int n, int64_t count) {
    constexpr int kU = kM >= 8 ? 1 : 8 / kM;
    for (int64_t i = threadIdx.x; i < count; i += (int64_t)kReorderThreads * kU) {
        W v[kM][kU];
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            if (m >= n) break;
            const W* p = reinterpret_cast<const W*>(base + src[m] * row_stride);
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (i + u * kReorderThreads < count) v[m][u] = p[i + u * kReorderThreads];
        }
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            if (m >= n) break;
            W* p = reinterpret_cast<W*>(base + dst[m] * row_stride);
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (i + u * kReorderThreads < count) p[i + u * kReorderThreads] = v[m][u];
        }
    }
}

// kMost: beams of a group at most
template <typename W, int kMost>
__global__ void __launch_bounds__(kReorderThreads, kMost <= 4 ? 4 : 2) reorder_kernel(const __grid_constant__ ReorderArgs A) {
    __shared__ int dst[BORN_MAX_BEAMS], src[BORN_MAX_BEAMS];
    __shared__ int n_moves;
    // (chunk, piece, buffer, group), the chunks of a piece first
    int64_t i = blockIdx.x;
    const int chunk = (int)(i % A.chunks);
    i /= A.chunks;
    const int plane = (int)(i % A.planes);
    i /= A.planes;
    const int buffer = (int)(i % A.n_buffers);
    const int n = (int)(i / A.n_buffers);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t used = A.positions;
    if (A.lens) {
        const int64_t len = A.lens[n];
        used = len < 0 ? 0 : len < used ? len : used;
    }
    used *= A.position_bytes;
    const int64_t at = chunk * A.chunk;
    if (at >= used) return;
    if (threadIdx.x < 32) {
        const int b = threadIdx.x;
        int p = b < A.K ? A.parents[(int64_t)n * A.K + b] : b;
        if (p < 0 || p >= A.K) p = b;
        const uint32_t moves = __ballot_sync(0xffffffffu, p != b);
        if (p != b) {
            const int k = __popc(moves & ((1u << b) - 1u));
            dst[k] = b;
            src[k] = p;
        }
        if (b == 0) n_moves = __popc(moves);
    }
    __syncthreads();
    const int m = n_moves;
    if (m == 0) return;
    const int64_t bytes = used - at < A.chunk ? used - at : A.chunk;
    uint8_t* base = A.buffers[buffer] + (int64_t)n * A.K * A.row_stride + plane * A.plane_stride + at;
    const int64_t count = bytes / (int64_t)sizeof(W);
    if (m == 1) move_bytes<W, 1>(base, A.row_stride, dst, src, m, count);
    else if (m == 2) move_bytes<W, 2>(base, A.row_stride, dst, src, m, count);
    else if (kMost <= 4 || m <= 4) move_bytes<W, 4>(base, A.row_stride, dst, src, m, count);
    else if (m <= 8) move_bytes<W, kMost <= 4 ? 4 : 8>(base, A.row_stride, dst, src, m, count);
    else move_bytes<W, kMost <= 4 ? 4 : 16>(base, A.row_stride, dst, src, m, count);
    if constexpr (sizeof(W) > 1) {
        const int64_t rest = bytes - count * (int64_t)sizeof(W);
        if (rest) move_bytes<uint8_t, kMost>(base + count * (int64_t)sizeof(W), A.row_stride, dst, src, m, rest);
    }
}

}  // namespace born
