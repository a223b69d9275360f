// Sequences of hypotheses out of the tables that the steps of a beam search wrote.
//
// Following the parents back is a chain of dependent reads, one per step.  A step's parents are a map of
// at most 16 beams to 16 beams, 64 bits; maps compose, so a CTA (one per group) cuts the steps into a
// chunk per thread, composes each chunk's map, and from tables of the maps over 2, 4, 8, ... chunks
// every thread learns in eight look-ups at which beam each hypothesis enters its chunk.  The walks inside
// the chunks then run side by side.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "beam_launch.cuh"

namespace born {

constexpr int kSeqThreads = 256;
constexpr int kSeqLevels = 8;
constexpr unsigned long long kIdentity = 0xfedcba9876543210ull;

// A map of beams: nibble b holds the beam that b came from; bit b of bad: it came from none.
struct BeamMap {
    unsigned long long to;
    uint32_t bad;
};
__device__ __forceinline__ int map_at(unsigned long long to, int b) { return (int)(to >> (4 * b)) & 15; }
// first `a` (later steps), then `b` (earlier ones)
__device__ __forceinline__ BeamMap compose(const BeamMap& a, const BeamMap& b) {
    BeamMap r;
    r.to = 0;
    r.bad = a.bad;
#pragma unroll
    for (int i = 0; i < BORN_MAX_BEAMS; ++i) {
        const int m = map_at(a.to, i);
        r.to |= (unsigned long long)map_at(b.to, m) << (4 * i);
        r.bad |= ((b.bad >> m) & 1u) << i;
    }
    return r;
}

struct SeqShared {
    unsigned long long to[kSeqLevels][kSeqThreads];
    uint16_t bad[kSeqLevels][kSeqThreads];
    int entry[BORN_MAX_BEAMS];   // beam at the bottom of the chunk in which the hypothesis ends, -1 = bad
    int end[BORN_MAX_BEAMS], first[BORN_MAX_BEAMS];
};

__global__ void __launch_bounds__(kSeqThreads) sequences_kernel(const SequencesArgs A) {
    extern __shared__ unsigned long long step_to[];  // [T], then step_bad [T] (16 bits each)
    __shared__ SeqShared sh;
    uint16_t* step_bad = reinterpret_cast<uint16_t*>(step_to + A.T);
    const int n = blockIdx.x, tid = threadIdx.x;
    const int K = A.K, T = A.T, H = A.H;
    const int32_t* parents = A.parents + (int64_t)n * K;
    const int32_t* tokens = A.tokens + (int64_t)n * K;
    const int C = (T + kSeqThreads - 1) / kSeqThreads;  // steps of a thread

    // Map of step t: beam of step t -> beam of step t - 1 (there is none before step 0: the identity).
    for (int t = tid; t < T; t += kSeqThreads) {
        unsigned long long to = t ? 0 : kIdentity;
        uint32_t bad = 0;
        for (int b = 0; b < K && t; ++b) {
            const int p = parents[t * A.table_stride + b];
            if (p < 0 || p >= K) bad |= 1u << b;
            else to |= (unsigned long long)p << (4 * b);
        }
        step_to[t] = to;
        step_bad[t] = (uint16_t)bad;
    }
    __syncthreads();
    // Map of chunk c: beam of its last step -> beam of the step before its first.
    {
        BeamMap m = {kIdentity, 0};
        for (int t = min(T, (tid + 1) * C) - 1; t >= tid * C; --t) m = compose(m, BeamMap{step_to[t], step_bad[t]});
        sh.to[0][tid] = m.to;
        sh.bad[0][tid] = (uint16_t)m.bad;
    }
    __syncthreads();
    // level l: the maps of 2^l chunks, the last of which is c
    for (int l = 1; l < kSeqLevels; ++l) {
        const int d = 1 << (l - 1);
        if (tid >= 2 * d - 1) {
            const BeamMap m = compose(BeamMap{sh.to[l - 1][tid], sh.bad[l - 1][tid]}, BeamMap{sh.to[l - 1][tid - d], sh.bad[l - 1][tid - d]});
            sh.to[l][tid] = m.to;
            sh.bad[l][tid] = (uint16_t)m.bad;
        }
        __syncthreads();
    }
    // The hypotheses: from their end to the bottom of its chunk, then all the way to see that no link is missing.
    if (tid < H) {
        int e = A.end_step[(int64_t)n * H + tid];
        const int p = A.end_parent[(int64_t)n * H + tid];
        if (e < 0 || e >= T || p < 0 || p >= K) e = -1;
        int b = p, low = -1;
        if (e >= 0) {
            int t = e - 1;
            const int c = t >= 0 ? t / C : 0;
            for (; t >= c * C && b >= 0; --t) b = (step_bad[t] >> b) & 1 ? -1 : map_at(step_to[t], b);
            low = b;
            int at = c - 1;
            for (int l = kSeqLevels - 1; l >= 0 && b >= 0; --l) {
                if (at + 1 < (1 << l)) continue;
                b = (sh.bad[l][at] >> b) & 1 ? -1 : map_at(sh.to[l][at], b);
                at -= 1 << l;
            }
            if (b < 0) e = -1;
        }
        sh.end[tid] = e;
        sh.first[tid] = p;
        sh.entry[tid] = low;
        A.out_lens[(int64_t)n * H + tid] = e + 1;
    }
    __syncthreads();
    const int lo = tid * C, hi = min(T, lo + C);
    for (int h = 0; h < H; ++h) {
        const int e = sh.end[h];
        int32_t* out = A.out_tokens + ((int64_t)n * H + h) * A.out_stride;
        int b = -1;
        if (e - 1 >= lo && e - 1 < hi) b = sh.first[h];
        else if (e - 1 >= hi) {
            b = sh.entry[h];
            int at = (e - 1) / C - 1;
            for (int l = kSeqLevels - 1; l >= 0; --l) {
                if (at - tid < (1 << l)) continue;
                b = map_at(sh.to[l][at], b);
                at -= 1 << l;
            }
        }
        for (int t = hi - 1; t >= lo; --t) {
            int32_t v = A.pad;
            if (t == e) v = A.end_token[(int64_t)n * H + h];
            else if (t < e) {
                v = tokens[t * A.table_stride + b];
                b = map_at(step_to[t], b);
            }
            out[t] = v;
        }
    }
}

}  // namespace born
