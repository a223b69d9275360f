// Sequences of hypotheses out of the tables that the steps of a beam search wrote.
//
// Following the parents back is a chain of dependent reads, one per step: 4096 steps would take a
// millisecond of latency.  A step's parents are a map of at most 16 beams to 16 beams, and maps compose.  So a group's
// CTAs (one, for long tables a cluster of two or four) bring parents and tokens of a tile of steps into shared memory, cut the
// steps into 32 chunks each, a half warp per chunk, and compose every chunk's map; a lane per hypothesis walks over all
// chunks' maps; then all chunks are walked at once, and the tokens are picked and written along the steps.  Longer
// tables go tile by tile, from the end.
// Bound by a chain of phases: of the 20 us that 64 groups of 8 beams and 4096 steps take (their bytes 3.9) the tables' short
// pieces (a group's beams of each row) are 5.6, the chunks' maps and their exchange 3.4, the look-up over 128 chunks and the second
// walk 5.2, the tokens 2.2, start and end 2.4 (clock stamps).  47 us when every chunk reads its own parents and tokens as it
// walks, 36 with the parents alone in shared memory, 26 with all of it in one CTA.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "beam_launch.cuh"
#include "scan_common.cuh"

namespace born {

constexpr int kSeqThreads = 512;
constexpr int kSeqChunks = kSeqThreads / 16;  // of a CTA
constexpr int kSeqRanks = 4;                  // CTAs of a group at most
constexpr uint32_t kNoLink = 0x80u;

__global__ void __launch_bounds__(kSeqThreads, 2) sequences_kernel(const SequencesArgs A) {
    extern __shared__ __align__(16) int32_t token_at[];  // [tile][width] tokens; then parents and beams, a byte each
    __shared__ __align__(16) int8_t map[kSeqRanks * kSeqChunks][BORN_MAX_BEAMS];  // beam of a chunk's last step -> beam below its first
    __shared__ int8_t entry[kSeqRanks * kSeqChunks][BORN_MAX_BEAMS];  // beam of hypothesis h at a chunk's last step
    __shared__ int8_t low[BORN_MAX_BEAMS];                // ... below the chunk in which it ends
    __shared__ int8_t carry[BORN_MAX_BEAMS];              // ... at the last step of the tile that comes next
    __shared__ int ends[BORN_MAX_BEAMS];
    __shared__ int32_t last[BORN_MAX_BEAMS];
    const int R = A.ranks, n = (int)blockIdx.x / R, rank = (int)blockIdx.x % R;
    const int tid = threadIdx.x, chunk = rank * kSeqChunks + (tid >> 4), l = tid & 15;
    const int K = A.K, T = A.T, H = A.H, shift = A.shift, W = 1 << shift;
    uint8_t* link = reinterpret_cast<uint8_t*>(token_at + A.tile * W);  // a step's parents; kNoLink: none
    uint8_t* beam = link + A.tile * W;                                  // beams of the hypotheses at a step
    const int turn = 5 - shift;  // tokens of a step are turned round, so that a beam's are in different banks
    __syncwarp();
    cluster_arrive();  // (the others' shared memory is there)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int32_t* parents = A.parents + (int64_t)n * K;
    const int32_t* tokens = A.tokens + (int64_t)n * K;
    int32_t* out = A.out_tokens + (int64_t)n * H * A.out_stride;
    // hypothesis l: its last step (-1: empty) and the beam before it
    int e = -1, first = 0;
    if (l < H) {
        e = A.end_step[(int64_t)n * H + l];
        first = A.end_parent[(int64_t)n * H + l];
        if (tid < 16) last[l] = A.end_token[(int64_t)n * H + l];
    }
    if (e < 0 || e >= T || first < 0 || first >= K) e = -1;
    if (tid < 16) {
        ends[l] = e;
        carry[l] = 0;
    }
    bool first_tile = true;
    for (int tile = (T - 1) / (A.tile * R); tile >= 0; --tile) {
        // the cluster's steps base0 ..., of them this CTA's base ...; chunks in the cluster's numbers
        const int base0 = tile * A.tile * R, all = min(A.tile * R, T - base0);
        const int C = (all + kSeqChunks * R - 1) / (kSeqChunks * R), from = min(rank * kSeqChunks * C, all);
        const int base = base0 + from, steps = min(kSeqChunks * C, all - from);
        const int lo = (tid >> 4) * C, hi = min(steps, lo + C);
        // ---- the tables' rows; before step 0 a beam's parent is itself
        for (int i0 = tid; i0 < steps << shift; i0 += 8 * kSeqThreads) {
            int32_t p[8], v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u * kSeqThreads, t = i >> shift, b = i & (W - 1);
                const bool ok = t < steps && b < K;
                p[u] = ok ? parents[(int64_t)(base + t) * A.table_stride + b] : 0;
                v[u] = ok ? tokens[(int64_t)(base + t) * A.table_stride + b] : 0;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u * kSeqThreads, t = i >> shift, b = i & (W - 1);
                if (t >= steps) break;
                link[i] = (uint8_t)(base + t == 0 ? b : p[u] < 0 || p[u] >= K ? kNoLink : p[u]);
                token_at[(t << shift) + ((b + (t >> turn)) & (W - 1))] = v[u];
            }
        }
        __syncthreads();
        if (first_tile) cluster_wait();
        first_tile = false;
        // ---- the chunks' maps, and the hypotheses from their end to the bottom of its chunk
        const int at = e - 1 - base, at0 = e - 1 - base0;  // the hypothesis joins here
        const bool joins = e > 0 && at0 >= 0 && at0 < all;
        {
            uint32_t r = l & (W - 1), b = 0, bad_r = 0, bad_b = 0;
            const uint8_t* row = link + (hi << shift);
            for (int t = hi - 1; t >= lo; --t) {
                row -= W;
                if (t == at) {
                    b = first;
                    bad_b = 0;
                }
                r = row[r];
                b = row[b];
                bad_r |= r;
                bad_b |= b;
                r &= 15u;
                b &= 15u;
            }
            map[chunk][l] = (int8_t)(bad_r & kNoLink ? -1 : (int)r);
            if (joins && at0 / C == chunk)
                for (int k = 0; k < R; ++k) *cluster_map(&low[l], k) = (int8_t)(bad_b & kNoLink ? -1 : (int)b);
        }
        __syncwarp();
        if (l < R && l != rank) *cluster_map(reinterpret_cast<uint4*>(map[chunk]), l) = *reinterpret_cast<const uint4*>(map[chunk]);
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        // ---- from chunk to chunk; a missing link empties the hypothesis.  (A lane holds a map's entry for its beam and
        // looks the beam it is at up in the others' registers: the maps are read ahead of the chain.)
        if (tid < 16) {
            const int top = (all - 1) / C;
            const bool walks = joins || e - 1 >= base0 + all;
            int c0 = -2, b = 0;  // where it starts: below chunk c0 + 1, at b
            if (walks) {
                c0 = joins ? at0 / C - 1 : top;
                b = joins ? low[l] : carry[l];
            }
#pragma unroll 4
            for (int c = top; c >= 0; --c) {
                const int to = map[c][l];
                entry[c][l] = (int8_t)b;
                const int below = __shfl_sync(0xffffu, to, b & 15, 16);
                if (c <= c0 && b >= 0) b = below;
            }
            if (walks) {
                carry[l] = (int8_t)max(b, 0);
                if (b < 0) ends[l] = e = -2;  // (written before it was known: see below)
            }
        }
        __syncthreads();
        if (ends[l] < 0) e = ends[l];
        // ---- the hypotheses' beams, step by step
        {
            uint32_t b = e - 1 >= base + hi ? entry[chunk][l] : 0;
            int i = hi << shift;
            for (int t = hi - 1; t >= lo; --t) {
                i -= W;
                if (t == at) b = first;
                if (l < H) beam[i + l] = (uint8_t)b;
                b = link[i + b] & 15u;
            }
        }
        __syncthreads();
        // ---- the tokens
        for (int h = 0; h < H; ++h) {
            const int eh = ends[h] - base;
            for (int t = tid; t < steps; t += kSeqThreads)
                out[h * A.out_stride + base + t] = t < eh ? token_at[(t << shift) + ((beam[(t << shift) + h] + (t >> turn)) & (W - 1))] : t == eh ? last[h] : A.pad;
        }
        __syncwarp();
        cluster_arrive();  // (maps that are still walked over; and nothing is written into a CTA that has ended)
        cluster_wait();
    }
    if (rank != 0) return;
    if (tid < H) A.out_lens[(int64_t)n * H + tid] = max(ends[tid], -1) + 1;
    // hypotheses whose missing link lay in an earlier tile than tokens already written
    if (T > A.tile * R)
        for (int h = 0; h < H; ++h)
            if (ends[h] == -2)
                for (int t = tid; t < T; t += kSeqThreads) out[h * A.out_stride + t] = A.pad;
}

}  // namespace born
