// One step of beam search over [groups * beams, vocab] logits, in one launch.
//
// Every row is cut into slices, a CTA each.  A CTA streams its slice once: the running maximum m and
// s = sum exp((z - m)/T) per thread, and per warp the best `beams` tokens as a sorted list held
// across the lanes.  It leaves (m, s, list) as a record; the CTA of a group that draws the group's
// last ticket ranks the candidates of all rows by
//     score[b] + (z - m_b)/T - log s_b
// in 64 bits, arranges the children and writes them out.  No CTA waits for another one.
//
// The normaliser of a row is the only rounded part of that value: tokens of one row order by their
// logits alone.  It comes from 32-bit exponentials, off by less than A.slack / 2 (beam_slack); where two
// candidates of different rows are nearer than A.slack and the order matters, the CTA recomputes the
// normalisers of those rows in 64 bits (row_normaliser), so that the order is that of the definition.
//
// What bounds it: the bytes of the logits.
#pragma once
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include "beam_launch.cuh"
#include "scan_common.cuh"

namespace born {

constexpr int kBeamWarps = kThreads / 32;
constexpr uint32_t kNoCandidate = 0xffffffffu;

struct BeamShared {
    unsigned long long lists[kBeamWarps][BORN_MAX_BEAMS];  // the warps' lists; then the rows' lists
    unsigned long long row_list[BORN_MAX_BEAMS][BORN_MAX_BEAMS];
    double value[BORN_MAX_BEAMS * (BORN_MAX_BEAMS + BORN_MAX_STOPS)];
    uint32_t flat[BORN_MAX_BEAMS * (BORN_MAX_BEAMS + BORN_MAX_STOPS)];  // beam << 24 | token of the candidate
    double offset[BORN_MAX_BEAMS];  // score - log s of the rows
    float row_max[BORN_MAX_BEAMS];
    double dsum[kBeamWarps];
    float fmx[kBeamWarps];
    unsigned long long thr;  // the best of the warps' last list entries: no token below it matters
    float stop_z[BORN_MAX_STOPS];
    float row_stop[BORN_MAX_BEAMS][BORN_MAX_STOPS];
    int32_t status[BORN_MAX_BEAMS];
    int32_t sel_parent[BORN_MAX_BEAMS], sel_token[BORN_MAX_BEAMS];
    double sel_value[BORN_MAX_BEAMS];
    int32_t end_parent[BORN_MAX_BEAMS], end_token[BORN_MAX_BEAMS];
    double end_value[BORN_MAX_BEAMS];
    int32_t fin_parent[BORN_MAX_BEAMS], fin_token[BORN_MAX_BEAMS];
    uint32_t refine;
    int n_sel, n_end;
    int last;
    int32_t hist[BORN_MAX_HISTORY];
};

template <typename T> __device__ __forceinline__ float logit_at(const T* p);
template <> __device__ __forceinline__ float logit_at<float>(const float* p) { return __ldg(p); }
template <> __device__ __forceinline__ float logit_at<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(__ldg(p)); }

__device__ __forceinline__ bool mask_bit(const BeamArgs& A, int64_t row, int t) {
    return !A.mask || ((A.mask[row * A.mask_stride + (t >> 5)] >> (t & 31)) & 1u);
}

// Puts nk into the warp's list (descending over lanes 0 .. K-1, 0 = free).
__device__ __forceinline__ void list_insert(unsigned long long& key, unsigned long long nk, int K) {
    const int lane = (int)threadIdx.x & 31;
    const int pos = __popc(__ballot_sync(0xffffffffu, lane < K && key > nk));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, key, 1);
    if (lane > pos) key = up;
    if (lane == pos) key = nk;
    if (lane >= K) key = 0;
}

__device__ __forceinline__ bool is_stop(const BeamArgs& A, int t) {
    for (int j = 0; j < A.n_stop; ++j)
        if (A.stop_ids[j] == t) return true;
    return false;
}

// Valid ids of the row's history, in sh.hist; ends with a barrier.
__device__ __forceinline__ int load_history(const BeamArgs& A, int64_t row, BeamShared& sh) {
    int len = A.history_len ? A.history_len[row] : A.history_stride;
    len = max(0, min(len, A.history_stride));
    for (int i = threadIdx.x; i < A.history_stride; i += kThreads) sh.hist[i] = i < len ? A.history[row * A.history_stride + i] : -1;
    __syncthreads();
    return len;
}

// If hist[i] is the first occurrence of a token of [lo, hi): its count, else 0.
__device__ __forceinline__ int first_count(const BeamShared& sh, int len, int i, int lo, int hi) {
    const int id = sh.hist[i];
    if (id < lo || id >= hi) return 0;
    int n = 0;
    for (int j = 0; j < len; ++j) {
        if (sh.hist[j] == id) {
            if (j < i) return 0;
            ++n;
        }
    }
    return n;
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0;
    for (int w = 0; w < kBeamWarps; ++w) t += sh[w];
    return t;
}

// log sum exp((z - m)/T) of a row in 64 bits, by the whole CTA, in an order that depends on the token
// indices alone (equal rows give equal bits).  Rare: about 60 us for a row of 128256 tokens.
template <typename T>
__device__ double row_normaliser(const BeamArgs& A, int64_t row, float m, BeamShared& sh, uint32_t* bits) {
    const T* z = reinterpret_cast<const T*>(A.logits) + row * A.row_stride;
    const double invT = 1.0 / (double)A.temperature;
    double s = 0;
    const int len = A.history ? load_history(A, row, sh) : 0;
    const int chunk = A.history ? A.bit_words * 32 : A.V;
    for (int lo = 0; lo < A.V; lo += chunk) {
        const int hi = min(A.V, lo + chunk);
        if (A.history) {
            __syncthreads();
            for (int i = threadIdx.x; i < A.bit_words; i += kThreads) bits[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < len; i += kThreads)
                if (sh.hist[i] >= lo && sh.hist[i] < hi) atomicOr(&bits[(sh.hist[i] - lo) >> 5], 1u << ((sh.hist[i] - lo) & 31));
            __syncthreads();
        }
        for (int t = lo + (int)threadIdx.x; t < hi; t += kThreads) {
            if (A.history && ((bits[(t - lo) >> 5] >> ((t - lo) & 31)) & 1u)) continue;
            if (mask_bit(A, row, t)) s += exp(((double)logit_at<T>(z + t) - (double)m) * invT);
        }
    }
    for (int i = threadIdx.x; i < len; i += kThreads) {
        const int n = first_count(sh, len, i, 0, A.V);
        if (n == 0) continue;
        const int t = sh.hist[i];
        if (mask_bit(A, row, t)) s += exp(((double)penalise(A.params, logit_at<T>(z + t), n) - (double)m) * invT);
    }
    return log(block_sum(s, sh.dsum));
}

// Ranks every candidate: the first K tokens of every row's list, then the rows' stop tokens.  Fills
// sel_* / end_* and, where `check`, the rows whose normalisers have to be exact.
__device__ void rank_candidates(const BeamArgs& A, BeamShared& sh, bool check) {
    const int K = A.K, n_list = K * K, n = n_list + K * A.n_stop;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        double v = -INFINITY;
        uint32_t f = kNoCandidate;
        if (i < n_list) {
            const int b = i / K;
            const unsigned long long k = sh.row_list[b][i - b * K];
            if (k) {
                f = (uint32_t)b << 24 | (uint32_t)ck_idx(k);
                v = sh.offset[b] + ((double)ck_z(k) - (double)sh.row_max[b]) / (double)A.temperature;
            }
        } else {
            const int b = (i - n_list) / A.n_stop, j = (i - n_list) - b * A.n_stop;
            const float z = sh.row_stop[b][j];
            if (z > -INFINITY) {
                f = (uint32_t)b << 24 | (uint32_t)A.stop_ids[j];
                v = sh.offset[b] + ((double)z - (double)sh.row_max[b]) / (double)A.temperature;
            }
        }
        sh.value[i] = v;
        sh.flat[i] = f;
    }
    if (threadIdx.x < (unsigned)K) {
        const int r = threadIdx.x;
        sh.sel_parent[r] = r;
        sh.sel_token[r] = -1;
        sh.sel_value[r] = -INFINITY;
        sh.end_parent[r] = -1;
        sh.end_token[r] = -1;
        sh.end_value[r] = -INFINITY;
    }
    if (threadIdx.x == 0) sh.n_sel = sh.n_end = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t f = sh.flat[i];
        if (f == kNoCandidate) continue;
        const double v = sh.value[i];
        int going = 0, stopping = 0;
        uint32_t near = 0;
        for (int j = 0; j < n; ++j) {
            const uint32_t g = sh.flat[j];  // (no candidate: value -inf)
            const double w = sh.value[j];
            const bool ahead = w > v || (w == v && g < f);
            if (j < n_list) going += ahead;
            else stopping += ahead;
            if (((f ^ g) >> 24) != 0 && fabs(w - v) < A.slack) near |= 1u << (g >> 24);
        }
        const int b = (int)(f >> 24), t = (int)(f & kIdxMask);
        if (i < n_list) {
            if (going < K) {
                sh.sel_parent[going] = b;
                sh.sel_token[going] = t;
                sh.sel_value[going] = v;
                atomicAdd(&sh.n_sel, 1);
            }
        } else if (going + stopping < K) {
            sh.end_parent[stopping] = b;
            sh.end_token[stopping] = t;
            sh.end_value[stopping] = v;
            atomicAdd(&sh.n_end, 1);
        }
        if (check && going < K && near) atomicOr(&sh.refine, near | (1u << b));
    }
    __syncthreads();
}

// The ended hypotheses join the pool, best first; thread 0.
__device__ void update_pool(const BeamArgs& A, const BeamShared& sh, int n) {
    const int K = A.K;
    float* ps = A.pool_score + n * K;
    int held = 0;
    while (held < K && A.pool_step[n * K + held] >= 0) ++held;
    for (int e = 0; e < sh.n_end; ++e) {
        const float v = (float)(sh.end_value[e] / A.length_norm);
        if (held == K && !(v > ps[K - 1])) continue;
        int at = held < K ? held++ : K - 1;
        while (at > 0 && v > ps[at - 1]) {
            const int64_t d = (int64_t)n * K + at;
            A.pool_score[d] = A.pool_score[d - 1];
            A.pool_step[d] = A.pool_step[d - 1];
            A.pool_parent[d] = A.pool_parent[d - 1];
            A.pool_token[d] = A.pool_token[d - 1];
            --at;
        }
        const int64_t d = (int64_t)n * K + at;
        A.pool_score[d] = v;
        A.pool_step[d] = A.step;
        A.pool_parent[d] = sh.end_parent[e];
        A.pool_token[d] = sh.end_token[e];
    }
    bool done = sh.n_sel == 0;
    if (held == K) done = done || (A.flags & BORN_BEAM_EARLY_STOP) || !((float)(sh.sel_value[0] / A.length_norm) > ps[K - 1]);
    if (done) A.done[n] = 1;
}

// The histories of the group's rows follow the beams, then take their tokens.  Every thread reads its
// places of all rows before it writes them.
__device__ void move_history(const BeamArgs& A, const BeamShared& sh, int n) {
    const int K = A.K, cap = A.ring_cap;
    const int64_t r0 = (int64_t)n * K;
    for (int i = threadIdx.x; i < cap; i += kThreads) {
        int32_t v[BORN_MAX_BEAMS];
#pragma unroll
        for (int b = 0; b < BORN_MAX_BEAMS; ++b)
            if (b < K) v[b] = A.ring[(r0 + sh.fin_parent[b]) * cap + i];
#pragma unroll
        for (int b = 0; b < BORN_MAX_BEAMS; ++b)
            if (b < K && sh.fin_parent[b] != b) A.ring[(r0 + b) * cap + i] = v[b];
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int b = threadIdx.x;
        const int from = b < K ? sh.fin_parent[b] : 0;
        const int total = A.ring_total[r0 + from], len = A.ring_len[r0 + from];
        __syncwarp();
        if (b < K) {
            const int tok = sh.fin_token[b];
            if (tok >= 0) {
                A.ring[(r0 + b) * cap + total % cap] = tok;
                A.ring_total[r0 + b] = total + 1;
                A.ring_len[r0 + b] = min(total + 1, cap);
            } else if (from != b) {
                A.ring_total[r0 + b] = total;
                A.ring_len[r0 + b] = len;
            }
        }
    }
}

// The group's last CTA: merges the records, ranks, arranges, writes.
template <typename T>
__device__ void finish_group(const BeamArgs& A, int n, BeamShared& sh, uint32_t* bits) {
    const int K = A.K, S = A.slices;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool done = A.done && A.done[n];
    for (int b = warp; b < K; b += kBeamWarps) {
        const int64_t row = (int64_t)n * K + b;
        const float score = A.scores[row];
        int status = done ? BORN_ROW_FINISHED : score == -INFINITY ? BORN_ROW_DEAD : score != score ? BORN_ROW_NAN : score == INFINITY ? BORN_ROW_POS_INF : BORN_ROW_OK;
        unsigned long long mine = 0;  // lane j: j-th best of the row
        double offset = 0;
        float m = -INFINITY;
        if (status == BORN_ROW_OK) {
            const BeamRecord* rec = A.records + row * S;
            const BeamRecord* r0 = lane < S ? rec + lane : nullptr;
            const BeamRecord* r1 = lane + 32 < S ? rec + lane + 32 : nullptr;
            const float m0 = r0 ? __ldcg(&r0->max) : -INFINITY, m1 = r1 ? __ldcg(&r1->max) : -INFINITY;
            m = max_nan(m0, m1);
            for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
            if (m != m) status = BORN_ROW_NAN;
            else if (m == INFINITY) status = BORN_ROW_POS_INF;
            else if (m == -INFINITY) status = BORN_ROW_ALL_MASKED;
            else {
                const double invT = 1.0 / (double)A.temperature;
                double s = 0;
                if (m0 > -INFINITY) s += __ldcg(&r0->sum) * exp(((double)m0 - (double)m) * invT);
                if (m1 > -INFINITY) s += __ldcg(&r1->sum) * exp(((double)m1 - (double)m) * invT);
                for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                offset = (double)score - log(s);
                int at0 = 0, at1 = 0;
                unsigned long long h0 = r0 ? __ldcg(&r0->list[0]) : 0, h1 = r1 ? __ldcg(&r1->list[0]) : 0;
                for (int k = 0; k < K; ++k) {
                    const unsigned long long head = h0 > h1 ? h0 : h1;
                    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 24));
                    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 24) == hi ? (uint32_t)(head & kIdxMask) : 0u);
                    const unsigned long long best = ((unsigned long long)hi << 24) | lo;
                    if (hi == 0) break;
                    if (lane == k) mine = best;
                    if (head == best) {
                        if (h0 == best) h0 = ++at0 < K ? __ldcg(&r0->list[at0]) : 0;
                        else h1 = ++at1 < K ? __ldcg(&r1->list[at1]) : 0;
                    }
                }
            }
        }
        if (lane < K) sh.row_list[b][lane] = mine;
        if (lane < A.n_stop) {
            float z = -INFINITY;
            if (status == BORN_ROW_OK)
                for (int s = 0; s < S; ++s) z = fmaxf(z, __ldcg(&A.records[row * S + s].stop_z[lane]));
            sh.row_stop[b][lane] = z;
        }
        if (lane == 0) {
            sh.offset[b] = offset;
            sh.row_max[b] = m;
            sh.status[b] = status;
        }
    }
    if (tid == 0) sh.refine = 0;
    __syncthreads();
    rank_candidates(A, sh, true);
    if (sh.refine) {
        for (int b = 0; b < K; ++b) {
            if (!((sh.refine >> b) & 1u)) continue;
            const int64_t row = (int64_t)n * K + b;
            const double l = row_normaliser<T>(A, row, sh.row_max[b], sh, bits);
            if (tid == 0) sh.offset[b] = (double)A.scores[row] - l;
        }
        __syncthreads();
        rank_candidates(A, sh, false);
    }
    if (warp == 0) {
        const bool in = lane < K;
        const bool lives = lane < sh.n_sel;
        int parent = in ? sh.sel_parent[lane] : 0, slot = lane;
        if (A.flags & BORN_BEAM_KEEP_SLOTS) {
            const uint32_t same = __match_any_sync(0xffffffffu, lives ? parent : 64 + lane);
            const bool stays = lives && (same & ((1u << lane) - 1u)) == 0;
            uint32_t taken = 0;
            for (int r = 0; r < K; ++r) {
                const int p = __shfl_sync(0xffffffffu, stays ? parent : -1, r);
                if (p >= 0) taken |= 1u << p;
            }
            const uint32_t others = __ballot_sync(0xffffffffu, in && !stays);
            uint32_t open = ~taken;
            for (int i = __popc(others & ((1u << lane) - 1u)); i > 0; --i) open &= open - 1u;
            slot = stays ? parent : __ffs(open) - 1;
        }
        if (in) {
            if (!lives) parent = slot;
            const int64_t row = (int64_t)n * K + slot;
            sh.fin_parent[slot] = parent;
            sh.fin_token[slot] = sh.sel_token[lane];
            A.out_parent[row] = parent;
            A.out_token[row] = sh.sel_token[lane];
            A.out_score[row] = (float)sh.sel_value[lane];
            if (A.out_status) A.out_status[(int64_t)n * K + lane] = sh.status[lane];
            if (A.out_end_parent) {
                A.out_end_parent[(int64_t)n * K + lane] = sh.end_parent[lane];
                A.out_end_token[(int64_t)n * K + lane] = sh.end_token[lane];
                A.out_end_score[(int64_t)n * K + lane] = (float)sh.end_value[lane];
            }
        }
    }
    __syncthreads();
    if (A.pool_score && !done && tid == 0) update_pool(A, sh, n);
    if (A.ring && !done) move_history(A, sh, n);
}

// kBits: a mask or a history is present; bit i of `bits` says that token a0 + i of the slice is
// allowed and not in the history (history tokens are added back with their penalised values).
template <typename T, bool kBits>
__global__ void __launch_bounds__(kThreads) beam_kernel(const BeamArgs A) {
    constexpr int kVec = 16 / (int)sizeof(T);
    constexpr int kU = 16 / kVec;      // vectors of a lane per turn: 16 values
    constexpr int kAhead = kVec == 4 ? 1 : 2;
    extern __shared__ uint32_t bits[];
    __shared__ BeamShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / A.slices;
    const int slice = blockIdx.x - (int)row * A.slices;
    const int n = (int)(row / A.K);
    const int K = A.K;
    const float score = A.scores[row];
    const bool live = score > -INFINITY && score < INFINITY && !(A.done && A.done[n]);
    if (live) {
        const T* z = reinterpret_cast<const T*>(A.logits) + row * A.row_stride;
        // the row's 16-byte vectors, dealt to the slices in equal parts; the tokens in front of them go
        // with the first slice, those behind with the last
        const int head = min(A.V, (int)(((16u - ((uint32_t)reinterpret_cast<uintptr_t>(z) & 15u)) & 15u) / sizeof(T)));
        const int nvec = (A.V - head) / kVec;
        const int per = (nvec + A.slices - 1) / A.slices;
        const int v0 = min(nvec, per * slice), v1 = min(nvec, v0 + per);
        const int a0 = head + v0 * kVec;                        // first token of the slice's vectors
        const int a1 = head + v1 * kVec;
        const int lo = slice == 0 ? 0 : a0;                     // the slice's tokens: [lo, hi)
        const int hi = slice == A.slices - 1 ? A.V : a1;
        const int n_front = a0 - lo, n_back = hi - a1;
        uint32_t* edge = bits + ((a1 - a0 + 31) >> 5);          // word 0: the tokens in front, word 1: those behind
        int hlen = 0;
        if (tid == 0) sh.thr = 0;
        if (tid < BORN_MAX_STOPS) {
            const int t = tid < A.n_stop ? A.stop_ids[tid] : -1;
            sh.stop_z[tid] = t >= lo && t < hi && mask_bit(A, row, t) ? logit_at<T>(z + t) : -INFINITY;
        }
        if constexpr (kBits) {
            const uint32_t* mw = A.mask ? A.mask + row * A.mask_stride : nullptr;
            const int words = (a1 - a0 + 31) >> 5, last = (A.V - 1) >> 5;
            for (int w = tid; w < words + 2; w += kThreads) {
                const int t = w < words ? a0 + 32 * w : w == words ? lo : a1;
                uint32_t v = 0xffffffffu;
                if (mw) v = __funnelshift_r(mw[min(last, t >> 5)], mw[min(last, (t >> 5) + 1)], (uint32_t)t & 31u);
                bits[w] = v;
            }
            if (A.history) hlen = load_history(A, row, sh);
            __syncthreads();
            for (int i = tid; i < hlen; i += kThreads) {
                const int id = sh.hist[i];
                if (id < lo || id >= hi) continue;
                if (id < a0) atomicAnd(&edge[0], ~(1u << (id - lo)));
                else if (id >= a1) atomicAnd(&edge[1], ~(1u << (id - a1)));
                else atomicAnd(&bits[(id - a0) >> 5], ~(1u << ((id - a0) & 31)));
            }
        }
        __syncthreads();

        // a contiguous part of the vectors for every warp, in turns of 32 * kU vectors
        const int turns = (v1 - v0 + kBeamWarps * 32 * kU - 1) / (kBeamWarps * 32 * kU);
        const int w0 = v0 + warp * turns * 32 * kU;
        const uint4* zv = reinterpret_cast<const uint4*>(z + head);
        const uint32_t ninf = kVec == 4 ? 0xff800000u : 0xff80ff80u;
        auto load = [&](int turn, uint4 (&q)[kU]) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int v = w0 + (turn * kU + u) * 32 + lane;
                bool ok = turn < turns && v < v1;
                if constexpr (kBits) {
                    if (ok) {
                        const int o = (v - v0) * kVec;
                        ok = ((bits[o >> 5] >> (o & 31)) & ((1u << kVec) - 1u)) != 0;
                    }
                }
                q[u] = ok ? __ldg(zv + v) : make_uint4(ninf, ninf, ninf, ninf);
            }
        };
        const float c = A.scale_log2e;
        float m = -INFINITY, mm = -INFINITY, s = 0.0f;
        unsigned long long list = 0;
        // turns, then the tokens in front and behind, then the history's
        const int extra = (warp == 0 && n_front + n_back > 0) ? 1 : 0;
        const int rounds = kBits && A.history ? (hlen + kThreads - 1) / kThreads : 0;
        const int total = turns + 1 + rounds;
        uint4 q0[kU], q1[kU];
        load(0, q0);
        if constexpr (kAhead == 2) load(1, q1);
        for (int it = 0; it < total; ++it) {
            float v[16];
            int t0;
            if (it < turns) {
                uint4 cur[kU];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    cur[u] = q0[u];
                    if constexpr (kAhead == 2) q0[u] = q1[u];
                }
                if constexpr (kAhead == 2) load(it + 2, q1);
                else load(it + 1, q0);
                const int vec = w0 + it * kU * 32 + lane;
                t0 = head + vec * kVec;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    if constexpr (kVec == 4) {
                        v[4 * u] = __uint_as_float(cur[u].x); v[4 * u + 1] = __uint_as_float(cur[u].y);
                        v[4 * u + 2] = __uint_as_float(cur[u].z); v[4 * u + 3] = __uint_as_float(cur[u].w);
                    } else {
                        const uint32_t w[4] = {cur[u].x, cur[u].y, cur[u].z, cur[u].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v[8 * u + 2 * i] = __uint_as_float(w[i] << 16);
                            v[8 * u + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                        }
                    }
                    if constexpr (kBits) {
                        const int o = (vec + u * 32 - v0) * kVec;
                        const uint32_t b = vec + u * 32 < v1 ? bits[o >> 5] >> (o & 31) : 0u;
#pragma unroll
                        for (int i = 0; i < kVec; ++i)
                            if (!((b >> i) & 1u)) v[kVec * u + i] = -INFINITY;
                    }
                }
            } else {
                if (it == turns && !extra) continue;
#pragma unroll
                for (int i = 1; i < 16; ++i) v[i] = -INFINITY;
                v[0] = -INFINITY;
                t0 = 0;
                if (it == turns) {
                    if (lane < n_front + n_back) {
                        const bool front = lane < n_front;
                        const int k = front ? lane : lane - n_front;
                        t0 = front ? lo + k : a1 + k;
                        bool ok = true;
                        if constexpr (kBits) ok = (edge[front ? 0 : 1] >> k) & 1u;
                        if (ok) v[0] = logit_at<T>(z + t0);
                    }
                } else {
                    const int i = (it - turns - 1) * kThreads + tid;
                    const int cnt = i < hlen ? first_count(sh, hlen, i, lo, hi) : 0;
                    if (cnt) {
                        t0 = sh.hist[i];
                        if (mask_bit(A, row, t0)) v[0] = penalise(A.params, logit_at<T>(z + t0), cnt);
                        for (int j = 0; j < A.n_stop; ++j)
                            if (A.stop_ids[j] == t0) sh.stop_z[j] = v[0];
                    }
                }
            }
            float mx = max3_nan(max3_nan(max3_nan(v[0], v[1], v[2]), v[3], v[4]), max3_nan(v[5], v[6], v[7]), max3_nan(v[8], v[9], v[10]));
            mx = max3_nan(mx, max3_nan(v[11], v[12], v[13]), max_nan(v[14], v[15]));
            mm = max_nan(mm, mx);
            // m follows the maximum only once it is 2^8 behind: what a change rounds is then negligible
            if ((mx - m) * c > 8.0f) {
                s *= ex2_approx((m - mx) * c);
                m = mx;
            }
            const float base = m == -INFINITY ? 0.0f : m;
            float e[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[i], v[i + 1]), make_float2(-base, -base)), make_float2(c, c));
                e[i] = ex2_approx(x.x);
                e[i + 1] = ex2_approx(x.y);
            }
#pragma unroll
            for (int d = 8; d; d >>= 1)
#pragma unroll
                for (int i = 0; i < d; ++i) e[i] += e[i + d];
            s += e[0];

            // candidates: best first, until none is ahead of the CTA's threshold
            unsigned long long thr = *(volatile unsigned long long*)&sh.thr;
            float tz = thr ? ck_z(thr) : -INFINITY;
            int tt = thr ? ck_idx(thr) : 0;
            while (true) {
                const bool pass = mx > tz || (mx == tz && t0 < tt);
                const uint32_t who = __ballot_sync(0xffffffffu, pass);
                if (!who) break;
                const uint32_t zk = pass ? zkey(mx) : 0u;
                const uint32_t top = __reduce_max_sync(0xffffffffu, zk);
                const int src = __ffs(__ballot_sync(0xffffffffu, zk == top)) - 1;
                int at = -1;
                if (lane == src) {
#pragma unroll
                    for (int i = 15; i >= 0; --i)
                        if (v[i] == mx) at = i;
                    float next = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (i == at) v[i] = -INFINITY;
                        next = max_nan(next, v[i]);
                    }
                    at = t0 + (at / kVec) * 32 * kVec + at % kVec;
                    mx = next;
                }
                const int tok = __shfl_sync(0xffffffffu, at, src);
                const unsigned long long nk = ((unsigned long long)top << 24) | (kIdxMask - (uint32_t)tok);
                if (nk > thr && !is_stop(A, tok)) {
                    list_insert(list, nk, K);
                    const unsigned long long kth = __shfl_sync(0xffffffffu, list, K - 1);
                    if (kth > thr) {
                        thr = kth;
                        tz = ck_z(thr);
                        tt = ck_idx(thr);
                        if (lane == 0 && thr > *(volatile unsigned long long*)&sh.thr) *(volatile unsigned long long*)&sh.thr = thr;
                    }
                }
            }
        }

        // the CTA's statistics and its best K
        float cm = m;
        for (int d = 16; d; d >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, d));
        for (int d = 16; d; d >>= 1) mm = max_nan(mm, __shfl_xor_sync(0xffffffffu, mm, d));
        if (lane == 0) sh.fmx[warp] = mm;
        if (lane < K) sh.lists[warp][lane] = list;
        __syncthreads();
        float bm = sh.fmx[0];
        for (int w = 1; w < kBeamWarps; ++w) bm = max_nan(bm, sh.fmx[w]);
        const double part = m > -INFINITY ? (double)s * (double)ex2_approx((m - bm) * c) : 0.0;
        const double sum = block_sum(part, sh.dsum);
        BeamRecord* rec = A.records + row * A.slices + slice;
        if (tid == 0) {
            rec->max = bm;
            rec->sum = sum;
        }
        if (tid < BORN_MAX_STOPS) rec->stop_z[tid] = sh.stop_z[tid];
        if (warp == 0) {
            // K rounds over the heads of the warps' lists
            int at = 0;
            unsigned long long h = lane < kBeamWarps ? sh.lists[lane][0] : 0;
            for (int k = 0; k < K; ++k) {
                const uint32_t hk = __reduce_max_sync(0xffffffffu, (uint32_t)(h >> 24));
                const uint32_t lk = __reduce_max_sync(0xffffffffu, (uint32_t)(h >> 24) == hk ? (uint32_t)(h & kIdxMask) : 0u);
                const unsigned long long best = ((unsigned long long)hk << 24) | lk;
                if (lane == 0) rec->list[k] = hk ? best : 0;
                if (hk && h == best) h = ++at < K ? sh.lists[lane][at] : 0;
            }
        }
    }

    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const uint32_t parts = (uint32_t)(K * A.slices);
        sh.last = atomicAdd(&A.tickets[n], 1u) == parts - 1u;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    if (tid == 0) A.tickets[n] = 0;
    finish_group<T>(A, n, sh, bits);
}

}  // namespace born
