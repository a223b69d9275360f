// One step of beam search over [groups * beams, vocab] logits, in one launch.
//
// The rows are cut into blocks of 1024 tokens, the blocks of all rows dealt to the CTAs (two per SM) in equal
// ranges; the part of a row inside a range is a segment.  Warps stream blocks through rings of their own
// (warp_ring.cuh), without a barrier from one segment to the next.  Streaming keeps per thread the running
// maximum and the sum of exponentials, and per group of 32 tokens the upper half of its maximum's
// key.  Afterwards, for all segments side by side, the warps' best groups tell a key that at least `beams` tokens
// reach; the few groups that reach it are read again and their tokens ranked.  A segment leaves (maximum, sum,
// best tokens) as a record; the CTA that draws a group's last ticket merges the records of its rows, ranks
// the candidates by
//     score[b] + (z - m_b)/T - log sum exp((z_j - m_b)/T)
// in 64 bits, arranges the children and writes them out.  No CTA waits for another one.
//
// The normaliser of a row is the only rounded part of that value: tokens of one row order by their
// logits alone.  It comes from 32-bit exponentials, off by less than A.slack / 2 (beam_slack); where two
// candidates of different rows are nearer than A.slack and the order matters, the CTA recomputes the
// normalisers of those rows in 64 bits (row_normaliser), so that the order is that of the definition.  The scores
// of other rows are reported with the 32-bit normaliser: up to 6e-7 off, 1e-7 as measured, about their own rounding.
//
// What bounds it: the bytes of the logits (64 groups of 4 rows of 128256 fp32: 20.1 us of 41.5; the stream ends after
// 23) and the chain of round trips behind them, about a microsecond each: bound, groups again, ranking, ticket, records,
// candidates, which a CTA goes through for its two segments side by side, for two groups that it finishes one after the
// other.  Few rows are the chain alone: one group of 4 x 32000 13 us.
// 512 history ids per row cost 11 us: their bits before the stream, their logits and exponentials behind it.  Repeated
// ids are counted over the list of all later occurrences, once per id: 1 to 4 us at 512 ids as a text repeats them (156
// of them), 10 to 15 at 1024 (385).  A pool costs 1.2 to 2.4 us (one thread).  Moving the histories costs 4 to 11 us at
// 512 ids, 7 to 33 at 1024.
// bf16 rows are bound by the exponentials, a multiply-add, a conversion and an ex2 per logit: 32 groups of 8 rows of
// 128256 take 40 us, 10 of them for the bytes.  Masked ones (151936, one token in twenty: 47 us of 12.6) wait: with four
// warps per scheduler 9.3 cycles pass between two instructions of a warp, and the first copies come behind the mask.
// Kept apart by measurement: none of the tail's lists and closures live on the stack, for L1 is small beside the rings
// (history 64 us instead of 54); at 128 registers a thread still spills 20 to 90 bytes.  Two segments side by side
// rather than one after the other, a team of warps each (42 -> 40.5, history 54 -> 50).
#pragma once
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include "beam_launch.cuh"
#include "scan_common.cuh"
#include "warp_ring.cuh"

namespace born {

constexpr int kBeamWarps = kThreads / 32;
constexpr uint32_t kStopBit = 0x80000000u;
constexpr int kBeamSegs = 2;        // segments that a CTA takes at a time
constexpr int kBeamCand = 384;      // candidates of a segment that are ranked at once (more: slow_list)
constexpr int kBeamGroups = 256;    // groups that are read again
constexpr int kBeamSparse = 8;      // allowed tokens of a group that are taken one by one
constexpr int kBeamPool = 64;       // W warps leave (24 + W - 1) / W + 2 keys each at most

struct BeamShared {
    union {
        struct {  // the selection in a segment
            unsigned long long pool[kBeamPool];  // the best keys of every warp's groups
            unsigned long long cand[kBeamCand];
            uint16_t groups[kBeamGroups];        // numbers of the segment's groups
        } seg[kBeamSegs];
        struct {  // the group's ranking
            unsigned long long row_list[BORN_MAX_BEAMS][BORN_MAX_BEAMS];  // the rows' best tokens, 0-terminated
            double value[BORN_MAX_BEAMS * (BORN_MAX_BEAMS + BORN_MAX_STOPS)];  // of the candidates
            uint32_t flat[BORN_MAX_BEAMS * (BORN_MAX_BEAMS + BORN_MAX_STOPS)]; // beam << 24 | token, kStopBit: a stop token
        };
    };
    struct {
        double wsum[kBeamWarps];       // the warps' sums (BeamSum)
        float wz0[kBeamWarps];
        int wm[kBeamWarps];
        float wmax[kBeamWarps], hmax[kBeamWarps];  // maxima of the warps' blocks, of their threads' history tokens
        unsigned long long hist_mass;  // history tokens' exponentials, 2^-40 each
        float stop_z[BORN_MAX_STOPS];
        int n_pool, n_cand, n_groups;
        int n_own, n_dups;             // history: ids, later occurrences of one
        int lo, hi, s0, s1, q;         // tokens, blocks of the launch, piece
        int64_t row;                   // -1: has no candidates
    } sg[kBeamSegs];
    double offset[BORN_MAX_BEAMS];  // score - log sum of the rows
    float row_max[BORN_MAX_BEAMS];
    float row_stop[BORN_MAX_BEAMS][BORN_MAX_STOPS];
    int32_t status[BORN_MAX_BEAMS];
    double dsum[kBeamWarps];
    unsigned long long two_best[2 * BORN_MAX_BEAMS];  // value_key of the rows' best two
    double sel_value[BORN_MAX_BEAMS], end_value[BORN_MAX_BEAMS];
    int32_t sel_parent[BORN_MAX_BEAMS], sel_token[BORN_MAX_BEAMS];
    int32_t end_parent[BORN_MAX_BEAMS], end_token[BORN_MAX_BEAMS];
    int32_t fin_parent[BORN_MAX_BEAMS], fin_token[BORN_MAX_BEAMS];
    uint32_t refine;
    int n_cand;
    int failed;                     // a wait for a copy ran out
    int last[kBeamSegs];            // the group whose last ticket this was, -1 = none
};

__device__ __forceinline__ uint32_t smem_atom_and(uint32_t at, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared.and.b32 %0, [%1], %2;" : "=r"(old) : "r"(at), "r"(v) : "memory");
    return old;
}

template <typename T> __device__ __forceinline__ float logit_at(const T* p);
template <> __device__ __forceinline__ float logit_at<float>(const float* p) { return __ldg(p); }
template <> __device__ __forceinline__ float logit_at<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(__ldg(p)); }

__device__ __forceinline__ bool mask_bit(const BeamArgs& A, int64_t row, int t) {
    return !A.mask || ((A.mask[row * A.mask_stride + (t >> 5)] >> (t & 31)) & 1u);
}

// The largest key (56 bits) of the warp.
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 24));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 24) == hi ? (uint32_t)(k & kIdxMask) : 0u);
    return ((unsigned long long)hi << 24) | lo;
}

__device__ __forceinline__ bool is_stop(const BeamArgs& A, int t) {
    for (int j = 0; j < A.n_stop; ++j)
        if (A.stop_ids[j] == t) return true;
    return false;
}

// 2^k, k <= 0 (0 below 2^-1000)
__device__ __forceinline__ double pow2_down(int k) { return k < -1000 ? 0.0 : __hiloint2double((1023 + k) << 20, 0); }

// Sum of exp(z/T) as s * 2^m * exp(z0/T), m a whole number that trails the maximum of (z - z0) log2(e)/T.
// A value's exponent is split into the nearest whole number n of z log2(e)/T and the fraction, which a fused
// multiply-add gives from the exact product; ex2 takes the fraction, n - m goes into the exponent.  So a value is
// off by ex2's 2^-22 and by 2^-25 of the fraction, however far z is from the maximum, which a scaled difference
// from the maximum would not give.  Sums of 32 in 32 bits, beyond that in 64.  z0 is 0 but for logits so large
// that the whole numbers would not fit: those are taken relative to the maximum (what is near it is then exact,
// and only that counts).  For temperatures beyond 2^100 it is not defined (BeamArgs::exact).
struct BeamSum {
    float c, c_lo;   // log2(e)/T in two parts
    float z0;
    float least;     // z - z0 below it counts as it: 2^-100
    int m;           // INT_MIN: nothing is summed yet
    double s;
    __device__ __forceinline__ explicit BeamSum(const BeamArgs& A) : c(A.scale_log2e), c_lo(A.scale_lo), z0(0.0f), least(0.0f), m(INT_MIN), s(0) {}
    // m follows the maximum once that is 2^8 ahead; scaling the sum by a power of two rounds nothing
    __device__ __forceinline__ void follow(float mx) {
        if ((m != INT_MIN && !((mx - z0) * c > (float)m + 8.0f)) || mx == -INFINITY) return;
        const float z1 = fabsf(mx * c) > 1048576.0f ? mx : 0.0f;
        const int to = __float2int_ru((mx - z1) * c);
        if (m != INT_MIN) {
            if (z0 == z1) s *= pow2_down(min(m - to, 0));
            else s *= exp2((double)m - (double)to + ((double)z0 - (double)z1) * ((double)c + (double)c_lo));
        }
        z0 = z1;
        m = to;
        least = __fdividef((float)m - 100.0f, c);
    }
    // two values of z - z0
    __device__ __forceinline__ float2 two(float2 z) const {
        const float magic = (float)(12582912 + m);  // 1.5 * 2^23: magic - n has m - n in its low bits
        z.x = fmaxf(z.x, least);
        z.y = fmaxf(z.y, least);
        // (-c and -n rather than n: a packed operation has no sign to flip its operands with)
        const float2 r = __ffma2_rn(z, make_float2(-c, -c), make_float2(magic, magic));
        const float2 minus_n = __fadd2_rn(r, make_float2(-magic, -magic));
        float2 f = __ffma2_rn(z, make_float2(c, c), minus_n);
        f = __ffma2_rn(z, make_float2(c_lo, c_lo), f);
        return make_float2(scaled(ex2_approx(f.x), r.x), scaled(ex2_approx(f.y), r.y));
    }
    // n - m into the exponent: minus r's low bits (what is above them shifts out), in one multiply-add
    static __device__ __forceinline__ float scaled(float e, float r) {
        uint32_t o;
        asm("mad.lo.u32 %0, %1, 0xff800000, %2;" : "=r"(o) : "r"(__float_as_uint(r)), "r"(__float_as_uint(e)));
        return __uint_as_float(o);
    }
    template <int N>
    __device__ __forceinline__ void add(float (&v)[N], float mx) {
        follow(mx);
        if (m == INT_MIN) return;  // (nothing but -inf so far)
        if (z0 != 0.0f) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] -= z0;
        }
        // four sums of N/8 pairs each, then three levels: a value is rounded N/8 + 2 times at most
        float2 e[4];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 x = two(make_float2(v[2 * i], v[2 * i + 1]));
            if (i < 4) e[i] = x;
            else e[i & 3] = __fadd2_rn(e[i & 3], x);
        }
        e[0] = __fadd2_rn(__fadd2_rn(e[0], e[1]), __fadd2_rn(e[2], e[3]));
        s += (double)(e[0].x + e[0].y);
    }
};
// s * 2^m * exp(z0/T) in units of 2^m1 * exp(z1/T), which is no less
__device__ __forceinline__ double in_units(const BeamArgs& A, double s, int m, float z0, int m1, float z1) {
    if (m == INT_MIN) return 0.0;
    if (z0 == z1) return s * pow2_down(min(m - m1, 0));
    return s * exp2((double)m - (double)m1 + ((double)z0 - (double)z1) * ((double)A.scale_log2e + (double)A.scale_lo));
}
// The units for a maximum: 2^m * exp(z0/T) at least as large as exp(mx/T)
__device__ __forceinline__ void units_of(const BeamArgs& A, float mx, int& m, float& z0) {
    const float t = mx * A.scale_log2e;
    const bool large = !(fabsf(t) <= 1048576.0f);
    z0 = large ? mx : 0.0f;
    m = large ? 0 : __float2int_ru(t);
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
// indices alone (equal rows give equal bits).  Rare, and slow: tens of microseconds for a row of 128256 tokens.
template <typename T>
__device__ __noinline__ double row_normaliser(const BeamArgs& A, int64_t row, float m, BeamShared& sh, uint32_t* bits, int32_t* hist) {
    const T* z = reinterpret_cast<const T*>(A.logits) + row * A.row_stride;
    const double invT = A.inv_T;
    double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int len = 0;
    if (A.history) {
        len = A.history_len ? A.history_len[row] : A.history_stride;
        len = max(0, min(len, A.history_stride));
        for (int i = threadIdx.x; i < len; i += kThreads) hist[i] = A.history[row * A.history_stride + i];
        __syncthreads();
    }
    const int chunk = A.history ? A.bit_words * 32 : A.V;
    for (int lo = 0; lo < A.V; lo += chunk) {
        const int hi = min(A.V, lo + chunk);
        if (A.history) {
            __syncthreads();
            for (int i = threadIdx.x; i < A.bit_words; i += kThreads) bits[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < len; i += kThreads)
                if (hist[i] >= lo && hist[i] < hi) atomicOr(&bits[(hist[i] - lo) >> 5], 1u << ((hist[i] - lo) & 31));
            __syncthreads();
        }
        // (eight loads in flight per thread, then their exponentials, into sums of their own)
        for (int t0 = lo + (int)threadIdx.x; t0 < hi; t0 += 8 * kThreads) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int t = t0 + u * kThreads;
                const bool ok = t < hi && mask_bit(A, row, t) && !(A.history && ((bits[(t - lo) >> 5] >> ((t - lo) & 31)) & 1u));
                x[u] = ok ? logit_at<T>(z + t) : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) s[u] += exp(((double)x[u] - (double)m) * invT);
        }
    }
    for (int i = threadIdx.x; i < len; i += kThreads) {
        // the first occurrence of a token: with its count
        const int t = hist[i];
        if (t < 0 || t >= A.V || !mask_bit(A, row, t)) continue;
        int n = 0;
        bool first = true;
        for (int j = 0; j < len; ++j) {
            if (hist[j] != t) continue;
            first = first && j >= i;
            ++n;
        }
        if (first) s[0] += exp(((double)penalise(A.params, logit_at<T>(z + t), n) - (double)m) * invT);
    }
    return log(block_sum(((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])), sh.dsum));
}

// Value of a candidate of row b: equal logits of a row give equal bits.
__device__ __forceinline__ double beam_value(const BeamArgs& A, const BeamShared& sh, int b, float z) {
    return sh.offset[b] + ((double)z - (double)sh.row_max[b]) * A.inv_T;
}
// Order-preserving map of a value (above 0 for all of them), and back.
__device__ __forceinline__ unsigned long long value_key(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b ^ ((unsigned long long)((long long)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(unsigned long long k) {
    return __longlong_as_double((long long)((k >> 63) ? k ^ 0x8000000000000000ull : ~k));
}
__device__ __forceinline__ unsigned long long candidate_key(const BeamArgs& A, const BeamShared& sh, int b, unsigned long long k) {
    return k ? value_key(beam_value(A, sh, b, ck_z(k))) : 0;
}
// Which lane holds the largest key (the lowest of equal ones), 32 for none above 0.
__device__ __forceinline__ int warp_argmax(unsigned long long key) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
    uint32_t who = __ballot_sync(0xffffffffu, key != 0 && (uint32_t)(key >> 32) == hi);
    if (who & (who - 1)) {
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (who >> (threadIdx.x & 31)) & 1u ? (uint32_t)key : 0u);
        who = __ballot_sync(0xffffffffu, key != 0 && key == ((unsigned long long)hi << 32 | lo));
    }
    return who ? __ffs(who) - 1 : 32;
}

// The whole CTA: the beams that go on (sel_*, best first) and the hypotheses that end (end_*), by counting how many
// candidates are ahead of each.  Candidates are the rows' list entries and stop tokens that reach `bound`, below
// which there are K better ones.  check: leaves in sh.refine the rows whose normalisers have to be exact: those
// of candidates from different rows nearer to each other than A.slack, one of which is among the K best.
__device__ __noinline__ void rank_candidates(const BeamArgs& A, BeamShared& sh, bool check, double bound) {
    const int K = A.K, tid = threadIdx.x;
    if (tid < K) {
        sh.sel_parent[tid] = tid;
        sh.sel_token[tid] = -1;
        sh.sel_value[tid] = -INFINITY;
        sh.end_parent[tid] = -1;
        sh.end_token[tid] = -1;
        sh.end_value[tid] = -INFINITY;
    }
    if (tid == 0) sh.n_cand = sh.refine = 0;
    __syncthreads();
    const int b = tid >> 4, j = tid & 15;  // (a thread per list entry)
    if (b < K && j < K) {
        const unsigned long long k = sh.row_list[b][j];
        const double v = k ? beam_value(A, sh, b, ck_z(k)) : -INFINITY;
        if (v > -INFINITY && v >= bound) {
            const int at = atomicAdd(&sh.n_cand, 1);
            sh.value[at] = v;
            sh.flat[at] = (uint32_t)b << 24 | (uint32_t)ck_idx(k);
        }
    }
    for (int i = tid; i < BORN_MAX_BEAMS * A.n_stop; i += kThreads) {
        const int row = i & 15, stop = i >> 4;
        if (row >= K) continue;
        const float z = sh.row_stop[row][stop];
        const double v = z > -INFINITY ? beam_value(A, sh, row, z) : -INFINITY;
        if (v > -INFINITY && v >= bound) {
            const int at = atomicAdd(&sh.n_cand, 1);
            sh.value[at] = v;
            sh.flat[at] = kStopBit | (uint32_t)row << 24 | (uint32_t)A.stop_ids[stop];
        }
    }
    __syncthreads();
    const int n = sh.n_cand;
    for (int i = tid; i < n; i += kThreads) {
        const uint32_t fs = sh.flat[i], f = fs & ~kStopBit;
        const double v = sh.value[i];
        int going = 0, stopping = 0;
        uint32_t near = 0;
#pragma unroll 4
        for (int e = 0; e < n; ++e) {
            const uint32_t gs = sh.flat[e], g = gs & ~kStopBit;
            const double d = sh.value[e] - v;
            const bool ahead = d > 0.0 || (d == 0.0 && g < f);
            going += ahead && !(gs & kStopBit);
            stopping += ahead && (gs & kStopBit);
            if (fabs(d) < A.slack && (f ^ g) >> 24) near |= 1u << (g >> 24);
        }
        const int row = (int)(f >> 24), t = (int)(f & kIdxMask);
        if (!(fs & kStopBit)) {
            if (going < K) {
                sh.sel_parent[going] = row;
                sh.sel_token[going] = t;
                sh.sel_value[going] = v;
            }
        } else if (going + stopping < K) {
            sh.end_parent[stopping] = row;
            sh.end_token[stopping] = t;
            sh.end_value[stopping] = v;
        }
        if (check && going < K && near) atomicOr(&sh.refine, near | 1u << row);
    }
    __syncthreads();
}

// The ended hypotheses join the pool, best first; one thread.
__device__ __noinline__ void update_pool(const BeamArgs& A, const BeamShared& sh, int n) {
    const int K = A.K;
    float* ps = A.pool_score + n * K;
    int held = 0;
    while (held < K && A.pool_step[n * K + held] >= 0) ++held;
    for (int e = 0; e < K && sh.end_token[e] >= 0; ++e) {
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
    bool done = sh.sel_token[0] < 0;
    if (held == K) done = done || (A.flags & BORN_BEAM_EARLY_STOP) || !((float)(sh.sel_value[0] / A.length_norm) > ps[K - 1]);
    if (done) A.done[n] = 1;
}

// The histories of the group's rows follow the beams, then take their tokens.  Every thread reads its
// places of all rows before it writes them.
__device__ __noinline__ void move_history(const BeamArgs& A, const BeamShared& sh, int n) {
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

// The records of a row, a warp over them: lane i walks down the list of record i.
struct RowHeads {
    unsigned long long h, next;  // the list's entry, and the one behind it
    int rec, at;                 // the lane's record; entry behind those
    // (the list's first two entries, with everything else of a record in one round trip)
    __device__ __forceinline__ void load_list(const BeamArgs& A, int i, bool has) {
        rec = i;
        ulonglong2 a = make_ulonglong2(0, 0);
        if (has) a = __ldcg(reinterpret_cast<const ulonglong2*>(A.records[i].list));
        h = a.x;
        next = A.K > 1 ? a.y : 0;
        at = 2;
    }
    __device__ __forceinline__ void step(const BeamArgs& A) {
        h = next;
        next = next && at < A.K ? __ldcg(&A.records[rec].list[at]) : 0;
        ++at;
    }
};

// A warp: the statistics of row b of group n and its best two tokens; returns the lists for more (one record per
// lane), or false where all K are found already (more than 32 records).
__device__ __forceinline__ bool merge_row(const BeamArgs& A, int n, int b, bool done, BeamShared& sh, RowHeads& heads) {
    const int K = A.K, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)n * K + b;
    const int q0 = (int)row * A.pieces;
    const int first = A.record_of(q0 * A.pb), last = A.record_of((q0 + A.pieces) * A.pb - 1);
    const float score = A.scores[row];
    float m = -INFINITY;
    int failed = 0;
    const BeamRecord* r = A.records + first + lane;
    const bool has = first + lane <= last;  // (read whether or not the row is alive: one round trip)
    double rs = 0;
    float rz0 = 0, stop = -INFINITY;
    int rm = INT_MIN;
    if (has) {
        m = __ldcg(&r->max);
        failed = __ldcg(&r->failed);
        rs = __ldcg(&r->sum);
        rm = __ldcg(&r->m);
        rz0 = __ldcg(&r->z0);
    }
    heads.load_list(A, first + lane, has);
    if (lane < A.n_stop) {
        const int blk = A.stop_ids[lane] / kBlkTok;
        stop = __ldcg(&A.records[A.record_of((q0 + blk / A.pb) * A.pb + blk % A.pb)].stop_z[lane]);
    }
    int status = done ? BORN_ROW_FINISHED : score == -INFINITY ? BORN_ROW_DEAD : score != score ? BORN_ROW_NAN : score == INFINITY ? BORN_ROW_POS_INF : BORN_ROW_OK;
    const bool live = status == BORN_ROW_OK;
    for (int i = first + lane + 32; live && i <= last; i += 32) {
        m = max_nan(m, __ldcg(&A.records[i].max));
        failed |= __ldcg(&A.records[i].failed);
    }
    for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (live && __any_sync(0xffffffffu, failed)) status = 100 + BORN_ERR_DEVICE_TIMEOUT;
    else if (live) status = m != m ? BORN_ROW_NAN : m == INFINITY ? BORN_ROW_POS_INF : m == -INFINITY ? BORN_ROW_ALL_MASKED : BORN_ROW_OK;
    unsigned long long kept = 0;  // lane j: j-th best of the row
    double offset = 0;
    const bool many = last - first >= 32;
    if (status == BORN_ROW_OK) {
        int m1;
        float z1;
        units_of(A, m, m1, z1);
        double s = in_units(A, rs, rm, rz0, m1, z1);
        const int pops = many ? K : min(K, 2);
        for (int k = 0; k < pops; ++k) {
            const int src = warp_argmax(heads.h << 8);
            if (src == 32) break;
            const unsigned long long best = __shfl_sync(0xffffffffu, heads.h, src);
            if (lane == k) kept = best;
            if (lane == src) heads.step(A);
        }
        for (int base = first + 32; base <= last; base += 32) {
            // the best of the records before are a 33rd list
            const bool more = base + lane <= last;
            r = A.records + base + lane;
            if (more) s += in_units(A, __ldcg(&r->sum), __ldcg(&r->m), __ldcg(&r->z0), m1, z1);
            heads.load_list(A, base + lane, more);
            const unsigned long long old = kept;
            int at_old = 0;
            kept = 0;
            for (int k = 0; k < K; ++k) {
                const unsigned long long prev = __shfl_sync(0xffffffffu, old, at_old), head = warp_max_key(heads.h);
                const unsigned long long best = head > prev ? head : prev;
                if (best == 0) break;
                if (lane == k) kept = best;
                if (prev == best) ++at_old;
                else if (heads.h == best) heads.step(A);
            }
        }
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        // log sum exp((z - m)/T): the units are 2^m1 exp(z1/T)
        const double c = (double)A.scale_log2e + (double)A.scale_lo;
        offset = (double)score - (log(s) + ((double)m1 - ((double)m - (double)z1) * c) * M_LN2);
    }
    if (lane < K) sh.row_list[b][lane] = kept;
    if (lane < A.n_stop) sh.row_stop[b][lane] = status == BORN_ROW_OK ? stop : -INFINITY;
    if (lane == 0) {
        sh.offset[b] = A.exact ? 0.0 : offset;  // (a number)
        sh.row_max[b] = m;
        sh.status[b] = status;
    }
    __syncwarp();
    if (lane < 2) sh.two_best[2 * b + lane] = candidate_key(A, sh, b, kept);
    return status == BORN_ROW_OK && !many;
}

// A warp: the tokens of row b behind its best two that reach `bound` (a value).
__device__ __forceinline__ void extend_row(const BeamArgs& A, int b, double bound, BeamShared& sh, RowHeads& heads) {
    const int K = A.K, lane = threadIdx.x & 31;
    for (int k = 2; k < K; ++k) {
        const int src = warp_argmax(heads.h << 8);
        if (src == 32) break;
        bool ends = false;
        if (lane == src) {
            const double v = beam_value(A, sh, b, ck_z(heads.h));
            ends = !(v >= bound);
            if (!ends) {
                sh.row_list[b][k] = heads.h;
                heads.step(A);
            }
        }
        if (__any_sync(0xffffffffu, ends)) break;
    }
}

// The group's last CTA: merges the records, ranks, arranges, writes.
template <typename T>
__device__ __forceinline__ void finish_group(const BeamArgs& A, int n, BeamShared& sh, uint32_t* bits, int32_t* hist) {
    const int K = A.K;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool done = A.done && A.done[n];
    static_assert(BORN_MAX_BEAMS <= 2 * kBeamWarps, "two rows a warp");
    RowHeads heads[2];
    bool more[2] = {false, false};
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (warp + i * kBeamWarps < K) more[i] = merge_row(A, n, warp + i * kBeamWarps, done, sh, heads[i]);
    __syncthreads();
    // the K-th best of all rows' best two: what is not near it or above is no candidate
    const unsigned long long key = lane < 2 * K ? sh.two_best[lane] : 0;
    int ahead = 0;
    for (int i = 0; i < 2 * K; ++i) {
        const unsigned long long o = sh.two_best[i];
        ahead += o > key || (o == key && i < lane);
    }
    const uint32_t who = __ballot_sync(0xffffffffu, key != 0 && ahead == K - 1);
    double bound = who && !A.exact ? key_value(__shfl_sync(0xffffffffu, key, __ffs(who) - 1)) - A.slack : -INFINITY;
    if (K > 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (more[i]) extend_row(A, warp + i * kBeamWarps, bound, sh, heads[i]);
    }
    rank_candidates(A, sh, true, bound);
    if (const uint32_t refine = A.exact && !done ? ~0u : sh.refine) {
        for (int b = 0; b < K; ++b) {
            if (!((refine >> b) & 1u)) continue;
            const int64_t row = (int64_t)n * K + b;
            const double l = row_normaliser<T>(A, row, sh.row_max[b], sh, bits, hist);
            if (tid == 0) sh.offset[b] = (double)A.scores[row] - l;
        }
        __syncthreads();
        rank_candidates(A, sh, false, bound - A.slack);
    }
    int parent = 0, token = -1;
    double value = 0;
    if (lane < K) {
        parent = sh.sel_parent[lane];
        token = sh.sel_token[lane];
        value = sh.sel_value[lane];
    }
    if (warp == 0) {
        const bool in = lane < K, lives = token >= 0 && in;
        int slot = lane;
        if (A.flags & BORN_BEAM_KEEP_SLOTS) {
            const uint32_t same = __match_any_sync(0xffffffffu, lives ? parent : 64 + lane);
            const bool stays = lives && (same & ((1u << lane) - 1u)) == 0;
            const uint32_t taken = __reduce_or_sync(0xffffffffu, stays ? 1u << parent : 0u);
            const uint32_t others = __ballot_sync(0xffffffffu, in && !stays);
            uint32_t open = ~taken;
            for (int i = __popc(others & ((1u << lane) - 1u)); i > 0; --i) open &= open - 1u;
            slot = stays ? parent : __ffs(open) - 1;
        }
        if (in) {
            if (!lives) parent = slot;
            const int64_t row = (int64_t)n * K + slot;
            sh.fin_parent[slot] = parent;
            sh.fin_token[slot] = token;
            A.out_parent[row] = parent;
            A.out_token[row] = token;
            A.out_score[row] = (float)value;
            const int64_t at = (int64_t)n * K + lane;
            if (A.out_status) A.out_status[at] = sh.status[lane];
            if (A.out_end_parent) {
                A.out_end_parent[at] = sh.end_parent[lane];
                A.out_end_token[at] = sh.end_token[lane];
                A.out_end_score[at] = (float)sh.end_value[lane];
            }
        }
        if (A.pool_score && !done && lane == 0) update_pool(A, sh, n);
    }
    if (A.ring && !done) {
        __syncthreads();
        move_history(A, sh, n);
    }
}

// Programmatic dependent launch: set-up runs while the launch before ends, nothing is read before its results are there.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The group's bits in the order in which load_half hands out its values (group_pos): bit 16 h + i for v[i] of half h.
template <typename T, bool kAligned>
__device__ __forceinline__ uint32_t in_load_order(uint32_t w) {
    const uint32_t lane = threadIdx.x & 31u;
    // bytes, then nibbles, pairs and bits change places with those of the other number in one binary digit
    const uint32_t x = kAligned ? (sizeof(T) == 4 ? (lane & 7u) << 2 : ((lane >> 1) & 3u) << 3) : lane;
    w = __byte_perm(w, 0, 0x3210u ^ ((x >> 3) * 0x1111u));
    if (!kAligned || sizeof(T) == 4)
        if (x & 4u) w = ((w & 0x0f0f0f0fu) << 4) | ((w >> 4) & 0x0f0f0f0fu);
    if (!kAligned) {
        if (x & 2u) w = ((w & 0x33333333u) << 2) | ((w >> 2) & 0x33333333u);
        if (x & 1u) w = ((w & 0x55555555u) << 1) | ((w >> 1) & 0x55555555u);
    }
    return w;
}

// The K best tokens of a segment by K rounds over all its values: where the candidates overflow, as when a
// few threads hold nearly all the large values.  key_of(i), i < count, enumerates the calling thread's keys (0: none).
template <typename F>
__device__ __forceinline__ void slow_list(unsigned long long* scratch, unsigned long long* list, int K, int count, const F& key_of) {
    unsigned long long below = ~0ull;
    for (int k = 0; k < K; ++k) {
        unsigned long long best = 0;
        if (below)
            for (int i = 0; i < count; ++i) {
                const unsigned long long q = key_of(i);
                if (q < below && q > best) best = q;
            }
        best = warp_max_key(best);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = best;
        __syncthreads();
        best = 0;
        for (int w = 0; w < kBeamWarps; ++w) best = max(best, scratch[w]);
        if (threadIdx.x == 0) list[k] = best;
        below = best;
    }
}

// kBits: a mask or a history is present; bit i of `bits` says that token i of the CTA's blocks is allowed and not
// in the history (history tokens are added back with their penalised values).  kAligned: every row starts
// on a 16-byte boundary.
template <typename T, bool kBits, bool kAligned>
__global__ void __launch_bounds__(kThreads, 2) beam_kernel(const __grid_constant__ BeamArgs A) {
    extern __shared__ __align__(128) uint8_t dyn[];  // rings, bits, group keys, histories
    __shared__ BeamShared sh;
    __shared__ uint64_t bars[kBeamWarps * kBeamMaxSlots];
    uint32_t* bits = reinterpret_cast<uint32_t*>(dyn + A.bits_at);
    uint16_t* gkey = reinterpret_cast<uint16_t*>(dyn + A.gkeys_at);
    // histories of the segments: ids that are the first of their token in the segment (else -1) and their penalised
    // logits; later occurrences
    int32_t* own = reinterpret_cast<int32_t*>(dyn + A.hist_at);
    float* own_z = reinterpret_cast<float*>(own + kBeamSegs * A.hist_cap);
    int32_t* dups = own + 2 * kBeamSegs * A.hist_cap;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int K = A.K, slots = A.slots;
    const bool hist = kBits && A.history;
    const uint32_t ring0 = smem_u32(dyn) + (uint32_t)(warp * slots * A.slot_bytes), bar0 = smem_u32(bars + warp * slots);
    if (lane == 0)
        for (int i = 0; i < slots; ++i)  // (the test hook's waits for an arrival that never comes)
            mbar_init(bars + warp * slots + i, i + tid == 0 && (int)blockIdx.x == A.debug_stuck_cta ? 2 : 1);
    if (tid == 0) {
        sh.failed = 0;
        mbar_fence_init();
    }
    __syncthreads();
    grid_wait();
    grid_launch();

    const int t0 = A.range_start((int)blockIdx.x), t1 = A.range_start((int)blockIdx.x + 1);
    auto live = [&](int row) {
        const float score = A.scores[row];
        return score > -INFINITY && score < INFINITY && !(A.done && A.done[row / K]);
    };
    // The warp's blocks are t0 + warp, + 8, ...; lane 0 keeps `slots` copies in flight.  The next one: block bi of
    // piece qi, which is piece pi of the row at `from` (NULL: nothing to stream).
    int ti = t0 + warp, si = 0, in_flight = 0;
    int qi = ti / A.pb, bi = ti - qi * A.pb, pi = 0;
    const uint8_t* from = nullptr;
    auto look_up = [&] {
        const int row = qi / A.pieces;
        pi = qi - row * A.pieces;
        from = ti < t1 && live(row) ? reinterpret_cast<const uint8_t*>(A.logits) + (int64_t)row * A.row_stride * (int64_t)sizeof(T) : nullptr;
    };
    look_up();
    auto issue_next = [&] {
        while (ti < t1) {
            const int tok = (pi * A.pb + bi) * kBlkTok;
            const bool there = from && tok < A.V;
            if (there && lane == 0)
                ring_issue(ring0 + (uint32_t)(si * A.slot_bytes), bar0 + (uint32_t)si * 8u, from, tok, min(kBlkTok, A.V - tok), (int)sizeof(T));
            ti += kBeamWarps;
            bi += kBeamWarps;
            if (bi >= A.pb) {
                do { bi -= A.pb; ++qi; } while (bi >= A.pb);
                look_up();
            }
            if (there) {
                ++in_flight;
                if (++si == slots) si = 0;
                return;
            }
        }
    };
    bool started = false;
    int sc = 0, tc = t0 + warp;
    uint32_t phase = 0;
    bool failed = false;  // of this warp

    const int want = K + A.n_stop;
    for (int q0 = t0 / A.pb; q0 * A.pb < t1; q0 += kBeamSegs) {
        const int ns = min(kBeamSegs, (t1 - 1) / A.pb - q0 + 1);
        const int bits0 = max(t0, q0 * A.pb);  // block whose bits and group keys come first
        // ---- the segments
        if (tid < ns) {
            const int q = q0 + tid;
            auto& G = sh.sg[tid];
            G.q = q;
            G.s0 = max(t0, q * A.pb);
            G.s1 = min(t1, (q + 1) * A.pb);
            const int row = q / A.pieces;
            const int blk0 = (q - row * A.pieces) * A.pb + (G.s0 - q * A.pb);  // its first block in the row
            G.lo = min(blk0 * kBlkTok, A.V);
            G.hi = min((blk0 + G.s1 - G.s0) * kBlkTok, A.V);
            G.row = live(row) ? row : -1;
            G.hist_mass = 0;
            G.n_pool = G.n_cand = G.n_groups = G.n_dups = 0;
        }
        __syncthreads();
        // ---- their bits and histories, and the stop tokens' logits
        constexpr int kIds = BORN_MAX_HISTORY / kThreads;
        if (hist) {
            int32_t id[kBeamSegs][kIds];
#pragma unroll
            for (int g = 0; g < kBeamSegs; ++g) {
                const int64_t row = g < ns ? sh.sg[g].row : -1;
#pragma unroll
                for (int j = 0; j < kIds; ++j)
                    id[g][j] = row >= 0 && tid + j * kThreads < A.history_stride ? A.history[row * A.history_stride + tid + j * kThreads] : -1;
                if (tid == 0) sh.sg[g].n_own = row < 0 ? 0 : max(0, min(A.history_len ? A.history_len[row] : A.history_stride, A.history_stride));
            }
#pragma unroll
            for (int g = 0; g < kBeamSegs; ++g)
#pragma unroll
                for (int j = 0; j < kIds; ++j)
                    if (tid + j * kThreads < A.hist_cap) own[g * A.hist_cap + tid + j * kThreads] = id[g][j];
        }
        if constexpr (kBits) {
#pragma unroll 1
            for (int g = 0; g < ns; ++g) {
                const auto& G = sh.sg[g];
                if (G.row < 0) continue;
                uint32_t* b = bits + (G.s0 - bits0) * 32;
                const uint32_t* mw = A.mask ? A.mask + G.row * A.mask_stride + G.lo / 32 : nullptr;
                for (int w = tid; w < (G.hi - G.lo + 31) >> 5; w += kThreads) b[w] = mw ? mw[w] : 0xffffffffu;
            }
        }
        if (tid < kBeamSegs * BORN_MAX_STOPS) {
            const int g = tid / BORN_MAX_STOPS, j = tid % BORN_MAX_STOPS;
            if (g < ns && sh.sg[g].row >= 0) {
                auto& G = sh.sg[g];
                const int t = j < A.n_stop ? A.stop_ids[j] : -1;
                G.stop_z[j] = t >= G.lo && t < G.hi && mask_bit(A, G.row, t)
                                  ? logit_at<T>(reinterpret_cast<const T*>(A.logits) + G.row * A.row_stride + t) : -INFINITY;
            }
        }
        if constexpr (kBits) {
            __syncthreads();
            if (hist) {
                // whoever clears a token's bit owns it; later occurrences are listed, to be counted; masked tokens are
                // taken for later occurrences of nothing
                const uint32_t bits0_at = smem_u32(bits);
                int32_t t[kBeamSegs][kIds];
                uint32_t was[kBeamSegs][kIds];
#pragma unroll
                for (int g = 0; g < kBeamSegs; ++g) {
                    const auto& G = sh.sg[g < ns ? g : 0];
                    const int len = g < ns ? G.n_own : 0, o0 = (G.s0 - bits0) * kBlkTok - G.lo;
#pragma unroll
                    for (int j = 0; j < kIds; ++j) {
                        t[g][j] = tid + j * kThreads < len ? own[g * A.hist_cap + tid + j * kThreads] : -1;
                        const int o = o0 + t[g][j];
                        if (t[g][j] < 0 || t[g][j] < G.lo || t[g][j] >= G.hi) t[g][j] = -1;
                        else was[g][j] = smem_atom_and(bits0_at + (uint32_t)(o >> 5) * 4u, ~(1u << (o & 31))) >> (o & 31);
                    }
                }
#pragma unroll
                for (int g = 0; g < kBeamSegs; ++g) {
#pragma unroll
                    for (int j = 0; j < kIds; ++j) {
                        const bool again = t[g][j] >= 0 && !(was[g][j] & 1u);
                        if (again) dups[g * A.hist_cap + atomicAdd(&sh.sg[g].n_dups, 1)] = t[g][j];
                        if (again || t[g][j] < 0)
                            if (tid + j * kThreads < A.hist_cap) own[g * A.hist_cap + tid + j * kThreads] = -1;
                    }
                }
                __syncthreads();
            }
        }
        // (the first copies behind the preparation, whose reads would wait for them)
        if (!started) {
            started = true;
            for (int i = 0; i < slots; ++i) issue_next();
        }

        // ---- the stream: a lane has 32 consecutive tokens of a block
#pragma unroll 1
        for (int g = 0; g < ns; ++g) {
            auto& G = sh.sg[g];
            const int s0 = G.s0, s1 = G.s1;
            if (G.row < 0) {
                while (tc < s1) tc += kBeamWarps;
                continue;
            }
            const T* z = reinterpret_cast<const T*>(A.logits) + G.row * A.row_stride;
            const int lo = G.lo;
            BeamSum sum(A);
            float mm = -INFINITY, top = -INFINITY;
            int top_tok = 0;
            for (; tc < s1; tc += kBeamWarps) {
                const int tok0 = lo + (tc - s0) * kBlkTok;
                if (tok0 >= A.V || failed) continue;
                const uint32_t slot = ring0 + (uint32_t)(sc * A.slot_bytes);
                if (!ring_wait(bar0 + (uint32_t)sc * 8u, phase, A.timeout_ns)) {
                    failed = true;
                    sh.failed = 1;
                    continue;
                }
                --in_flight;
                const int at = (tc - bits0) * 32 + lane;
                uint32_t w = 0xffffffffu;
                if constexpr (kBits) w = bits[at];
                if (tok0 + kBlkTok > A.V) {  // the row's last block
                    const int rest = A.V - tok0 - 32 * lane;
                    if (rest < 32) w &= rest <= 0 ? 0u : (1u << rest) - 1u;
                }
                const uint32_t mis = kAligned ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(z + tok0) & 15u);
                const bool all = __all_sync(0xffffffffu, w == 0xffffffffu);
                float gm = -INFINITY;
                if (kBits && !all && __reduce_max_sync(0xffffffffu, __popc(w)) <= kBeamSparse) {
                    // few tokens are allowed: one at a time, the others are not even looked at
                    float v[kBeamSparse];
#pragma unroll
                    for (int i = 0; i < kBeamSparse; ++i) {
                        const uint32_t at_i = slot + mis + (uint32_t)((lane * 32 + __ffs(w) - 1) * (int)sizeof(T));
                        v[i] = -INFINITY;
                        if (w) v[i] = sizeof(T) == 4 ? lds32f(at_i) : bf16_bits_to_f32(lds16u(at_i));
                        w &= w - 1;
                        gm = max_nan(gm, v[i]);
                    }
                    __syncwarp();
                    issue_next();
                    sum.add(v, gm);
                } else {
                    float v[32];
                    load_half<T, kAligned>(slot, mis, 0, reinterpret_cast<float(&)[16]>(v[0]));
                    load_half<T, kAligned>(slot, mis, 1, reinterpret_cast<float(&)[16]>(v[16]));
                    __syncwarp();
                    issue_next();  // the block is in registers: its slot takes the next copy
                    if (!all) {
                        const uint32_t mine = in_load_order<T, kAligned>(w);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(mine & (1u << i))) v[i] = -INFINITY;
                    }
                    float mx[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mx[i] = max3_nan(max3_nan(max3_nan(v[8 * i], v[8 * i + 1], v[8 * i + 2]), v[8 * i + 3], v[8 * i + 4]), max3_nan(v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]), -INFINITY);
                    gm = max3_nan(max_nan(mx[0], mx[1]), mx[2], mx[3]);
                    sum.add(v, gm);
                }
                if (++sc == slots) { sc = 0; phase ^= 1u; }
                gkey[at] = (uint16_t)(zkey(gm) >> 16);
                mm = max_nan(mm, gm);
                if (gm > top) {
                    top = gm;
                    top_tok = tok0 + 32 * lane + 31;
                }
            }
            // The warp's statistics, and the best of its lanes' best groups: no less than k distinct tokens reach the
            // k-th best of all those (a key names the group's last token, the true one is no smaller).
            for (int d = 16; d; d >>= 1) mm = max_nan(mm, __shfl_xor_sync(0xffffffffu, mm, d));
            int m1;
            float z1;
            units_of(A, mm, m1, z1);
            double part = mm < INFINITY ? in_units(A, sum.s, sum.m, sum.z0, m1, z1) : 0.0;
            for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
            if (lane == 0) {
                G.wmax[warp] = mm;
                G.wsum[warp] = part;
                G.wm[warp] = mm > -INFINITY && mm < INFINITY ? m1 : INT_MIN;
                G.wz0[warp] = z1;
            }
            unsigned long long left = top > -INFINITY ? make_ck(top, top_tok) : 0;
            const int busy = min(kBeamWarps, (G.hi - G.lo + kBlkTok - 1) / kBlkTok);
            for (int r = busy ? (want + busy - 1) / busy + 2 : 0; r > 0; --r) {
                const unsigned long long k = warp_max_key(left);
                if (k == 0) break;
                if (left == k) {
                    sh.seg[g].pool[atomicAdd(&G.n_pool, 1)] = k;
                    left = 0;
                }
            }
        }
        // ---- the history's tokens: their logits have just been streamed, so they come out of L2 (read before
        // the stream, from all over the row, they held it up for 6 us at 256 rows of 512 ids)
        if (hist) {
#pragma unroll 1
            for (int g = 0; g < ns; ++g) {
                auto& G = sh.sg[g];
                if (G.row < 0) continue;
                const int32_t* ids = own + g * A.hist_cap;
                float x[kIds], hm = -INFINITY;
#pragma unroll
                for (int j = 0; j < kIds; ++j) {
                    const int i = tid + j * kThreads, t = i < G.n_own ? ids[i] : -1;
                    x[j] = t >= 0 ? logit_at<T>(reinterpret_cast<const T*>(A.logits) + G.row * A.row_stride + t) : -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < kIds; ++j) {
                    const int i = tid + j * kThreads, t = i < G.n_own ? ids[i] : -1;
                    if (t < 0) continue;
                    int count = 1;
                    for (int k = 0; k < G.n_dups; ++k) count += dups[g * A.hist_cap + k] == t;
                    x[j] = penalise(A.params, x[j], count);
                    own_z[g * A.hist_cap + i] = x[j];
                    hm = max_nan(hm, x[j]);
                    for (int k = 0; k < A.n_stop; ++k)
                        if (A.stop_ids[k] == t) G.stop_z[k] = x[j];
                }
                for (int d = 16; d; d >>= 1) hm = max_nan(hm, __shfl_xor_sync(0xffffffffu, hm, d));
                if (lane == 0) G.hmax[warp] = hm;
            }
        }
        __syncthreads();

        // ---- a team of warps per segment: every warp its maximum and the key that at least K + n_stop tokens reach; a
        // share of the groups that reach it
        const int team = warp % ns, crew = kThreads / ns, me = warp / ns * 32 + lane;
        if (const int g = team; sh.sg[g].row >= 0) {
            auto& G = sh.sg[g];
            float bm = -INFINITY;
            if (lane < kBeamWarps) {
                bm = G.wmax[lane];
                if (hist) bm = max_nan(bm, G.hmax[lane]);
            }
            for (int d = 4; d; d >>= 1) bm = max_nan(bm, __shfl_xor_sync(0xffffffffu, bm, d));
            bm = __shfl_sync(0xffffffffu, bm, 0);
            int m1;
            float z1;
            units_of(A, bm, m1, z1);
            const int pooled = G.n_pool;
            unsigned long long bound = 1;
            if (pooled >= want) {
                const unsigned long long *pool = sh.seg[g].pool, k0 = lane < pooled ? pool[lane] : 0, k1 = lane + 32 < pooled ? pool[lane + 32] : 0;
                int a0 = 0, a1 = 0;
                for (int e = 0; e < pooled; ++e) {
                    const unsigned long long k = pool[e];
                    a0 += k > k0;
                    a1 += k > k1;
                }
                const unsigned long long mine = k0 && a0 == want - 1 ? k0 : k1 && a1 == want - 1 ? k1 : 0;
                bound = warp_max_key(mine);
            }
            auto add = [&](unsigned long long k) {
                if (k < bound || is_stop(A, ck_idx(k))) return;
                const int at = atomicAdd(&G.n_cand, 1);
                if (at < kBeamCand) sh.seg[g].cand[at] = k;
            };
            if (hist) {
                // (whole numbers: in which order the tokens come is a matter of chance, the sum must not be)
                BeamSum one(A);
                one.z0 = z1;
                one.m = m1;
                one.least = __fdividef((float)m1 - 100.0f, one.c);
                unsigned long long u = 0;
                for (int i = me; i < G.n_own; i += crew) {
                    const float x = own[g * A.hist_cap + i] >= 0 ? own_z[g * A.hist_cap + i] : -INFINITY;
                    if (!(x > -INFINITY)) continue;
                    u += __float2ull_rn(one.two(make_float2(x - z1, x - z1)).x * 1099511627776.0f);
                    add(make_ck(x, own[g * A.hist_cap + i]));
                }
                for (int d = 16; d; d >>= 1) u += __shfl_xor_sync(0xffffffffu, u, d);
                if (lane == 0 && u) atomicAdd(&G.hist_mass, u);
            }
            const uint32_t least = max((uint32_t)(bound >> 40), 0x80u);  // (0x7f is -inf)
            const int groups = (G.hi - G.lo + 31) / 32, first = (G.s0 - bits0) * 32;
            for (int i = me; i < groups; i += crew) {
                if (gkey[first + i] < least) continue;
                const int at = atomicAdd(&G.n_groups, 1);
                if (at < kBeamGroups) sh.seg[g].groups[at] = (uint16_t)i;
            }
            if (warp == g) {
                BeamRecord* rec = A.records + ((int)blockIdx.x + G.q);
                double sum = lane < kBeamWarps && bm < INFINITY ? in_units(A, G.wsum[lane], G.wm[lane], G.wz0[lane], m1, z1) : 0.0;
                for (int d = 4; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (lane == 0) {
                    rec->max = bm;
                    rec->failed = sh.failed;
                    rec->sum = sum;
                    rec->m = m1;
                    rec->z0 = z1;
                }
                if (lane < BORN_MAX_STOPS) rec->stop_z[lane] = G.stop_z[lane];
                // a range that begins with a piece leaves a gap in the row's records
                if (G.s0 == G.q * A.pb && G.s0 == t0 && G.q % A.pieces != 0) {
                    BeamRecord* gap = rec - 1;
                    if (lane == 0) {
                        gap->max = -INFINITY;
                        gap->m = INT_MIN;
                        gap->failed = 0;
                    }
                    if (lane < BORN_MAX_BEAMS) gap->list[lane] = 0;
                }
            }
            if (lane == 0 && warp == g) sh.seg[g].pool[kBeamPool - 1] = bound;
        }
        __syncthreads();
        // rank key of token `tok` of segment g, 0 = none
        auto key_at = [&](int g, int tok) {
            const auto& G = sh.sg[g];
            if (tok >= G.hi) return 0ull;
            if constexpr (kBits) {
                const int o = (G.s0 - bits0) * kBlkTok + tok - G.lo;
                if (!((bits[o >> 5] >> (o & 31)) & 1u)) return 0ull;
            }
            const float x = logit_at<T>(reinterpret_cast<const T*>(A.logits) + G.row * A.row_stride + tok);
            return x > -INFINITY ? (unsigned long long)make_ck(x, tok) : 0ull;
        };
        if (const int g = team; sh.sg[g].row >= 0) {
            auto& G = sh.sg[g];
            const unsigned long long bound = sh.seg[g].pool[kBeamPool - 1];
            if (warp == g && lane == 0 && hist) A.records[(int)blockIdx.x + G.q].sum += (double)G.hist_mass * 0x1p-40;
            const int listed = min(G.n_groups, kBeamGroups);
            for (int i = me >> 5; i < listed; i += crew >> 5) {
                const unsigned long long k = key_at(g, G.lo + (int)sh.seg[g].groups[i] * 32 + lane);
                if (k < bound || is_stop(A, ck_idx(k))) continue;
                const int at = atomicAdd(&G.n_cand, 1);
                if (at < kBeamCand) sh.seg[g].cand[at] = k;
            }
        }
        __syncthreads();
        const auto fits = [&](int g) { return sh.sg[g].n_cand <= kBeamCand && sh.sg[g].n_groups <= kBeamGroups; };
        if (const int g = team; sh.sg[g].row >= 0 && fits(g)) {
            unsigned long long* list = A.records[(int)blockIdx.x + sh.sg[g].q].list;
            const int found = sh.sg[g].n_cand;
            for (int i = me; i < found; i += crew) {
                const unsigned long long k = sh.seg[g].cand[i];
                int ahead = 0;
                for (int j = 0; j < found; ++j) ahead += sh.seg[g].cand[j] > k;
                if (ahead < K) list[ahead] = k;
            }
            if (me >= found && me < K) list[me] = 0;
        }
#pragma unroll 1
        for (int g = 0; g < ns; ++g) {
            const auto& G = sh.sg[g];
            if (G.row < 0 || fits(g)) continue;
            const int most = (G.hi - G.lo + kThreads - 1) / kThreads;
            slow_list(sh.seg[g].pool, A.records[(int)blockIdx.x + G.q].list, K, most + (hist ? BORN_MAX_HISTORY / kThreads : 0), [&](int i) {
                unsigned long long k = 0;
                if (i < most) k = key_at(g, G.lo + i * kThreads + tid);
                else if (const int e = (i - most) * kThreads + tid; e < G.n_own && own[g * A.hist_cap + e] >= 0 && own_z[g * A.hist_cap + e] > -INFINITY)
                    k = make_ck(own_z[g * A.hist_cap + e], own[g * A.hist_cap + e]);
                return k && !is_stop(A, ck_idx(k)) ? k : 0ull;
            });
        }
        __syncthreads();
        // ---- the groups' tickets, which count blocks
        if (tid < ns) {
            __threadfence();
            const int n = sh.sg[tid].q / A.pieces / K, add = sh.sg[tid].s1 - sh.sg[tid].s0;
            const bool mine = atomicAdd(&A.tickets[n], (uint32_t)add) == (uint32_t)(K * A.pieces * A.pb - add);
            if (mine) {
                A.tickets[n] = 0;
                __threadfence();
            }
            sh.last[tid] = mine ? n : -1;
        }
        __syncthreads();
#pragma unroll 1
        for (int g = 0; g < ns; ++g) {
            if (sh.last[g] < 0) continue;
            finish_group<T>(A, sh.last[g], sh, bits, own);
            __syncthreads();
        }
    }
    if (sh.failed) {
        // the copies in flight land before the CTA ends (bounded)
        if (tid == 0) atomicExch(A.dev_error, BORN_ERR_DEVICE_TIMEOUT);
        for (; in_flight > 0; --in_flight) {
            ring_wait(bar0 + (uint32_t)sc * 8u, phase, A.timeout_ns);
            if (++sc == slots) { sc = 0; phase ^= 1u; }
        }
    }
}

}  // namespace born
