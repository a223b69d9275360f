// Host-side entry points of the beam-search kernels, instantiated in beam.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "../../include/born_sampler.h"

namespace born {

constexpr int kBeamPiece = 256;     // blocks of a piece of a row at most
constexpr int kBeamMaxSlots = 8;    // ring slots of a warp

// What a segment leaves for the merge.
struct BeamRecord {
    double sum;  // sum exp(z/T) over the segment, in units of 2^m exp(z0/T)
    int32_t m;   // INT_MIN: nothing
    float z0;
    float max;   // NaN / +inf: the segment holds one
    int32_t failed;  // a wait for a copy ran out
    int32_t pad[2];
    float stop_z[BORN_MAX_STOPS];  // penalised logits of the stop tokens in the segment, -inf elsewhere
    unsigned long long list[BORN_MAX_BEAMS];  // rank keys of the best tokens, 0 = none
};

struct BeamArgs {
    int N, K, V;
    // A row is `pieces` pieces of `pb` blocks of 1024 tokens (the last ones may be empty); the `blocks` blocks of
    // all rows are dealt to `grid` CTAs in equal ranges.
    int pieces, pb, blocks, grid;
    int slots, slot_bytes, bits_at, gkeys_at, hist_at, hist_cap;  // shared memory
    const void* logits;
    int64_t row_stride;
    const uint32_t* mask;
    int64_t mask_stride;
    const int32_t* history;
    const int32_t* history_len;
    int history_stride;
    uint32_t flags;
    born_row_params params;
    float temperature;
    float scale_log2e, scale_lo;  // log2(e)/T in two parts
    int exact;  // T is above 2^100: at last log2(e)/T is no number of full length in 32 bits, and the bound below which weights count as
                // 2^-100 overflows (a masked token would make the sum NaN); all normalisers are computed in 64 bits
    double inv_T;   // 1/T
    double slack;   // two normalisers in 32 bits are off by less than this together
    int bit_words;  // words of a CTA's bit map
    const float* scores;
    int32_t stop_ids[BORN_MAX_STOPS];
    int n_stop, step;
    int32_t *out_parent, *out_token;
    float* out_score;
    int32_t* out_status;
    int32_t *out_end_parent, *out_end_token;
    float* out_end_score;
    float* pool_score;
    int32_t *pool_step, *pool_parent, *pool_token, *done;
    double length_norm;
    // workspace
    BeamRecord* records;
    uint32_t* tickets;
    int* dev_error;
    unsigned long long timeout_ns;
    int debug_stuck_cta;  // test hook: its first warp never sees its first copy land (-1: none)
    // device-resident history (born_beam_next)
    int32_t *ring, *ring_total, *ring_len;
    int ring_cap;

    // (cta <= grid <= 2 SMs, and beam_launch admits 2^32 / (2 SMs) blocks: products fit 32 bits)
    __host__ __device__ int range_start(int cta) const { return (int)((unsigned)cta * (unsigned)blocks / (unsigned)grid); }
    // A segment is a CTA and a piece; from one to the next the CTA or the piece goes up by one, or both, so their
    // sum numbers the segments.  Of the segment that holds block t:
    __host__ __device__ int record_of(int t) const { return (int)(((unsigned)(t + 1) * (unsigned)grid - 1u) / (unsigned)blocks) + t / pb; }
};

// Records that launches of up to max_batch rows of up to max_vocab tokens leave.
int64_t beam_max_records(int max_batch, int max_vocab, int num_sms);
cudaError_t beam_attrs();
// Fills in how the rows are dealt and launches; cudaErrorNotSupported: more rows than the numbering of the blocks holds.
cudaError_t beam_launch(BeamArgs& A, int dtype, bool aligned, int num_sms, cudaStream_t st);

// ---- born_beam_reorder ------------------------------------------------------------------------
struct ReorderArgs {
    int N, K, n_buffers, planes;
    int64_t row_stride, plane_stride, position_bytes, positions;
    int64_t chunk;   // bytes of a piece that a CTA moves
    int chunks;      // of a piece
    const int32_t* parents;
    const int32_t* lens;
    uint8_t* buffers[BORN_MAX_REORDER];
};
cudaError_t reorder_launch(ReorderArgs& A, cudaStream_t st);

// ---- born_beam_sequences ------------------------------------------------------------------------
struct SequencesArgs {
    int N, K, T, H;
    int64_t table_stride, out_stride;
    const int32_t *tokens, *parents, *end_step, *end_parent, *end_token;
    int32_t *out_tokens, *out_lens;
    int32_t pad;
    int tile, shift;  // steps that a CTA's shared memory holds at a time, 2^shift places each
    int ranks;        // CTAs of a group
};
cudaError_t sequences_attrs();
cudaError_t sequences_launch(SequencesArgs& A, int num_sms, cudaStream_t st);

}  // namespace born
