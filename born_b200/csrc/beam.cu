// Beam search (step, reordering of states, read-out of sequences): instantiations and launches.
#include "beam_kernel.cuh"
#include "reorder_kernel.cuh"
#include "sequences_kernel.cuh"

namespace born {

// A slice's bits fill at most 37.5 KB of shared memory.
static int least_slices(int vocab) { return (vocab + 299999) / 300000; }

// Slices of at least 4096 tokens, as many as give every SM four CTAs.
int beam_slices(int rows, int vocab, int num_sms) {
    int s = (4 * num_sms + rows - 1) / rows;
    const int most = (vocab + 4095) / 4096;
    if (s > most) s = most;
    if (s > kBeamMaxSlices) s = kBeamMaxSlices;
    const int least = least_slices(vocab);
    if (s < least) s = least;
    return s < 1 ? 1 : s;
}
int64_t beam_max_records(int max_batch, int max_vocab, int num_sms) {
    // rows * beam_slices(rows): less than 4 CTAs per SM and one more per row, or the least slices of every row
    const int64_t fill = 4 * (int64_t)num_sms + max_batch, least = (int64_t)max_batch * least_slices(max_vocab);
    return fill > least ? fill : least;
}

// The normaliser log sum exp of a row in 32 bits.  Every value's exponent t (base 2, relative to a maximum
// that may be 2^8 behind) rounds by 2^-24 |t| in the subtraction, in the scaling and through the scale's own
// rounding, and sum p |t| <= log2(V) + 8; ex2 is off by 2^-22, once per value and once per thread;
// a thread's sum rounds once per turn of 16 values after a tree of 16.  The rest is in 64 bits.
static double beam_slack(int vocab, int slices) {
    const double u = ldexp(1.0, -24);
    const double turns = (double)vocab / slices / (16.0 * kThreads) + 8.0;
    const double one = 3 * u * (log2((double)vocab) + 8.0) * M_LN2 + 8 * u + (turns + 4.0) * u;
    return 2.0 * one;
}

template <typename T, bool kBits>
static cudaError_t raise_limit() {
    return cudaFuncSetAttribute(beam_kernel<T, kBits>, cudaFuncAttributeMaxDynamicSharedMemorySize, 40 * 1024);
}
cudaError_t beam_attrs() {
    cudaError_t e = raise_limit<float, true>();
    return e != cudaSuccess ? e : raise_limit<uint16_t, true>();
}

cudaError_t beam_launch(BeamArgs& A, int dtype, cudaStream_t st) {
    const int grid = A.N * A.K * A.slices;
    const bool has_bits = A.mask || A.history;
    // vectors per slice, rounded up, and the two words of the tokens beside them
    const int vec = dtype == BORN_DTYPE_F32 ? 4 : 8;
    A.bit_words = has_bits ? ((A.V / vec + A.slices) / A.slices * vec + 31) / 32 + 2 : 0;
    A.slack = beam_slack(A.V, A.slices);
    const size_t smem = (size_t)A.bit_words * 4;
    if (dtype == BORN_DTYPE_F32) {
        if (has_bits) beam_kernel<float, true><<<grid, kThreads, smem, st>>>(A);
        else beam_kernel<float, false><<<grid, kThreads, 0, st>>>(A);
    } else {
        if (has_bits) beam_kernel<uint16_t, true><<<grid, kThreads, smem, st>>>(A);
        else beam_kernel<uint16_t, false><<<grid, kThreads, 0, st>>>(A);
    }
    return cudaGetLastError();
}

// The widest vectors that every row and piece is aligned to; ranges of 32 KB a CTA, smaller ones where
// those would not fill the GPU.
cudaError_t reorder_launch(ReorderArgs& A, cudaStream_t st) {
    const int64_t piece = A.positions * A.position_bytes;
    if (piece == 0) return cudaSuccess;
    uint64_t low = (uint64_t)A.row_stride | (uint64_t)(A.planes > 1 ? A.plane_stride : 0);
    for (int i = 0; i < A.n_buffers; ++i) low |= (uint64_t)(uintptr_t)A.buffers[i];
    const int64_t pieces = (int64_t)A.N * A.n_buffers * A.planes;
    A.chunk = 32768;
    while (A.chunk > 4096 && pieces * ((piece + A.chunk - 1) / A.chunk) < 1024) A.chunk /= 2;
    while (pieces * ((piece + A.chunk - 1) / A.chunk) > 0x7fffffff) A.chunk *= 2;
    A.chunks = (int)((piece + A.chunk - 1) / A.chunk);
    const unsigned grid = (unsigned)(pieces * A.chunks);
    if (low % 16 == 0) reorder_kernel<uint4><<<grid, kReorderThreads, 0, st>>>(A);
    else if (low % 4 == 0) reorder_kernel<uint32_t><<<grid, kReorderThreads, 0, st>>>(A);
    else if (low % 2 == 0) reorder_kernel<uint16_t><<<grid, kReorderThreads, 0, st>>>(A);
    else reorder_kernel<uint8_t><<<grid, kReorderThreads, 0, st>>>(A);
    return cudaGetLastError();
}

cudaError_t sequences_attrs() {
    return cudaFuncSetAttribute(sequences_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 10 * kSequenceMaxSteps);
}
cudaError_t sequences_launch(const SequencesArgs& A, cudaStream_t st) {
    sequences_kernel<<<A.N, kSeqThreads, (size_t)A.T * 10, st>>>(A);
    return cudaGetLastError();
}

}  // namespace born
