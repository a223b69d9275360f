// Beam search (step, reordering of states, read-out of sequences): instantiations and launches.
#include <string.h>
#include "beam_kernel.cuh"
#include "reorder_kernel.cuh"
#include "sequences_kernel.cuh"

namespace born {

// The fewest pieces of at most `most` blocks.
static void row_pieces(int vocab, int most, int& pieces, int& pb) {
    const int nb = (vocab + kBlkTok - 1) / kBlkTok;
    pieces = (nb + most - 1) / most;
    pb = (nb + pieces - 1) / pieces;
}
constexpr int kBeamLeastPiece = 48;  // blocks that a piece is not cut below for the sake of a longer ring
int64_t beam_max_records(int max_batch, int max_vocab, int num_sms) {
    int pieces, pb;
    row_pieces(max_vocab, kBeamLeastPiece, pieces, pb);
    return 2 * (int64_t)num_sms + (int64_t)max_batch * (pieces + 1);  // (CTAs and pieces; a CTA of its own for every piece)
}

// What the normalisers log sum exp of two rows are off by at most in 32 bits (BeamSum): every value by ex2's
// 2^-22 and 2^-25 of the fraction in the exponent, sums of 32 by their six rounded additions; the rest is in 64 bits.
static double beam_slack() {
    const double u = ldexp(1.0, -24);
    return 2.0 * (4 * u + 0.5 * u + 6 * u + 0.5 * u);
}

// Dynamic shared memory of a CTA, two of which share an SM's 228 KB.
constexpr int kBeamSmem = (228 * 1024 / 2 - 1024 - (int)sizeof(BeamShared) - 8 * kBeamWarps * kBeamMaxSlots - 16) & ~127;
template <typename T, bool kBits, bool kAligned>
static cudaError_t raise_limit() {
    return cudaFuncSetAttribute(beam_kernel<T, kBits, kAligned>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBeamSmem);
}
template <typename T>
static cudaError_t raise_limits() {
    cudaError_t e;
    if ((e = raise_limit<T, false, false>()) != cudaSuccess || (e = raise_limit<T, false, true>()) != cudaSuccess) return e;
    if ((e = raise_limit<T, true, false>()) != cudaSuccess) return e;
    return raise_limit<T, true, true>();
}
cudaError_t beam_attrs() {
    const cudaError_t e = raise_limits<float>();
    return e != cudaSuccess ? e : raise_limits<uint16_t>();
}

// A launch, in clusters of `cluster` CTAs, that may begin while the one before it ends (the kernels wait before they read).
template <typename... P, typename... Q>
static cudaError_t launch_clusters(int cluster, void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, const Q&... args) {
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... Q>
static cudaError_t launch_after(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t st, const Q&... args) {
    return launch_clusters(1, kernel, grid, threads, smem, st, args...);
}

template <typename T>
static cudaError_t beam_launch_as(const BeamArgs& A, bool has_bits, bool aligned, size_t smem, cudaStream_t st) {
    const unsigned grid = (unsigned)A.grid;
    if (has_bits)
        return aligned ? launch_after(beam_kernel<T, true, true>, grid, kThreads, smem, st, A) : launch_after(beam_kernel<T, true, false>, grid, kThreads, smem, st, A);
    return aligned ? launch_after(beam_kernel<T, false, true>, grid, kThreads, smem, st, A) : launch_after(beam_kernel<T, false, false>, grid, kThreads, smem, st, A);
}

cudaError_t beam_launch(BeamArgs& A, int dtype, bool aligned, int num_sms, cudaStream_t st) {
    const bool has_bits = A.mask || A.history;
    const int esz = dtype == BORN_DTYPE_F32 ? 4 : 2;
    A.slot_bytes = ring_slot_bytes(esz, aligned);
    A.hist_cap = A.history ? (A.history_stride + 31) / 32 * 32 : 0;  // ids, penalised logits and later occurrences of each segment
    const int hist_bytes = kBeamSegs * A.hist_cap * 12;
    int bit_bytes = 0, key_bytes = 0;
    // as few pieces as possible, more where two segments' bits and keys would leave a warp fewer than two ring slots
    for (int most = kBeamPiece;; most = most * 3 / 4 > kBeamLeastPiece ? most * 3 / 4 : kBeamLeastPiece) {
        row_pieces(A.V, most, A.pieces, A.pb);
        const int64_t pieces = (int64_t)A.N * A.K * A.pieces, blocks = pieces * A.pb;
        if (blocks > (int64_t)(0xffffffffu / (2u * (unsigned)num_sms))) return cudaErrorNotSupported;  // (range_start, record_of: 32 bits)
        A.blocks = (int)blocks;
        // a block per warp at least, a CTA of its own for every piece while the GPU holds them at once
        int64_t grid = (blocks + kBeamWarps - 1) / kBeamWarps;
        if (grid < pieces) grid = pieces;
        if (grid > 2 * num_sms) grid = 2 * num_sms;
        A.grid = (int)grid;
        const int range = (int)((blocks + grid - 1) / grid), seg = range < kBeamSegs * A.pb ? range : kBeamSegs * A.pb;  // blocks taken at a time
        bit_bytes = has_bits ? seg * 128 : 0;
        key_bytes = (seg * 64 + 127) & ~127;
        A.slots = (kBeamSmem - bit_bytes - key_bytes - hist_bytes) / (kBeamWarps * A.slot_bytes);
        const int need = (range + kBeamWarps - 1) / kBeamWarps;
        if (A.slots > need) A.slots = need;
        if (A.slots > kBeamMaxSlots) A.slots = kBeamMaxSlots;
        if (A.slots >= (need < 2 ? need : 2) || most == kBeamLeastPiece) break;
    }
    if (A.slots < 1) return cudaErrorInvalidValue;
    A.bit_words = bit_bytes / 4;
    A.bits_at = kBeamWarps * A.slots * A.slot_bytes;
    A.gkeys_at = A.bits_at + bit_bytes;
    A.slack = beam_slack();
    A.hist_at = A.gkeys_at + key_bytes;
    const size_t smem = (size_t)A.hist_at + hist_bytes;
    if (dtype == BORN_DTYPE_F32) return beam_launch_as<float>(A, has_bits, aligned, smem, st);
    return beam_launch_as<uint16_t>(A, has_bits, aligned, smem, st);
}

template <typename W>
static cudaError_t reorder_launch_as(const ReorderArgs& A, unsigned grid, cudaStream_t st) {
    if (A.K <= 4) return launch_after(reorder_kernel<W, 4>, grid, kReorderThreads, 0, st, A);
    return launch_after(reorder_kernel<W, BORN_MAX_BEAMS>, grid, kReorderThreads, 0, st, A);
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
    if (low % 16 == 0) return reorder_launch_as<uint4>(A, grid, st);
    if (low % 4 == 0) return reorder_launch_as<uint32_t>(A, grid, st);
    if (low % 2 == 0) return reorder_launch_as<uint16_t>(A, grid, st);
    return reorder_launch_as<uint8_t>(A, grid, st);
}

constexpr int kSeqSmem = 108 * 1024;  // two CTAs per SM
cudaError_t sequences_attrs() { return cudaFuncSetAttribute(sequences_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSeqSmem); }
cudaError_t sequences_launch(SequencesArgs& A, int num_sms, cudaStream_t st) {
    A.shift = 2;
    while ((1 << A.shift) < A.K || (1 << A.shift) < A.H) ++A.shift;
    A.ranks = 1;
    // A cluster costs 1.5 us with two CTAs, 2.5 to 4 with four, and shares out the tables' bytes: 64 groups of 8 take 11 / 10 /
    // 12 us for 1024 steps with one, two, four CTAs each, 38 / 25 / 20.5 us for 4096; one group of 4 8 / 8 / 9 and 21 / 14 / 11 us.
    // Clusters that do not fit the GPU at once lose (256 groups, 1024 steps: 13 / 21 / 40 us).
    while (A.ranks < kSeqRanks && A.ranks * A.N <= num_sms && A.T > A.ranks * 1024) A.ranks *= 2;
    const int each = (A.T + A.ranks * kSeqChunks - 1) / (A.ranks * kSeqChunks) * kSeqChunks;
    A.tile = kSeqSmem / (6 << A.shift) / kSeqChunks * kSeqChunks;  // a token and two bytes per beam
    if (A.tile > each) A.tile = each;
    return launch_clusters(A.ranks, sequences_kernel, (unsigned)(A.N * A.ranks), kSeqThreads, (size_t)A.tile * (6 << A.shift), st, A);
}

}  // namespace born
