// latent.h -- the paged latent cache of a batch of requests (internal).
//
// A key is a latent row (its value too) and a rope row; keys of a sequence are
// spread over pages that its table names.  A row is bf16 latent and rope values, or
// e2m1 codes of the latent values (32 to a power-of-two scale) and bf16 rope values.
#pragma once

#include "../../include/moonlight_kernels.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlh {

constexpr int kLatentMax = 512;       // values of a latent row
constexpr int kLatentRopeMax = 64;    // values of a rope row
constexpr int kLatentMaxHeads = 1024;
// A launch counts threads in 32 bits: a row of append is a workgroup, four of gather are.
constexpr int kLatentRowThreads = 256, kLatentGatherRows = 4;
constexpr int kLatentMaxAppend = 0xFFFFFFFFu / kLatentRowThreads;
constexpr int kLatentMaxGather = kLatentMaxAppend * kLatentGatherRows;
// Sequences are gone through in 32 bits, a workgroup's threads at a time, and counted with 2^27 tiles
// of 16 (row, head) pairs.
constexpr int kLatentMaxSeqs = 1 << 30;
constexpr int kFp4Group = 32;         // values of a scale
constexpr int kFp4ScaleBytes = 16;    // bytes of a row's scales
constexpr int kFp4Bias = 127;         // of a scale byte; 255: its values are NaN
constexpr int kFp4LeastExp = -100;    // (far from bf16's subnormals)

// Launches of `kernel` may ask for so much LDS beside its static arrays (else 64 KB).
template <class Kernel> inline bool allow_lds(Kernel kernel, int bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               bytes) == hipSuccess;
}

__host__ __device__ constexpr bool latent_widths_ok(int latent, int rope) {
    return latent > 0 && latent <= kLatentMax && latent % 64 == 0 && rope > 0 &&
           rope <= kLatentRopeMax && rope % 16 == 0;
}
// Bytes of a row's latent part, and of a row; a multiple of 16.
__host__ __device__ constexpr int latent_part_bytes(bool fp4, int latent) {
    return fp4 ? latent / 2 + kFp4ScaleBytes : 2 * latent;
}
__host__ __device__ constexpr int latent_row_bytes(bool fp4, int latent, int rope) {
    return latent_part_bytes(fp4, latent) + 2 * rope;
}

// The token rows of sequence s: rows begin .. begin + count - 1 of the batch, the last one
// key length - 1.  What the device's memory holds is not trusted; `begin` is below 0 where starts
// decrease, without which no row belongs to two sequences.
struct LatentSeq {
    int begin, count;
    int length;
};
__device__ __forceinline__ LatentSeq latent_seq(const MlkLatentBatch &b, int s, int rows) {
    const int length = b.lengths[s];
    if (!b.row_starts) return {s, s < rows ? 1 : 0, length};
    const int begin = b.row_starts[s], end = b.row_starts[s + 1];
    return {end < begin ? -1 : begin, begin >= 0 && begin < end && end <= rows ? end - begin : 0, length};
}

// The place of key j >= 0 of sequence s among the rows of all pages; -1: it has none.
__device__ __forceinline__ long latent_slot(const MlkLatentBatch &b, int s, unsigned j) {
    const unsigned at = j / (unsigned)b.page_size;
    if (at >= (unsigned)b.table_width) return -1;
    const int page = b.tables[(long)s * b.table_width + at];
    if ((unsigned)page >= (unsigned)b.pages) return -1;
    return (long)page * b.page_size + (j - at * (unsigned)b.page_size);
}

// Rows of type bf16 or f32 (`bf16`).
struct LatentAppend {
    bool bf16 = false;
    const void *kv = nullptr;
    long kv_stride = 0;
    const float *norm_w = nullptr;
    float eps = 0.0f;
    const float *inv_freq = nullptr;
    int rows = 0;
    const void *query = nullptr;
    long query_stride = 0;
    int heads = 0, head_width = 0;
    void *q = nullptr;
};
int latent_append(const MlkLatentBatch &b, const LatentAppend &p, hipStream_t stream);
int latent_gather(const MlkLatentBatch &b, bool bf16, int rows, void *out, hipStream_t stream);

struct LatentAttend {
    bool bf16 = false;
    const void *q = nullptr;
    void *out = nullptr;
    int rows = 0, heads = 0;
    float scale = 1.0f;
    void *workspace = nullptr;
};
size_t latent_attend_workspace();
int latent_attend(const MlkLatentBatch &b, const LatentAttend &p, int cu_count, hipStream_t stream);

// Log probabilities of rows of logits (logprobs.hip).
constexpr int kLogprobsMaxTop = 32;
constexpr int kLogprobsMaxVocab = 1 << 22;
struct TokenLogprobs {
    bool bf16 = false;
    const void *logits = nullptr;
    long stride = 0;
    int rows = 0, vocab = 0, top = 0;
    const int *tokens = nullptr;
    float *logprobs = nullptr, *entropy = nullptr;
    int *top_ids = nullptr;
    float *top_logprobs = nullptr;
    void *workspace = nullptr;
};
bool token_logprobs_fits(int rows, int vocab);  // into a launch
size_t token_logprobs_needs(int rows, int vocab, int top);      // of a call
size_t token_logprobs_workspace(int rows, int vocab, int top);  // of it and all smaller ones
int token_logprobs(const TokenLogprobs &p, hipStream_t stream);

}  // namespace mlh
