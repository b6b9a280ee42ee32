// latent_api.cpp -- the latent cache and log probability entry points of
// include/moonlight_kernels.h.
#include "entry_checks.h"
#include "latent.h"

#include <math.h>

using namespace mlh;

namespace {

constexpr long kMaxPairs = 0x7FFFFFFF - 15;  // (row, head) pairs, counted in 32 bits

int check_batch(const char *what, const MlkLatentBatch *b, int rows) {
    if (!b) return refuse(what, "batch is null");
    if (b->type != MLK_BF16 && b->type != MLK_FP4)
        return refuse(what, "the batch's type must be MLK_BF16 or MLK_FP4");
    if (!latent_widths_ok(b->latent, b->rope))
        return refuse(what, "latent must be a multiple of 64 up to 512, rope a multiple of 16 up to 64");
    if (b->pages <= 0 || b->page_size <= 0 || b->seqs < 0 || b->table_width <= 0)
        return refuse(what, "pages, page_size and table_width must be > 0, seqs >= 0");
    if (b->seqs > kLatentMaxSeqs) return refuse(what, "seqs must be at most 2^30", kErrSize);
    if (rows < 0) return refuse(what, "rows must be >= 0");
    if (!b->row_starts && rows < b->seqs)
        return refuse(what, "without row_starts every sequence needs a row");
    return kOk;
}

#define LATENT_BATCH_POINTERS(b)                                                            \
    {(b)->data, "data", 16, false}, {(b)->tables, "tables", 4, false},                      \
        {(b)->lengths, "lengths", 4, false}, {(b)->row_starts, "row_starts", 4, true}

}  // namespace

extern "C" {

size_t mlk_latent_row_bytes(int type, int latent, int rope) {
    if ((type != MLK_BF16 && type != MLK_FP4) || !latent_widths_ok(latent, rope)) return 0;
    return latent_row_bytes(type == MLK_FP4, latent, rope);
}

int mlk_latent_append(const MlkLatentBatch *batch, int type, const void *kv, long kv_stride,
                      const float *norm_w, float eps, const float *inv_freq, int rows,
                      const void *query, long query_stride, int heads, int head_width, void *q) {
    const char *what = "mlk_latent_append";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_batch(what, batch, rows)) return e;
    if (rows > kLatentMaxAppend) return refuse(what, "rows must be below 2^24", kErrSize);
    if (kv_stride < batch->latent + batch->rope)
        return refuse(what, "kv_stride must be at least latent + rope");
    if (!(eps >= 0.0f) || isinf(eps)) return refuse(what, "eps must be finite and >= 0");
    if (query) {
        if (heads <= 0 || heads > kLatentMaxHeads)
            return refuse(what, "heads must be > 0 and at most 1024");
        if (head_width < batch->rope) return refuse(what, "head_width must be at least rope");
        if (query_stride < (long)heads * head_width)
            return refuse(what, "query_stride must be at least heads * head_width");
        if (!q) return refuse(what, "q is null");
    }
    if (rows == 0 || batch->seqs == 0) return kOk;
    const unsigned size = size_of(type);
    const Pointer list[] = {LATENT_BATCH_POINTERS(batch),
                            {kv, "kv", size, false},
                            {norm_w, "norm_w", 4, true},
                            {inv_freq, "inv_freq", 4, false},
                            {query, "query", size, true},
                            {query ? q : nullptr, "q", size, true}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    LatentAppend p;
    p.bf16 = type == MLK_BF16;
    p.kv = kv;
    p.kv_stride = kv_stride;
    p.norm_w = norm_w;
    p.eps = eps;
    p.inv_freq = inv_freq;
    p.rows = rows;
    p.query = query;
    p.query_stride = query_stride;
    p.heads = heads;
    p.head_width = head_width;
    p.q = q;
    return finish(latent_append(*batch, p, st), what);
}

int mlk_latent_gather(const MlkLatentBatch *batch, int type, int rows, void *out) {
    const char *what = "mlk_latent_gather";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_batch(what, batch, rows)) return e;
    if (rows > kLatentMaxGather) return refuse(what, "rows must be at most 2^26 - 4", kErrSize);
    if (rows == 0 || batch->seqs == 0) return kOk;
    const Pointer list[] = {LATENT_BATCH_POINTERS(batch), {out, "out", size_of(type), false}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    return finish(latent_gather(*batch, type == MLK_BF16, rows, out, st), what);
}

size_t mlk_latent_attend_workspace(void) { return latent_attend_workspace(); }

int mlk_latent_attend(const MlkLatentBatch *batch, int type, const void *q, void *out, int rows,
                      int heads, float scale, void *workspace, size_t workspace_bytes) {
    const char *what = "mlk_latent_attend";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_batch(what, batch, rows)) return e;
    if (heads <= 0 || heads > kLatentMaxHeads)
        return refuse(what, "heads must be > 0 and at most 1024");
    if ((long)rows * heads > kMaxPairs)
        return refuse(what, "rows * heads must be below 2^31 - 15", kErrSize);
    // (times log2(e) it has to be an f32 too)
    if (!(fabsf(scale) < 0x1p127f)) return refuse(what, "scale must be finite and below 2^127");
    if (rows == 0 || batch->seqs == 0) return kOk;
    if (workspace_bytes < latent_attend_workspace())
        return refuse(what, "the workspace needs " + std::to_string(latent_attend_workspace()) + " bytes");
    const unsigned size = size_of(type);
    const Pointer list[] = {LATENT_BATCH_POINTERS(batch),
                            {q, "q", size, false},
                            {out, "out", size, false},
                            {workspace, "workspace", 16, false}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    LatentAttend p;
    p.bf16 = type == MLK_BF16;
    p.q = q;
    p.out = out;
    p.rows = rows;
    p.heads = heads;
    p.scale = scale;
    p.workspace = workspace;
    return finish(latent_attend(*batch, p, context()->cu_count, st), what);
}

size_t mlk_token_logprobs_workspace(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || vocab > kLogprobsMaxVocab || top < 0 || top > kLogprobsMaxTop) return 0;
    return token_logprobs_workspace(rows, vocab, top);
}

int mlk_token_logprobs(int type, const void *logits, long stride, int rows, int vocab,
                       const int *tokens, float *logprobs, float *entropy, int top, int *top_ids,
                       float *top_logprobs, void *workspace, size_t workspace_bytes) {
    const char *what = "mlk_token_logprobs";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (rows < 0) return refuse(what, "rows must be >= 0");
    if (vocab <= 0) return refuse(what, "vocab must be > 0");
    if (vocab > kLogprobsMaxVocab) return refuse(what, "vocab must be at most 2^22", kErrSize);
    if (stride < vocab) return refuse(what, "stride must be at least vocab");
    if (top < 0 || top > kLogprobsMaxTop || top > vocab)
        return refuse(what, "top must be between 0 and 32, and at most vocab");
    if (rows == 0) return kOk;
    if (!token_logprobs_fits(rows, vocab))
        return refuse(what, "too many rows of so many logits for one launch", kErrSize);
    const size_t need = token_logprobs_needs(rows, vocab, top);
    if (workspace_bytes < need)
        return refuse(what, "the workspace needs " + std::to_string(need) + " bytes");
    const unsigned size = size_of(type);
    const Pointer list[] = {{logits, "logits", size, false},
                            {tokens, "tokens", 4, false},
                            {logprobs, "logprobs", 4, false},
                            {entropy, "entropy", 4, true},
                            {top ? top_ids : nullptr, "top_ids", 4, top == 0},
                            {top ? top_logprobs : nullptr, "top_logprobs", 4, top == 0},
                            {need ? workspace : nullptr, "workspace", 16, need == 0}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    TokenLogprobs p;
    p.bf16 = type == MLK_BF16;
    p.logits = logits;
    p.stride = stride;
    p.rows = rows;
    p.vocab = vocab;
    p.tokens = tokens;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.top = top;
    p.top_ids = top_ids;
    p.top_logprobs = top_logprobs;
    p.workspace = workspace;
    return finish(token_logprobs(p, st), what);
}

}  // extern "C"
