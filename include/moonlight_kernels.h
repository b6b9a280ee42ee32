/*
 * moonlight_kernels.h -- kernel-level C ABI of the MI355X Moonlight library.
 *
 * These entry points take DEVICE pointers (from mlk_malloc) and run on the
 * library's HIP stream; they are what moonlight_hip.h's session runtime is
 * built from, exposed for callers that keep their own buffers in HBM (and for
 * the parity tests and bench).  Every function returns 0 on success or a
 * negative status (-1 bad arguments, -2 launch failure, -3 device error,
 * -4 size limit); mlk_last_error() describes the last failure.
 *
 * Reference interfaces replaced (paths in c4pt0r/floyd):
 *   mlk_gemv           moonlight_matmul_f32 / _q8_reduction / _q4
 *                      (moonlight_kernels.metal:43-130) as encoded by
 *                      encode_matmul_at (moonlight_metal.m:164-197)
 *   mlk_gemv_swiglu    gate + up matmuls + moonlight_silu_multiply
 *                      (moonlight_metal.m:459-472, moonlight_kernels.metal:533-541)
 *   mlk_route_topk     moonlight_route_sigmoid_topk (moonlight_kernels.metal:469-512)
 *                      = moe_route_select + moe_route_finalize (moe_route.h:47-99)
 *   mlk_quantize       quant_int8 / quant_int4 (tools/convert_moonlight.py:46-66)
 *   mlk_sample         choose_token (moonlight_chat.c:96-131), the caller-side
 *                      sampler, on device logits
 */
#ifndef MOONLIGHT_KERNELS_H
#define MOONLIGHT_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Weight formats of mlk_gemv; MLK_F32 and MLK_BF16 are also the types of the
 * values that the fp8 entry points take and return beside their codes. */
enum { MLK_F32 = 0, MLK_Q8 = 1, MLK_Q4 = 2, MLK_BF16 = 3 };

/* ---- device plumbing (no counterpart in the reference: Metal used shared
 *      memory buffers, moonlight_metal.m:733-755) ---------------------------- */
int mlk_init(void);
const char *mlk_device_name(void);
const char *mlk_last_error(void);
void *mlk_malloc(size_t bytes);
int mlk_free(void *ptr);
int mlk_memcpy_h2d(void *dst, const void *src, size_t bytes);
int mlk_memcpy_d2h(void *dst, const void *src, size_t bytes);
int mlk_memcpy_d2d(void *dst, const void *src, size_t bytes);
int mlk_memset(void *dst, int value, size_t bytes);
int mlk_synchronize(void);

/* ---- dequant matmul ------------------------------------------------------
 * y[b, o] = (sum_i xn[b, i] * W[o, i]) * s[o] (+ resid[b, o]) for b < rows,
 * with W f32 [O, I], int8 [O, I] or packed int4 [O, ceil(I/2)] and one f32
 * scale per output row; xn = RMSNorm(x) * norm_w when norm_w != NULL
 * (moonlight_kernels.metal:23-41), else x.  x, y, resid are dense [rows, *]. */
int mlk_gemv(int fmt, const void *w, const float *s, const float *x, float *y,
             int out_width, int in_width, int rows, const float *norm_w,
             float eps, const float *resid);
/* h[b, j] = silu(gate_j . xn_b) * (up_j . xn_b), gate/up of one format. */
int mlk_gemv_swiglu(int fmt, const void *w_gate, const float *s_gate,
                    const void *w_up, const float *s_up, const float *x,
                    float *h, int out_width, int in_width, int rows,
                    const float *norm_w, float eps);
/* Name of the kernel instantiation mlk_gemv (swiglu = 0) or mlk_gemv_swiglu
 * (swiglu = 1) launches for this shape, as profilers print it; written into
 * name[name_size]. */
int mlk_gemv_kernel_name(int fmt, int out_width, int in_width, int rows,
                         int swiglu, char *name, size_t name_size);
/* Average device time per launch (microseconds) of `iters` back-to-back
 * mlk_gemv launches that rotate over n_copies weight copies (defeats the
 * 256 MB last-level cache), measured with HIP events on the library stream.
 * use_graph != 0 replays the launches from one captured hipGraph. */
int mlk_time_gemv(int fmt, const void *const *w_copies,
                  const float *const *s_copies, int n_copies, const float *x,
                  float *y, int out_width, int in_width, int rows, int warmup,
                  int iters, int use_graph, double *avg_us);

/* Average device time per launch (microseconds) of a plain 16-byte streaming
 * copy of `bytes` (rotating over n_buffers source/destination pairs): the
 * measured HBM yardstick reported beside the GEMV roofline. */
int mlk_time_copy(void *const *src, void *const *dst, int n_buffers,
                  size_t bytes, int warmup, int iters, double *avg_us);

/* Same for a read-only stream of `bytes` split over `blocks` workgroups
 * (scratch: blocks * 4 words of device memory): the ceiling a GEMV reading
 * that many bytes can reach, launch ramp and tail included. */
int mlk_time_read(void *const *src, int n_buffers, size_t bytes, int blocks,
                  unsigned *scratch, int warmup, int iters, double *avg_us);

/* ---- routing --------------------------------------------------------------
 * Sigmoid top-k of rows x experts router logits: ids[r, k] is the expert with
 * the k-th largest sigmoid(logit) + bias (lower index on ties; NaN and -inf
 * never taken, -1 when fewer than top_k can be), weights[r, k] its sigmoid
 * score, divided by the row's sum (+ 1e-20) when normalize, times
 * routed_scale.  Runs the decode path's routing kernels and waits for them. */
int mlk_route_topk(const float *logits, const float *bias, int rows, int experts,
                   int top_k, int normalize, float routed_scale, int *ids,
                   float *weights);

/* ---- token choice ---------------------------------------------------------
 * The token choose_token (moonlight_chat.c:96-131) picks from `vocab` device
 * logits with the caller's draw u in [0, 1) (random_unit,
 * moonlight_chat.c:89-94): the first index of the maximum when temperature
 * <= 0, else the top-p draw.  The device sampler that
 * moonlight_session_sample runs; writes *token (host memory) and waits.
 * Non-finite logits under a top-p draw return -1 ("logits are not finite"). */
int mlk_sample(const float *logits, int vocab, float temperature, float top_p,
               double u, int *token);

/* ---- packing / synthetic weights ---------------------------------------- */
int mlk_quantize(int bits, const float *w, int rows, int cols, uint8_t *q,
                 float *s);
int mlk_fill_normal(float *out, int64_t n, uint64_t seed, float mean,
                    float std, int bf16);

/* ---- fp8 rows and products ------------------------------------------------
 * No counterpart in the reference, whose matrices are int8 or int4 with f32
 * activations.  Values are e4m3 codes (one byte; largest value 448) times an
 * f32 scale per block: 128 columns of one row for activations, 128 x 128 for
 * matrices, the form that fp8 checkpoints of this architecture come in.  A
 * [rows, cols] tensor of codes is dense, its scales are
 * [rows or ceil(rows / 128), ceil(cols / 128)] f32; the last block of a row
 * and of a column may be narrower.  Any width up to 2^30 and any alignment of
 * codes is taken; widths that are multiples of 16 at 16-byte addresses are
 * faster.  (A product of more than 2^23 - 16 tiles of 128 x 128 results, those
 * of a group its own, may be refused with -4.)
 *
 * Quantising: scale = max(amax / 448, 2^-126) with amax the block's largest
 * magnitude, code = the e4m3 value nearest to x * (1 / scale), ties to even;
 * quotients and product in f32.  A NaN keeps to its own code; a block that
 * holds an infinity gets an infinite scale, and all of it reads as NaN.
 *
 * Like mlk_gemv these queue their work on the library stream of the current
 * device and return (work of other streams on the same memory has to be
 * waited for by the caller, before and after); they allocate nothing and
 * keep nothing.  Pointers have to be memory of the current device (-1
 * otherwise), f32, bf16 and int values at addresses of their own size.
 * rows = 0 (entries = 0) writes nothing.  Outputs must not overlap inputs
 * unless stated. */

/* Codes and scales of x, f32 or bf16 [rows, cols] (type MLK_F32 or MLK_BF16):
 * block_rows = 1 for activations, 128 for matrices. */
int mlk_quantize_fp8(int type, const void *x, int rows, int cols,
                     int block_rows, uint8_t *q, float *s);
/* h = x + resid (resid == NULL: h = x), rounded to `type` and stored to sum
 * unless that is NULL; q, s = the codes and scales (block_rows = 1) of
 * RMSNorm(h) * norm_w, the norm as in mlk_gemv.  x, resid and sum are of one
 * type; sum may be x or resid itself. */
int mlk_rmsnorm_fp8(int type, const void *x, const void *resid,
                    const float *norm_w, float eps, int rows, int cols,
                    void *sum, uint8_t *q, float *s);
/* Codes and scales (block_rows = 1) of silu(gate) * up, gate_up [rows,
 * 2 * width] holding each row's gate values and then its up values. */
int mlk_swiglu_fp8(int type, const void *gate_up, int rows, int width,
                   uint8_t *q, float *s);
/* y[r, o] = sum_i x[r, i] W[o, i] (+ resid[r, o]) for codes x [rows, in_width]
 * with scales xs and codes w [out_width, in_width] with scales ws; y and
 * resid of out_type, MLK_F32 or MLK_BF16 (rounded once, resid added before;
 * y may be resid itself).  A block's product is scaled by its two scales'
 * product, which has to be finite in f32.
 * Sums are f32, with one exception: for MLK_BF16 outputs of many rows (which
 * calls those are is the library's choice, by their sizes) a block's products
 * come from the fp8 matrix instructions, which cut the 8 products of
 * neighbouring columns below 2^-13 of the largest before they add them.  That
 * is at most 2^-10 of the sum of these largest products: below the rounding of
 * an output of ordinary size, but an output that is small because large
 * products cancel in it may keep none of its bits, and a row's result may
 * depend on how many rows are in the call by as much.  Ask for MLK_F32 outputs
 * where that matters: theirs are always f32 sums. */
int mlk_matmul_fp8(int out_type, const uint8_t *w, const float *ws,
                   const uint8_t *x, const float *xs, void *y, int out_width,
                   int in_width, int rows, const void *resid);
/* The same with one matrix per group of rows (w [groups, out_width, in_width],
 * ws likewise): y [entries, out_width] holds the groups' rows one after the
 * other, group g's from offsets[g] to offsets[g + 1] (device memory,
 * groups + 1 numbers that do not decrease; a group may be empty).  Row j of
 * y is the product of x row row_ids[j], or of x row j where row_ids == NULL.
 * With row_ids x_rows * ceil(in_width / 128) has to be below 0x3C000000 (-4).
 * Rows of y before offsets[0] and from offsets[groups] on are left as they
 * were.  A row whose row_ids[j] is outside [0, x_rows) becomes NaN.  With
 * offsets that decrease or leave [0, entries] the rows of y are unspecified,
 * but nothing is read or written out of range. */
int mlk_matmul_fp8_grouped(int out_type, const uint8_t *w, const float *ws,
                           const uint8_t *x, const float *xs, int x_rows,
                           void *y, int out_width, int in_width, int groups,
                           const int *offsets, const int *row_ids,
                           int entries);

#ifdef __cplusplus
}
#endif
#endif
