// fp8_api.cpp -- the fp8 entry points of include/moonlight_kernels.h.
#include "entry_checks.h"
#include "fp8.h"

#include <math.h>

using namespace mlh;

namespace {

int check_rows(const char *what, int rows, const char *name, int width) {
    if (rows < 0) return refuse(what, "rows must be >= 0");
    if (width <= 0 || width > kFp8MaxWidth)
        return refuse(what, std::string(name) + " must be > 0 and at most 2^30");
    return kOk;
}

Fp8Rows rows_of(int type, const void *x, int rows, int cols, uint8_t *q, float *s) {
    Fp8Rows p;
    p.bf16 = type == MLK_BF16;
    p.x = x;
    p.rows = rows;
    p.cols = cols;
    p.q = q;
    p.scale = s;
    return p;
}

}  // namespace

extern "C" {

int mlk_quantize_fp8(int type, const void *x, int rows, int cols, int block_rows, uint8_t *q,
                     float *s) {
    const char *what = "mlk_quantize_fp8";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_rows(what, rows, "cols", cols)) return e;
    if (block_rows != 1 && block_rows != kFp8Block) return refuse(what, "block_rows must be 1 or 128");
    if (rows == 0) return kOk;
    const Pointer list[] = {{x, "x", size_of(type), false}, {q, "q", 1, false}, {s, "s", 4, false}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    return finish(fp8_quantize(rows_of(type, x, rows, cols, q, s), block_rows, st), what);
}

int mlk_rmsnorm_fp8(int type, const void *x, const void *resid, const float *norm_w, float eps,
                    int rows, int cols, void *sum, uint8_t *q, float *s) {
    const char *what = "mlk_rmsnorm_fp8";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_rows(what, rows, "cols", cols)) return e;
    if (!(eps >= 0.0f) || isinf(eps)) return refuse(what, "eps must be finite and >= 0");
    if (rows == 0) return kOk;
    const unsigned size = size_of(type);
    const Pointer list[] = {{x, "x", size, false},  {resid, "resid", size, true},
                            {norm_w, "norm_w", 4, false}, {sum, "sum", size, true},
                            {q, "q", 1, false},     {s, "s", 4, false}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    return finish(fp8_rmsnorm(rows_of(type, x, rows, cols, q, s), resid, norm_w, eps, sum, st), what);
}

int mlk_swiglu_fp8(int type, const void *gate_up, int rows, int width, uint8_t *q, float *s) {
    const char *what = "mlk_swiglu_fp8";
    if (!type_ok(type)) return refuse(what, "type must be MLK_F32 or MLK_BF16");
    if (int e = check_rows(what, rows, "width", width)) return e;
    if (rows == 0) return kOk;
    const Pointer list[] = {{gate_up, "gate_up", size_of(type), false}, {q, "q", 1, false},
                            {s, "s", 4, false}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    return finish(fp8_swiglu(rows_of(type, gate_up, rows, width, q, s), st), what);
}

int mlk_matmul_fp8(int out_type, const uint8_t *w, const float *ws, const uint8_t *x,
                   const float *xs, void *y, int out_width, int in_width, int rows,
                   const void *resid) {
    const char *what = "mlk_matmul_fp8";
    if (!type_ok(out_type)) return refuse(what, "out_type must be MLK_F32 or MLK_BF16");
    if (int e = check_rows(what, rows, "out_width", out_width)) return e;
    if (int e = check_rows(what, rows, "in_width", in_width)) return e;
    if (rows == 0) return kOk;
    const unsigned size = size_of(out_type);
    const Pointer list[] = {{w, "w", 1, false},   {ws, "ws", 4, false}, {x, "x", 1, false},
                            {xs, "xs", 4, false}, {y, "y", size, false}, {resid, "resid", size, true}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    Fp8Matmul p;
    p.w = w;
    p.ws = ws;
    p.x = x;
    p.xs = xs;
    p.y = y;
    p.resid = resid;
    p.bf16 = out_type == MLK_BF16;
    p.O = out_width;
    p.I = in_width;
    p.rows = rows;
    p.x_rows = rows;
    return finish(fp8_matmul(p, st), what);
}

int mlk_matmul_fp8_grouped(int out_type, const uint8_t *w, const float *ws, const uint8_t *x,
                           const float *xs, int x_rows, void *y, int out_width, int in_width,
                           int groups, const int *offsets, const int *row_ids, int entries) {
    const char *what = "mlk_matmul_fp8_grouped";
    if (!type_ok(out_type)) return refuse(what, "out_type must be MLK_F32 or MLK_BF16");
    if (entries < 0 || x_rows < 0 || groups <= 0)
        return refuse(what, "entries and x_rows must be >= 0, groups > 0");
    if (int e = check_rows(what, entries, "out_width", out_width)) return e;
    if (int e = check_rows(what, entries, "in_width", in_width)) return e;
    if (!row_ids && x_rows < entries)
        return refuse(what, "without row_ids x needs a row for each entry");
    if (row_ids && !fp8_scales_in_reach(x_rows, in_width))
        return refuse(what, "with row_ids x_rows * ceil(in_width / 128) must be below 0x3C000000",
                      kErrSize);
    if (entries == 0) return kOk;
    if (x_rows == 0) return refuse(what, "x has no rows");
    const Pointer list[] = {{w, "w", 1, false},   {ws, "ws", 4, false},
                            {x, "x", 1, false},   {xs, "xs", 4, false},
                            {y, "y", size_of(out_type), false}, {offsets, "offsets", 4, false},
                            {row_ids, "row_ids", 4, true}};
    if (int e = check_pointers(what, list)) return e;
    hipStream_t st;
    if (int e = check_device(what, list, &st)) return e;
    Fp8Matmul p;
    p.w = w;
    p.ws = ws;
    p.x = x;
    p.xs = xs;
    p.y = y;
    p.bf16 = out_type == MLK_BF16;
    p.O = out_width;
    p.I = in_width;
    p.rows = entries;
    p.groups = groups;
    p.offsets = offsets;
    p.row_ids = row_ids;
    p.x_rows = x_rows;
    return finish(fp8_matmul(p, st), what);
}

}  // extern "C"
