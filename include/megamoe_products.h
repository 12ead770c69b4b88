/*
 * megamoe_products.h — C ABI of the experts' matrix products outside the fused layer (gfx950).
 *
 * The layer of megamoe.h runs routing, experts and combine in one call with E4M3 or MXFP4
 * experts. The products here are its building blocks in the other types that experts come in:
 * bf16 and fp16 with gradients (training, adapting), and int8 with one scale for each token and
 * each output channel. Both libraries are one, libmegamoe.so; the status codes are megamoe.h's.
 *
 * Rows are grouped by expert: `counts` (int64 [groups], on the device) holds how many rows each
 * group has, in order. Group e's rows start where group e-1's end; rows from the sum of the
 * counts on belong to no group. Groups may be empty. Counts that are negative, or whose sum
 * passes `rows`, make every element of the result NaN (they are read on the device; nothing is
 * read or written outside the tensors).
 *
 * Conventions: all pointers are device pointers unless stated otherwise. Every call is
 * asynchronous on `stream` (a hipStream_t passed as void*; NULL is the default stream),
 * allocates nothing, needs no workspace, keeps nothing between calls, records one kernel (so it
 * may be captured in a graph) and throws nothing. Results are deterministic: the same inputs
 * give the same bits. Inputs are only read; the result may not overlap them.
 */
#ifndef MEGAMOE_PRODUCTS_H
#define MEGAMOE_PRODUCTS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum megamoe_product_type {
  MEGAMOE_BF16 = 0,
  MEGAMOE_FP16 = 1,
  MEGAMOE_FP32 = 2 /* results of megamoe_int8_mm and inputs of megamoe_quantize_rows_int8 only */
};

/* Geometry of one product. Limits beyond which MEGAMOE_ERR_UNSUPPORTED is returned: groups
 * 1024, rows 2^30, row strides 4 MiB (ldx, and ldy as if its elements had four bytes), and 131071
 * for k of an int8 product (its int32 sums cannot overflow up to there). */
typedef struct megamoe_product {
  int64_t rows;       /* rows of x and y, >= 0 */
  int32_t groups;     /* E >= 1 */
  int32_t n;          /* output features, >= 0 */
  int32_t k;          /* input features, >= 0 */
  int32_t dtype;      /* enum megamoe_product_type: of x, w and y (y alone for int8) */
  int32_t transposed; /* 0: w is [E, n, k]; 1: w is [E, k, n] (not for int8) */
  int32_t fill_rest;  /* 1: rows of no group become zero in y; 0: they are left as they were */
  int64_t ldx;        /* row stride of x in elements, >= k */
  int64_t ldy;        /* row stride of y (of dy in megamoe_grouped_mm_wgrad) in elements, >= n */
} megamoe_product;

/* y[r] = w[e(r)] @ x[r] (transposed 0) or x[r] @ w[e(r)] (transposed 1) for every row r of a
 * group e(r): x [rows, k], w [E, n, k] or [E, k, n] dense, y [rows, n]; bf16 or fp16, products
 * summed in fp32 and rounded once. The gradient of x is the same product of dy with the other
 * value of `transposed`. Rows of 16-byte aligned operands whose strides are multiples of 8
 * elements run on the tiled kernels; other alignments on a slower kernel of the same results up
 * to the order of the sums. */
int megamoe_grouped_mm(const megamoe_product* p, const void* x, const void* w, const int64_t* counts, void* y,
                       void* stream);

/* The gradient of w: dw[e] = sum over the rows r of group e of dy[r]^T x[r], dw [E, n, k] dense
 * (zero for an empty group); dy [rows, n] with row stride ldy, x [rows, k]. Sums in fp32, one
 * rounding to `dtype`. For a transposed w exchange dy and x (and n and k, ldx and ldy).
 * `transposed` and `fill_rest` are ignored. */
int megamoe_grouped_mm_wgrad(const megamoe_product* p, const void* dy, const void* x, const int64_t* counts, void* dw,
                             void* stream);

/* y[r, j] = (float(sum_i x[r, i] * w[e(r), j, i]) * x_scale[r]) * w_scale[e(r), j]: x int8
 * [rows, k], x_scale fp32 [rows], w int8 [E, n, k], w_scale fp32 [E, n], y [rows, n] in bf16,
 * fp16 or fp32 (`dtype`). The sum is exact in int32. counts NULL: one group of all the rows
 * (groups must be 1). */
int megamoe_int8_mm(const megamoe_product* p, const int8_t* x, const float* x_scale, const int8_t* w,
                    const float* w_scale, const int64_t* counts, void* y, void* stream);

/* Rows to int8 with one scale each: a = max(max_i |x[r, i]|, 2^-100), scale[r] = a / 127,
 * q[r, i] = x[r, i] * (127 / a) rounded to nearest even, in fp32. A row that holds NaN or an
 * infinity gets the scale NaN and zeros, so its products are NaN. x [rows, cols] in bf16, fp16 or
 * fp32 with row stride ldx (elements), q int8 [rows, cols] dense, scale fp32 [rows]. */
int megamoe_quantize_rows_int8(int64_t rows, int32_t cols, int64_t ldx, int32_t dtype, const void* x, int8_t* q,
                               float* scale, void* stream);

/* Version of the functions of this header: 1. */
int megamoe_products_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MEGAMOE_PRODUCTS_H */
