/*
 * C ABI of microscaled 4-bit floating point: rows to it and back, and dense projections whose weights are held in
 * it - plain ones, with activations rounded to it as well, and those of cp4/adapter.h with low-rank adapters.
 * No counterpart in the reference.
 *
 * A row of K values is ceil(K / 32) blocks.  A block's values share the scale 2^(s - 127), s a byte of `scales`
 * [rows][blocks]; a value is a code of 4 bits, the even one of two in the low half of a byte of `codes`
 * [rows][blocks][16]: a sign (8) and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1).  s is 255 for a block that is NaN.  Codes
 * behind a row's last value are zero.
 *
 * Rounding to it: s - 127 = floor(log2(largest magnitude)) - 2, from -127 on, a value to the nearest code, ties to the
 * even one, magnitudes beyond 6 to 6.  A block with an infinity or a NaN is NaN in whole.
 *
 * A projection reads W [N][K] as its values in the type of x, which they fit exactly in fp32 and bfloat16 (but that
 * a code times 2^126 or more may be infinite); in float16 values below 2^-14 are rounded to its steps and those of
 * 65536 and more are infinite.  Sums are fp32, outputs are rounded once.
 *
 * All pointers are device pointers, codes on 16-byte boundaries; outputs overlap nothing else.  Asynchronous on `stream`,
 * kernel launches only.  K and N: up to 2^22, T: up to 2^26.
 */
#ifndef CP4_MX4_H
#define CP4_MX4_H

#include "cp4/adapter.h"
#include "cp4/capi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cp4_mx4 {
  const void* codes;              /* [rows][ceil(K / 32)][16] */
  const unsigned char* scales;    /* [rows][ceil(K / 32)] */
} cp4_mx4;

/* x [T][K] of a cp4_dtype, rows ldx apart (0: contiguous). */
cp4_status cp4_mx4_quantize(size_t T, unsigned K, int dtype, const void* x, size_t ldx, void* codes,
                            unsigned char* scales, cp4_stream stream);
/* y [T][K], contiguous: the values, rounded to y's type. */
cp4_status cp4_mx4_dequantize(size_t T, unsigned K, int dtype, const cp4_mx4* q, void* y, cp4_stream stream);

/* y [T][N] = x W^T + bias.  x [T][K] of dtype, rows ldx apart; bias [N] fp32 or NULL.  workspace: device memory of
 * ..._workspace_bytes(), 256-byte aligned, its contents scratch. */
size_t cp4_mx4_forward_workspace_bytes(size_t T, unsigned K, unsigned N, int dtype);
cp4_status cp4_mx4_forward(size_t T, unsigned K, unsigned N, int dtype, const void* x, size_t ldx, const cp4_mx4* W,
                           const float* bias, void* y, void* workspace, size_t workspace_bytes, cp4_stream stream);
/* dx [T][K] = dy W, dy [T][N] rows lddy apart. */
size_t cp4_mx4_backward_workspace_bytes(size_t T, unsigned K, unsigned N, int dtype);
cp4_status cp4_mx4_backward(size_t T, unsigned K, unsigned N, int dtype, const void* dy, size_t lddy, const cp4_mx4* W,
                            void* dx, void* workspace, size_t workspace_bytes, cp4_stream stream);

/* How the projection of a call with W in 4 bits (backward != 0: that of dx) would run now, for reports and tests, as
 * cp4_adapter_plan_query has it.  G: adapters beside it, 0: none.  aligned: whether rows of x (dy) start on 16-byte
 * boundaries.  room: the bytes of its workspace for the partial sums of a split depth, and for W's values where aligned
 * calls read those instead of its codes (0: they do not). */
cp4_status cp4_mx4_plan_query(size_t T, unsigned K, unsigned N, unsigned G, int dtype, int backward, int aligned,
                              cp4_adapter_launch launches[2], size_t room[2]);

/* y [T][N] = X W^T + bias, both operands in 4 bits, on the scaled matrix instructions; y of dtype.  (cp4_mx4_quantize
 * makes X of activations.) */
size_t cp4_mx4_product_workspace_bytes(size_t T, unsigned K, unsigned N);
cp4_status cp4_mx4_product(size_t T, unsigned K, unsigned N, int dtype, const cp4_mx4* X, const cp4_mx4* W,
                           const float* bias, void* y, void* workspace, size_t workspace_bytes, cp4_stream stream);

/* cp4_adapter_forward and cp4_adapter_backward with W in 4 bits (shape->ldw is not used). */
size_t cp4_adapter_mx4_forward_workspace_bytes(const cp4_adapter_shape* shape, int dtype);
cp4_status cp4_adapter_mx4_forward(const cp4_adapter_shape* shape, int dtype, const void* x,
                                   const cp4_mx4* W, const void* A, const void* B, const int* ids,
                                   const float* scale, const float* bias, void* y, float* kept,
                                   void* workspace, size_t workspace_bytes, cp4_stream stream);
size_t cp4_adapter_mx4_backward_workspace_bytes(const cp4_adapter_shape* shape, int dtype);
cp4_status cp4_adapter_mx4_backward(const cp4_adapter_shape* shape, int dtype, const void* dy,
                                    const void* x, const cp4_mx4* W, const void* A, const void* B,
                                    const int* ids, const float* scale, const float* kept, void* dx,
                                    void* dA, void* dB, void* workspace, size_t workspace_bytes,
                                    cp4_stream stream);

#ifdef __cplusplus
}
#endif
#endif
