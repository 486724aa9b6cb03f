/*
 * C ABI of a dense projection with the low-rank adapters of many requests beside it, for prompts,
 * single tokens and training.  No counterpart in the reference, whose layers are convolutions.
 *
 *   y[t] = W x[t] + bias + s_a B_a (A_a x[t]),   a = ids[t]
 *
 * x [T, K], W [N, K], A [G, R, K], B [G, N, R] and y [T, N] of one cp4_dtype; scale [G] and bias
 * [N] fp32.  ids[t] says whose adapter token t goes through, in any order; an id outside 0 .. G - 1
 * is a token without one.  W and bias are not trained.  Gradients of dy [T, N], with
 * dh[t] = s_a B_a^T dy[t] and h[t] = s_a A_a x[t]:
 *
 *   dx[t] = W^T dy[t] + A_a^T dh[t]    dA_a = sum_{ids[t] = a} dh[t] x[t]^T
 *                                      dB_a = sum_{ids[t] = a} dy[t] h[t]^T
 *
 * All sums are fp32; h and dh stay fp32 in memory and enter the second product as two bfloat16 parts
 * (16 bits) where the layer's type has 16 bits.  Outputs are rounded once, to nearest-even.  No
 * atomics: results do not change from call to call.  An adapter that no token uses has zero
 * gradients.  What is not finite stays with its own: a token's x and dy with that token's rows of y and dx and with its
 * adapter's gradients, an adapter with its own tokens and gradients.  (An infinity may come out as NaN: in an fp32
 * operand anywhere, in a 16-bit one wherever it meets an adapter.  fp32 operands, h, dh and float16 ranks are taken
 * apart into bfloat16 parts, of which an infinity's are an infinity and NaN, and places that fill up a block of
 * products are multiplied by zero.)
 *
 * All pointers are device pointers.  Rows of x, W and dy may be further apart than they are long
 * (ldx, ldw, lddy, in elements); A, B, y, dx, dA and dB are contiguous.  Any alignment of the
 * element type runs; rows that start on 16-byte boundaries (K and N multiples of 8 in 16 bits, of 4
 * in fp32) run faster.  Asynchronous on `stream`, kernel launches only.
 */
#ifndef CP4_ADAPTER_H
#define CP4_ADAPTER_H

#include "cp4/capi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct cp4_adapter_shape {
  size_t T;               /* tokens, up to 2^26; 0: gradients of A and B are zero, nothing else is written */
  unsigned K, N;          /* inputs, outputs, up to 2^22 each */
  unsigned R, G;          /* rank of the adapters (up to 256), how many there are (up to 65535) */
  size_t ldx, ldw, lddy;  /* row strides of x, W and dy; 0: contiguous */
} cp4_adapter_shape;

/* What a forward call leaves for the backward call: h, cp4_adapter_kept_bytes() of device memory. */
size_t cp4_adapter_kept_bytes(const cp4_adapter_shape* shape, int dtype);

/* `kept` may be NULL (inference).  scale NULL: all 1; bias may be NULL.  workspace: device memory of
 * cp4_adapter_forward_workspace_bytes(), 256-byte aligned, its contents scratch. */
size_t cp4_adapter_forward_workspace_bytes(const cp4_adapter_shape* shape, int dtype);
cp4_status cp4_adapter_forward(const cp4_adapter_shape* shape, int dtype, const void* x,
                               const void* W, const void* A, const void* B, const int* ids,
                               const float* scale, const float* bias, void* y, float* kept,
                               void* workspace, size_t workspace_bytes, cp4_stream stream);

/* dx, or dA and dB together, may be NULL (not wanted). */
size_t cp4_adapter_backward_workspace_bytes(const cp4_adapter_shape* shape, int dtype);
cp4_status cp4_adapter_backward(const cp4_adapter_shape* shape, int dtype, const void* dy,
                                const void* x, const void* W, const void* A, const void* B,
                                const int* ids, const float* scale, const float* kept, void* dx,
                                void* dA, void* dB, void* workspace, size_t workspace_bytes,
                                cp4_stream stream);

/* How the shared projection of a call (backward != 0: that of dx) would run now, for reports and tests: its
 * launches, the second one for the rows that whole tiles leave over, where those are cheaper on their
 * own.  aligned: whether its operands' rows start on 16-byte boundaries. */
typedef struct cp4_adapter_launch {
  size_t rows;                /* tokens; 0: there is no such launch */
  int tile_rows, tile_cols;   /* 0 and 0: the kernel of few rows, without tiles */
  int splits;                 /* parts of the depth */
} cp4_adapter_launch;
cp4_status cp4_adapter_plan_query(const cp4_adapter_shape* shape, int dtype, int backward,
                                  int aligned, cp4_adapter_launch launches[2]);

#ifdef __cplusplus
}
#endif
#endif
