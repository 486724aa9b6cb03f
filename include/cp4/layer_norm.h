/*
 * C ABI of the layer norm of rows, forward and backward, as it stands before the projections of
 * cp4/adapter.h.  No counterpart in the reference, whose layers are convolutions.
 *
 *   y[t] = (x[t] - m_t) r_t weight + bias,   m_t = mean(x[t]),  r_t = 1 / sqrt(mean((x[t] - m_t)^2) + eps)
 *
 *   dh = dy[t] weight,  h = (x[t] - m_t) r_t
 *   dx[t] = r_t (dh - mean(dh) - h mean(dh h))    dweight = sum_t dy[t] h    dbias = sum_t dy[t]
 *
 * x, y, dy and dx [T, D] of one cp4_dtype; weight, bias and their gradients [D] fp32, the statistics and all sums
 * fp32.  The mean is corrected by the mean of what it leaves, the variance is the sum of squares about it: a row far
 * from zero loses nothing that x itself has.  Squares are fp32: a row with values beyond some 1e19 from its
 * mean is bias in y (NaN where its sum is infinite) and 0 in dx.  Outputs are rounded once, to nearest-even.  No atomics: results do not
 * change from call to call.  What is not finite stays with its row of y and dx, and with its columns of the gradients
 * (a row with an infinity or a NaN is NaN in y and dx; weight's gradient is then NaN throughout).
 *
 * All pointers are device pointers.  Rows of x and dy may be further apart than they are long (ldx, lddy, in
 * elements; 0: contiguous); y and dx are contiguous.  Any alignment of the element type runs.  y may be a contiguous x
 * itself; otherwise outputs overlap nothing else.  Asynchronous on `stream`, kernel launches only.  D: up to 32768.
 */
#ifndef CP4_LAYER_NORM_H
#define CP4_LAYER_NORM_H

#include "cp4/capi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* weight NULL: all 1; bias NULL: none.  stats: NULL, or 2 T floats, m_t and r_t of each row, for the backward call. */
cp4_status cp4_layer_norm_forward(size_t T, unsigned D, int dtype, const void* x, size_t ldx, const float* weight,
                                  const float* bias, float eps, void* y, float* stats, cp4_stream stream);

/* dx, dweight and dbias: each may be NULL (not wanted).  T == 0: the gradients of weight and bias are zero.
 * workspace: cp4_layer_norm_backward_workspace_bytes() of device memory, 16-byte aligned, its contents scratch; may be
 * NULL where only dx is wanted. */
size_t cp4_layer_norm_backward_workspace_bytes(size_t T, unsigned D);
cp4_status cp4_layer_norm_backward(size_t T, unsigned D, int dtype, const void* dy, size_t lddy, const void* x,
                                   size_t ldx, const float* weight, const float* stats, void* dx, float* dweight,
                                   float* dbias, void* workspace, size_t workspace_bytes, cp4_stream stream);

#ifdef __cplusplus
}
#endif
#endif
