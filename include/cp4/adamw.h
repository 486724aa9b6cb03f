/*
 * C ABI of the AdamW step over many tensors, for the factors, biases and adapters that the
 * library's gradients belong to.  No counterpart in the reference, whose training loop is its
 * framework's.
 *
 *   g  = c * grad
 *   m  = beta1 m + (1 - beta1) g           v = beta2 v + (1 - beta2) g^2
 *   p  = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 *
 * in fp32 whatever the types in memory, every operation rounded as the formula shows it (no fused
 * multiply-adds), so that a value's step has the same bits wherever it lies.  c is
 * grad_scale, with max_norm > 0 times min(1, max_norm / (norm + 1e-6)), norm the 2-norm of all
 * grad_scale * grad together.
 *
 * 8-bit moments: each 256 consecutive values of a tensor (the last ones of a tensor: what is
 * left) share one fp32 scale for m and one for v, their largest magnitude.  m's code is an int8
 * q for sign(q) q^2 scale / 127^2, v's a uint8 q for q^4 scale_sq / 255^4, both rounded to
 * nearest-even in q; a v above zero has a code of at least 1, so that a small second moment never
 * becomes none (it reads as 2^-149 or more, the least fp32 value).  The step itself uses m and v
 * before they are rounded.  A block in which a
 * moment is infinite or NaN has NaN scales (all of its moments read as NaN); one whose largest
 * magnitude is below the smallest normal number has the scale zero.
 */
#ifndef CP4_ADAMW_H
#define CP4_ADAMW_H

#include "cp4/capi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One tensor of a step; all pointers are device pointers to contiguous values. */
typedef struct cp4_adamw_tensor {
  void* param;        /* n values of param_dtype, updated */
  const void* grad;   /* n values of grad_dtype */
  void* exp_avg;      /* m: n floats, or n int8 codes (bits == 8); updated */
  void* exp_avg_sq;   /* v: n floats, or n uint8 codes; updated */
  float* scale;       /* bits == 8: ceil(n / 256) floats for m and ... */
  float* scale_sq;    /* ... for v; updated.  Otherwise ignored. */
  void* copy;         /* NULL, or n values of copy_dtype: the new parameters, rounded */
  size_t n;           /* 0: nothing is read or written */
  int param_dtype, grad_dtype, copy_dtype;   /* cp4_dtype */
  int bits;                                  /* 32 or 8 */
  unsigned group;                            /* whose rates: an index into `groups` */
} cp4_adamw_tensor;

/* Tensors that share their rates and their count of steps.  counter: four doubles on the device,
 * {t, beta1^t, beta2^t, 0} of the steps done so far (a new one: {0, 1, 1, 0}); the step reads and
 * advances it there, so that a captured graph counts its replays. */
typedef struct cp4_adamw_group {
  double lr, beta1, beta2, eps, weight_decay;
  double* counter;
} cp4_adamw_group;

/* One step.  Each group has a counter of its own; steps that share one must not overlap in time.
 * grad_scale: what all gradients are multiplied by (1: as they are).  With max_norm > 0 the norm of
 * all gradients of the call is written to *norm (device memory; may be NULL), and a step whose norm
 * is infinite or NaN changes nothing, the counters included.  Asynchronous on `stream`: one launch
 * for up to 75 (8-bit moments: 57) tensors of the same group and types; with max_norm, one more before them for up to 192
 * of the same gradient type.  `workspace`: cp4_adamw_workspace_bytes() of device memory, 16-byte
 * aligned; with max_norm == 0 it may be NULL.  Tensors must not overlap one another. */
size_t cp4_adamw_workspace_bytes(void);
cp4_status cp4_adamw_step(const cp4_adamw_tensor* tensors, size_t count,
                          const cp4_adamw_group* groups, size_t n_groups, float grad_scale,
                          float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                          cp4_stream stream);

/* What 8-bit moments stand for: values[i] and values_sq[i] receive tensors[i].n floats each
 * (device memory).  Reads exp_avg, exp_avg_sq, scale, scale_sq and n of each tensor. */
cp4_status cp4_adamw_moments(const cp4_adamw_tensor* tensors, size_t count, float* const* values,
                             float* const* values_sq, cp4_stream stream);
/* The other way: the codes and scales of tensors[i] from values[i] and values_sq[i]. */
cp4_status cp4_adamw_set_moments(const cp4_adamw_tensor* tensors, size_t count,
                                 const float* const* values, const float* const* values_sq,
                                 cp4_stream stream);

#ifdef __cplusplus
}
#endif
#endif
