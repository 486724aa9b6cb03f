/*
 * C ABI of the Muon step over many matrices: each is moved along its momentum, orthogonalised by
 * Newton-Schulz products.  For the CP factors, adapters and dense layers that the library's gradients belong
 * to, beside the AdamW step of cp4/adamw.h.  No counterpart in the reference.
 *
 *   m = momentum m + grad           u = grad + momentum m  (nesterov), or m
 *   X = u / (|u| + eps)             |u| the root of the sum of squares
 *   X = a X + (b A + c A A) X,      A = X X^T  (X transposed where it has more rows than columns), `steps` times,
 *                                   a, b, c = 3.4445, -4.7750, 2.0315
 *   p = p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) X
 *
 * The polynomial takes every singular value from 0.01 or so up into 0.68 .. 1.21 in five steps and keeps it there.
 * m, p's step and all sums are fp32 or wider whatever the types in memory.  Matrices with a side of up to 64 go through
 * their Gram matrix, summed and iterated in fp64 (and past 5 steps applied in it, so that directions a matrix does not
 * have stay nothing however often they are multiplied by 3.4445); larger ones through products of values in two float16 parts
 * (22 bits, of fp32's 24; accumulated in fp32), whose range moves with the norm where that is far below eps.  What they are
 * off 64 bits by in five steps, in norm, is 2e-6 of noise (an iteration in fp32: 3e-6) and of few directions, whose
 * roundings are multiplied by 3.4445 a step, 1.2e-4 of one (1.7e-4), 4.4e-5 of 8 (3.6e-5), 2.4e-5 of 64 (1.5e-5; 512 x 768).  No atomics: results do not change from call to call.  A matrix whose u has
 * an infinity or a NaN becomes NaN in whole; others are not touched by it.
 */
#ifndef CP4_MUON_H
#define CP4_MUON_H

#include "cp4/capi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* `count` matrices of the same shape, one behind the other; all pointers are device pointers to
 * contiguous, row-major values, aligned to their type. */
typedef struct cp4_muon_matrix {
  void* param;          /* of param_dtype, updated; NULL: no step is taken */
  const void* grad;     /* of grad_dtype */
  float* momentum;      /* updated; NULL: u is grad */
  void* copy;           /* NULL, or of copy_dtype: the new parameters, rounded; without param X itself; with neither the
                           momentum alone is updated */
  size_t count;
  unsigned rows, cols;  /* up to 65536 each; nothing is read or written where one of the three is 0 */
  int param_dtype, grad_dtype, copy_dtype;   /* cp4_dtype */
} cp4_muon_matrix;

/* One step.  Asynchronous on `stream`, kernel launches only: three for up to 72 entries whose shorter sides round up to
 * the same multiple of 16 up to 64, and 3 steps + 2 (long ones: 4 steps + 2) for up to 16 larger ones whose scratch memory
 * stays below 1 GiB together (a larger matrix on its own).  steps: 1 to 16.  eps: 1e-30 or more.  workspace:
 * cp4_muon_workspace_bytes() of device memory, 256-byte aligned, its contents scratch.  What is written must not overlap
 * anything else, but that `copy` without a param may be grad itself, of its type. */
size_t cp4_muon_workspace_bytes(const cp4_muon_matrix* matrices, size_t count);
cp4_status cp4_muon_step(const cp4_muon_matrix* matrices, size_t count, double lr, double momentum,
                         int nesterov, double weight_decay, double eps, unsigned steps,
                         void* workspace, size_t workspace_bytes, cp4_stream stream);

#ifdef __cplusplus
}
#endif
#endif
