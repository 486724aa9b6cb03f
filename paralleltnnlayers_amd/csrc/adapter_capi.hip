// C ABI of the adapters beside a shared projection (include/cp4/adapter.h): checks, workspace, launches.
#include <algorithm>

#include "adapter.h"

namespace {

using cp4::fail_hip;
using cp4::fail_with;
using namespace cp4::adapter;

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
int padded(const cp4_adapter_shape& s) { return (int)((s.R + 15) / 16 * 16); }
size_t value_bytes(int dtype) { return dtype == CP4_DTYPE_F32 ? 4 : 2; }

cp4_status check_shape(const cp4_adapter_shape* s, int dtype) {
  if (!s) return fail_with(CP4_ERR_NULL_POINTER, "shape is NULL");
  if (dtype != CP4_DTYPE_F32 && dtype != CP4_DTYPE_BF16 && dtype != CP4_DTYPE_F16)
    return fail_with(CP4_ERR_SHAPE, "unknown dtype");
  if (!s->K || !s->N || !s->R || !s->G) return fail_with(CP4_ERR_SHAPE, "K, N, R and G must be 1 or more");
  if (s->R > 256) return fail_with(CP4_ERR_SHAPE, "adapters of a rank above 256");
  if (s->G > 65535) return fail_with(CP4_ERR_SHAPE, "more than 65535 adapters");
  if (s->K > 1u << 22 || s->N > 1u << 22) return fail_with(CP4_ERR_SHAPE, "K or N above 2^22");
  if (s->T > (size_t)1 << 26) return fail_with(CP4_ERR_SHAPE, "more than 2^26 tokens");
  if ((s->ldx && s->ldx < s->K) || (s->ldw && s->ldw < s->K) || (s->lddy && s->lddy < s->N))
    return fail_with(CP4_ERR_SHAPE, "a row stride is smaller than the row");
  if (std::max({s->ldx, s->ldw, s->lddy}) > (size_t)1 << 30)
    return fail_with(CP4_ERR_SHAPE, "a row stride above 2^30");
  return CP4_OK;
}
cp4_status check_pointers(size_t bytes, std::initializer_list<const void*> values,
                          std::initializer_list<const void*> floats) {
  for (const void* p : values)
    if ((size_t)p % bytes) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  for (const void* p : floats)
    if ((size_t)p & 3) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  return CP4_OK;
}

size_t h_bytes(const cp4_adapter_shape& s) { return s.T * padded(s) * 4; }

struct BackwardPlan {
  int splits, dh_planes;
  size_t part_at, part_b, total;                       // (dh comes first; B's partial sums: floats behind A's)
};
BackwardPlan backward_plan(const cp4_adapter_shape& s, int dtype) {
  BackwardPlan p{};
  p.splits = grad_splits(s.T, (int)s.K, (int)s.N, (int)s.R, (int)s.G);
  p.dh_planes = shrink_planes(s.T, (int)s.N, dtype);
  p.part_at = align256(p.dh_planes * h_bytes(s));
  p.part_b = p.splits > 1 ? (size_t)p.splits * s.G * s.R * s.K : 0;
  const size_t parts = p.splits > 1 ? (p.part_b + (size_t)p.splits * s.G * s.R * s.N) * 4 : 0;
  p.total = p.part_at + align256(std::max(parts, project_part_bytes(s.T, (int)s.N, (int)s.K, (int)s.G, dtype, true)));  // (one after the other)
  return p;
}

}  // namespace

extern "C" size_t cp4_adapter_kept_bytes(const cp4_adapter_shape* s, int dtype) {
  return check_shape(s, dtype) == CP4_OK ? h_bytes(*s) : 0;
}

extern "C" size_t cp4_adapter_forward_workspace_bytes(const cp4_adapter_shape* s, int dtype) {
  if (check_shape(s, dtype) != CP4_OK) return 0;
  return align256(shrink_planes(s->T, (int)s->K, dtype) * h_bytes(*s)) + align256(project_part_bytes(s->T, (int)s->K, (int)s->N, (int)s->G, dtype, false));
}

extern "C" cp4_status cp4_adapter_forward(const cp4_adapter_shape* s, int dtype, const void* x, const void* W,
                                          const void* A, const void* B, const int* ids, const float* scale,
                                          const float* bias, void* y, float* kept, void* workspace,
                                          size_t workspace_bytes, cp4_stream stream) {
  if (const cp4_status rc = check_shape(s, dtype)) return rc;
  if (!s->T) return CP4_OK;
  if (!x || !W || !A || !B || !ids || !y) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  if (const cp4_status rc = check_pointers(value_bytes(dtype), {x, W, A, B, y}, {ids, scale, bias})) return rc;
  const size_t need = cp4_adapter_forward_workspace_bytes(s, dtype);
  if (!workspace || workspace_bytes < need || ((size_t)workspace & 255))
    return fail_with(CP4_ERR_WORKSPACE, "workspace missing, too small or not aligned to 256 bytes");
  if ((size_t)kept & 15) return fail_with(CP4_ERR_WORKSPACE, "kept is not aligned to 16 bytes");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  float* const planes = static_cast<float*>(workspace);
  ShrinkArgs sh{};
  sh.z = x; sh.f = A; sh.ids = ids; sh.scale = scale;
  sh.T = s->T; sh.ldz = s->ldx ? s->ldx : s->K;
  sh.K = (int)s->K; sh.R = (int)s->R; sh.Rp = padded(*s); sh.G = (int)s->G;
  sh.fr = (int)s->K; sh.fk = 1; sh.planes = shrink_planes(s->T, (int)s->K, dtype);
  sh.h = sh.planes == 1 && kept ? kept : planes;
  if (const hipError_t e = shrink_launch(sh, dtype, st)) return fail_hip(e, "cp4_adapter_forward");
  ProjectArgs p{};
  p.z = x; p.w = W; p.f = B; p.h = sh.h; p.bias = bias; p.ids = ids; p.y = y;
  p.T = s->T; p.ldz = sh.ldz; p.ldw = s->ldw ? s->ldw : s->K;
  p.K = (int)s->K; p.N = (int)s->N; p.R = (int)s->R; p.Rp = sh.Rp; p.G = (int)s->G;
  p.fn = (int)s->R; p.fr = 1; p.planes = sh.planes; p.plane = p.T * p.Rp;
  if (p.planes > 1 && project_sums_planes(p, dtype, false)) {
    p.keep = kept;
  } else if (p.planes > 1) {
    float* const h = kept ? kept : planes;
    if (const hipError_t e = planes_join(h, planes, p.plane, p.planes, st)) return fail_hip(e, "cp4_adapter_forward");
    p.h = h;
    p.planes = 1;
  }
  float* const part = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(sh.planes * h_bytes(*s)));
  if (const hipError_t e = project_launch(p, part, dtype, false, st)) return fail_hip(e, "cp4_adapter_forward");
  return CP4_OK;
}

extern "C" size_t cp4_adapter_backward_workspace_bytes(const cp4_adapter_shape* s, int dtype) {
  if (check_shape(s, dtype) != CP4_OK) return 0;
  return backward_plan(*s, dtype).total;
}

extern "C" cp4_status cp4_adapter_backward(const cp4_adapter_shape* s, int dtype, const void* dy, const void* x,
                                           const void* W, const void* A, const void* B, const int* ids,
                                           const float* scale, const float* kept, void* dx, void* dA, void* dB,
                                           void* workspace, size_t workspace_bytes, cp4_stream stream) {
  if (const cp4_status rc = check_shape(s, dtype)) return rc;
  if (!dA != !dB) return fail_with(CP4_ERR_NULL_POINTER, "dA without dB");
  if (s->T) {
    if (!dy || !W || !A || !B || !ids || (dA && (!x || !kept)))
      return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
    if (const cp4_status rc = check_pointers(value_bytes(dtype), {dy, x, W, A, B, dx, dA, dB}, {ids, scale})) return rc;
    if ((size_t)kept & 15) return fail_with(CP4_ERR_WORKSPACE, "kept is not aligned to 16 bytes");
  }
  const BackwardPlan plan = backward_plan(*s, dtype);
  if (plan.total && (!workspace || workspace_bytes < plan.total || ((size_t)workspace & 255)))
    return fail_with(CP4_ERR_WORKSPACE, "workspace missing, too small or not aligned to 256 bytes");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  float* const dh = static_cast<float*>(workspace);
  float* const part = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.part_at);
  const int Rp = padded(*s);
  const size_t lddy = s->lddy ? s->lddy : s->N, ldx = s->ldx ? s->ldx : s->K;
  if (s->T && (dx || dA)) {
    ShrinkArgs sh{};
    sh.z = dy; sh.f = B; sh.ids = ids; sh.scale = scale; sh.h = dh;
    sh.T = s->T; sh.ldz = lddy;
    sh.K = (int)s->N; sh.R = (int)s->R; sh.Rp = Rp; sh.G = (int)s->G;
    sh.fr = 1; sh.fk = (int)s->R; sh.planes = plan.dh_planes;
    if (const hipError_t e = shrink_launch(sh, dtype, st)) return fail_hip(e, "cp4_adapter_backward");
    if (sh.planes > 1)
      if (const hipError_t e = planes_join(dh, dh, s->T * Rp, sh.planes, st)) return fail_hip(e, "cp4_adapter_backward");
  }
  if (s->T && dx) {
    ProjectArgs p{};
    p.z = dy; p.w = W; p.f = A; p.h = dh; p.ids = ids; p.y = dx;
    p.T = s->T; p.ldz = lddy; p.ldw = s->ldw ? s->ldw : s->K;
    p.K = (int)s->N; p.N = (int)s->K; p.R = (int)s->R; p.Rp = Rp; p.G = (int)s->G;
    p.fn = 1; p.fr = (int)s->K; p.planes = 1;
    if (const hipError_t e = project_launch(p, part, dtype, true, st)) return fail_hip(e, "cp4_adapter_backward");
  }
  if (dA) {
    GradArgs ga{};
    ga.ids = ids; ga.T = s->T; ga.R = (int)s->R; ga.Rp = Rp; ga.G = (int)s->G; ga.splits = plan.splits;
    GradArgs gb = ga;
    ga.p = dh; ga.z = x; ga.out = dA; ga.part = part; ga.ldz = ldx; ga.C = (int)s->K; ga.outr = (int)s->K; ga.outc = 1;
    gb.p = kept; gb.z = dy; gb.out = dB; gb.part = part + plan.part_b; gb.ldz = lddy; gb.C = (int)s->N; gb.outr = 1; gb.outc = (int)s->R;
    if (const hipError_t e = grad_launch(ga, gb, dtype, st)) return fail_hip(e, "cp4_adapter_backward");
  }
  return CP4_OK;
}

extern "C" cp4_status cp4_adapter_plan_query(const cp4_adapter_shape* s, int dtype, int backward, int aligned,
                                             cp4_adapter_launch launches[2]) {
  if (const cp4_status rc = check_shape(s, dtype)) return rc;
  if (!launches) return fail_with(CP4_ERR_NULL_POINTER, "launches is NULL");
  cp4_adapter_launch l[2];
  const int K = (int)(backward ? s->N : s->K), N = (int)(backward ? s->K : s->N);
  project_plan(s->T, K, N, (int)s->G, dtype, backward != 0, aligned != 0, l);
  launches[0] = l[0];
  launches[1] = l[1];
  return CP4_OK;
}
