// PyTorch binding of the C ABI (module paralleltnnlayers_amd._binding): the three passes and
// the differentiable layer as native calls.
//
// A small layer's pass takes 4 - 8 us on the device; through ctypes and a Python
// autograd.Function one call cost 11 us (a pass), 20 us (a layer's inference) and some 150 us
// of a training step (forward and backward, each with its own tensors, workspace query and
// argument conversions).  Here the arguments are parsed in place, outputs come straight from
// the caching allocator and the layer is a C++ autograd function, whose backward runs without
// the interpreter.
//
// The semantics are the Python functions' of capi.py / torch_ops.py that call this module.
// Stands where the reference registers its op with a framework (Kernels/cp4_conv_nchw.cc:6-108).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <algorithm>
#include <optional>
#include <string>
#include <vector>

#include "cp4/adamw.h"
#include "cp4/adapter.h"
#include "cp4/capi.h"
#include "cp4/layer_norm.h"
#include "cp4/muon.h"
#include "cp4/mx4.h"

namespace {

using at::Tensor;

PyObject* g_error = nullptr;                    // capi.Cp4Error(status, message)
std::atomic<bool> g_check_backward{false};      // torch_ops.set_device_checks

// ---- errors ---------------------------------------------------------------------

void set_status_error(cp4_status rc) {
  const std::string text =
      std::string(cp4_status_string(rc)) + ": " + cp4_last_error_message();
  PyObject* args = Py_BuildValue("(is)", (int)rc, text.c_str());
  PyObject* err = args && g_error ? PyObject_CallObject(g_error, args) : nullptr;
  Py_XDECREF(args);
  if (err) {
    PyErr_SetObject(g_error, err);
    Py_DECREF(err);
  } else if (!PyErr_Occurred()) {
    PyErr_SetString(PyExc_RuntimeError, text.c_str());
  }
}
// From any thread, with or without the interpreter lock (the autograd engine's threads run
// without it): the Python exception travels through the engine as it is.
void check(cp4_status rc) {
  if (rc == CP4_OK) return;
  PyGILState_STATE gil = PyGILState_Ensure();
  set_status_error(rc);
  python_error e;
  e.persist();
  PyGILState_Release(gil);
  throw e;
}
[[noreturn]] void fail(PyObject* type, const char* what) {
  PyGILState_STATE gil = PyGILState_Ensure();
  PyErr_SetString(type, what);
  python_error e;
  e.persist();
  PyGILState_Release(gil);
  throw e;
}
void require(bool ok, const char* what = "") {
  if (!ok) fail(PyExc_AssertionError, what);
}

// The interpreter lock is given up around allocations and launches, as a ctypes call does: a
// launch that waits for room in a full queue must not keep other Python threads from running.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// ---- arguments --------------------------------------------------------------------

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) fail(PyExc_AssertionError, "expected a tensor");
  return THPVariable_Unpack(o);
}
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
float* f32(const Tensor& t) {
  require(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous(),
          "expected a contiguous float32 device tensor");
  return static_cast<float*>(t.data_ptr());
}
void* stream_of(PyObject* o) {
  if (o && o != Py_None) {
    PyObject* h = PyObject_GetAttrString(o, "cuda_stream");
    if (!h) throw python_error();
    void* s = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    return s;
  }
  return c10::hip::getCurrentHIPStream().stream();
}
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
// Device memory of `bytes` (the allocator's blocks lie on 512-byte boundaries); undefined for 0.
Tensor scratch(size_t bytes, const Tensor& like) {
  return bytes ? empty({(int64_t)bytes}, at::kByte, like) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Factors {
  const Tensor &FK, &FC, &FH, &FW;
};
// tensor_shape as CP::Conv2dForward / Conv2dBackwardData derive it (Cuda_kernels/cp4Conv2d.cu:21-30)
cp4_shape shape_for(const Tensor& act, const Factors& f, long pad) {
  require(act.dim() == 4 && f.FK.dim() >= 2 && f.FC.dim() >= 1 && f.FH.dim() >= 1 && f.FW.dim() >= 1,
          "expected an activation [N, C, H, W] and factors [rows, rank]");
  cp4_shape s;
  s.N = (unsigned)act.size(0); s.H = (unsigned)act.size(2); s.W = (unsigned)act.size(3);
  s.pad = (unsigned)pad;
  s.T = (unsigned)f.FK.size(0); s.C = (unsigned)f.FC.size(0); s.Y = (unsigned)f.FH.size(0);
  s.X = (unsigned)f.FW.size(0); s.Rank = (unsigned)f.FK.size(1);
  // (rows and rank count, not the form: at rank 1 a vector holds a factor as well)
  for (const Tensor* t : {&f.FK, &f.FC, &f.FH, &f.FW})
    require(t->numel() >= t->size(0) * (int64_t)s.Rank, "a factor holds fewer than rows * rank entries");
  return s;
}

// ---- the three passes (capi.conv2d_forward, _backward_data, _backward_filter) --------
// (Outputs and scratch come from the current stream's memory: a caller that names another
// stream makes it current around the call, as capi.py does.)

// (x, FK, FC, FH, FW, pad, out, variant, stream) -> y
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 9);
  const Tensor& x = tensor(a[0]);
  const Factors f{tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4])};
  const cp4_shape s = shape_for(x, f, integer(a[5]));
  require(x.size(1) == s.C && f.FC.dim() >= 2 && f.FC.size(1) == s.Rank,
          "x or FC does not match the factors");
  const int variant = (int)integer(a[7]);
  void* st = stream_of(a[8]);
  Tensor y = a[6] != Py_None ? tensor(a[6]) : Tensor();
  {
    NoGil unlocked;
    const float *px = f32(x), *pK = f32(f.FK), *pC = f32(f.FC), *pH = f32(f.FH), *pW = f32(f.FW);
    if (!y.defined()) y = empty({s.N, s.T, s.H, s.W}, at::kFloat, x);
    require(y.numel() >= (int64_t)s.N * s.T * s.H * s.W, "out is smaller than the result");
    check(cp4_conv2d_forward_variant(&s, px, pK, pC, pH, pW, f32(y), variant, st));
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (dy, FK, FC, FH, FW, pad, out, stream) -> dx
PyObject* backward_data(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 8);
  const Tensor& dy = tensor(a[0]);
  const Factors f{tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4])};
  const cp4_shape s = shape_for(dy, f, integer(a[5]));
  require(dy.size(1) == s.T);
  void* st = stream_of(a[7]);
  Tensor dx = a[6] != Py_None ? tensor(a[6]) : Tensor();
  {
    NoGil unlocked;
    const float *pdy = f32(dy), *pK = f32(f.FK), *pC = f32(f.FC), *pH = f32(f.FH), *pW = f32(f.FW);
    if (!dx.defined()) dx = empty({s.N, s.C, s.H, s.W}, at::kFloat, dy);
    require(dx.numel() >= (int64_t)s.N * s.C * s.H * s.W, "out is smaller than the result");
    check(cp4_conv2d_backward_data(&s, pdy, pK, pC, pH, pW, f32(dx), st));
  }
  return THPVariable_Wrap(std::move(dx));
  END_HANDLE_TH_ERRORS
}

PyObject* wrap_four(Tensor (&t)[4]) {
  PyObject* out = PyTuple_New(4);
  if (!out) throw python_error();
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(t[i])));
  return out;
}

// (x, dy, FK, FC, FH, FW, pad, workspace, stream, variant) -> (dFK, dFC, dFH, dFW)
PyObject* backward_filter(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 10);
  const Tensor &x = tensor(a[0]), &dy = tensor(a[1]);
  const Factors f{tensor(a[2]), tensor(a[3]), tensor(a[4]), tensor(a[5])};
  const cp4_shape s = shape_for(x, f, integer(a[6]));
  require(dy.dim() == 4 && dy.size(0) == s.N && dy.size(1) == s.T && dy.size(2) == s.H &&
          dy.size(3) == s.W && x.size(1) == s.C);
  const int variant = (int)integer(a[9]);
  void* st = stream_of(a[8]);
  Tensor ws = a[7] != Py_None ? tensor(a[7]) : Tensor();
  Tensor grads[4];
  {
    NoGil unlocked;
    const float *px = f32(x), *pdy = f32(dy), *pK = f32(f.FK), *pC = f32(f.FC), *pH = f32(f.FH),
                *pW = f32(f.FW);
    const Tensor* fac[4] = {&f.FK, &f.FC, &f.FH, &f.FW};
    for (int i = 0; i < 4; ++i) grads[i] = empty(fac[i]->sizes(), at::kFloat, x);
    if (ws.defined()) {
      require(ws.is_cuda() && ws.is_contiguous(), "the workspace must be a contiguous device tensor");
    } else {
      const size_t need = cp4_conv2d_backward_filter_workspace_bytes(&s);
      ws = scratch(need ? need : 4, x);
    }
    check(cp4_conv2d_backward_filter_variant(&s, px, pdy, pK, pC, pH, pW, f32(grads[0]),
                                             f32(grads[1]), f32(grads[2]), f32(grads[3]),
                                             ws.data_ptr(), (size_t)ws.numel() * ws.element_size(),
                                             variant, st));
  }
  return wrap_four(grads);
  END_HANDLE_TH_ERRORS
}

// ---- the differentiable layer (torch_ops.cp4_conv2d) -----------------------------------

struct LayerSpec {
  cp4_shape shape;
  cp4_geometry geometry;
  bool has_geometry, has_bias;
  int dtype, activation;
  int kept_parts;                               // what the forward pass left in the last saved tensor
  const cp4_geometry* g() const { return has_geometry ? &geometry : nullptr; }
};

Tensor as_f32(const Tensor& t) {
  if (t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
  return t.contiguous().to(at::kFloat);
}

// wanted: CP4_WANT_* of the backward pass that will follow (0: none); kept and parts: what the forward
// pass leaves for it, the memory of which outlives the call as the saved tensors do.
Tensor layer_forward(const LayerSpec& l, const Tensor& x, const Factors& f, const Tensor& bias,
                     int wanted = 0, Tensor* kept = nullptr, int* parts = nullptr) {
  const cp4_shape& s = l.shape;
  const int64_t oh = l.has_geometry ? l.geometry.out_h : s.H, ow = l.has_geometry ? l.geometry.out_w : s.W;
  Tensor y = empty({s.N, s.T, oh, ow}, x.scalar_type(), x);
  const size_t need = l.dtype == CP4_DTYPE_F32
                          ? 0 : cp4_layer_forward_workspace_bytes(&s, l.g(), l.dtype);
  const Tensor ws = scratch(need, x);
  if (const size_t room = wanted ? cp4_layer_kept_bytes(&s, l.g(), l.dtype, l.activation, wanted) : 0) {
    *kept = scratch(room, x);
    check(cp4_layer_forward_keeping(&s, l.g(), l.dtype, x.data_ptr(), f32(f.FK), f32(f.FC), f32(f.FH),
                                    f32(f.FW), bias.defined() ? f32(bias) : nullptr, l.activation,
                                    wanted, y.data_ptr(), kept->data_ptr(), room, parts, ptr(ws), need,
                                    c10::hip::getCurrentHIPStream(x.device().index()).stream()));
    if (!*parts) *kept = Tensor();
    return y;
  }
  check(cp4_layer_forward(&s, l.g(), l.dtype, x.data_ptr(), f32(f.FK), f32(f.FC), f32(f.FH),
                          f32(f.FW), bias.defined() ? f32(bias) : nullptr, l.activation,
                          y.data_ptr(), ptr(ws), need,
                          c10::hip::getCurrentHIPStream(x.device().index()).stream()));
  return y;
}

struct LayerFunction : torch::autograd::Function<LayerFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& FK,
                        const Tensor& FC, const Tensor& FH, const Tensor& FW,
                        const std::optional<Tensor>& bias, LayerSpec l) {
    const Factors f{as_f32(FK), as_f32(FC), as_f32(FH), as_f32(FW)};
    const Tensor b = bias ? as_f32(*bias) : Tensor();
    const bool factors = FK.requires_grad() || FC.requires_grad() || FH.requires_grad() || FW.requires_grad();
    const int wanted = (x.requires_grad() ? CP4_WANT_DX : 0) | (factors ? CP4_WANT_FACTORS : 0) |
                       (bias && bias->requires_grad() ? CP4_WANT_BIAS : 0);
    Tensor kept;
    Tensor y = layer_forward(l, x, f, b, factors ? wanted : 0, &kept, &l.kept_parts);
    const bool relu = l.activation == CP4_ACT_RELU;
    torch::autograd::variable_list saved{x, f.FK, f.FC, f.FH, f.FW, relu ? y : Tensor()};
    if (kept.defined()) saved.push_back(kept);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["spec"] = c10::IValue(std::string(reinterpret_cast<const char*>(&l), sizeof l));
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &FK = saved[1], &FC = saved[2], &FH = saved[3], &FW = saved[4];
    LayerSpec l;
    {
      const std::string& raw = ctx->saved_data["spec"].toStringRef();
      memcpy(&l, raw.data(), sizeof l);
    }
    torch::autograd::variable_list out(7);
    if (!grad[0].defined()) return out;
    Tensor dy = grad[0].contiguous();
    if (dy.scalar_type() != x.scalar_type()) dy = dy.to(x.scalar_type());
    const bool want_dx = ctx->needs_input_grad(0), want_bias = l.has_bias && ctx->needs_input_grad(5);
    bool want_factor[4], want_factors = false;
    for (int i = 0; i < 4; ++i) want_factors |= want_factor[i] = ctx->needs_input_grad(1 + i);
    const Tensor* fac[4] = {&FK, &FC, &FH, &FW};
    Tensor dx, grads[4], dbias;
    // create_graph: the bias gradient is linear in dy and stays differentiable (the other
    // gradients are the library's and are not)
    const bool bias_graph = want_bias && at::GradMode::is_enabled() && grad[0].requires_grad();
    if (want_dx) dx = empty(x.sizes(), x.scalar_type(), x);
    if (want_factors)
      for (int i = 0; i < 4; ++i) grads[i] = empty(fac[i]->sizes(), at::kFloat, x);
    if (want_bias && !bias_graph) dbias = empty({(int64_t)l.shape.T}, at::kFloat, x);
    const int wanted = (want_dx ? CP4_WANT_DX : 0) | (want_factors ? CP4_WANT_FACTORS : 0) |
                       (dbias.defined() ? CP4_WANT_BIAS : 0);
    const size_t need =
        cp4_layer_backward_workspace_bytes(&l.shape, l.g(), l.dtype, l.activation, wanted);
    const Tensor ws = scratch(need, x);
    void* st = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    // (what hooks on saved tensors give back in another form than bytes on this device is left alone)
    const Tensor kept = saved.size() > 6 && saved[6].defined() && saved[6].device() == x.device() &&
                                saved[6].scalar_type() == at::kByte && saved[6].is_contiguous()
                            ? saved[6] : Tensor();
    check(cp4_layer_backward_kept(&l.shape, l.g(), l.dtype, x.data_ptr(), ptr(saved[5]), dy.data_ptr(),
                             f32(FK), f32(FC), f32(FH), f32(FW), l.activation, ptr(dx),
                             static_cast<float*>(ptr(grads[0])), static_cast<float*>(ptr(grads[1])),
                             static_cast<float*>(ptr(grads[2])), static_cast<float*>(ptr(grads[3])),
                             static_cast<float*>(ptr(dbias)), ptr(kept),
                             kept.defined() ? (size_t)kept.numel() : 0, l.kept_parts, ptr(ws), need, st));
    if (g_check_backward.load(std::memory_order_relaxed)) check(cp4_device_status(st, nullptr));
    if (bias_graph) {
      const Tensor d = saved[5].defined() ? grad[0] * (saved[5] > 0) : grad[0];
      dbias = d.to(at::kFloat).sum(at::IntArrayRef{0, 2, 3});
    }
    out[0] = dx;
    for (int i = 0; i < 4; ++i)
      if (want_factor[i]) out[1 + i] = grads[i];
    out[5] = dbias;
    return out;
  }
};

int activation_of(PyObject* o) {
  if (o == Py_None) return CP4_ACT_NONE;
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "relu") == 0) return CP4_ACT_RELU;
    if (PyUnicode_CompareWithASCIIString(o, "none") == 0) return CP4_ACT_NONE;
  }
  PyErr_SetObject(PyExc_KeyError, o);
  throw python_error();
}

// Python's o == 1.
bool equals_one(PyObject* o) {
  if (PyLong_Check(o)) return integer(o) == 1;
  PyObject* one = PyLong_FromLong(1);
  const int eq = one ? PyObject_RichCompareBool(o, one, Py_EQ) : -1;
  Py_XDECREF(one);
  if (eq < 0) throw python_error();
  return eq != 0;
}

// An int or a pair of ints.
void int_pair(PyObject* o, long* h, long* w) {
  if (PyLong_Check(o)) {
    *h = *w = integer(o);
    return;
  }
  PyObject* seq = PySequence_Fast(o, "expected an int or an (h, w) pair");
  if (!seq) throw python_error();
  const bool two = PySequence_Fast_GET_SIZE(seq) == 2;
  if (two) {
    *h = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, 0));
    *w = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, 1));
  }
  Py_DECREF(seq);
  if (PyErr_Occurred()) throw python_error();
  if (!two) fail(PyExc_ValueError, "expected an int or an (h, w) pair");
}

// (x, FK, FC, FH, FW, pad, bias, activation, stride, padding) -> y; see torch_ops.cp4_conv2d
PyObject* layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 10);
  const Tensor& x_in = tensor(a[0]);
  const Factors f{tensor(a[1]), tensor(a[2]), tensor(a[3]), tensor(a[4])};
  LayerSpec l{};
  l.activation = activation_of(a[7]);
  PyObject* padding = a[9] == Py_None ? a[5] : a[9];
  const bool same = PyUnicode_Check(padding) && PyUnicode_CompareWithASCIIString(padding, "same") == 0;
  const bool valid = PyUnicode_Check(padding) && PyUnicode_CompareWithASCIIString(padding, "valid") == 0;
  l.shape = shape_for(x_in, f, 0);
  const long Y = l.shape.Y, X = l.shape.X;
  // the reference's own layer runs its three passes as they are (whatever number says stride 1)
  bool plain = equals_one(a[8]) && Y == X;
  if (plain && PyLong_Check(padding)) plain = 2 * integer(padding) + 1 == Y;
  else plain = plain && same && Y % 2 == 1;
  if (plain) {
    l.shape.pad = (unsigned)(Y / 2);
  } else {
    l.has_geometry = true;
    long sh, sw;
    int_pair(a[8], &sh, &sw);
    if (same) {
      check(cp4_geometry_same(&l.shape, (unsigned)sh, (unsigned)sw, &l.geometry));
    } else if (valid) {
      check(cp4_geometry_valid(&l.shape, (unsigned)sh, (unsigned)sw, &l.geometry));
    } else {
      long ph, pw;
      int_pair(padding, &ph, &pw);
      check(cp4_geometry_symmetric(&l.shape, (unsigned)sh, (unsigned)sw, (unsigned)ph, (unsigned)pw,
                                   &l.geometry));
    }
  }
  const at::ScalarType t = x_in.scalar_type();
  const bool half = plain && (t == at::kBFloat16 || t == at::kHalf);
  l.dtype = !half ? CP4_DTYPE_F32 : t == at::kBFloat16 ? CP4_DTYPE_BF16 : CP4_DTYPE_F16;
  const Tensor x = half ? x_in.contiguous() : as_f32(x_in);
  require(x.is_cuda() && x.size(1) == l.shape.C && f.FC.dim() >= 2 && f.FC.size(1) == l.shape.Rank,
          "expected a device tensor [N, C, H, W] that matches the factors");
  std::optional<Tensor> bias;
  if (a[6] != Py_None) {
    bias = tensor(a[6]);
    // (a layer with a geometry and a float16 one take any form that holds T entries)
    require(l.has_geometry || l.dtype == CP4_DTYPE_F16
                ? bias->numel() >= l.shape.T
                : bias->dim() == 1 && bias->size(0) == l.shape.T,
            "bias does not match the layer's output channels");
    l.has_bias = true;
  }
  const c10::DeviceGuard guard(x.device());
  // What carries a forward-mode tangent goes through the autograd function too, which refuses it.
  auto tracked = [](const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
  };
  const bool track = tracked(x) || tracked(f.FK) || tracked(f.FC) || tracked(f.FH) ||
                     tracked(f.FW) || (bias && tracked(*bias));
  Tensor y;
  {
    NoGil unlocked;
    if (track) {
      y = LayerFunction::apply(x, f.FK, f.FC, f.FH, f.FW, bias, l);
    } else {
      const Tensor FK = as_f32(f.FK), FC = as_f32(f.FC), FH = as_f32(f.FH), FW = as_f32(f.FW);
      y = layer_forward(l, x, Factors{FK, FC, FH, FW}, bias ? as_f32(*bias) : Tensor());
    }
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- adapters beside a shared projection (capi.adapter_*, torch_ops.adapter_linear) ---------

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CP4_DTYPE_F32;
    case at::kBFloat16: return CP4_DTYPE_BF16;
    case at::kHalf: return CP4_DTYPE_F16;
    default: fail(PyExc_AssertionError, "expected float32, bfloat16 or float16");
  }
}
std::optional<Tensor> optional_tensor(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return tensor(o);
}
// [..., cols] as rows that lie `stride` apart; copied where its last dimensions do not allow that.
Tensor rows_of(const Tensor& t, size_t* stride) {
  const int64_t cols = t.size(-1);
  const bool one = t.dim() == 2 && t.size(0) == 1;  // (a single row's stride says nothing, and may be anything)
  if (t.dim() == 2 && (cols == 1 || t.stride(1) == 1) && (one || t.stride(0) >= cols)) {
    *stride = (size_t)(one ? cols : t.stride(0));
    return t;
  }
  *stride = (size_t)cols;
  return t.contiguous();
}

// The bytes from a tensor's first value to behind its last one, and whether two tensors' overlap.
std::pair<const char*, const char*> extent(const Tensor& t) {
  const char* const first = static_cast<const char*>(t.data_ptr());
  if (!t.numel()) return {first, first};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {first, first + (last + 1) * t.element_size()};
}
bool overlap(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return false;
  const auto x = extent(a), y = extent(b);
  return x.first < y.second && y.first < x.second;
}
// An output that the caller gave is none of the operands'.
void check_apart(const Tensor& out, std::initializer_list<const Tensor*> operands) {
  for (const Tensor* t : operands) require(!overlap(out, *t), "out overlaps an operand");
}

// The weights of a projection [N, K]: a tensor, or microscaled 4-bit floating point (capi.Mx4: codes, scales, K).
struct Weight {
  Tensor W, scales;                                // (scales undefined: W is the tensor)
  int64_t K = 0;
  bool four() const { return scales.defined(); }
  cp4_mx4 mx4() const { return cp4_mx4{W.data_ptr(), static_cast<const unsigned char*>(scales.data_ptr())}; }
};
// Rows held in 4 bits as the C ABI takes them: contiguous, codes on a 16-byte boundary.
Weight packed(const Tensor& codes, const Tensor& scales, int64_t K) {
  const int64_t blocks = (K + 31) / 32;
  require(K >= 1 && K <= 1 << 22 && codes.is_cuda() && scales.is_cuda() && scales.device() == codes.device() &&
              codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.dim() >= 1 &&
              codes.dim() == scales.dim() && codes.size(-1) == blocks * 16 && scales.size(-1) == blocks &&
              codes.sizes().slice(0, codes.dim() - 1) == scales.sizes().slice(0, codes.dim() - 1),
          "expected uint8 codes [..., ceil(K / 32) * 16] and scales [..., ceil(K / 32)] on one device");
  Weight w;
  w.W = codes.contiguous();
  if ((size_t)w.W.data_ptr() & 15) w.W = w.W.clone();
  w.scales = scales.contiguous();
  w.K = K;
  return w;
}
bool is_packed(PyObject* o) { return PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3; }
Weight packed_of(PyObject* o) {
  require(is_packed(o), "expected codes, scales and the number of values of a row");
  const Tensor &codes = tensor(PyTuple_GET_ITEM(o, 0)), &scales = tensor(PyTuple_GET_ITEM(o, 1));
  return packed(codes, scales, integer(PyTuple_GET_ITEM(o, 2)));
}
Weight weight_of(PyObject* o) {
  if (is_packed(o)) return packed_of(o);
  Weight w;
  w.W = tensor(o);
  if (w.W.dim() == 2) w.K = w.W.size(1);
  return w;
}

struct Adapters {
  cp4_adapter_shape shape{};
  int dtype = 0;
  bool four = false;
  Tensor x, W, scales, A, B, ids, scale, bias;     // as the C ABI takes them
  cp4_mx4 mx4() const { return cp4_mx4{W.data_ptr(), static_cast<const unsigned char*>(scales.data_ptr())}; }
};
// Checks the operands of an adapter call; x: [..., K] (dy of a backward call: [..., N]).
Adapters adapters(const Tensor& x, const Weight& w, const Tensor& A, const Tensor& B, const Tensor& ids,
                  const std::optional<Tensor>& scale, const std::optional<Tensor>& bias, bool is_dy = false) {
  Adapters p;
  const Tensor& W = w.W;
  require(x.dim() >= 1 && W.dim() == 2 && A.dim() == 3 && B.dim() == 3,
          "expected x [..., K], W [N, K], A [adapters, R, K] and B [adapters, N, R]");
  const int64_t N = W.size(0), K = w.K, G = A.size(0), R = A.size(1);
  require(x.size(-1) == (is_dy ? N : K) && A.size(2) == K && B.size(0) == G && B.size(1) == N && B.size(2) == R,
          "x, W, A and B do not match");
  for (const Tensor* t : {&x, &W, &A, &B})
    require(t->is_cuda() && t->device() == x.device() && (t->scalar_type() == x.scalar_type() || (t == &W && w.four())),
            "x, W, A and B must be of one type on one device");
  p.dtype = dtype_of(x);
  for (const auto& t : {scale, bias})
    require(!t || (t->is_cuda() && t->device() == x.device() && t->scalar_type() == at::kFloat && t->dim() == 1),
            "scale and bias must be float32 vectors on x's device");
  require(!scale || scale->size(0) == G, "scale holds one value an adapter");
  require(!bias || bias->size(0) == N, "bias does not match W");
  const int64_t rows = x.numel() / std::max<int64_t>(1, x.size(-1));
  require(ids.is_cuda() && ids.device() == x.device() && ids.numel() == (x.size(-1) ? rows : ids.numel()) &&
              (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
          "ids must be one int32 or int64 a token, on x's device");
  require(N <= 1 << 22 && K <= 1 << 22 && G <= 65535 && R <= 256, "adapters: K, N <= 2^22, R <= 256, G <= 65535");
  p.shape.T = (size_t)ids.numel();
  p.shape.K = (unsigned)K; p.shape.N = (unsigned)N; p.shape.R = (unsigned)R; p.shape.G = (unsigned)G;
  p.x = rows_of(x, is_dy ? &p.shape.lddy : &p.shape.ldx);
  p.W = w.four() ? W : rows_of(W, &p.shape.ldw);
  p.scales = w.scales;
  p.four = w.four();
  p.A = A.contiguous();
  p.B = B.contiguous();
  p.ids = ids.contiguous();
  if (ids.scalar_type() == at::kLong)                // (an id beyond 32 bits is no adapter's)
    p.ids = at::where((p.ids >= 0).logical_and(p.ids < G), p.ids, at::full({}, -1, p.ids.options())).to(at::kInt);
  if (scale) p.scale = scale->contiguous();
  if (bias) p.bias = bias->contiguous();
  return p;
}
const float* floats(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; }
const int* ints(const Tensor& t) { return static_cast<const int*>(t.data_ptr()); }
std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s = sizes.vec();
  s.back() = last;
  return s;
}

// y, and where `kept` is given what the backward call needs.
Tensor adapter_run(const Adapters& p, at::IntArrayRef sizes, Tensor y, Tensor* kept, void* st) {
  if (!y.defined()) y = empty(with_last(sizes, p.shape.N), p.x.scalar_type(), p.x);
  if (kept) *kept = empty({(int64_t)(cp4_adapter_kept_bytes(&p.shape, p.dtype) / 4)}, at::kFloat, p.x);
  const size_t need = p.four ? cp4_adapter_mx4_forward_workspace_bytes(&p.shape, p.dtype)
                             : cp4_adapter_forward_workspace_bytes(&p.shape, p.dtype);
  const Tensor ws = scratch(need, p.x);
  float* const keep = kept ? static_cast<float*>(ptr(*kept)) : nullptr;
  if (p.four) {
    const cp4_mx4 w = p.mx4();
    check(cp4_adapter_mx4_forward(&p.shape, p.dtype, ptr(p.x), &w, ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale),
                                  floats(p.bias), ptr(y), keep, ptr(ws), need, st));
  } else {
    check(cp4_adapter_forward(&p.shape, p.dtype, ptr(p.x), ptr(p.W), ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale),
                              floats(p.bias), ptr(y), keep, ptr(ws), need, st));
  }
  return y;
}
// dx, dA, dB as far as they are wanted; p.x is dy.
void adapter_run_backward(const Adapters& p, const Tensor& x_in, const Tensor& kept, at::IntArrayRef sizes, Tensor* dx,
                          Tensor* dA, Tensor* dB, void* st) {
  cp4_adapter_shape s = p.shape;
  Tensor x;
  if (dA) {
    require(x_in.is_cuda() && x_in.device() == p.x.device() && x_in.scalar_type() == p.x.scalar_type() &&
                x_in.dim() >= 1 && x_in.size(-1) == (int64_t)s.K && x_in.numel() == (int64_t)(s.T * s.K),
            "x does not match dy");
    x = rows_of(x_in, &s.ldx);
    require(kept.defined() && kept.is_cuda() && kept.scalar_type() == at::kFloat && kept.is_contiguous() &&
                (size_t)kept.numel() * 4 == cp4_adapter_kept_bytes(&s, p.dtype),
            "kept is not what the forward call left");
    *dA = empty({(int64_t)s.G, (int64_t)s.R, (int64_t)s.K}, p.x.scalar_type(), p.x);
    *dB = empty({(int64_t)s.G, (int64_t)s.N, (int64_t)s.R}, p.x.scalar_type(), p.x);
  }
  if (dx) *dx = empty(with_last(sizes, s.K), p.x.scalar_type(), p.x);
  const size_t need = p.four ? cp4_adapter_mx4_backward_workspace_bytes(&s, p.dtype) : cp4_adapter_backward_workspace_bytes(&s, p.dtype);
  const Tensor ws = scratch(need, p.x);
  void *const to_x = dx ? ptr(*dx) : nullptr, *const to_A = dA ? ptr(*dA) : nullptr, *const to_B = dB ? ptr(*dB) : nullptr;
  const float* const h = static_cast<const float*>(ptr(kept));
  if (p.four) {
    const cp4_mx4 w = p.mx4();
    check(cp4_adapter_mx4_backward(&s, p.dtype, ptr(p.x), ptr(x), &w, ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale), h, to_x,
                                   to_A, to_B, ptr(ws), need, st));
  } else {
    check(cp4_adapter_backward(&s, p.dtype, ptr(p.x), ptr(x), ptr(p.W), ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale), h, to_x,
                               to_A, to_B, ptr(ws), need, st));
  }
}

// (x, W, A, B, ids, scale, bias, out, keep, stream) -> y, or (y, kept)
PyObject* adapter_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 10);
  const Tensor &x = tensor(a[0]), &A = tensor(a[2]), &B = tensor(a[3]), &ids = tensor(a[4]);
  const Weight W = weight_of(a[1]);
  const auto scale = optional_tensor(a[5]), bias = optional_tensor(a[6]);
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  Tensor y = a[7] != Py_None ? tensor(a[7]) : Tensor(), kept;
  const bool keep = PyObject_IsTrue(a[8]) == 1;
  void* st = stream_of(a[9]);
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    const Adapters p = adapters(x, W, A, B, ids, scale, bias);
    require(!y.defined() || (y.is_cuda() && y.device() == x.device() && y.scalar_type() == x.scalar_type() &&
                             y.is_contiguous() && y.numel() == (int64_t)(p.shape.T * p.shape.N)),
            "out does not match the result");
    const Tensor none;
    check_apart(y, {&x, &W.W, &W.scales, &A, &B, &ids, scale ? &*scale : &none, bias ? &*bias : &none});
    y = adapter_run(p, x.sizes(), y, keep ? &kept : nullptr, st);
  }
  if (a[7] != Py_None && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();   // (what autograd saved of it is out of date)
  PyObject* py = THPVariable_Wrap(std::move(y));
  return keep ? Py_BuildValue("(NN)", py, THPVariable_Wrap(std::move(kept))) : py;
  END_HANDLE_TH_ERRORS
}

// (dy, x, W, A, B, ids, scale, kept, want_dx, want_factors, stream) -> (dx, dA, dB)
PyObject* adapter_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 11);
  const Tensor &dy = tensor(a[0]), &A = tensor(a[3]), &B = tensor(a[4]), &ids = tensor(a[5]);
  const Weight W = weight_of(a[2]);
  const auto x = optional_tensor(a[1]), scale = optional_tensor(a[6]), kept = optional_tensor(a[7]);
  const bool want_dx = PyObject_IsTrue(a[8]) == 1, want = PyObject_IsTrue(a[9]) == 1;
  require(!want || (x && kept), "the adapters' gradients need x and what the forward call kept");
  require(dy.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(dy.device());
  void* st = stream_of(a[10]);
  Tensor g[3];
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    const Adapters p = adapters(dy, W, A, B, ids, scale, std::nullopt, true);
    adapter_run_backward(p, want ? *x : Tensor(), want ? *kept : Tensor(), dy.sizes(), want_dx ? &g[0] : nullptr,
                         want ? &g[1] : nullptr, want ? &g[2] : nullptr, st);
  }
  PyObject* out = PyTuple_New(3);
  if (!out) throw python_error();
  for (int i = 0; i < 3; ++i) {
    PyObject* o = Py_None;
    if (g[i].defined()) o = THPVariable_Wrap(std::move(g[i]));
    else Py_INCREF(o);
    PyTuple_SET_ITEM(out, i, o);
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// In a backward pass that is captured into a graph: a leaf whose gradient torch would add up on the default stream, since an
// eager graph that uses the leaf still lives, would pull that stream into the capture, which ends the process.
void check_captured_leaves(const Tensor& grad) {
  const auto current = c10::hip::getCurrentHIPStream(grad.device().index());
  const auto none = c10::hip::getDefaultHIPStream(grad.device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (current == none || hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const auto& next = node->next_edge(i).function;
    if (!next || !node->task_should_compute_output(i) || !dynamic_cast<torch::autograd::AccumulateGrad*>(next.get())) continue;
    const auto stream = next->stream();                              // (on a device of type cuda, where HIP's own are of type hip)
    TORCH_CHECK(!stream || stream->id() != none.id(),
                "a backward pass is being captured while an eager graph of the same leaves lives: drop what was computed from them first");
  }
}

struct AdapterFunction : torch::autograd::Function<AdapterFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& W, const Tensor& A,
                        const Tensor& B, const Tensor& ids, const std::optional<Tensor>& scale,
                        const std::optional<Tensor>& bias, const std::optional<Tensor>& scales, int64_t K) {
    const Adapters p = adapters(x, Weight{W, scales ? *scales : Tensor(), K}, A, B, ids, scale, bias);
    const bool factors = A.requires_grad() || B.requires_grad();
    Tensor kept;
    Tensor y = adapter_run(p, x.sizes(), Tensor(), factors ? &kept : nullptr,
                           c10::hip::getCurrentHIPStream(x.device().index()).stream());
    ctx->save_for_backward({factors ? x : Tensor(), W, A, B, ids, scale ? *scale : Tensor(), kept, scales ? *scales : Tensor()});
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(9);
    if (!grad[0].defined()) return out;
    check_captured_leaves(grad[0]);
    Tensor dy = grad[0];
    if (dy.scalar_type() != s[2].scalar_type()) dy = dy.to(s[2].scalar_type());
    const bool want_dx = ctx->needs_input_grad(0), want = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    const std::optional<Tensor> scale = s[5].defined() ? std::optional<Tensor>(s[5]) : std::nullopt;
    Weight W{s[1], s[7], s[2].size(2)};
    if (W.four()) W = packed(s[1], s[7], W.K);                       // (hooks may have given back something else)
    const Adapters p = adapters(dy, W, s[2], s[3], s[4], scale, std::nullopt, true);
    Tensor dx, dA, dB;
    void* st = c10::hip::getCurrentHIPStream(dy.device().index()).stream();
    adapter_run_backward(p, s[0], s[6], dy.sizes(), want_dx ? &dx : nullptr, want ? &dA : nullptr,
                         want ? &dB : nullptr, st);
    out[0] = dx;
    if (ctx->needs_input_grad(2)) out[2] = dA;
    if (ctx->needs_input_grad(3)) out[3] = dB;
    // create_graph: the gradients are the library's and have none of their own; who asks for those is told
    if (at::GradMode::is_enabled())
      for (int i : {0, 2, 3})
        if (out[i].defined())
          out[i] = (*std::make_shared<torch::autograd::DelayedError>(
              "the gradients of adapter_linear cannot be differentiated again", 1))({out[i].detach().set_requires_grad(true)})[0];
    return out;
  }
};

// (x, W, A, B, ids, scale, bias) -> y; see torch_ops.adapter_linear
PyObject* adapter_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 7);
  const Tensor &x = tensor(a[0]), &A = tensor(a[2]), &B = tensor(a[3]), &ids = tensor(a[4]);
  const Weight W = weight_of(a[1]);
  const auto scale = optional_tensor(a[5]), bias = optional_tensor(a[6]);
  auto tracked = [](const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
  };
  if (tracked(W.W) || (bias && tracked(*bias)) || (scale && tracked(*scale)))
    fail(PyExc_ValueError, "the projection, its bias and the scales are not trained: detach them");
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  Tensor y;
  {
    NoGil unlocked;
    if (tracked(x) || tracked(A) || tracked(B)) {
      y = AdapterFunction::apply(x, W.W, A, B, ids, scale, bias, W.four() ? std::optional<Tensor>(W.scales) : std::nullopt, W.K);
    } else {
      const Adapters p = adapters(x, W, A, B, ids, scale, bias);
      y = adapter_run(p, x.sizes(), Tensor(), nullptr, c10::hip::getCurrentHIPStream(x.device().index()).stream());
    }
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- layer norm (capi.layer_norm_*, torch_ops.layer_norm) -----------------------------------------

struct NormRows {
  size_t T = 0, ld = 0;
  unsigned D = 0;
  int dtype = 0;
  Tensor x, weight, bias;                          // as the C ABI takes them
};
// Checks the operands of a layer norm; x: [..., D].
NormRows norm_rows(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias) {
  NormRows p;
  require(x.is_cuda(), "expected device tensors");
  require(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 32768, "expected x [..., D], D from 1 to 32768");
  for (const auto& t : {weight, bias})
    require(!t || (t->is_cuda() && t->device() == x.device() && t->scalar_type() == at::kFloat && t->dim() == 1 &&
                   t->size(0) == x.size(-1)),
            "weight and bias must be float32 vectors of x's last dimension, on x's device");
  p.dtype = dtype_of(x);
  p.D = (unsigned)x.size(-1);
  p.T = (size_t)(x.numel() / x.size(-1));
  p.x = rows_of(x, &p.ld);
  if (weight) p.weight = weight->contiguous();
  if (bias) p.bias = bias->contiguous();
  return p;
}
Tensor norm_run(const NormRows& p, at::IntArrayRef sizes, float eps, Tensor y, Tensor* stats, void* st) {
  if (!y.defined()) y = empty(sizes, p.x.scalar_type(), p.x);
  if (stats) *stats = empty({(int64_t)p.T, 2}, at::kFloat, p.x);
  check(cp4_layer_norm_forward(p.T, p.D, p.dtype, ptr(p.x), p.ld, floats(p.weight), floats(p.bias), eps, ptr(y),
                               stats ? static_cast<float*>(ptr(*stats)) : nullptr, st));
  return y;
}
// dx, dweight, dbias as far as they are wanted.
void norm_run_backward(const Tensor& dy_in, const Tensor& x, const std::optional<Tensor>& weight, const Tensor& stats,
                       Tensor* dx, Tensor* dw, Tensor* db, void* st) {
  const NormRows p = norm_rows(x, weight, std::nullopt);
  require(dy_in.is_cuda() && dy_in.device() == x.device() && dy_in.scalar_type() == x.scalar_type() &&
              dy_in.sizes() == x.sizes(),
          "dy does not match x");
  require(stats.defined() && stats.is_cuda() && stats.device() == x.device() && stats.scalar_type() == at::kFloat &&
              stats.is_contiguous() && (size_t)stats.numel() == 2 * p.T,
          "stats is not what the forward call left");
  size_t lddy = 0;
  const Tensor dy = rows_of(dy_in, &lddy);
  if (dx) *dx = empty(x.sizes(), x.scalar_type(), x);
  for (Tensor* t : {dw, db})
    if (t) *t = empty({(int64_t)p.D}, at::kFloat, x);
  const size_t need = dw || db ? cp4_layer_norm_backward_workspace_bytes(p.T, p.D) : 0;
  const Tensor ws = scratch(need, x);
  check(cp4_layer_norm_backward(p.T, p.D, p.dtype, ptr(dy), lddy, ptr(p.x), p.ld, floats(p.weight), floats(stats),
                                dx ? ptr(*dx) : nullptr, dw ? static_cast<float*>(ptr(*dw)) : nullptr,
                                db ? static_cast<float*>(ptr(*db)) : nullptr, ptr(ws), need, st));
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}
PyObject* or_none(Tensor&& t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}

// (x, weight, bias, eps, out, keep, stream) -> y, or (y, stats)
PyObject* layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 7);
  const Tensor& x = tensor(a[0]);
  const auto weight = optional_tensor(a[1]), bias = optional_tensor(a[2]);
  const float eps = real(a[3]);
  Tensor y = a[4] != Py_None ? tensor(a[4]) : Tensor(), stats;
  const bool keep = PyObject_IsTrue(a[5]) == 1;
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  void* st = stream_of(a[6]);
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    const NormRows p = norm_rows(x, weight, bias);
    require(!y.defined() || (y.is_cuda() && y.device() == x.device() && y.scalar_type() == x.scalar_type() &&
                             y.is_contiguous() && y.numel() == x.numel()),
            "out does not match the result");
    const Tensor none;
    const bool in_place = y.defined() && x.is_contiguous() && y.data_ptr() == x.data_ptr();
    check_apart(y, {in_place ? &none : &x, weight ? &*weight : &none, bias ? &*bias : &none});
    y = norm_run(p, x.sizes(), eps, y, keep ? &stats : nullptr, st);
  }
  if (a[4] != Py_None && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  PyObject* py = THPVariable_Wrap(std::move(y));
  return keep ? Py_BuildValue("(NN)", py, THPVariable_Wrap(std::move(stats))) : py;
  END_HANDLE_TH_ERRORS
}

// (dy, x, weight, stats, want_dx, want_weight, want_bias, stream) -> (dx, dweight, dbias)
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 8);
  const Tensor &dy = tensor(a[0]), &x = tensor(a[1]), &stats = tensor(a[3]);
  const auto weight = optional_tensor(a[2]);
  const bool want[3] = {PyObject_IsTrue(a[4]) == 1, PyObject_IsTrue(a[5]) == 1, PyObject_IsTrue(a[6]) == 1};
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  void* st = stream_of(a[7]);
  Tensor g[3];
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    norm_run_backward(dy, x, weight, stats, want[0] ? &g[0] : nullptr, want[1] ? &g[1] : nullptr, want[2] ? &g[2] : nullptr, st);
  }
  return Py_BuildValue("(NNN)", or_none(std::move(g[0])), or_none(std::move(g[1])), or_none(std::move(g[2])));
  END_HANDLE_TH_ERRORS
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    const NormRows p = norm_rows(x, weight, bias);
    Tensor stats;
    Tensor y = norm_run(p, x.sizes(), (float)eps, Tensor(), &stats,
                        c10::hip::getCurrentHIPStream(x.device().index()).stream());
    ctx->save_for_backward({x, weight ? *weight : Tensor(), stats});
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(4);
    if (!grad[0].defined()) return out;
    check_captured_leaves(grad[0]);
    const Tensor dy = grad[0].scalar_type() == s[0].scalar_type() ? grad[0] : grad[0].to(s[0].scalar_type());
    const std::optional<Tensor> weight = s[1].defined() ? std::optional<Tensor>(s[1]) : std::nullopt;
    Tensor g[3];
    // (needs_input_grad counts the tensors that are there)
    const bool want_weight = weight && ctx->needs_input_grad(1);
    const bool want_bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight ? 2 : 1);
    norm_run_backward(dy, s[0], weight, s[2], ctx->needs_input_grad(0) ? &g[0] : nullptr, want_weight ? &g[1] : nullptr,
                      want_bias ? &g[2] : nullptr, c10::hip::getCurrentHIPStream(dy.device().index()).stream());
    for (int i = 0; i < 3; ++i) {
      out[i] = g[i];
      if (g[i].defined() && at::GradMode::is_enabled())            // (create_graph: as adapter_linear's)
        out[i] = (*std::make_shared<torch::autograd::DelayedError>(
            "the gradients of layer_norm cannot be differentiated again", 1))({g[i].detach().set_requires_grad(true)})[0];
    }
    return out;
  }
};

// (x, weight, bias, eps) -> y; see torch_ops.layer_norm
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 4);
  const Tensor& x = tensor(a[0]);
  const auto weight = optional_tensor(a[1]), bias = optional_tensor(a[2]);
  const float eps = real(a[3]);
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  auto tracked = [](const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
  };
  Tensor y;
  {
    NoGil unlocked;
    if (tracked(x) || (weight && tracked(*weight)) || (bias && tracked(*bias)))
      y = LayerNormFunction::apply(x, weight, bias, eps);
    else
      y = norm_run(norm_rows(x, weight, bias), x.sizes(), eps, Tensor(), nullptr,
                   c10::hip::getCurrentHIPStream(x.device().index()).stream());
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- microscaled 4-bit floating point (capi.mx4_*, torch_ops.mx4_linear) ---------------------------

at::ScalarType type_of(PyObject* o) {
  require(THPDtype_Check(o), "expected a dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
Weight mx4_round(const Tensor& x, void* st) {
  require(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 1 << 22, "expected a device tensor [..., K], K from 1 to 2^22");
  Weight w;
  w.K = x.size(-1);
  const int64_t blocks = (w.K + 31) / 32;
  size_t ld = 0;
  const int dtype = dtype_of(x);
  const Tensor rows = rows_of(x, &ld);
  w.W = empty(with_last(x.sizes(), blocks * 16), at::kByte, x);
  w.scales = empty(with_last(x.sizes(), blocks), at::kByte, x);
  check(cp4_mx4_quantize((size_t)(x.numel() / w.K), (unsigned)w.K, dtype, ptr(rows), ld, w.W.data_ptr(),
                         static_cast<unsigned char*>(w.scales.data_ptr()), st));
  return w;
}

// (x, stream) -> (codes, scales)
PyObject* mx4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 2);
  const Tensor& x = tensor(a[0]);
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  void* st = stream_of(a[1]);
  Weight w;
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    w = mx4_round(x, st);
  }
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(w.W)), THPVariable_Wrap(std::move(w.scales)));
  END_HANDLE_TH_ERRORS
}

// (q, dtype, out, stream) -> values
PyObject* mx4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 4);
  const Weight q = packed_of(a[0]);
  Tensor y = a[2] != Py_None ? tensor(a[2]) : Tensor();
  const at::ScalarType type = y.defined() ? y.scalar_type() : type_of(a[1]);
  const c10::DeviceGuard guard(q.W.device());
  void* st = stream_of(a[3]);
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    const std::vector<int64_t> sizes = with_last(q.W.sizes(), q.K);
    if (!y.defined()) y = empty(sizes, type, q.W);
    require(y.is_cuda() && y.device() == q.W.device() && y.is_contiguous() && y.sizes() == at::IntArrayRef(sizes), "out does not match the result");
    check_apart(y, {&q.W, &q.scales});
    const cp4_mx4 m = q.mx4();
    check(cp4_mx4_dequantize((size_t)(q.scales.numel() / q.scales.size(-1)), (unsigned)q.K, dtype_of(y), &m, ptr(y), st));
  }
  if (a[2] != Py_None && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

Tensor bias_of(const std::optional<Tensor>& bias, int64_t N, const Tensor& like) {
  require(!bias || (bias->is_cuda() && bias->device() == like.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                    bias->size(0) == N),
          "bias must be a float32 vector of W's rows, on x's device");
  return bias ? bias->contiguous() : Tensor();
}
void check_weight(const Weight& w, const Tensor& like) {
  require(w.W.dim() == 2 && w.W.size(0) >= 1 && w.W.size(0) <= 1 << 22, "expected codes of W [N, K], N from 1 to 2^22");
  require(w.W.device() == like.device(), "x and W must be on one device");
}
Tensor output(const std::vector<int64_t>& sizes, at::ScalarType type, const Tensor& like, Tensor y, const Tensor& scales, const Weight& w,
              const std::optional<Tensor>& bias) {
  if (!y.defined()) return empty(sizes, type, like);
  int64_t n = 1;
  for (int64_t d : sizes) n *= d;
  require(y.is_cuda() && y.device() == like.device() && y.scalar_type() == type && y.is_contiguous() && y.numel() == n,
          "out does not match the result");
  const Tensor none;
  check_apart(y, {&like, &scales, &w.W, &w.scales, bias ? &*bias : &none});
  return y;
}
// x in its own type
Tensor mx4_run(const Tensor& x, const Weight& w, const std::optional<Tensor>& bias_in, Tensor y, void* st) {
  require(x.is_cuda() && x.dim() >= 1 && x.size(-1) == w.K, "x and W do not match");
  check_weight(w, x);
  const int64_t N = w.W.size(0);
  const Tensor bias = bias_of(bias_in, N, x);
  const int dtype = dtype_of(x);
  size_t ld = 0;
  const Tensor rows = rows_of(x, &ld);
  y = output(with_last(x.sizes(), N), x.scalar_type(), x, y, Tensor(), w, bias_in);
  const size_t T = (size_t)(x.numel() / w.K), need = cp4_mx4_forward_workspace_bytes(T, (unsigned)w.K, (unsigned)N, dtype);
  const Tensor ws = scratch(need, x);
  const cp4_mx4 m = w.mx4();
  check(cp4_mx4_forward(T, (unsigned)w.K, (unsigned)N, dtype, ptr(rows), ld, &m, floats(bias), ptr(y), ptr(ws), need, st));
  return y;
}
Tensor mx4_run_backward(const Tensor& dy, const Weight& w, void* st) {
  check_weight(w, dy);
  const int64_t N = w.W.size(0);
  require(dy.is_cuda() && dy.dim() >= 1 && dy.size(-1) == N, "dy and W do not match");
  const int dtype = dtype_of(dy);
  size_t ld = 0;
  const Tensor rows = rows_of(dy, &ld);
  Tensor dx = empty(with_last(dy.sizes(), w.K), dy.scalar_type(), dy);
  const size_t T = (size_t)(dy.numel() / N), need = cp4_mx4_backward_workspace_bytes(T, (unsigned)w.K, (unsigned)N, dtype);
  const Tensor ws = scratch(need, dy);
  const cp4_mx4 m = w.mx4();
  check(cp4_mx4_backward(T, (unsigned)w.K, (unsigned)N, dtype, ptr(rows), ld, &m, ptr(dx), ptr(ws), need, st));
  return dx;
}
// x in 4 bits
Tensor mx4_run_product(const Weight& x, const Weight& w, const std::optional<Tensor>& bias_in, at::ScalarType type, Tensor y, void* st) {
  require(x.K == w.K, "x and W do not match");
  check_weight(w, x.W);
  const int64_t N = w.W.size(0);
  const Tensor bias = bias_of(bias_in, N, x.W);
  y = output(with_last(x.W.sizes(), N), type, x.W, y, x.scales, w, bias_in);
  const size_t T = (size_t)(x.scales.numel() / x.scales.size(-1)), need = cp4_mx4_product_workspace_bytes(T, (unsigned)w.K, (unsigned)N);
  const Tensor ws = scratch(need, x.W);
  const cp4_mx4 mx = x.mx4(), mw = w.mx4();
  check(cp4_mx4_product(T, (unsigned)w.K, (unsigned)N, dtype_of(y), &mx, &mw, floats(bias), ptr(y), ptr(ws), need, st));
  return y;
}

// (x or q, W, bias, round, dtype or None, out, stream) -> y
PyObject* mx4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 7);
  const bool is_four = is_packed(a[0]), round = PyObject_IsTrue(a[3]) == 1;
  const Weight w = packed_of(a[1]);
  const Weight q = is_four ? packed_of(a[0]) : Weight();
  const Tensor x = is_four ? Tensor() : tensor(a[0]);
  const auto bias = optional_tensor(a[2]);
  Tensor y = a[5] != Py_None ? tensor(a[5]) : Tensor();
  const Tensor& like = is_four ? q.W : x;
  require(like.is_cuda(), "expected device tensors");
  const at::ScalarType type = a[4] != Py_None ? type_of(a[4]) : is_four ? (y.defined() ? y.scalar_type() : at::kFloat) : x.scalar_type();
  require(is_four || type == x.scalar_type() || round, "y is of x's type");
  const c10::DeviceGuard guard(like.device());
  void* st = stream_of(a[6]);
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    if (is_four) {
      y = mx4_run_product(q, w, bias, type, y, st);
    } else if (round) {
      require(x.dim() >= 1 && x.size(-1) == w.K, "x and W do not match");
      y = mx4_run_product(mx4_round(x, st), w, bias, type, y, st);
    } else {
      y = mx4_run(x, w, bias, y, st);
    }
  }
  if (a[5] != Py_None && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (dy, W, stream) -> dx
PyObject* mx4_linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 3);
  const Tensor& dy = tensor(a[0]);
  const Weight w = packed_of(a[1]);
  require(dy.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(dy.device());
  void* st = stream_of(a[2]);
  Tensor dx;
  {
    NoGil unlocked;
    const at::NoGradGuard no_grad;
    dx = mx4_run_backward(dy, w, st);
  }
  return THPVariable_Wrap(std::move(dx));
  END_HANDLE_TH_ERRORS
}

struct Mx4LinearFunction : torch::autograd::Function<Mx4LinearFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t K,
                        const std::optional<Tensor>& bias) {
    Tensor y = mx4_run(x, Weight{codes, scales, K}, bias, Tensor(), c10::hip::getCurrentHIPStream(x.device().index()).stream());
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["K"] = K;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(5);
    if (!grad[0].defined()) return out;
    check_captured_leaves(grad[0]);
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const Tensor dy = grad[0].scalar_type() == type ? grad[0] : grad[0].to(type);
    const Weight w = packed(s[0], s[1], ctx->saved_data["K"].toInt());               // (as in adapter_linear's)
    if (at::GradMode::is_enabled() && grad[0].requires_grad())       // (create_graph: dx is linear in dy, but for W it has no rule)
      out[0] = (*std::make_shared<torch::autograd::DelayedError>("the gradients of mx4_linear cannot be differentiated again", 1))(
          {mx4_run_backward(dy.detach(), w, c10::hip::getCurrentHIPStream(dy.device().index()).stream()).set_requires_grad(true)})[0];
    else
      out[0] = mx4_run_backward(dy, w, c10::hip::getCurrentHIPStream(dy.device().index()).stream());
    return out;
  }
};

// (x, W, bias) -> y; see torch_ops.mx4_linear
PyObject* mx4_linear_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 3);
  const Tensor& x = tensor(a[0]);
  const Weight w = packed_of(a[1]);
  const auto bias = optional_tensor(a[2]);
  auto tracked = [](const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
  };
  if (bias && tracked(*bias)) fail(PyExc_ValueError, "the projection and its bias are not trained: detach them");
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  Tensor y;
  {
    NoGil unlocked;
    if (tracked(x)) y = Mx4LinearFunction::apply(x, w.W, w.scales, w.K, bias);
    else y = mx4_run(x, w, bias, Tensor(), c10::hip::getCurrentHIPStream(x.device().index()).stream());
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// ---- AdamW over many tensors (optim.py) --------------------------------------------------------

// The tensors of a list or tuple, held by a tuple of their own (a Tensor's count of owners is an atomic: 65
// parameters with their gradients and moments cost 6 us of those); where there may be holes, None is none.
class TensorList {
 public:
  TensorList(PyObject* o, size_t count, const char* what, bool holes = false) : count_(count) {
    if (o == Py_None && holes) return;
    items_ = PySequence_Tuple(o);
    if (!items_) throw python_error();
    bool good = (size_t)PyTuple_GET_SIZE(items_) == count;
    for (size_t i = 0; good && i < count; ++i) {
      PyObject* v = PyTuple_GET_ITEM(items_, i);
      good = THPVariable_Check(v) || (holes && v == Py_None);
    }
    if (!good) {
      Py_CLEAR(items_);
      fail(PyExc_AssertionError, what);
    }
  }
  ~TensorList() { Py_XDECREF(items_); }              // (with the interpreter lock)
  TensorList(const TensorList&) = delete;
  TensorList& operator=(const TensorList&) = delete;
  bool has(size_t i) const { return items_ && PyTuple_GET_ITEM(items_, i) != Py_None; }
  const Tensor& operator[](size_t i) const { return has(i) ? THPVariable_Unpack(PyTuple_GET_ITEM(items_, i)) : none_; }
  size_t size() const { return count_; }

 private:
  PyObject* items_ = nullptr;
  size_t count_;
  Tensor none_;
};
size_t length(PyObject* o) {
  const Py_ssize_t n = PySequence_Size(o);
  if (n < 0) throw python_error();
  return (size_t)n;
}
void* dense(const Tensor& t, int64_t n, const Tensor& like, const char* what) {
  require(t.is_cuda() && t.device() == like.device() && t.numel() == n && t.is_contiguous(), what);
  return t.data_ptr();
}
constexpr int64_t kMomentBlock = 256;
// The moments of tensor i: 32 bits, or 8 with their scales [2, blocks].
void moments_of(cp4_adamw_tensor& t, const Tensor& m, const Tensor& v, const Tensor& scales, const Tensor& like) {
  const int64_t n = (int64_t)t.n;
  t.exp_avg = dense(m, n, like, "a moment does not match its tensor");
  t.exp_avg_sq = dense(v, n, like, "a moment does not match its tensor");
  if (m.scalar_type() == at::kFloat) {
    require(v.scalar_type() == at::kFloat, "moments are float32 both, or int8 and uint8");
    t.bits = 32;
    return;
  }
  require(m.scalar_type() == at::kChar && v.scalar_type() == at::kByte, "moments are float32 both, or int8 and uint8");
  const int64_t blocks = (n + kMomentBlock - 1) / kMomentBlock;
  require(scales.defined() && scales.is_cuda() && scales.device() == like.device() &&
              scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == 2 &&
              scales.size(1) == blocks && (blocks <= 1 || scales.stride(1) == 1),
          "8-bit moments have float32 scales [2, ceil(n / 256)]");
  t.bits = 8;
  t.scale = static_cast<float*>(scales.data_ptr());
  t.scale_sq = t.scale + scales.stride(0);
}
// What autograd has saved of a tensor that is written here is out of date (where: those that are, or all).
void written(const TensorList& list, const TensorList* where = nullptr) {
  for (size_t i = 0; i < list.size(); ++i)
    if (list.has(i) && (!where || where->has(i)) && !list[i].is_inference())
      list[i].unsafeGetTensorImpl()->bump_version();
}

// (params, grads, exp_avgs, exp_avg_sqs, scales, copies, group of each or None,
//  [(lr, beta1, beta2, eps, weight_decay, counter)], max_norm, grad_scale, stream) -> norm or None
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  require(n_args == 11);
  const size_t n = length(a[0]), n_groups = length(a[7]);
  const TensorList params(a[0], n, "expected a list of tensors"), grads(a[1], n, "one gradient a parameter", true);
  const TensorList ms(a[2], n, "one first moment a parameter"), vs(a[3], n, "one second moment a parameter");
  const TensorList scales(a[4], n, "one pair of scales (or None) a parameter", true);
  const TensorList copies(a[5], n, "one copy (or None) a parameter", true);
  std::vector<cp4_adamw_group> groups(n_groups);
  std::vector<Tensor> counters(n_groups);
  PyObject* seq = PySequence_Fast(a[7], "expected a list of groups");
  if (!seq) throw python_error();
  for (size_t k = 0; k < n_groups; ++k) {
    cp4_adamw_group& g = groups[k];
    PyObject* counter;
    if (!PyArg_ParseTuple(PySequence_Fast_GET_ITEM(seq, k), "dddddO", &g.lr, &g.beta1, &g.beta2, &g.eps,
                          &g.weight_decay, &counter)) {
      Py_DECREF(seq);
      throw python_error();
    }
    if (THPVariable_Check(counter)) counters[k] = THPVariable_Unpack(counter);
  }
  Py_DECREF(seq);
  require(n_groups > 0, "at least one group");
  const Tensor& like = counters[0];
  for (size_t k = 0; k < n_groups; ++k) {
    const Tensor& c = counters[k];
    require(c.defined() && c.is_cuda() && c.device() == like.device() && c.scalar_type() == at::kDouble &&
                c.numel() == 4 && c.is_contiguous(),
            "a counter is four contiguous float64 on the tensors' device");
    groups[k].counter = static_cast<double*>(c.data_ptr());
  }
  std::vector<cp4_adamw_tensor> list;
  list.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    if (!grads.has(i)) continue;
    cp4_adamw_tensor t{};
    t.n = (size_t)params[i].numel();
    t.param = dense(params[i], (int64_t)t.n, like, "a parameter is not a contiguous tensor on the counter's device");
    t.param_dtype = dtype_of(params[i]);
    t.grad = dense(grads[i], (int64_t)t.n, like, "a gradient does not match its parameter");
    t.grad_dtype = dtype_of(grads[i]);
    if (copies.has(i)) {
      t.copy = dense(copies[i], (int64_t)t.n, like, "a copy does not match its parameter");
      t.copy_dtype = dtype_of(copies[i]);
    }
    moments_of(t, ms[i], vs[i], scales[i], like);
    if (a[6] != Py_None) {
      PyObject* g = PySequence_GetItem(a[6], (Py_ssize_t)i);
      if (!g) throw python_error();
      const long k = PyLong_AsLong(g);
      Py_DECREF(g);
      if (PyErr_Occurred()) throw python_error();
      require(k >= 0 && (size_t)k < n_groups, "a parameter of a group that is not there");
      t.group = (unsigned)k;
    }
    list.push_back(t);
  }
  const float max_norm = a[8] == Py_None ? 0.0f : (float)PyFloat_AsDouble(a[8]);
  const double grad_scale = PyFloat_AsDouble(a[9]);
  if (PyErr_Occurred()) throw python_error();
  require(a[8] == Py_None || max_norm > 0, "max_norm must be above 0 (in float32)");
  const c10::DeviceGuard guard(like.device());
  void* st = stream_of(a[10]);
  Tensor norm;
  {
    NoGil unlocked;
    size_t need = 0;
    Tensor ws;
    if (max_norm > 0) {
      need = cp4_adamw_workspace_bytes();
      ws = scratch(need, like);
      norm = empty({}, at::kFloat, like);
    }
    check(cp4_adamw_step(list.data(), list.size(), groups.data(), n_groups, (float)grad_scale, max_norm,
                         static_cast<float*>(ptr(norm)), ptr(ws), need, st));
  }
  for (const auto* l : {&params, &ms, &vs, &scales, &copies}) written(*l, &grads);
  for (const Tensor& c : counters)
    if (!c.is_inference()) c.unsafeGetTensorImpl()->bump_version();
  if (!norm.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

// (exp_avgs, exp_avg_sqs, scales, values, values_sq, encode, stream): codes to values, or back
PyObject* adamw_moments(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  require(n_args == 7);
  const size_t n = length(a[0]);
  const TensorList ms(a[0], n, "expected a list of tensors"), vs(a[1], n, "one second moment a first");
  const TensorList scales(a[2], n, "one pair of scales a moment");
  const TensorList to_m(a[3], n, "one tensor of values a moment"), to_v(a[4], n, "one tensor of values a moment");
  const bool encode = PyObject_IsTrue(a[5]) == 1;
  if (!n) Py_RETURN_NONE;
  std::vector<cp4_adamw_tensor> list(n);
  std::vector<float*> pm(n), pv(n);
  for (size_t i = 0; i < n; ++i) {
    list[i].n = (size_t)ms[i].numel();
    moments_of(list[i], ms[i], vs[i], scales[i], ms[0]);
    require(list[i].bits == 8, "expected 8-bit moments");
    require(to_m[i].scalar_type() == at::kFloat && to_v[i].scalar_type() == at::kFloat, "values are float32");
    pm[i] = static_cast<float*>(dense(to_m[i], (int64_t)list[i].n, ms[0], "values do not match their moment"));
    pv[i] = static_cast<float*>(dense(to_v[i], (int64_t)list[i].n, ms[0], "values do not match their moment"));
  }
  const c10::DeviceGuard guard(ms[0].device());
  void* st = stream_of(a[6]);
  {
    NoGil unlocked;
    check(encode ? cp4_adamw_set_moments(list.data(), n, pm.data(), pv.data(), st)
                 : cp4_adamw_moments(list.data(), n, pm.data(), pv.data(), st));
  }
  if (encode)
    for (const auto* l : {&ms, &vs, &scales}) written(*l);
  else
    for (const auto* l : {&to_m, &to_v}) written(*l);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// ---- Muon over many matrices (optim.py) ----------------------------------------------------------

// (params or None, grads, momenta or None, copies or None, outs or None, lr, momentum, nesterov, weight_decay, eps, steps,
//  stream): a parameter without a gradient is left alone
PyObject* muon_step(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  require(n_args == 12);
  const size_t n = length(a[1]);
  const TensorList params(a[0], n, "one parameter a gradient", true), grads(a[1], n, "expected a list of tensors", true);
  const TensorList momenta(a[2], n, "one momentum a parameter", true), copies(a[3], n, "one copy (or None) a parameter", true);
  const TensorList outs(a[4], n, "one output a matrix", true);
  double of[4];
  for (int k = 0; k < 4; ++k) {
    PyObject* const o = a[k < 2 ? 5 + k : 6 + k];
    of[k] = PyFloat_AsDouble(o);
    if (of[k] == -1.0 && PyErr_Occurred()) throw python_error();
  }
  const bool nesterov = PyObject_IsTrue(a[7]) == 1;
  const long steps = integer(a[10]);
  require(steps >= 1 && steps <= 16, "1 to 16 steps");
  std::vector<cp4_muon_matrix> list;
  list.reserve(n);
  struct Place { const char *first, *last; bool written; };
  std::vector<Place> places;
  const auto place = [&](const Tensor& t, bool is_written) {
    const auto e = extent(t);
    if (e.first != e.second) places.push_back(Place{e.first, e.second, is_written});
  };
  const Tensor* like = nullptr;
  for (size_t i = 0; i < n; ++i) {
    if (!grads.has(i)) continue;
    const Tensor& g = grads[i];
    if (!like) like = &g;
    require(g.dim() >= 2, "matrices have two dimensions or more: [..., rows, cols]");
    require(g.size(-1) <= 65536 && g.size(-2) <= 65536, "matrices of up to 65536 rows and columns");
    cp4_muon_matrix m{};
    m.rows = (unsigned)g.size(-2);
    m.cols = (unsigned)g.size(-1);
    m.count = m.rows && m.cols ? (size_t)(g.numel() / g.size(-1) / g.size(-2)) : 0;
    const auto of_shape = [&](const Tensor& t, const char* what) {
      require(t.sizes() == g.sizes(), what);
      return dense(t, g.numel(), *like, what);
    };
    m.grad = of_shape(g, "a gradient is not a contiguous tensor on the others' device");
    m.grad_dtype = dtype_of(g);
    if (params.has(i)) {
      m.param = of_shape(params[i], "a parameter is not contiguous or does not match its gradient");
      m.param_dtype = dtype_of(params[i]);
    }
    if (copies.has(i)) {
      require(m.param, "a copy without a parameter");
      m.copy = of_shape(copies[i], "a copy is not contiguous or does not match its parameter");
      m.copy_dtype = dtype_of(copies[i]);
    }
    if (momenta.has(i)) {
      require(momenta[i].scalar_type() == at::kFloat, "a momentum is float32");
      m.momentum = static_cast<float*>(of_shape(momenta[i], "a momentum is not contiguous or does not match its parameter"));
    }
    if (outs.has(i)) {
      require(!m.param && !m.copy, "an output beside a parameter");
      m.copy = of_shape(outs[i], "an output is not contiguous or does not match its matrix");
      m.copy_dtype = dtype_of(outs[i]);
    }
    if (m.copy != m.grad || m.copy_dtype != m.grad_dtype) place(g, false);     // (an output may take its matrix's place)
    for (const auto* l : {&params, &momenta, &copies, &outs})
      if (l->has(i)) place((*l)[i], true);
    list.push_back(m);
  }
  // (one after the other in memory; of all that came before only the one that reaches furthest matters, and of those written)
  std::sort(places.begin(), places.end(), [](const Place& a, const Place& b) { return a.first < b.first; });
  const char *reached = nullptr, *reached_written = nullptr;
  for (const Place& p : places) {
    require(p.first >= (p.written ? reached : reached_written), "what is written overlaps another tensor of the step");
    reached = std::max(reached, p.last);
    if (p.written) reached_written = std::max(reached_written, p.last);
  }
  if (list.empty()) Py_RETURN_NONE;
  const c10::DeviceGuard guard(like->device());
  void* st = stream_of(a[11]);
  {
    NoGil unlocked;
    const size_t need = cp4_muon_workspace_bytes(list.data(), list.size());
    const Tensor ws = scratch(need, *like);
    check(cp4_muon_step(list.data(), list.size(), of[0], of[1], nesterov, of[2], of[3], (unsigned)steps, ptr(ws), need, st));
  }
  for (const auto* l : {&params, &momenta, &copies, &outs}) written(*l, &grads);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_XINCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}
PyObject* set_check_backward(PyObject*, PyObject* on) {
  g_check_backward.store(PyObject_IsTrue(on) == 1);
  Py_RETURN_NONE;
}

#define FAST(fn) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL
PyMethodDef kMethods[] = {
    {"forward", FAST(forward), nullptr},
    {"backward_data", FAST(backward_data), nullptr},
    {"backward_filter", FAST(backward_filter), nullptr},
    {"layer", FAST(layer), nullptr},
    {"adapter_forward", FAST(adapter_forward), nullptr},
    {"adapter_backward", FAST(adapter_backward), nullptr},
    {"adapter_linear", FAST(adapter_linear), nullptr},
    {"layer_norm_forward", FAST(layer_norm_forward), nullptr},
    {"layer_norm_backward", FAST(layer_norm_backward), nullptr},
    {"layer_norm", FAST(layer_norm), nullptr},
    {"mx4_quantize", FAST(mx4_quantize), nullptr},
    {"mx4_dequantize", FAST(mx4_dequantize), nullptr},
    {"mx4_linear", FAST(mx4_linear), nullptr},
    {"mx4_linear_backward", FAST(mx4_linear_backward), nullptr},
    {"mx4_linear_grad", FAST(mx4_linear_grad), nullptr},
    {"adamw_step", FAST(adamw_step), nullptr},
    {"adamw_moments", FAST(adamw_moments), nullptr},
    {"muon_step", FAST(muon_step), nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {"set_check_backward", set_check_backward, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
