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
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <optional>
#include <string>
#include <vector>

#include "cp4/adamw.h"
#include "cp4/adapter.h"
#include "cp4/capi.h"

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

struct Adapters {
  cp4_adapter_shape shape{};
  int dtype = 0;
  Tensor x, W, A, B, ids, scale, bias;             // as the C ABI takes them
};
// Checks the operands of an adapter call; x: [..., K] (dy of a backward call: [..., N]).
Adapters adapters(const Tensor& x, const Tensor& W, const Tensor& A, const Tensor& B, const Tensor& ids,
                  const std::optional<Tensor>& scale, const std::optional<Tensor>& bias, bool is_dy = false) {
  Adapters p;
  require(x.dim() >= 1 && W.dim() == 2 && A.dim() == 3 && B.dim() == 3,
          "expected x [..., K], W [N, K], A [adapters, R, K] and B [adapters, N, R]");
  const int64_t N = W.size(0), K = W.size(1), G = A.size(0), R = A.size(1);
  require(x.size(-1) == (is_dy ? N : K) && A.size(2) == K && B.size(0) == G && B.size(1) == N && B.size(2) == R,
          "x, W, A and B do not match");
  for (const Tensor* t : {&x, &W, &A, &B})
    require(t->is_cuda() && t->device() == x.device() && t->scalar_type() == x.scalar_type(),
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
  p.W = rows_of(W, &p.shape.ldw);
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
  const size_t need = cp4_adapter_forward_workspace_bytes(&p.shape, p.dtype);
  const Tensor ws = scratch(need, p.x);
  check(cp4_adapter_forward(&p.shape, p.dtype, ptr(p.x), ptr(p.W), ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale),
                            floats(p.bias), ptr(y), kept ? static_cast<float*>(ptr(*kept)) : nullptr, ptr(ws), need, st));
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
  const size_t need = cp4_adapter_backward_workspace_bytes(&s, p.dtype);
  const Tensor ws = scratch(need, p.x);
  check(cp4_adapter_backward(&s, p.dtype, ptr(p.x), ptr(x), ptr(p.W), ptr(p.A), ptr(p.B), ints(p.ids), floats(p.scale),
                             static_cast<const float*>(ptr(kept)), dx ? ptr(*dx) : nullptr, dA ? ptr(*dA) : nullptr,
                             dB ? ptr(*dB) : nullptr, ptr(ws), need, st));
}

// (x, W, A, B, ids, scale, bias, out, keep, stream) -> y, or (y, kept)
PyObject* adapter_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  require(n == 10);
  const Tensor &x = tensor(a[0]), &W = tensor(a[1]), &A = tensor(a[2]), &B = tensor(a[3]), &ids = tensor(a[4]);
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
  const Tensor &dy = tensor(a[0]), &W = tensor(a[2]), &A = tensor(a[3]), &B = tensor(a[4]), &ids = tensor(a[5]);
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

struct AdapterFunction : torch::autograd::Function<AdapterFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& W, const Tensor& A,
                        const Tensor& B, const Tensor& ids, const std::optional<Tensor>& scale,
                        const std::optional<Tensor>& bias) {
    const Adapters p = adapters(x, W, A, B, ids, scale, bias);
    const bool factors = A.requires_grad() || B.requires_grad();
    Tensor kept;
    Tensor y = adapter_run(p, x.sizes(), Tensor(), factors ? &kept : nullptr,
                           c10::hip::getCurrentHIPStream(x.device().index()).stream());
    ctx->save_for_backward({factors ? x : Tensor(), W, A, B, ids, scale ? *scale : Tensor(), kept});
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(7);
    if (!grad[0].defined()) return out;
    Tensor dy = grad[0];
    if (dy.scalar_type() != s[1].scalar_type()) dy = dy.to(s[1].scalar_type());
    const bool want_dx = ctx->needs_input_grad(0), want = ctx->needs_input_grad(2) || ctx->needs_input_grad(3);
    const std::optional<Tensor> scale = s[5].defined() ? std::optional<Tensor>(s[5]) : std::nullopt;
    const Adapters p = adapters(dy, s[1], s[2], s[3], s[4], scale, std::nullopt, true);
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
  const Tensor &x = tensor(a[0]), &W = tensor(a[1]), &A = tensor(a[2]), &B = tensor(a[3]), &ids = tensor(a[4]);
  const auto scale = optional_tensor(a[5]), bias = optional_tensor(a[6]);
  auto tracked = [](const Tensor& t) {
    return (at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined();
  };
  if (tracked(W) || (bias && tracked(*bias)) || (scale && tracked(*scale)))
    fail(PyExc_ValueError, "the projection, its bias and the scales are not trained: detach them");
  require(x.is_cuda(), "expected device tensors");
  const c10::DeviceGuard guard(x.device());
  Tensor y;
  {
    NoGil unlocked;
    if (tracked(x) || tracked(A) || tracked(B)) {
      y = AdapterFunction::apply(x, W, A, B, ids, scale, bias);
    } else {
      const Adapters p = adapters(x, W, A, B, ids, scale, bias);
      y = adapter_run(p, x.sizes(), Tensor(), nullptr, c10::hip::getCurrentHIPStream(x.device().index()).stream());
    }
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
    {"adamw_step", FAST(adamw_step), nullptr},
    {"adamw_moments", FAST(adamw_moments), nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {"set_check_backward", set_check_backward, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
