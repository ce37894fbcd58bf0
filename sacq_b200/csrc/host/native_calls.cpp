// The host side of a layer call as one native function per entry point.
//
// A decode-sized call is 3-9 us of GPU work.  Walked in Python -- argument checks, torch.empty,
// data_ptr(), a ctypes call with a dozen converted arguments, a device context -- its host side took
// 15 us (and 12-20 us more for every quantizer or GEMM entry point called by itself), so the GPU
// waited for the host at every size below a few hundred tokens.  Here the checks, the output
// allocation, the workspace lookup and the library call are one METH_FASTCALL function.
//
// Every function handles the plain case -- bf16 CUDA tensors of the layer's device with unit inner
// stride, shapes that match -- and returns None otherwise without having launched anything; the
// caller (linear.py, activation.py) then takes the general route, which converts what can be
// converted and raises the errors.  The calls only enqueue work and keep the GIL, which keeps the two
// launches of a forward together when two threads share a stream.  forward_host releases it: a copy from
// or to pageable memory waits for the stream, and a lock per scratch set keeps its launches together.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <map>
#include <mutex>
#include <optional>
#include <unordered_map>
#include <utility>

#include "internal.h"

namespace {

// ---------------------------------------------------------------- scratch per (device, stream)
// Calls on one stream are ordered and share a set; calls on different streams may overlap on the
// GPU, so each stream has its own.  Grown on demand, at most one set per stream of the process
// (PyTorch hands out a fixed pool of streams).  Never destroyed at exit: the tensors must not
// outlive the CUDA context's teardown order.
struct Workspace {
  at::Tensor ws;            // zero-initialised: arrival counters lead, then kernel scratch
  at::Tensor q, scale;      // quantized activations of a forward
  at::Tensor host_scratch;  // everything a host-buffer forward needs on the device
  std::mutex host_lock;     // ... and whose turn it is to use it; taken without the GIL only
};

std::map<std::pair<int, cudaStream_t>, Workspace>& pool() {
  static auto* p = new std::map<std::pair<int, cudaStream_t>, Workspace>();
  return *p;
}

at::Tensor new_tensor(at::IntArrayRef size, at::ScalarType t, int dev) {
  return at::Tensor(at::detail::empty_cuda(size, t, c10::Device(c10::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}

at::Tensor zeroed(int64_t bytes, int dev) { return new_tensor({bytes}, at::kByte, dev).zero_(); }

Workspace& workspace(int dev, cudaStream_t s) {
  static thread_local std::pair<int, cudaStream_t> last_key{-1, nullptr};
  static thread_local Workspace* last = nullptr;
  const std::pair<int, cudaStream_t> key{dev, s};
  if (last == nullptr || key != last_key) {
    last = &pool()[key];                              // map nodes do not move
    last_key = key;
  }
  return *last;
}

at::Tensor& scratch(Workspace& w, int64_t bytes, int dev) {
  if (!w.ws.defined() || w.ws.numel() < bytes) w.ws = zeroed(bytes > (1 << 20) ? bytes : (1 << 20), dev);
  return w.ws;
}

void act_buffers(Workspace& w, int64_t m, int64_t k, int dev) {
  if (!w.q.defined() || w.q.numel() < m * k) w.q = new_tensor({m * k > (1 << 16) ? m * k : (1 << 16)}, at::kByte, dev);
  if (!w.scale.defined() || w.scale.numel() < m) w.scale = new_tensor({m > 1024 ? m : 1024}, at::kFloat, dev);
}

// ---------------------------------------------------------------- small helpers
PyObject* g_error_class = nullptr;   // sacq_b200._lib.SacqError(code, message)

PyObject* raise_status(int rc) {
  PyObject* args = Py_BuildValue("(is)", rc, sacq_last_error());
  if (args != nullptr) {
    PyObject* e = PyObject_CallObject(g_error_class ? g_error_class : PyExc_RuntimeError, args);
    Py_DECREF(args);
    if (e != nullptr) {
      PyErr_SetObject((PyObject*)Py_TYPE(e), e);
      Py_DECREF(e);
    }
  }
  return nullptr;
}

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on_device(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

// A 2-D tensor whose rows are contiguous (the inner stride of rows of one element means nothing).
bool whole_rows(const at::Tensor& t) { return t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1); }

// bf16 [m, k] rows with unit inner stride
bool bf16_rows(const at::Tensor& t, int dev) {
  return t.scalar_type() == at::kBFloat16 && on_device(t, dev) && whole_rows(t);
}

bool f32_vector(const at::Tensor& t, int64_t n, int dev) {
  return t.scalar_type() == at::kFloat && on_device(t, dev) && t.numel() == n && t.is_contiguous();
}

bool byte_matrix(const at::Tensor& t, int64_t k, int dev) {
  return t.element_size() == 1 && on_device(t, dev) && t.dim() == 2 && t.size(1) == k && t.is_contiguous();
}

// The stream work of a device goes to, and that device made current while the object lives.
struct Target {
  int dev;
  cudaStream_t stream;
  std::optional<c10::cuda::CUDAGuard> guard;
  explicit Target(int d) : dev(d), stream(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)d).stream()) {
    if (c10::cuda::current_device() != d) guard.emplace((c10::DeviceIndex)d);
  }
};

// A C++ exception leaves as the Python exception that PyTorch makes of it (an allocation that fails as
// torch.OutOfMemoryError, which callers catch to free memory and try again).
#define NATIVE_TRY try {
#define NATIVE_CATCH                                                                            \
  }                                                                                             \
  catch (...) {                                                                                 \
    if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());      \
    return nullptr;                                                                             \
  }

// Activations of a forward: any [..., K] bf16 tensor whose rows can be addressed with one pitch.
struct Rows {
  const void* ptr;
  int64_t m, pitch;
};

bool rows_of(const at::Tensor& x, int64_t k, int dev, Rows& r) {
  const int64_t nd = x.dim();
  if (nd < 1 || x.scalar_type() != at::kBFloat16 || !on_device(x, dev) || x.size(nd - 1) != k) return false;
  if (nd == 2) {
    if (!whole_rows(x)) return false;
    r = {x.data_ptr(), x.size(0), x.stride(0)};
  } else {
    if (!x.is_contiguous()) return false;
    r = {x.data_ptr(), k > 0 ? x.numel() / k : 0, k};
  }
  return r.m > 0;
}

// [..., n] like x, for a fresh [m, n] result
at::Tensor result_like(const at::Tensor& x, int64_t m, int64_t n, int dev) {
  if (x.dim() == 2) return new_tensor({m, n}, at::kBFloat16, dev);
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  return new_tensor(shape, at::kBFloat16, dev);
}

// ---------------------------------------------------------------- one layer
enum NeedKind { kNeedA8 = 0, kNeedInt8 = 1, kNeedHost = 2, kNeedKinds = 3 };

struct LayerObject {
  PyObject_HEAD
  sacq_layer_t* handle;      // borrowed from the Python module that owns both
  int dev;
  int64_t k, n;
  std::unordered_map<int64_t, int64_t>* need;   // workspace bytes by 3 * M + kind
};

int64_t need_bytes(LayerObject* L, int64_t m, NeedKind kind) {
  const int64_t key = m * kNeedKinds + kind;
  auto it = L->need->find(key);
  if (it != L->need->end()) return it->second;
  const int64_t b = kind == kNeedA8     ? sacq_workspace_bytes(L->handle, m)
                    : kind == kNeedInt8 ? sacq_workspace_bytes_int8(L->handle, m)
                                        : sacq_host_forward_scratch_bytes(L->handle, m);
  if (L->need->size() > 4096) L->need->clear();       // a program with ragged token counts does not grow it without end
  L->need->emplace(key, b);
  return b;
}

// out (None, or a bf16 [m, n] tensor with unit inner stride on the device) -> the tensor to write, or undefined
at::Tensor out_or_new(PyObject* out, int64_t m, int64_t n, int dev) {
  if (out == Py_None) return new_tensor({m, n}, at::kBFloat16, dev);
  const at::Tensor* t = tensor_of(out);
  if (t == nullptr || !bf16_rows(*t, dev) || t->size(0) != m || t->size(1) != n) return at::Tensor();
  return *t;
}

PyObject* layer_forward(LayerObject* L, PyObject* x_obj) {
  NATIVE_TRY
  const at::Tensor* x = tensor_of(x_obj);
  Rows r;
  if (x == nullptr || L->n <= 0 || !rows_of(*x, L->k, L->dev, r)) Py_RETURN_NONE;
  Target at_(L->dev);
  Workspace& w = workspace(L->dev, at_.stream);
  at::Tensor& ws = scratch(w, need_bytes(L, r.m, kNeedA8), L->dev);
  act_buffers(w, r.m, L->k, L->dev);
  at::Tensor y = result_like(*x, r.m, L->n, L->dev);
  const int rc = sacq_forward_call(L->handle, r.ptr, r.pitch, r.m, 0, nullptr, 0, w.q.data_ptr(), (float*)w.scale.data_ptr(),
                                   y.data_ptr(), L->n, ws.data_ptr(), ws.numel(), at_.stream);
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : raise_status(rc);
  NATIVE_CATCH
}

PyObject* layer_forward_residual(LayerObject* L, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor *x = n == 2 ? tensor_of(a[0]) : nullptr, *res = n == 2 ? tensor_of(a[1]) : nullptr;
  Rows r, rr;
  if (x == nullptr || res == nullptr || L->n <= 0 || !rows_of(*x, L->k, L->dev, r) || !rows_of(*res, L->n, L->dev, rr) ||
      rr.m != r.m)
    Py_RETURN_NONE;
  Target at_(L->dev);
  Workspace& w = workspace(L->dev, at_.stream);
  at::Tensor& ws = scratch(w, need_bytes(L, r.m, kNeedA8), L->dev);
  act_buffers(w, r.m, L->k, L->dev);
  at::Tensor y = result_like(*x, r.m, L->n, L->dev);
  const int rc = sacq_forward_call(L->handle, r.ptr, r.pitch, r.m, 0, rr.ptr, rr.pitch, w.q.data_ptr(),
                                   (float*)w.scale.data_ptr(), y.data_ptr(), L->n, ws.data_ptr(), ws.numel(), at_.stream);
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : raise_status(rc);
  NATIVE_CATCH
}

PyObject* layer_forward_int8(LayerObject* L, PyObject* x_obj) {
  NATIVE_TRY
  const at::Tensor* x = tensor_of(x_obj);
  Rows r;
  if (x == nullptr || L->n <= 0 || !rows_of(*x, L->k, L->dev, r)) Py_RETURN_NONE;
  Target at_(L->dev);
  Workspace& w = workspace(L->dev, at_.stream);
  at::Tensor& ws = scratch(w, need_bytes(L, r.m, kNeedInt8), L->dev);
  act_buffers(w, r.m, L->k, L->dev);
  at::Tensor y = result_like(*x, r.m, L->n, L->dev);
  const int rc = sacq_forward_call(L->handle, r.ptr, r.pitch, r.m, 1, nullptr, 0, w.q.data_ptr(), (float*)w.scale.data_ptr(),
                                   y.data_ptr(), L->n, ws.data_ptr(), ws.numel(), at_.stream);
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : raise_status(rc);
  NATIVE_CATCH
}

// linear_a8(q, scale, out, residual, int8)
PyObject* layer_linear_a8(LayerObject* L, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor *q = n == 5 ? tensor_of(a[0]) : nullptr, *s = n == 5 ? tensor_of(a[1]) : nullptr;
  if (q == nullptr || s == nullptr || L->n <= 0 || !byte_matrix(*q, L->k, L->dev)) Py_RETURN_NONE;
  const int64_t m = q->size(0);
  const bool int8 = a[4] == Py_True;
  if (m == 0 || !f32_vector(*s, m, L->dev) || (int8 && q->scalar_type() != at::kChar)) Py_RETURN_NONE;
  const at::Tensor* res = nullptr;
  if (a[3] != Py_None) {
    res = tensor_of(a[3]);
    if (res == nullptr || int8 || !bf16_rows(*res, L->dev) || res->size(0) != m || res->size(1) != L->n) Py_RETURN_NONE;
  }
  Target at_(L->dev);
  at::Tensor y = out_or_new(a[2], m, L->n, L->dev);
  if (!y.defined()) Py_RETURN_NONE;
  at::Tensor& ws = scratch(workspace(L->dev, at_.stream), need_bytes(L, m, int8 ? kNeedInt8 : kNeedA8), L->dev);
  const void* qp = q->data_ptr();
  const float* sp = (const float*)s->data_ptr();
  const int rc =
      int8 ? sacq_linear_a8i(L->handle, qp, sp, m, y.data_ptr(), y.stride(0), ws.data_ptr(), ws.numel(), at_.stream)
      : res ? sacq_linear_a8_residual(L->handle, qp, sp, m, res->data_ptr(), res->stride(0), y.data_ptr(), y.stride(0),
                                      ws.data_ptr(), ws.numel(), at_.stream)
            : sacq_linear_a8(L->handle, qp, sp, m, y.data_ptr(), y.stride(0), ws.data_ptr(), ws.numel(), at_.stream);
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : raise_status(rc);
  NATIVE_CATCH
}

// linear_w8a8(q, scale, weight_row_scale, out, int8)
PyObject* layer_linear_w8a8(LayerObject* L, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor *q = n == 5 ? tensor_of(a[0]) : nullptr, *s = n == 5 ? tensor_of(a[1]) : nullptr,
                   *sw = n == 5 ? tensor_of(a[2]) : nullptr;
  if (q == nullptr || s == nullptr || sw == nullptr || L->n <= 0 || !byte_matrix(*q, L->k, L->dev)) Py_RETURN_NONE;
  const int64_t m = q->size(0);
  const bool int8 = a[4] == Py_True;
  const at::ScalarType t = q->scalar_type();
  if (m == 0 || !f32_vector(*s, m, L->dev) || !f32_vector(*sw, L->n, L->dev) ||
      !(int8 ? t == at::kChar : (t == at::kFloat8_e4m3fn || t == at::kByte)))
    Py_RETURN_NONE;
  Target at_(L->dev);
  at::Tensor y = out_or_new(a[3], m, L->n, L->dev);
  if (!y.defined()) Py_RETURN_NONE;
  at::Tensor& ws = scratch(workspace(L->dev, at_.stream), sacq_workspace_bytes_w8a8(L->handle, m), L->dev);
  const int rc = (int8 ? sacq_linear_w8a8_int8 : sacq_linear_w8a8_fp8)(
      L->handle, q->data_ptr(), (const float*)s->data_ptr(), (const float*)sw->data_ptr(), m, y.data_ptr(), y.stride(0),
      ws.data_ptr(), ws.numel(), at_.stream);
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : raise_status(rc);
  NATIVE_CATCH
}

// forward_host(x_host, out_host): both CPU bf16, contiguous
PyObject* layer_forward_host(LayerObject* L, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor *x = n == 2 ? tensor_of(a[0]) : nullptr, *y = n == 2 ? tensor_of(a[1]) : nullptr;
  if (x == nullptr || y == nullptr || L->n <= 0 || !x->is_cpu() || !y->is_cpu() || x->scalar_type() != at::kBFloat16 ||
      y->scalar_type() != at::kBFloat16 || x->dim() != 2 || y->dim() != 2 || !x->is_contiguous() || !y->is_contiguous() ||
      x->size(1) != L->k || x->size(0) <= 0 || y->size(0) != x->size(0) || y->size(1) != L->n)
    Py_RETURN_NONE;
  const int64_t m = x->size(0);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)L->dev).stream();
  Workspace& w = workspace(L->dev, stream);
  const int64_t need = need_bytes(L, m, kNeedHost);
  if (!w.host_scratch.defined() || w.host_scratch.numel() < need) {
    Target at_(L->dev);
    w.host_scratch = zeroed(need > (1 << 22) ? need : (1 << 22), L->dev);
  }
  // the call's own references: another thread may let go of its tensors, or grow the scratch, meanwhile
  const at::Tensor xt = *x, yt = *y, scratch_t = w.host_scratch;
  const void* xp = xt.data_ptr();
  void *yp = yt.data_ptr(), *sp = scratch_t.data_ptr();
  const int64_t bytes = scratch_t.numel();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  {
    std::lock_guard<std::mutex> turn(w.host_lock);
    // the library switches to the layer's device itself
    rc = sacq_linear_bf16_host(L->handle, xp, m, yp, sp, bytes, stream);
  }
  Py_END_ALLOW_THREADS
  if (rc != 0) return raise_status(rc);
  Py_INCREF(a[1]);
  return a[1];
  NATIVE_CATCH
}

PyObject* layer_forget(LayerObject* L, PyObject*) {   // the kernel choice changed: so may the workspace sizes
  L->need->clear();
  Py_RETURN_NONE;
}

PyMethodDef layer_methods[] = {
    {"forward", (PyCFunction)layer_forward, METH_O, nullptr},
    {"forward_residual", (PyCFunction)(void*)layer_forward_residual, METH_FASTCALL, nullptr},
    {"forward_int8", (PyCFunction)layer_forward_int8, METH_O, nullptr},
    {"linear_a8", (PyCFunction)(void*)layer_linear_a8, METH_FASTCALL, nullptr},
    {"linear_w8a8", (PyCFunction)(void*)layer_linear_w8a8, METH_FASTCALL, nullptr},
    {"forward_host", (PyCFunction)(void*)layer_forward_host, METH_FASTCALL, nullptr},
    {"forget_sizes", (PyCFunction)layer_forget, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyObject* layer_new(PyTypeObject* type, PyObject* args, PyObject*) {
  unsigned long long handle = 0;
  int dev = 0;
  long long n = 0, k = 0;
  if (!PyArg_ParseTuple(args, "KiLL", &handle, &dev, &n, &k)) return nullptr;
  LayerObject* L = (LayerObject*)type->tp_alloc(type, 0);
  if (L == nullptr) return nullptr;
  L->handle = (sacq_layer_t*)(uintptr_t)handle;
  L->dev = dev;
  L->n = n;
  L->k = k;
  L->need = new std::unordered_map<int64_t, int64_t>();
  return (PyObject*)L;
}

void layer_dealloc(LayerObject* L) {
  delete L->need;
  Py_TYPE(L)->tp_free((PyObject*)L);
}

PyTypeObject LayerType = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---------------------------------------------------------------- quantizers
PyObject* pair_of(at::Tensor q, at::Tensor s) {
  PyObject* t = PyTuple_New(2);
  PyObject *a = THPVariable_Wrap(std::move(q)), *b = THPVariable_Wrap(std::move(s));
  if (t == nullptr || a == nullptr || b == nullptr) {
    Py_XDECREF(t);
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}

// Fresh (q [m, k], scale [m, 1])
struct Encoded {
  at::Tensor q, s;
  Encoded(int64_t m, int64_t k, bool int8, int dev)
      : q(new_tensor({m, k}, int8 ? at::kChar : at::kFloat8_e4m3fn, dev)), s(new_tensor({m, 1}, at::kFloat, dev)) {}
};

// The 2-D bf16 CUDA input of a quantizer, not empty
const at::Tensor* quantizer_input(PyObject* o) {
  const at::Tensor* x = tensor_of(o);
  if (x == nullptr || !x->is_cuda() || !bf16_rows(*x, x->get_device()) || x->numel() == 0) return nullptr;
  return x;
}

// A bf16 vector of k contiguous elements, null for None; false: not that
bool vector_or_none(PyObject* o, int64_t k, int dev, const void** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor_of(o);
  if (t == nullptr || t->scalar_type() != at::kBFloat16 || !on_device(*t, dev) || t->numel() != k || !t->is_contiguous())
    return false;
  *p = t->data_ptr();
  return true;
}

// quantize_rows(x, int8)
PyObject* py_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* x = n == 2 ? quantizer_input(a[0]) : nullptr;
  if (x == nullptr) Py_RETURN_NONE;
  const bool int8 = a[1] == Py_True;
  Target at_(x->get_device());
  Encoded e(x->size(0), x->size(1), int8, at_.dev);
  const int rc = (int8 ? sacq_quant_act_int8 : sacq_quant_act_fp8)(x->data_ptr(), x->stride(0), x->size(0), x->size(1),
                                                                   e.q.data_ptr(), (float*)e.s.data_ptr(), at_.stream);
  return rc == 0 ? pair_of(std::move(e.q), std::move(e.s)) : raise_status(rc);
  NATIVE_CATCH
}

// act_quantize_rows(kind, a, b)
PyObject* py_act_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* x = n == 3 ? quantizer_input(a[1]) : nullptr;
  if (x == nullptr) Py_RETURN_NONE;
  const long kind = PyLong_AsLong(a[0]);
  const at::Tensor* b = nullptr;
  if (kind == SACQ_ACT_SILU_MUL) {
    b = tensor_of(a[2]);
    if (b == nullptr || !bf16_rows(*b, x->get_device()) || b->sizes() != x->sizes()) Py_RETURN_NONE;
  }
  Target at_(x->get_device());
  Encoded e(x->size(0), x->size(1), false, at_.dev);
  const int rc = sacq_act_quant_fp8((int)kind, x->data_ptr(), x->stride(0), b ? b->data_ptr() : nullptr,
                                    b ? b->stride(0) : 0, x->size(0), x->size(1), e.q.data_ptr(), (float*)e.s.data_ptr(),
                                    at_.stream);
  return rc == 0 ? pair_of(std::move(e.q), std::move(e.s)) : raise_status(rc);
  NATIVE_CATCH
}

// modulate_quantize_rows(x, scale, shift)
PyObject* py_modulate_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* x = n == 3 ? quantizer_input(a[0]) : nullptr;
  const void *sc = nullptr, *sh = nullptr;
  if (x == nullptr || !vector_or_none(a[1], x->size(1), x->get_device(), &sc) ||
      !vector_or_none(a[2], x->size(1), x->get_device(), &sh) || sc == nullptr || sh == nullptr)
    Py_RETURN_NONE;
  Target at_(x->get_device());
  Encoded e(x->size(0), x->size(1), false, at_.dev);
  const int rc = sacq_modulate_quant_fp8(x->data_ptr(), x->stride(0), sc, sh, x->size(0), x->size(1), e.q.data_ptr(),
                                         (float*)e.s.data_ptr(), at_.stream);
  return rc == 0 ? pair_of(std::move(e.q), std::move(e.s)) : raise_status(rc);
  NATIVE_CATCH
}

// layernorm_quantize_rows(x, weight, bias, eps, mod_scale, mod_shift, return_normalized)
PyObject* py_layernorm_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* x = n == 7 ? quantizer_input(a[0]) : nullptr;
  if (x == nullptr) Py_RETURN_NONE;
  const int64_t m = x->size(0), k = x->size(1);
  const int dev = x->get_device();
  const void* v[4];
  static const int at_arg[4] = {1, 2, 4, 5};
  for (int i = 0; i < 4; ++i)
    if (!vector_or_none(a[at_arg[i]], k, dev, &v[i])) Py_RETURN_NONE;
  if ((v[2] == nullptr) != (v[3] == nullptr)) Py_RETURN_NONE;
  const double eps = PyFloat_AsDouble(a[3]);
  if (eps == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const int want_y = PyObject_IsTrue(a[6]);            // any truth value, as the general route takes it
  if (want_y < 0) return nullptr;
  Target at_(dev);
  Encoded e(m, k, false, dev);
  at::Tensor y;
  if (want_y) y = new_tensor({m, k}, at::kBFloat16, dev);
  const int rc = sacq_layernorm_quant_fp8(x->data_ptr(), x->stride(0), v[0], v[1], (float)eps, v[2], v[3], m, k,
                                          y.defined() ? y.data_ptr() : nullptr, k, e.q.data_ptr(), (float*)e.s.data_ptr(),
                                          at_.stream);
  if (rc != 0) return raise_status(rc);
  if (!y.defined()) return pair_of(std::move(e.q), std::move(e.s));
  PyObject *q = THPVariable_Wrap(std::move(e.q)), *s = THPVariable_Wrap(std::move(e.s)), *yy = THPVariable_Wrap(std::move(y));
  PyObject* t = (q && s && yy) ? PyTuple_Pack(3, q, s, yy) : nullptr;
  Py_XDECREF(q);
  Py_XDECREF(s);
  Py_XDECREF(yy);
  return t;
  NATIVE_CATCH
}

// ---------------------------------------------------------------- the steps between projections
// Whether autograd would expect a backward pass through this call, or a tangent out of it: refused by the general route.
bool wants_grad(const at::Tensor& t) { return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(/*level=*/0).defined(); }

// bf16 [tokens, heads, dim] with unit inner stride and strides that go forwards
const at::Tensor* heads_of(PyObject* o, int dev) {
  const at::Tensor* t = tensor_of(o);
  if (t == nullptr || t->scalar_type() != at::kBFloat16 || t->dim() != 3 || !t->is_cuda() || (dev >= 0 && t->get_device() != dev) ||
      (t->stride(2) != 1 && t->size(2) > 1) || wants_grad(*t))
    return nullptr;
  return t;
}

// Whether two tensors share memory.  Views of one buffer whose elements take turns (the query and the key heads of a fused
// projection) do not: where a stride S of either divides the larger strides of both, their places modulo S are two spans, and those
// may lie apart.
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const at::Tensor* const both[2] = {&a, &b};
  auto places = [&](int64_t step, int64_t (&span)[2]) {      // bytes from a tensor's first to its last place modulo `step` bytes
    for (int t = 0; t < 2; ++t) {
      const int64_t size = both[t]->element_size();
      span[t] = size;
      for (int64_t i = 0; i < both[t]->dim(); ++i) {
        const int64_t stride = both[t]->stride(i) * size;
        if (both[t]->size(i) == 1 || (step != 0 && stride % step == 0)) continue;
        if (step != 0 && stride > step) return false;
        span[t] += (both[t]->size(i) - 1) * stride;
      }
    }
    return true;
  };
  const char *const pa = (const char*)a.data_ptr(), *const pb = (const char*)b.data_ptr();
  int64_t span[2];
  places(0, span);
  if (pa >= pb + span[1] || pb >= pa + span[0]) return false;
  for (const at::Tensor* t : both)
    for (int64_t i = 0; i < t->dim(); ++i) {
      const int64_t step = t->stride(i) * t->element_size();
      if (t->size(i) == 1 || step <= 0 || !places(step, span)) continue;
      const int64_t apart = ((pb - pa) % step + step) % step;
      if (apart >= span[0] && apart + span[1] <= step) return false;
    }
  return true;
}

// overlaps(a, (b, ...))
PyObject* py_overlaps(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* t = n == 2 ? tensor_of(a[0]) : nullptr;
  if (t == nullptr || !PyTuple_Check(a[1])) Py_RETURN_FALSE;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[1]); ++i) {
    const at::Tensor* b = tensor_of(PyTuple_GET_ITEM(a[1], i));
    if (b != nullptr && overlap(*t, *b)) Py_RETURN_TRUE;
  }
  Py_RETURN_FALSE;
  NATIVE_CATCH
}

PyObject* tuple_of(std::initializer_list<at::Tensor> list) {
  PyObject* t = PyTuple_New((Py_ssize_t)list.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& x : list) {
    PyObject* o = t == nullptr ? nullptr : x.defined() ? THPVariable_Wrap(x) : Py_NewRef(Py_None);
    if (o == nullptr) {
      Py_XDECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

// A result that can be written: no two of its elements are one
bool writable(const at::Tensor& t) { return at::has_internal_overlap(t) != at::MemOverlap::Yes; }

bool offsets_of(const at::Tensor* t, int dev) {
  return t != nullptr && t->scalar_type() == at::kInt && on_device(*t, dev) && t->dim() == 1 && t->numel() >= 1 && t->is_contiguous();
}

// attention_packed(q, k, v, cu_q, cu_k, causal, scale, out, return_lse)
PyObject* py_attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* q = n == 9 ? heads_of(a[0], -1) : nullptr;
  if (q == nullptr) Py_RETURN_NONE;
  const int dev = q->get_device();
  const at::Tensor *k = heads_of(a[1], dev), *v = heads_of(a[2], dev), *cu_q = tensor_of(a[3]),
                   *cu_k = a[4] == Py_None ? cu_q : tensor_of(a[4]);
  if (k == nullptr || v == nullptr || k->sizes() != v->sizes() || !offsets_of(cu_q, dev) || !offsets_of(cu_k, dev) ||
      cu_q->numel() != cu_k->numel())
    Py_RETURN_NONE;
  const int64_t h = q->size(1), d = q->size(2), hk = k->size(1);
  if (d < 1 || d > 256 || h < 1 || hk < 1 || h % hk != 0 || k->size(2) != d || h > 65536) Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt((double)d);
  if (a[6] != Py_None) {
    scale = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) PyErr_Clear();
    if (!(scale > 0.0 && (float)scale > 0.f && std::isfinite((float)scale))) Py_RETURN_NONE;
  }
  Target at_(dev);
  at::Tensor out;
  if (a[7] == Py_None) {
    out = new_tensor({q->size(0), h, d}, at::kBFloat16, dev);
  } else {
    const at::Tensor* o = heads_of(a[7], dev);
    if (o == nullptr || o->sizes() != q->sizes() || !writable(*o) || overlap(*o, *q) || overlap(*o, *k) || overlap(*o, *v)) Py_RETURN_NONE;
    out = *o;
  }
  const bool want_lse = a[8] == Py_True;
  at::Tensor lse, ws;
  if (want_lse) lse = new_tensor({q->size(0), h}, at::kFloat, dev);
  sacq_attention_desc c = {};
  c.struct_size = sizeof(c);
  c.causal = a[5] == Py_True;
  c.q = q->data_ptr();
  c.k = k->data_ptr();
  c.v = v->data_ptr();
  c.out = out.data_ptr();
  c.lse = want_lse ? (float*)lse.data_ptr() : nullptr;
  c.q_token = q->stride(0); c.q_head = q->stride(1);
  c.k_token = k->stride(0); c.k_head = k->stride(1);
  c.v_token = v->stride(0); c.v_head = v->stride(1);
  c.out_token = out.stride(0); c.out_head = out.stride(1);
  c.tokens_q = q->size(0); c.tokens_k = k->size(0);
  c.cu_q = (const int32_t*)cu_q->data_ptr();
  c.cu_k = (const int32_t*)cu_k->data_ptr();
  c.sequences = (int32_t)(cu_q->numel() - 1);
  c.heads = (int32_t)h;
  c.kv_heads = (int32_t)hk;
  c.head_dim = (int32_t)d;
  c.scale = (float)scale;
  // partial results belong to the call: a captured graph keeps its own
  c.workspace_bytes = sacq_attention_workspace_bytes(&c);
  if (c.workspace_bytes < 0) return raise_status((int)c.workspace_bytes);
  if (c.workspace_bytes > 0) {
    ws = new_tensor({c.workspace_bytes}, at::kByte, dev);
    c.workspace = ws.data_ptr();
  }
  const int rc = sacq_attention_packed(&c, at_.stream);
  if (rc != 0) return raise_status(rc);
  if (want_lse) return pair_of(std::move(out), std::move(lse));
  return THPVariable_Wrap(std::move(out));
  NATIVE_CATCH
}

// other: the call's other input, null if there is none.  In place means the same places, so `other` is still looked at
bool fill_heads(const at::Tensor* x, const at::Tensor* other, PyObject* out_obj, int dev, sacq_head_rows& r, at::Tensor& out) {
  if (out_obj == Py_None) {
    out = new_tensor(x->sizes(), at::kBFloat16, dev);
  } else {
    const at::Tensor* o = heads_of(out_obj, dev);
    if (o == nullptr || o->sizes() != x->sizes() || !writable(*o)) return false;
    const bool same = o->data_ptr() == x->data_ptr() && o->strides() == x->strides();
    if ((!same && overlap(*o, *x)) || (other != nullptr && overlap(*o, *other))) return false;
    out = *o;
  }
  r.in = x->data_ptr();
  r.out = out.data_ptr();
  r.in_token = x->stride(0); r.in_head = x->stride(1);
  r.out_token = out.stride(0); r.out_head = out.stride(1);
  r.heads = (int32_t)x->size(1);
  return true;
}

// rotate_heads(q, k, positions, inv_freq, layout, amplitude, q_out, k_out)
PyObject* py_rotate_heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor* q = n == 8 ? heads_of(a[0], -1) : nullptr;
  if (q == nullptr) Py_RETURN_NONE;
  const int dev = q->get_device();
  const at::Tensor *k = nullptr, *pos = tensor_of(a[2]), *freq = tensor_of(a[3]);
  if (a[1] != Py_None) {
    k = heads_of(a[1], dev);
    if (k == nullptr || k->size(0) != q->size(0) || k->size(2) != q->size(2)) Py_RETURN_NONE;
  } else if (a[7] != Py_None) {
    Py_RETURN_NONE;
  }
  if (pos == nullptr || freq == nullptr || !on_device(*pos, dev) || !on_device(*freq, dev) || pos->dim() != 1 || freq->dim() != 1 ||
      !pos->is_contiguous() || !freq->is_contiguous() || pos->numel() != q->size(0) ||
      (pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong) || freq->scalar_type() != at::kDouble ||
      freq->numel() < 1 || 2 * freq->numel() > q->size(2))
    Py_RETURN_NONE;
  Target at_(dev);
  sacq_rotary_desc c = {};
  c.struct_size = sizeof(c);
  at::Tensor q_out, k_out;
  if (!fill_heads(q, k, a[6], dev, c.q, q_out) || (k != nullptr && !fill_heads(k, q, a[7], dev, c.k, k_out))) Py_RETURN_NONE;
  if (k != nullptr && a[6] != Py_None && a[7] != Py_None && overlap(q_out, k_out)) Py_RETURN_NONE;
  c.layout = (int32_t)PyLong_AsLong(a[4]);
  c.tokens = q->size(0);
  c.head_dim = (int32_t)q->size(2);
  c.rotary_dim = (int32_t)(2 * freq->numel());
  c.positions = pos->data_ptr();
  c.position_bytes = pos->scalar_type() == at::kLong ? 8 : 4;
  c.amplitude = (float)PyFloat_AsDouble(a[5]);
  c.inv_freq = (const double*)freq->data_ptr();
  if (PyErr_Occurred()) return nullptr;
  const int rc = sacq_rotate_heads(&c, at_.stream);
  return rc == 0 ? tuple_of({q_out, k_out}) : raise_status(rc);
  NATIVE_CATCH
}

// residual_norm_quantize_rows(branch, residual, weight, bias, post_weight, post_bias, gate, mod_scale, mod_shift, vector_rows, norm,
// post_norm, eps, residual_scale, quantize, return_normalized)
PyObject* py_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  const at::Tensor *x = n == 16 ? quantizer_input(a[0]) : nullptr, *res = n == 16 ? tensor_of(a[1]) : nullptr;
  if (x == nullptr || res == nullptr || res->dim() != 2 || res->sizes() != x->sizes()) Py_RETURN_NONE;
  const int dev = x->get_device();
  const int64_t m = x->size(0), k = x->size(1);
  if (!bf16_rows(*res, dev) || wants_grad(*x) || wants_grad(*res)) Py_RETURN_NONE;
  if ((m > 1 && (x->stride(0) < k || res->stride(0) < k))) Py_RETURN_NONE;
  sacq_residual_norm_desc c = {};
  c.struct_size = sizeof(c);
  const void** vec[4] = {&c.weight, &c.bias, &c.post_weight, &c.post_bias};
  for (int i = 0; i < 4; ++i) {
    if (!vector_or_none(a[2 + i], k, dev, vec[i])) Py_RETURN_NONE;
    if (a[2 + i] != Py_None && wants_grad(*tensor_of(a[2 + i]))) Py_RETURN_NONE;
  }
  const at::Tensor* rows = a[9] == Py_None ? nullptr : tensor_of(a[9]);
  if (a[9] != Py_None && (rows == nullptr || rows->scalar_type() != at::kInt || !on_device(*rows, dev) || rows->numel() != m ||
                          !rows->is_contiguous()))
    Py_RETURN_NONE;
  const void** table[3] = {&c.gate, &c.mod_scale, &c.mod_shift};
  for (int i = 0; i < 3; ++i) {
    const at::Tensor* t = a[6 + i] == Py_None ? nullptr : tensor_of(a[6 + i]);
    if (a[6 + i] == Py_None) continue;
    if (t == nullptr || t->scalar_type() != at::kBFloat16 || !on_device(*t, dev) || !t->is_contiguous() || wants_grad(*t)) Py_RETURN_NONE;
    if (rows == nullptr ? t->numel() != k : (t->dim() != 2 || t->size(1) != k || t->size(0) < 1)) Py_RETURN_NONE;
    if (rows != nullptr && c.vectors != 0 && c.vectors != t->size(0)) Py_RETURN_NONE;
    if (rows != nullptr) c.vectors = t->size(0);
    *table[i] = t->data_ptr();
  }
  if (rows != nullptr && c.vectors == 0) Py_RETURN_NONE;
  c.norm = (int32_t)PyLong_AsLong(a[10]);
  c.post_norm = (int32_t)PyLong_AsLong(a[11]);
  c.eps = (float)PyFloat_AsDouble(a[12]);
  c.residual_scale = (float)PyFloat_AsDouble(a[13]);
  if (PyErr_Occurred()) return nullptr;
  if (!(c.eps >= 0.f) || (c.mod_scale == nullptr) != (c.mod_shift == nullptr) ||
      (c.post_norm == SACQ_NORM_NONE && (c.post_weight || c.post_bias)))
    Py_RETURN_NONE;
  const bool quantize = a[14] == Py_True, want_h = !quantize || a[15] == Py_True;
  Target at_(dev);
  at::Tensor r = new_tensor({m, k}, at::kBFloat16, dev), h, q, s;
  if (want_h) h = new_tensor({m, k}, at::kBFloat16, dev);
  if (quantize) {
    Encoded e(m, k, false, dev);
    q = std::move(e.q);
    s = std::move(e.s);
    c.q_out = q.data_ptr();
    c.scale_out = (float*)s.data_ptr();
  }
  c.M = m;
  c.K = k;
  c.branch = x->data_ptr();
  c.residual = res->data_ptr();
  c.branch_pitch = m > 1 ? x->stride(0) : k;
  c.residual_pitch = m > 1 ? res->stride(0) : k;
  c.vector_rows = rows ? (const int32_t*)rows->data_ptr() : nullptr;
  c.residual_out = r.data_ptr();
  c.normalized_out = want_h ? h.data_ptr() : nullptr;
  const int rc = sacq_residual_norm(&c, at_.stream);
  if (rc != 0) return raise_status(rc);
  return !quantize ? tuple_of({r, h}) : want_h ? tuple_of({r, q, s, h}) : tuple_of({r, q, s});
  NATIVE_CATCH
}

// ---------------------------------------------------------------- several layers on one input
constexpr int kMostSiblings = 16;

struct Siblings {
  LayerObject* L[kMostSiblings];
  int n = 0;
};

// A list of modules that carry a Layer as `_native`, all of one device and input width
bool siblings_of(PyObject* list, Siblings& out) {
  static PyObject* name = PyUnicode_InternFromString("_native");
  if (!PyList_Check(list)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  if (n < 1 || n > kMostSiblings) return false;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyObject_GetAttr(PyList_GET_ITEM(list, i), name);
    if (o == nullptr) {
      PyErr_Clear();
      return false;
    }
    const bool ok = Py_TYPE(o) == &LayerType;
    Py_DECREF(o);                                     // the module keeps it
    if (!ok) return false;
    out.L[i] = (LayerObject*)o;
    if (out.L[i]->k != out.L[0]->k || out.L[i]->dev != out.L[0]->dev || out.L[i]->n <= 0) return false;
  }
  out.n = (int)n;
  return true;
}

PyObject* run_siblings(const Siblings& sb, const void* q, const float* s, int64_t m, const at::Tensor* like,
                       const Target& at_) {
  int64_t need = 0;
  const sacq_layer_t* handles[kMostSiblings];
  void* ys[kMostSiblings];
  int64_t ldys[kMostSiblings];
  at::Tensor outs[kMostSiblings];
  for (int i = 0; i < sb.n; ++i) {
    LayerObject* L = sb.L[i];
    need = std::max(need, need_bytes(L, m, kNeedA8));
    handles[i] = L->handle;
    outs[i] = like ? result_like(*like, m, L->n, L->dev) : new_tensor({m, L->n}, at::kBFloat16, L->dev);
    ys[i] = outs[i].data_ptr();
    ldys[i] = L->n;
  }
  at::Tensor& ws = scratch(workspace(at_.dev, at_.stream), need, at_.dev);
  const int rc = sacq_linear_a8_multi(handles, sb.n, q, s, m, ys, ldys, ws.data_ptr(), ws.numel(), at_.stream);
  if (rc != 0) return raise_status(rc);
  PyObject* list = PyList_New(sb.n);
  for (int i = 0; i < sb.n && list != nullptr; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(outs[i]));
    if (o == nullptr) {
      Py_DECREF(list);
      return nullptr;
    }
    PyList_SET_ITEM(list, i, o);
  }
  return list;
}

// linear_a8_multi(layers, q, scale)
PyObject* py_linear_a8_multi(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  Siblings sb;
  const at::Tensor *q = n == 3 ? tensor_of(a[1]) : nullptr, *s = n == 3 ? tensor_of(a[2]) : nullptr;
  if (q == nullptr || s == nullptr || !siblings_of(a[0], sb) || !byte_matrix(*q, sb.L[0]->k, sb.L[0]->dev) ||
      q->size(0) == 0 || !f32_vector(*s, q->size(0), sb.L[0]->dev))
    Py_RETURN_NONE;
  Target at_(sb.L[0]->dev);
  return run_siblings(sb, q->data_ptr(), (const float*)s->data_ptr(), q->size(0), nullptr, at_);
  NATIVE_CATCH
}

// forward_shared(layers, x)
PyObject* py_forward_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NATIVE_TRY
  Siblings sb;
  Rows r;
  const at::Tensor* x = n == 2 ? tensor_of(a[1]) : nullptr;
  if (x == nullptr || !siblings_of(a[0], sb) || !rows_of(*x, sb.L[0]->k, sb.L[0]->dev, r)) Py_RETURN_NONE;
  Target at_(sb.L[0]->dev);
  Workspace& w = workspace(at_.dev, at_.stream);
  act_buffers(w, r.m, sb.L[0]->k, at_.dev);
  const int rc = sacq_quant_act_fp8(r.ptr, r.pitch, r.m, sb.L[0]->k, w.q.data_ptr(), (float*)w.scale.data_ptr(), at_.stream);
  if (rc != 0) return raise_status(rc);
  return run_siblings(sb, w.q.data_ptr(), (const float*)w.scale.data_ptr(), r.m, x, at_);
  NATIVE_CATCH
}

// ---------------------------------------------------------------- the pool, for the general route
// workspace(device, bytes): the current stream's kernel scratch, grown to `bytes`
PyObject* py_workspace(PyObject*, PyObject* args) {
  NATIVE_TRY
  int dev = 0;
  long long bytes = 0;
  if (!PyArg_ParseTuple(args, "iL", &dev, &bytes)) return nullptr;
  Target at_(dev);
  return THPVariable_Wrap(scratch(workspace(dev, at_.stream), bytes, dev));
  NATIVE_CATCH
}

// host_scratch(device, bytes): device scratch of the current stream's host-buffer forwards
PyObject* py_host_scratch(PyObject*, PyObject* args) {
  NATIVE_TRY
  int dev = 0;
  long long bytes = 0;
  if (!PyArg_ParseTuple(args, "iL", &dev, &bytes)) return nullptr;
  Target at_(dev);
  Workspace& w = workspace(dev, at_.stream);
  if (!w.host_scratch.defined() || w.host_scratch.numel() < bytes)
    w.host_scratch = zeroed(bytes > (1 << 22) ? bytes : (1 << 22), dev);
  return THPVariable_Wrap(w.host_scratch);
  NATIVE_CATCH
}

PyObject* py_set_error_class(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error_class, cls);
  Py_RETURN_NONE;
}

PyMethodDef module_methods[] = {
    {"quantize_rows", (PyCFunction)(void*)py_quantize_rows, METH_FASTCALL, nullptr},
    {"act_quantize_rows", (PyCFunction)(void*)py_act_quantize_rows, METH_FASTCALL, nullptr},
    {"modulate_quantize_rows", (PyCFunction)(void*)py_modulate_quantize_rows, METH_FASTCALL, nullptr},
    {"layernorm_quantize_rows", (PyCFunction)(void*)py_layernorm_quantize_rows, METH_FASTCALL, nullptr},
    {"attention_packed", (PyCFunction)(void*)py_attention_packed, METH_FASTCALL, nullptr},
    {"rotate_heads", (PyCFunction)(void*)py_rotate_heads, METH_FASTCALL, nullptr},
    {"residual_norm_quantize_rows", (PyCFunction)(void*)py_residual_norm, METH_FASTCALL, nullptr},
    {"overlaps", (PyCFunction)(void*)py_overlaps, METH_FASTCALL, nullptr},
    {"linear_a8_multi", (PyCFunction)(void*)py_linear_a8_multi, METH_FASTCALL, nullptr},
    {"forward_shared", (PyCFunction)(void*)py_forward_shared, METH_FASTCALL, nullptr},
    {"workspace", py_workspace, METH_VARARGS, nullptr},
    {"host_scratch", py_host_scratch, METH_VARARGS, nullptr},
    {"set_error_class", py_set_error_class, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, module_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
  LayerType.tp_name = "sacq_b200._native.Layer";
  LayerType.tp_basicsize = sizeof(LayerObject);
  LayerType.tp_flags = Py_TPFLAGS_DEFAULT;
  LayerType.tp_new = layer_new;
  LayerType.tp_dealloc = (destructor)layer_dealloc;
  LayerType.tp_methods = layer_methods;
  if (PyType_Ready(&LayerType) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (m == nullptr) return nullptr;
  Py_INCREF(&LayerType);
  if (PyModule_AddObject(m, "Layer", (PyObject*)&LayerType) < 0) {
    Py_DECREF(&LayerType);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
