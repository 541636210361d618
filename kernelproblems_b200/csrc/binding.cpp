// binding.cpp — a compiled way into libfrag.so for the calls whose time is the
// host's: small rows, and lists of hundreds of tensors.
//
// Each function takes the arguments of an operator of ops.py and does what its
// Python does for the ordinary call: plain tensors on the current device,
// contiguous, of the types that belong together, no workspace of the caller's.  For
// that call it checks the arguments, makes the outputs and calls the C ABI on the
// current stream.  For any other it returns None, having done nothing, and the
// Python path goes on from there, with the same kernels and with the errors of the
// refusals.  An int is the C ABI's status.  130 gradients of 4096: the checks and
// pointers that take Python's maps 65 us take 2 here; a layer norm of eight
// rows with four outputs 19 us through ctypes.
//
// libfrag.so's entry points are given as addresses at load (bind), so this file
// needs no linking with it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "frag.h"

namespace {

struct Entries {
  decltype(&frag_layernorm_fwd) layernorm_fwd;
  decltype(&frag_layernorm_bwd) layernorm_bwd;
  decltype(&frag_layernorm_bwd_workspace_bytes) layernorm_bwd_workspace;
  decltype(&frag_grad_norm) grad_norm;
  decltype(&frag_grad_norm_workspace_bytes) grad_norm_workspace;
  decltype(&frag_adamw_update) adamw;
} entries;

// A plain torch.Tensor (or Parameter) on the current device, contiguous, holding
// its values as they are (and holding them: what a function transform wraps does not).
const at::Tensor* plain(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.has_storage() || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != device ||
      !t.is_contiguous() || t.is_neg() || t.is_conj())
    return nullptr;
  return &t;
}
// The current device, where `o` is a tensor on it; otherwise -1 (and CUDA is not
// touched for a CPU tensor).
int device_of(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return -1;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.has_storage() || !t.is_cuda() || t.get_device() != c10::cuda::current_device()) return -1;
  return t.get_device();
}
int code(const at::Tensor& t) {
  const auto d = t.scalar_type();
  return d == at::kBFloat16 ? FRAG_DT_BF16 : d == at::kFloat ? FRAG_DT_F32 : -1;
}
bool absent(PyObject* o) { return o == Py_None; }

at::Tensor like(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
  return at::detail::empty_cuda(shape, type, t.device(), std::nullopt);
}
PyObject* wrapped(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <class... Ts>
PyObject* tuple(const Ts&... ts) {
  PyObject* out = PyTuple_New(sizeof...(ts));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  bool ok = true;
  auto put = [&](const at::Tensor& t) {
    PyObject* o = ok ? wrapped(t) : nullptr;
    ok = o != nullptr;
    PyTuple_SET_ITEM(out, i++, o);
  };
  (put(ts), ...);
  if (!ok) {
    Py_DECREF(out);
    return nullptr;
  }
  return out;
}
// (Pointers are asked for ahead of a call without the interpreter's lock: an exception
// may not leave that.)
void* data(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* given(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
frag_stream_t stream_of(int device) {
  return reinterpret_cast<frag_stream_t>(c10::cuda::getCurrentCUDAStream(device).stream());
}

// Weight or bias: `t` stays undefined where there is none.
bool vector(PyObject* o, int device, int64_t N, int* type, at::Tensor& t) {
  if (absent(o)) return true;
  const at::Tensor* v = plain(o, device);
  if (!v || v->numel() != N || code(*v) < 0 || (*type >= 0 && code(*v) != *type)) return false;
  *type = code(*v);
  t = *v;
  return true;
}

// (x, weight, bias, eps, residual, write_h, save_stats)
PyObject* layernorm_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const int device = device_of(a[0]);
  const at::Tensor* x = device < 0 ? nullptr : plain(a[0], device);
  if (!x || x->dim() < 1 || x->numel() == 0 || code(*x) < 0) Py_RETURN_NONE;
  const int64_t N = x->size(-1), M = x->numel() / N;
  int type = -1;
  at::Tensor w, b, h, mean, rstd;
  if (!vector(a[1], device, N, &type, w) || !vector(a[2], device, N, &type, b)) Py_RETURN_NONE;
  const double eps = PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* res = nullptr;
  if (!absent(a[4])) {
    res = plain(a[4], device);
    if (!res || res->scalar_type() != x->scalar_type() || res->sizes() != x->sizes()) Py_RETURN_NONE;
  }
  const int write_h = PyObject_IsTrue(a[5]), stats = PyObject_IsTrue(a[6]);
  if (write_h < 0 || stats < 0) return nullptr;
  const at::Tensor y = like(*x, x->sizes(), x->scalar_type());
  if (res && write_h) h = like(*x, x->sizes(), x->scalar_type());
  if (stats) {
    const auto rows = x->sizes().slice(0, x->dim() - 1);
    mean = like(*x, rows, at::kFloat);
    rstd = like(*x, rows, at::kFloat);
  }
  const void *xp = x->const_data_ptr(), *rp = res ? res->const_data_ptr() : nullptr, *wp = given(w), *bp = given(b);
  void *yp = data(y), *hp = data(h);
  float *mp = static_cast<float*>(data(mean)), *sp = static_cast<float*>(data(rstd));
  const int dtype = code(*x);
  const frag_stream_t stream = stream_of(device);
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = entries.layernorm_fwd(xp, N, rp, N, wp, bp, yp, hp, mp, sp, M, N, static_cast<float>(eps), dtype,
                             type < 0 ? FRAG_DT_F32 : type, stream);
  Py_END_ALLOW_THREADS
  return st ? PyLong_FromLong(st) : tuple(y, h, mean, rstd);
  END_HANDLE_TH_ERRORS
}

// (dy, x, mean, rstd, weight, dres, compute_dw, compute_db)
PyObject* layernorm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const int device = device_of(a[1]);
  if (device < 0) Py_RETURN_NONE;
  const at::Tensor *dy = plain(a[0], device), *x = plain(a[1], device), *mean = plain(a[2], device),
                   *rstd = plain(a[3], device);
  if (!dy || !x || !mean || !rstd || x->dim() < 1 || x->numel() == 0 || code(*x) < 0) Py_RETURN_NONE;
  const int64_t N = x->size(-1), M = x->numel() / N;
  if (dy->scalar_type() != x->scalar_type() || dy->sizes() != x->sizes() || mean->scalar_type() != at::kFloat ||
      rstd->scalar_type() != at::kFloat || mean->numel() != M || rstd->numel() != M)
    Py_RETURN_NONE;
  int type = -1;
  at::Tensor w, dw, db, ws;
  if (!vector(a[4], device, N, &type, w)) Py_RETURN_NONE;
  const at::Tensor* dres = nullptr;
  if (!absent(a[5])) {
    dres = plain(a[5], device);
    if (!dres || dres->scalar_type() != x->scalar_type() || dres->sizes() != x->sizes()) Py_RETURN_NONE;
  }
  const int want_dw = PyObject_IsTrue(a[6]), want_db = PyObject_IsTrue(a[7]);
  if (want_dw < 0 || want_db < 0) return nullptr;
  const at::Tensor dx = like(*x, x->sizes(), x->scalar_type());
  if (want_dw && w.defined()) dw = like(*x, {N}, at::kFloat);
  if (want_db) db = like(*x, {N}, at::kFloat);
  size_t bytes = 0;
  if (dw.defined() || db.defined()) {
    bytes = entries.layernorm_bwd_workspace(M, N);
    ws = like(*x, {static_cast<int64_t>(bytes)}, at::kByte);
  }
  const void *yp = dy->const_data_ptr(), *xp = x->const_data_ptr(), *wp = given(w),
             *rp = dres ? dres->const_data_ptr() : nullptr;
  const float *mp = static_cast<const float*>(mean->const_data_ptr()),
              *sp = static_cast<const float*>(rstd->const_data_ptr());
  void *dxp = data(dx), *wsp = data(ws);
  float *dwp = static_cast<float*>(data(dw)), *dbp = static_cast<float*>(data(db));
  const int dtype = code(*x);
  const frag_stream_t stream = stream_of(device);
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = entries.layernorm_bwd(yp, N, xp, N, mp, sp, wp, rp, N, dxp, dwp, dbp, M, N, dtype, type < 0 ? FRAG_DT_F32 : type,
                             wsp, bytes, stream);
  Py_END_ALLOW_THREADS
  return st ? PyLong_FromLong(st) : tuple(dx, dw, db);
  END_HANDLE_TH_ERRORS
}

// A list's or tuple's items; null for anything else.
PyObject** items(PyObject* o, Py_ssize_t* n) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return nullptr;
  *n = PySequence_Fast_GET_SIZE(o);
  return PySequence_Fast_ITEMS(o);
}

// (grads, max_norm or None)
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) Py_RETURN_NONE;
  Py_ssize_t count = 0;
  PyObject** grads = items(a[0], &count);
  if (!grads) Py_RETURN_NONE;
  double top = 1.0;
  if (!absent(a[1])) {
    top = PyFloat_AsDouble(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (!(top > 0) || !std::isfinite(static_cast<float>(top)) || static_cast<float>(top) <= 0.f) Py_RETURN_NONE;
  }
  Py_ssize_t first = 0;
  while (first < count && absent(grads[first])) ++first;
  const int device = first < count ? device_of(grads[first]) : -1;
  if (device < 0) Py_RETURN_NONE;
  std::vector<const void*> ptrs;
  std::vector<int64_t> numel;
  std::vector<int32_t> codes;
  ptrs.reserve(count);
  numel.reserve(count);
  codes.reserve(count);
  const at::Tensor* one = nullptr;
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (absent(grads[i])) continue;
    const at::Tensor* g = plain(grads[i], device);
    if (!g || code(*g) < 0) Py_RETURN_NONE;
    one = g;
    ptrs.push_back(g->const_data_ptr());
    numel.push_back(g->numel());
    codes.push_back(code(*g));
  }
  if (!one) Py_RETURN_NONE;
  const at::Tensor norm = like(*one, {}, at::kFloat);
  at::Tensor scale;
  if (!absent(a[1])) scale = like(*one, {}, at::kFloat);
  const int64_t bytes = static_cast<int64_t>(entries.grad_norm_workspace(ptrs.size()));
  const at::Tensor ws = like(norm, {bytes}, at::kByte);
  float *np = static_cast<float*>(data(norm)), *sp = static_cast<float*>(data(scale));
  void* wsp = data(ws);
  const frag_stream_t stream = stream_of(device);
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = entries.grad_norm(ptrs.data(), numel.data(), codes.data(), ptrs.size(), static_cast<float>(top), np, sp, wsp,
                         bytes, stream);
  Py_END_ALLOW_THREADS
  return st ? PyLong_FromLong(st) : tuple(norm, scale);
  END_HANDLE_TH_ERRORS
}

// One value on the device: 1 there, 0 none given, -1 something else.
int word(PyObject* o, int device, at::ScalarType type, const void** p) {
  *p = nullptr;
  if (absent(o)) return 0;
  const at::Tensor* t = plain(o, device);
  if (!t || t->scalar_type() != type || t->numel() != 1) return -1;
  *p = t->const_data_ptr();
  return 1;
}

// (written, places, kinds, numel, grads, table, m, v, m_scale, v_scale, total, lr,
//  lr_device, beta1, beta2, eps, step, step_device, grad_scale)
// written: the parameters and, behind them, their copies, as the table was made for
// them; places, kinds, numel: addresses of uint64, int32 and int64 arrays of what
// each was then.
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 19) Py_RETURN_NONE;
  Py_ssize_t total_written = 0, count = 0;
  PyObject **written = items(a[0], &total_written), **grads = items(a[4], &count);
  if (!written || !grads || count > total_written) Py_RETURN_NONE;
  const auto* places = static_cast<const uint64_t*>(PyLong_AsVoidPtr(a[1]));
  const auto* kinds = static_cast<const int32_t*>(PyLong_AsVoidPtr(a[2]));
  const auto* numel = static_cast<const int64_t*>(PyLong_AsVoidPtr(a[3]));
  const auto* table = static_cast<const frag_adamw_tensor*>(PyLong_AsVoidPtr(a[5]));
  const int64_t total = PyLong_AsLongLong(a[10]), step = PyLong_AsLongLong(a[16]);
  const double lr = PyFloat_AsDouble(a[11]), b1 = PyFloat_AsDouble(a[13]), b2 = PyFloat_AsDouble(a[14]),
               eps = PyFloat_AsDouble(a[15]);
  if (PyErr_Occurred()) return nullptr;
  const int device = total_written ? device_of(written[0]) : -1;
  if (device < 0) Py_RETURN_NONE;
  std::vector<const void*> ptrs(count);
  std::vector<int32_t> codes(count);
  for (Py_ssize_t i = 0; i < total_written; ++i) {
    const at::Tensor* p = plain(written[i], device);
    if (!p || reinterpret_cast<uint64_t>(p->mutable_data_ptr()) != places[i] || p->numel() != numel[i] ||
        code(*p) != kinds[i])
      Py_RETURN_NONE;
    if (i >= count || absent(grads[i])) continue;
    const at::Tensor* g = plain(grads[i], device);
    if (!g || code(*g) < 0 || g->sizes() != p->sizes()) Py_RETURN_NONE;
    ptrs[i] = g->const_data_ptr();
    codes[i] = code(*g);
  }
  void* held[4];
  for (int i = 0; i < 4; ++i) {
    held[i] = nullptr;
    if (i >= 2 && absent(a[6 + i])) continue;
    const at::Tensor* t = plain(a[6 + i], device);
    const auto type = i < 2 && !absent(a[8]) ? at::kFloat8_e4m3fn : at::kFloat;
    if (!t || t->scalar_type() != type || t->numel() != (i < 2 ? total : total / 128)) Py_RETURN_NONE;
    held[i] = t->mutable_data_ptr();
  }
  const void *lr_p, *step_p, *scale_p;
  if (word(a[12], device, at::kFloat, &lr_p) < 0 || word(a[17], device, at::kLong, &step_p) < 0 ||
      word(a[18], device, at::kFloat, &scale_p) < 0)
    Py_RETURN_NONE;
  const frag_stream_t stream = stream_of(device);
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = entries.adamw(table, ptrs.data(), codes.data(), count, held[0], held[1], static_cast<float*>(held[2]),
                     static_cast<float*>(held[3]), lr, static_cast<const float*>(lr_p), b1, b2, eps, step,
                     static_cast<const int64_t*>(step_p), static_cast<const float*>(scale_p), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
  END_HANDLE_TH_ERRORS
}

// The addresses of Entries' members, in their order.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[6];
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
    return nullptr;
  }
  for (int i = 0; i < 6; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  entries = {reinterpret_cast<decltype(entries.layernorm_fwd)>(p[0]),
             reinterpret_cast<decltype(entries.layernorm_bwd)>(p[1]),
             reinterpret_cast<decltype(entries.layernorm_bwd_workspace)>(p[2]),
             reinterpret_cast<decltype(entries.grad_norm)>(p[3]),
             reinterpret_cast<decltype(entries.grad_norm_workspace)>(p[4]),
             reinterpret_cast<decltype(entries.adamw)>(p[5])};
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}

PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, nullptr},
    {"layernorm_fwd", fast(layernorm_fwd), METH_FASTCALL, nullptr},
    {"layernorm_bwd", fast(layernorm_bwd), METH_FASTCALL, nullptr},
    {"grad_norm", fast(grad_norm), METH_FASTCALL, nullptr},
    {"adamw", fast(adamw), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__binding() { return PyModule_Create(&module_def); }
