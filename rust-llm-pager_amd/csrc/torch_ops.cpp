// Call path of the operator API for plain tensors: the Python functions of
// pager_hf/streaming_attention.py, pager_hf/rotary.py and pager_hf/heavy_hitter_cache.py hand their
// arguments to these before anything else.
//
// Each function checks that its arguments are what the kernels take as they are (exact
// torch.Tensor objects without functorch, functionalization or lazy-bit keys, one GPU, one
// dtype, contiguous (rotary and cache operands: head_dim contiguous), matching shapes), allocates the
// workspace or outputs from torch's current allocator, and calls the C entry point of libpgr.so. It
// returns the entry point's status, or None where any check fails: the caller then runs its general
// Python path, which converts, copies or refuses as it always has. So this file decides nothing but speed: checks in Python,
// one attribute object at a time, and a ctypes call of 19 arguments held the GPU up. A call of one
// query (init, fold, finalize; 28/4 heads, D 128, fp16, 64 tokens) 30.6 -> 16.8 us, 4133 tokens
// the same; the two-pass run of 12 calls (32/4, D 64, batch 4, 8209 tokens) 151 -> 84.6 us.
// q and k of one token turned (14/2 heads, D 64) 17.9 -> 8.0 us, an append to a full cache of 256 tokens 13.4
// -> 7.3 us, attention over 256 tokens (28/4, D 128) 10.8 -> 7.1 us.
//
// libpgr.so's entry points come as addresses (bind), so that the library the Python package has
// loaded is the one called.
#include <Python.h>

#include "../../include/pgr.h"

#include <ATen/ATen.h>
#include <ATen/detail/CUDAHooksInterface.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <exception>

namespace {

using Tensor = at::Tensor;

size_t (*g_workspace_bytes)(int64_t, int64_t, int64_t, int64_t, int64_t, int, int64_t);
int (*g_step)(const void*, const void*, const void*, const int32_t*, const int32_t*, float*, float*, float*, int64_t,
              int64_t, int64_t, int64_t, int64_t, int, float, float, void*, size_t, void*);
int (*g_stats)(const void*, const void*, const int32_t*, const int32_t*, float*, float*, int64_t, int64_t, int64_t,
               int64_t, int64_t, int, float, float, void*, size_t, void*);
int (*g_accumulate)(const void*, const void*, const void*, const int32_t*, const int32_t*, const float*, const float*,
                    float*, float*, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int, float,
                    float, void*, size_t, void*);
int (*g_fold_fixed)(const void*, const void*, const void*, const int32_t*, const float*, const float*, float*, int64_t,
                    int64_t, int64_t, int64_t, int64_t, int, float, float, void*, size_t, void*);
int (*g_state_init)(float*, float*, float*, int64_t, int64_t, void*);
int (*g_finalize)(const float*, const float*, void*, int64_t, int64_t, int, void*);
decltype(&pgr_rotary) g_rotary;
decltype(&pgr_hh_append) g_append;
decltype(&pgr_hh_attend) g_attend;
decltype(&pgr_hh_prompt_weights) g_prompt_weights;
decltype(&pgr_hh_prompt_weights_workspace_bytes) g_prompt_weights_bytes;
decltype(&pgr_hh_load_prompt) g_load_prompt;
decltype(&pgr_hh_load_prompt_workspace_bytes) g_load_prompt_bytes;
PyObject* g_raw_stream;     // torch._C._cuda_getCurrentRawStream
PyObject* g_out_of_memory;  // torch.OutOfMemoryError

enum Mode : int { kFold = 0, kStats = 1, kAccumulate = 2, kFoldFixed = 3 };  // PGR_MODE_* (pgr.h)

// The dispatch keys of an ordinary GPU tensor. A tensor with any other key (functorch wrappers,
// functionalization, Python subclasses, the negative bit) takes the general path.
bool plain_keys(const Tensor& t) {
  static const c10::DispatchKeySet allowed =
      c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView}) |
      c10::getAutogradRelatedKeySetFromBackend(c10::BackendComponent::CUDABit) |
      c10::getAutocastRelatedKeySetFromBackend(c10::BackendComponent::CUDABit);
  return (t.key_set().raw_repr() & ~allowed.raw_repr()) == 0;  // (operator- would keep backend bits)
}

const Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && plain_keys(t) && t.has_storage() && t.is_contiguous() ? &t : nullptr;
}

bool is_f32(const Tensor* t, const c10::Device& dev, at::IntArrayRef shape) {
  return t && t->scalar_type() == at::kFloat && t->device() == dev && t->sizes() == shape;
}

// An optional 0/1 mask: *out is its data or null. False: not in the form the kernels read.
bool mask(PyObject* o, const c10::Device& dev, at::IntArrayRef shape, const int32_t** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const Tensor* t = plain(o);
  if (!t || t->scalar_type() != at::kInt || t->device() != dev || t->sizes() != shape) return false;
  *out = t->const_data_ptr<int32_t>();
  return true;
}

// None or an exact Python float.
bool number(PyObject* o, double none_value, double* out) {
  if (o == Py_None) {
    *out = none_value;
    return true;
  }
  if (PyFloat_CheckExact(o)) {
    *out = PyFloat_AS_DOUBLE(o);
    return true;
  }
  return false;
}

bool integer(PyObject* o, int64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool current_stream(const c10::Device& dev, void** out) {
  PyObject* idx = PyLong_FromLong(dev.index());
  if (!idx) return false;
  PyObject* s = PyObject_CallFunctionObjArgs(g_raw_stream, idx, nullptr);
  Py_DECREF(idx);
  if (!s) return false;
  *out = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return !PyErr_Occurred();
}

// Everything a launch needs, resolved while the GIL is held.
struct Call {
  const void *q, *k, *v = nullptr;
  float *m, *l, *acc = nullptr;
  const int32_t *valid = nullptr, *active = nullptr;
  int64_t b, hq, hkv, tc, d;
  int code;
  float scale, softcap;
  void* stream;
  c10::Device dev{c10::DeviceType::CUDA};
};

int dtype_code(at::ScalarType t) {
  return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1;  // PGR_DTYPE_*
}

float* f32(const Tensor* t) { return static_cast<float*>(t->mutable_data_ptr()); }

// The operands that every mode takes; v and acc are null for the statistics pass.
bool prepare(Call& c, PyObject* q_, PyObject* k_, PyObject* v_, PyObject* m_, PyObject* l_, PyObject* acc_,
             PyObject* valid_, PyObject* active_, PyObject* scale_, PyObject* softcap_) {
  const Tensor *q = plain(q_), *k = plain(k_);
  if (!q || !k || q->dim() != 3 || k->dim() != 4) return false;
  c.dev = q->device();
  c.b = q->size(0);
  c.hq = q->size(1);
  c.d = q->size(2);
  c.hkv = k->size(1);
  c.tc = k->size(2);
  c.code = dtype_code(q->scalar_type());
  if (c.code < 0 || k->scalar_type() != q->scalar_type() || k->device() != c.dev) return false;
  if (c.b <= 0 || c.tc <= 0 || c.hkv <= 0 || c.hq <= 0 || c.hq % c.hkv != 0 || c.hq / c.hkv > 16 ||
      k->size(0) != c.b || k->size(3) != c.d)
    return false;
  if (v_) {
    const Tensor* v = plain(v_);
    if (!v || v->scalar_type() != q->scalar_type() || v->device() != c.dev || v->sizes() != k->sizes()) return false;
    c.v = v->const_data_ptr();
  }
  const Tensor *m = plain(m_), *l = plain(l_), *acc = acc_ ? plain(acc_) : nullptr;
  if (!is_f32(m, c.dev, {c.b, c.hq}) || !is_f32(l, c.dev, {c.b, c.hq})) return false;
  if (acc_ && !is_f32(acc, c.dev, {c.b, c.hq, c.d})) return false;
  if (!mask(valid_, c.dev, {c.b, c.tc}, &c.valid)) return false;
  if (active_ && !mask(active_, c.dev, {c.b}, &c.active)) return false;
  double scale = 0.0, softcap = 0.0;
  if (!number(scale_, 1.0 / std::pow((double)c.d, 0.5), &scale) || !number(softcap_, 0.0, &softcap)) return false;
  c.scale = (float)scale;
  c.softcap = (float)softcap;
  c.q = q->const_data_ptr();
  c.k = k->const_data_ptr();
  c.m = f32(m);
  c.l = f32(l);
  if (acc_) c.acc = f32(acc);
  return true;
}

// Runs `launch(workspace, bytes)` with the workspace of the call's mode. New reference or null.
template <class F>
PyObject* run(Call& c, int mode, int64_t tpb, F launch) {
  if (!current_stream(c.dev, &c.stream)) return nullptr;
  int rc = 0;
  {
    const c10::DeviceGuard guard(c.dev);
    const size_t bytes = g_workspace_bytes(c.b, c.hq, c.hkv, c.tc, c.d, mode, tpb);
    // Freed on return, behind this stream's work, as a tensor of this size would be, and from the
    // allocator that torch.empty uses (c10::GetAllocator is the native one also where
    // torch.cuda.memory.change_current_allocator has put another in its place).
    const c10::DataPtr ws =
        at::detail::getCUDAHooks().getCUDADeviceAllocator()->allocate(bytes ? bytes : 1);
    Py_BEGIN_ALLOW_THREADS;
    rc = launch(ws.get(), bytes);
    Py_END_ALLOW_THREADS;
  }
  return PyLong_FromLong(rc);
}

// C++ exceptions (an allocation that fails, a torch check) end as Python exceptions.
template <class F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g_out_of_memory, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

bool ready(Py_ssize_t n, Py_ssize_t want) {
  if (n == want && g_raw_stream) return true;
  PyErr_SetString(PyExc_TypeError, g_raw_stream ? "wrong number of arguments" : "bind was not called");
  return false;
}

// A torch dispatch or function mode sees what the general path calls.
bool modes_active() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled();
}

// step(q, k, v, m, l, acc, valid, active, scale, softcap)
PyObject* py_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 10)) return nullptr;
  return guarded([&]() -> PyObject* {
    Call c;
    if (modes_active() || !prepare(c, a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9])) Py_RETURN_NONE;
    return run(c, kFold, 16, [&](void* ws, size_t bytes) {
      return g_step(c.q, c.k, c.v, c.valid, c.active, c.m,
                    c.l, c.acc, c.b, c.hq, c.hkv, c.tc, c.d, c.code, c.scale, c.softcap, ws,
                    bytes, c.stream);
    });
  });
}

// stats_step(q, k, m, l, valid, active, scale, softcap)
PyObject* py_stats(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    Call c;
    if (modes_active() || !prepare(c, a[0], a[1], nullptr, a[2], a[3], nullptr, a[4], a[5], a[6], a[7]))
      Py_RETURN_NONE;
    return run(c, kStats, 16, [&](void* ws, size_t bytes) {
      return g_stats(c.q, c.k, c.valid, c.active, c.m, c.l, c.b, c.hq,
                     c.hkv, c.tc, c.d, c.code, c.scale, c.softcap, ws, bytes, c.stream);
    });
  });
}

// accumulate_step(q, k, v, m, l, acc, block_mass, block_id_offset, tokens_per_block, valid,
// active, scale, softcap)
PyObject* py_accumulate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 13)) return nullptr;
  return guarded([&]() -> PyObject* {
    Call c;
    int64_t offset = 0, tpb = 0;
    if (modes_active() || !prepare(c, a[0], a[1], a[2], a[3], a[4], a[5], a[9], a[10], a[11], a[12]) ||
        !integer(a[7], &offset) || !integer(a[8], &tpb) || tpb <= 0)
      Py_RETURN_NONE;
    const Tensor* mass = plain(a[6]);
    if (!mass || mass->scalar_type() != at::kFloat || mass->device() != c.dev || mass->dim() != 3 ||
        mass->size(0) != c.b || mass->size(1) != c.hq)
      Py_RETURN_NONE;
    const int64_t max_blocks = mass->size(2);
    float* const mass_data = f32(mass);
    return run(c, kAccumulate, tpb, [&](void* ws, size_t bytes) {
      return g_accumulate(c.q, c.k, c.v, c.valid, c.active,
                          c.m, c.l, c.acc, mass_data, max_blocks, offset, tpb, c.b, c.hq, c.hkv, c.tc,
                          c.d, c.code, c.scale, c.softcap, ws, bytes, c.stream);
    });
  });
}

// fold_fixed_step(q, k, v, m, l, acc, valid, scale, softcap)
PyObject* py_fold_fixed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    Call c;
    if (modes_active() || !prepare(c, a[0], a[1], a[2], a[3], a[4], a[5], a[6], nullptr, a[7], a[8])) Py_RETURN_NONE;
    return run(c, kFoldFixed, 16, [&](void* ws, size_t bytes) {
      return g_fold_fixed(c.q, c.k, c.v, c.valid, c.m,
                          c.l, c.acc, c.b, c.hq, c.hkv, c.tc, c.d, c.code, c.scale, c.softcap,
                          ws, bytes, c.stream);
    });
  });
}

// state_init(batch, query_heads, head_dim, device) -> (status, m, l, acc) or None. The device has
// an index and torch's GPU state exists: the caller sees to both.
PyObject* py_state_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 4)) return nullptr;
  return guarded([&]() -> PyObject* {
    int64_t b = 0, hq = 0, d = 0;
    if (modes_active() || !THPDevice_Check(a[3])) Py_RETURN_NONE;
    const c10::Device dev = reinterpret_cast<THPDevice*>(a[3])->device;
    if (!dev.is_cuda() || !dev.has_index() || !integer(a[0], &b) || !integer(a[1], &hq) || !integer(a[2], &d) ||
        b <= 0 || hq <= 0 || d <= 0)
      Py_RETURN_NONE;
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(at::kFloat).device(dev);
    Tensor m = at::empty({b, hq}, opt), l = at::empty({b, hq}, opt), acc = at::empty({b, hq, d}, opt);
    if (!plain_keys(m)) Py_RETURN_NONE;  // a mode or transform is active: the general path
    float *pm = f32(&m), *pl = f32(&l), *pacc = f32(&acc);
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_state_init(pm, pl, pacc, b * hq, d, stream);
    Py_END_ALLOW_THREADS;
    return Py_BuildValue("(iNNN)", rc, THPVariable_Wrap(m), THPVariable_Wrap(l), THPVariable_Wrap(acc));
  });
}

// finalize(acc, l, dtype) -> (status, out) or None
PyObject* py_finalize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 3)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor *acc = plain(a[0]), *l = plain(a[1]);
    if (modes_active() || !acc || !l || !THPDtype_Check(a[2]) || acc->dim() < 1) Py_RETURN_NONE;
    const at::ScalarType type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    const int code = dtype_code(type);
    if (code < 0 || acc->numel() == 0 || !is_f32(acc, acc->device(), acc->sizes()) ||
        !is_f32(l, acc->device(), acc->sizes().slice(0, acc->dim() - 1)))
      Py_RETURN_NONE;
    void* stream = nullptr;
    if (!current_stream(acc->device(), &stream)) return nullptr;
    const c10::DeviceGuard guard(acc->device());
    Tensor out = at::empty(acc->sizes(), at::TensorOptions().dtype(type).device(acc->device()));
    if (!plain_keys(out)) Py_RETURN_NONE;
    const float *pacc = f32(acc), *pl = f32(l);
    void* pout = out.mutable_data_ptr();
    const int64_t rows = l->numel(), d = acc->size(-1);
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_finalize(pacc, pl, pout, rows, d, code, stream);
    Py_END_ALLOW_THREADS;
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(out));
  });
}

// bind(workspace_bytes, step, stats, accumulate, fold_fixed, state_init, finalize: addresses;
// raw_stream: callable(device index) -> hipStream_t; out_of_memory: exception class)
PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long p[7];
  PyObject *raw = nullptr, *oom = nullptr;
  if (!PyArg_ParseTuple(args, "KKKKKKKOO", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &raw, &oom))
    return nullptr;
  auto set = [](auto& fn, unsigned long long addr) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addr); };
  set(g_workspace_bytes, p[0]);
  set(g_step, p[1]);
  set(g_stats, p[2]);
  set(g_accumulate, p[3]);
  set(g_fold_fixed, p[4]);
  set(g_state_init, p[5]);
  set(g_finalize, p[6]);
  Py_INCREF(raw);
  Py_XSETREF(g_raw_stream, raw);
  Py_INCREF(oom);
  Py_XSETREF(g_out_of_memory, oom);
  Py_RETURN_NONE;
}

// ---- rotary positions and the bounded cache --------------------------------------------
// Whether a call would lose a gradient that is being recorded, or a forward-mode tangent.
bool differentiated(const Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(/*level=*/0).defined();
}

// An operand whose last dimension is contiguous, the others strided at will. Null: not plain, or its
// gradient is being recorded (the general path refuses it).
const Tensor* viewed(PyObject* o, int64_t dims) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || !plain_keys(t) || !t.has_storage() || t.dim() != dims) return nullptr;
  if (t.stride(-1) != 1 && t.size(-1) != 1) return nullptr;
  return differentiated(t) ? nullptr : &t;
}

bool shaped(const Tensor* t, const Tensor* like, at::IntArrayRef shape) {
  return t && t->scalar_type() == like->scalar_type() && t->device() == like->device() && t->sizes() == shape;
}

bool truth(PyObject* o, int* out) {
  if (!PyBool_Check(o)) return false;
  *out = o == Py_True;
  return true;
}

// inv_freq: None, or the frequencies of at most head_dim / 2 pairs.
bool frequencies(PyObject* o, const c10::Device& dev, int64_t head_dim, const float** data, int64_t* rotary) {
  *data = nullptr;
  *rotary = 0;
  if (o == Py_None) return true;
  const Tensor* t = plain(o);
  if (!t || t->scalar_type() != at::kFloat || t->device() != dev || t->dim() != 1 || 2 * t->size(0) > head_dim ||
      differentiated(*t))
    return false;
  *data = t->const_data_ptr<float>();
  *rotary = 2 * t->size(0);
  return true;
}

bool whole_numbers(const Tensor* t, const c10::Device& dev) {
  return t && (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong) && t->device() == dev;
}

// rotary(q, k or None, positions, inv_freq, interleaved, factor, inverse) -> (status, q', k') or None
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 7)) return nullptr;
  return guarded([&]() -> PyObject* {
    if (modes_active() || !THPVariable_CheckExact(a[0])) Py_RETURN_NONE;
    const int64_t dims = THPVariable_Unpack(a[0]).dim();
    if (dims != 3 && dims != 4) Py_RETURN_NONE;
    const Tensor *q = viewed(a[0], dims), *k = a[1] == Py_None ? nullptr : viewed(a[1], dims);
    if (!q || (a[1] != Py_None && !k) || !THPVariable_CheckExact(a[2])) Py_RETURN_NONE;
    const c10::Device dev = q->device();
    const Tensor* pos = &THPVariable_Unpack(a[2]);
    if (!pos->defined() || !pos->is_cuda() || !plain_keys(*pos) || !whole_numbers(pos, dev)) Py_RETURN_NONE;
    // [B, H, D] is [B, H, 1, D], its positions [B] are [B, 1].
    const int64_t b = q->size(0), hq = q->size(1), t = dims == 4 ? q->size(2) : 1, d = q->size(-1);
    const int code = dtype_code(q->scalar_type());
    if (code < 0 || b == 0 || t == 0 || hq == 0 || d == 0 || pos->dim() != dims - 2) Py_RETURN_NONE;
    if (dims == 4 ? (pos->size(0) != b && pos->size(0) != 1) || pos->size(1) != t : pos->size(0) != b) Py_RETURN_NONE;
    const int64_t hk = k ? k->size(1) : 0;
    if (k && (k->scalar_type() != q->scalar_type() || k->device() != dev || k->size(0) != b ||
              (dims == 4 && k->size(2) != t) || k->size(-1) != d))
      Py_RETURN_NONE;
    const float* freq = nullptr;
    int64_t turning = 0;
    int interleaved = 0, inverse = 0;
    double factor = 0.0;
    if (a[3] == Py_None || !frequencies(a[3], dev, d, &freq, &turning) || !truth(a[4], &interleaved) ||
        !PyFloat_CheckExact(a[5]) || !number(a[5], 1.0, &factor) || !truth(a[6], &inverse))
      Py_RETURN_NONE;
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    const auto opt = at::TensorOptions().dtype(q->scalar_type()).device(dev);
    Tensor qo = at::empty(q->sizes(), opt), ko;
    if (k) ko = at::empty(k->sizes(), opt);
    if (!plain_keys(qo)) Py_RETURN_NONE;
    const int64_t qs[3] = {q->stride(0), q->stride(1), dims == 4 ? q->stride(2) : 0};
    const int64_t ks[3] = {k ? k->stride(0) : 0, k ? k->stride(1) : 0, k && dims == 4 ? k->stride(2) : 0};
    const int64_t ps[2] = {dims == 4 && pos->size(0) == 1 ? 0 : pos->stride(0), dims == 4 ? pos->stride(1) : 0};
    const void *pq = q->const_data_ptr(), *pk = k ? k->const_data_ptr() : nullptr, *pp = pos->const_data_ptr();
    void *pqo = qo.mutable_data_ptr(), *pko = k ? ko.mutable_data_ptr() : nullptr;
    const int long_pos = pos->scalar_type() == at::kLong;
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_rotary(pq, qs, pqo, hq, pk, ks, pko, hk, pp, long_pos, ps, freq, turning, b, t, d, code, interleaved,
                  (float)factor, inverse, stream);
    Py_END_ALLOW_THREADS;
    if (!k) return Py_BuildValue("(iNO)", rc, THPVariable_Wrap(qo), Py_None);
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(qo), THPVariable_Wrap(ko));
  });
}

// The cache of a call: the address of its pgr_hh_cache_t, which the Python object holds.
const pgr_hh_cache_t* cache_at(PyObject* o) {
  return PyLong_CheckExact(o) ? static_cast<const pgr_hh_cache_t*>(PyLong_AsVoidPtr(o)) : nullptr;
}

// t is a [batch, heads, head_dim] token operand of the cache on device `index`.
bool token(const Tensor* t, const pgr_hh_cache_t* c, int64_t heads, int64_t index) {
  return t && dtype_code(t->scalar_type()) == c->dtype && t->device().index() == index &&
         t->sizes() == at::IntArrayRef({c->batch, heads, c->head_dim});
}

// Whether an index operand views the cache's own state, which a call changes while it reads the operand: the
// general path copies it.
bool in_state(const pgr_hh_cache_t* c, const void* p) {
  const size_t rows = (size_t)(c->batch * c->kv_heads), slots = rows * (size_t)c->capacity;
  auto within = [p](const void* base, size_t count) {
    return (uintptr_t)p >= (uintptr_t)base && (uintptr_t)p - (uintptr_t)base < count * 4;
  };
  return p != nullptr && (within(c->seen, rows) || within(c->lengths, rows) || within(c->order, slots) ||
                          within(c->weights, slots));
}

// append(cache, device index, q, k, v, inv_freq or None, positions or None, interleaved, factor) -> (status, q')
// or None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    const pgr_hh_cache_t* c = cache_at(a[0]);
    int64_t index = 0;
    if (modes_active() || !c || !integer(a[1], &index)) Py_RETURN_NONE;
    const Tensor *q = viewed(a[2], 3), *k = viewed(a[3], 3), *v = viewed(a[4], 3);
    if (!token(q, c, c->query_heads, index) || !token(k, c, c->kv_heads, index) || !token(v, c, c->kv_heads, index))
      Py_RETURN_NONE;
    const c10::Device dev = q->device();
    const float* freq = nullptr;
    int64_t turning = 0;
    int interleaved = 0;
    double factor = 0.0;
    if (!frequencies(a[5], dev, c->head_dim, &freq, &turning) || !truth(a[7], &interleaved) ||
        !PyFloat_CheckExact(a[8]) || !number(a[8], 1.0, &factor))
      Py_RETURN_NONE;
    const void* positions = nullptr;
    int long_pos = 0;
    if (a[6] != Py_None) {
      const Tensor* pos = plain(a[6]);
      if (!whole_numbers(pos, dev) || pos->sizes() != at::IntArrayRef({c->batch})) Py_RETURN_NONE;
      positions = pos->const_data_ptr();
      if (in_state(c, positions)) Py_RETURN_NONE;
      long_pos = pos->scalar_type() == at::kLong;
    }
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    Tensor qo;
    void* pqo = nullptr;
    if (a[5] != Py_None) {
      qo = at::empty(q->sizes(), at::TensorOptions().dtype(q->scalar_type()).device(dev));
      if (!plain_keys(qo)) Py_RETURN_NONE;
      pqo = qo.mutable_data_ptr();
    }
    const int64_t qs[2] = {q->stride(0), q->stride(1)}, ks[2] = {k->stride(0), k->stride(1)},
                  vs[2] = {v->stride(0), v->stride(1)};
    const void *pq = q->const_data_ptr(), *pk = k->const_data_ptr(), *pv = v->const_data_ptr();
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_append(c, pq, qs, pk, ks, pv, vs, pqo, positions, long_pos, freq, turning, interleaved, (float)factor,
                  stream);
    Py_END_ALLOW_THREADS;
    if (!pqo) return Py_BuildValue("(iO)", rc, a[2]);
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(qo));
  });
}

// attend(cache, device index, workspace bytes, q, scale, softcap) -> (status, out) or None
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const pgr_hh_cache_t* c = cache_at(a[0]);
    int64_t index = 0, bytes = 0;
    if (modes_active() || !c || !integer(a[1], &index) || !integer(a[2], &bytes)) Py_RETURN_NONE;
    const Tensor* q = viewed(a[3], 3);
    double scale = 0.0, softcap = 0.0;
    if (!token(q, c, c->query_heads, index) || !number(a[4], 1.0 / std::pow((double)c->head_dim, 0.5), &scale) ||
        !number(a[5], 0.0, &softcap))
      Py_RETURN_NONE;
    const c10::Device dev = q->device();
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    Tensor out = at::empty(q->sizes(), at::TensorOptions().dtype(q->scalar_type()).device(dev));
    if (!plain_keys(out)) Py_RETURN_NONE;
    c10::DataPtr ws;
    if (bytes > 0) ws = at::detail::getCUDAHooks().getCUDADeviceAllocator()->allocate((size_t)bytes);
    const int64_t qs[2] = {q->stride(0), q->stride(1)};
    const void* pq = q->const_data_ptr();
    void* po = out.mutable_data_ptr();
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_attend(c, pq, qs, po, (float)scale, (float)softcap, ws.get(), (size_t)bytes, stream);
    Py_END_ALLOW_THREADS;
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(out));
  });
}

// lo: None, or int32 [batch].
bool first_columns(PyObject* o, const c10::Device& dev, int64_t batch, const int32_t** out) {
  return mask(o, dev, {batch}, out);
}

// prompt_weights(q, k, lo or None, scale, softcap) -> (status, weights) or None
PyObject* py_prompt_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    if (modes_active()) Py_RETURN_NONE;
    const Tensor *q = viewed(a[0], 4), *k = viewed(a[1], 4);
    if (!q || !k) Py_RETURN_NONE;
    const c10::Device dev = q->device();
    const int64_t b = q->size(0), hq = q->size(1), w = q->size(2), d = q->size(3), hkv = k->size(1), t = k->size(2);
    const int code = dtype_code(q->scalar_type());
    const int32_t* lo = nullptr;
    double scale = 0.0, softcap = 0.0;
    if (!shaped(k, q, {b, hkv, t, d}) || code < 0 || code == 2 || b == 0 || t == 0 ||
        !first_columns(a[2], dev, b, &lo) || !number(a[3], 1.0 / std::pow((double)d, 0.5), &scale) ||
        !number(a[4], 0.0, &softcap))
      Py_RETURN_NONE;
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    const size_t bytes = g_prompt_weights_bytes(b, hq, hkv, t, w, d);
    if (bytes == 0) Py_RETURN_NONE;  // refused: the general path says why
    Tensor out = at::empty({b, hkv, t}, at::TensorOptions().dtype(at::kFloat).device(dev));
    if (!plain_keys(out)) Py_RETURN_NONE;
    const c10::DataPtr ws = at::detail::getCUDAHooks().getCUDADeviceAllocator()->allocate(bytes);
    const int64_t qs[3] = {q->stride(0), q->stride(1), q->stride(2)}, ks[3] = {k->stride(0), k->stride(1), k->stride(2)};
    const void *pq = q->const_data_ptr(), *pk = k->const_data_ptr();
    float* po = f32(&out);
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_prompt_weights(pq, qs, pk, ks, lo, po, b, hq, hkv, t, w, d, code, (float)scale, (float)softcap, ws.get(),
                          bytes, stream);
    Py_END_ALLOW_THREADS;
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(out));
  });
}

// load_prompt(cache, device index, k, v, weights, lo or None) -> status or None
PyObject* py_load_prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!ready(n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const pgr_hh_cache_t* c = cache_at(a[0]);
    int64_t index = 0;
    if (modes_active() || !c || !integer(a[1], &index)) Py_RETURN_NONE;
    const Tensor *k = viewed(a[2], 4), *v = viewed(a[3], 4), *w = plain(a[4]);
    if (!k || !v || dtype_code(k->scalar_type()) != c->dtype || k->device().index() != index) Py_RETURN_NONE;
    const c10::Device dev = k->device();
    const int64_t t = k->size(2);
    const int32_t* lo = nullptr;
    if (t == 0 || k->sizes() != at::IntArrayRef({c->batch, c->kv_heads, t, c->head_dim}) || !shaped(v, k, k->sizes()) ||
        !is_f32(w, dev, {c->batch, c->kv_heads, t}) || differentiated(*w) ||
        !first_columns(a[5], dev, c->batch, &lo) || in_state(c, lo))
      Py_RETURN_NONE;
    void* stream = nullptr;
    if (!current_stream(dev, &stream)) return nullptr;
    const c10::DeviceGuard guard(dev);
    const size_t bytes = g_load_prompt_bytes(c, t);
    if (bytes == 0) Py_RETURN_NONE;
    const c10::DataPtr ws = at::detail::getCUDAHooks().getCUDADeviceAllocator()->allocate(bytes);
    const int64_t ks[3] = {k->stride(0), k->stride(1), k->stride(2)}, vs[3] = {v->stride(0), v->stride(1), v->stride(2)};
    const void *pk = k->const_data_ptr(), *pv = v->const_data_ptr();
    const float* pw = w->const_data_ptr<float>();
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS;
    rc = g_load_prompt(c, pk, ks, pv, vs, pw, lo, t, ws.get(), bytes, stream);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(rc);
  });
}

// bind_cache(rotary, append, attend, prompt_weights, its workspace size, load_prompt, its workspace size: addresses)
PyObject* py_bind_cache(PyObject*, PyObject* args) {
  unsigned long long p[7];
  if (!PyArg_ParseTuple(args, "KKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6])) return nullptr;
  auto set = [](auto& fn, unsigned long long addr) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addr); };
  set(g_rotary, p[0]);
  set(g_append, p[1]);
  set(g_attend, p[2]);
  set(g_prompt_weights, p[3]);
  set(g_prompt_weights_bytes, p[4]);
  set(g_load_prompt, p[5]);
  set(g_load_prompt_bytes, p[6]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"step", (PyCFunction)(void (*)(void))py_step, METH_FASTCALL, nullptr},
    {"stats_step", (PyCFunction)(void (*)(void))py_stats, METH_FASTCALL, nullptr},
    {"accumulate_step", (PyCFunction)(void (*)(void))py_accumulate, METH_FASTCALL, nullptr},
    {"fold_fixed_step", (PyCFunction)(void (*)(void))py_fold_fixed, METH_FASTCALL, nullptr},
    {"state_init", (PyCFunction)(void (*)(void))py_state_init, METH_FASTCALL, nullptr},
    {"finalize", (PyCFunction)(void (*)(void))py_finalize, METH_FASTCALL, nullptr},
    {"bind_cache", py_bind_cache, METH_VARARGS, nullptr},
    {"rotary", (PyCFunction)(void (*)(void))py_rotary, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void (*)(void))py_append, METH_FASTCALL, nullptr},
    {"attend", (PyCFunction)(void (*)(void))py_attend, METH_FASTCALL, nullptr},
    {"prompt_weights", (PyCFunction)(void (*)(void))py_prompt_weights, METH_FASTCALL, nullptr},
    {"load_prompt", (PyCFunction)(void (*)(void))py_load_prompt, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pgr_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pgr_ops() { return PyModule_Create(&module); }
