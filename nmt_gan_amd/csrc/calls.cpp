// The operators' calls on torch tensors for nmt_gan_amd/ops.py: arguments checked, outputs and scratch allocated by torch's
// caching allocator, the entry point of include/nmtgan.h called on the current stream of the tensors' device.  In C++ because
// a call of one token is over sooner than Python reads twenty tensor attributes: 5.6 us of GPU time, 12 us of host time
// when these checks were written in Python.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/nmtgan.h"

namespace {

using at::Tensor;

// the entry points of the library that the package has loaded, set by bind()
struct Entry {
  decltype(&nmtgan_attn_span) attn_span;
  decltype(&nmtgan_attn_span_step_workspace_bytes) attn_span_step_workspace_bytes;
  decltype(&nmtgan_attn_span_step) attn_span_step;
  decltype(&nmtgan_attn_span_grads_workspace_bytes) attn_span_grads_workspace_bytes;
  decltype(&nmtgan_attn_span_grads) attn_span_grads;
  decltype(&nmtgan_linear_xent_workspace_bytes) linear_xent_workspace_bytes;
  decltype(&nmtgan_linear_xent) linear_xent;
  decltype(&nmtgan_linear_xent_grads) linear_xent_grads;
  decltype(&nmtgan_global_norm_workspace_bytes) global_norm_workspace_bytes;
  decltype(&nmtgan_global_norm) global_norm;
  decltype(&nmtgan_clip_global_norm) clip_global_norm;
} entry;

[[noreturn]] void refuse(const char* what, const std::string& text) {
  PyErr_Format(PyExc_ValueError, "%s: %s", what, text.c_str());
  throw python_error();
}

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    default: return c10::toString(t);
  }
}
std::string shape_of(const Tensor& t) { return c10::str(t.sizes()); }

const Tensor& tensor(const char* what, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(what, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
long integer(const char* what, const char* name, PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be an integer");
  }
  return v;
}
double number(const char* what, const char* name, PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be a number");
  }
  return v;
}

// What all tensors of a call share
struct Common {
  const char* what;
  at::Device device;
  at::ScalarType type;
  int code, size;
};
Common common(const char* what, const char* name, PyObject* o) {
  const Tensor& t = tensor(what, name, o);
  if (!t.is_cuda()) refuse(what, "tensors on a GPU are needed");
  const at::ScalarType s = t.scalar_type();
  if (s != at::kBFloat16 && s != at::kHalf && s != at::kFloat)
    refuse(what, std::string("bfloat16, float16 or float32 expected, got ") + type_name(s));
  return {what, t.device(), s, s == at::kBFloat16 ? NMTGAN_BF16 : s == at::kHalf ? NMTGAN_F16 : NMTGAN_F32, s == at::kFloat ? 4 : 2};
}

struct Rows { void* at; int64_t ld; };
// a [rows, width] matrix whose rows are contiguous and 16-byte aligned
Rows rows(const Common& c, const char* name, const Tensor& t, int64_t width) {
  if (t.dim() != 2 || t.size(1) != width)
    refuse(c.what, std::string(name) + " must be [rows, " + std::to_string(width) + "], is " + shape_of(t));
  if (t.scalar_type() != c.type || t.device() != c.device)
    refuse(c.what, std::string(name) + " is " + type_name(t.scalar_type()) + " on " + t.device().str() + ", expected " +
                       type_name(c.type) + " on " + c.device.str());
  const int64_t step = t.size(0) < 2 ? width : t.stride(0);
  void* at = t.data_ptr();
  if ((t.stride(1) != 1 && width > 1) || step < width || step * c.size % 16 || (uintptr_t)at % 16)
    refuse(c.what, std::string(name) + " needs contiguous rows that start at 16-byte boundaries");
  return {at, step};
}
void* vector(const Common& c, const char* name, const Tensor& t, int64_t n, at::ScalarType type) {
  if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != type || t.device() != c.device || (n > 1 && t.stride(0) != 1))
    refuse(c.what, std::string(name) + " must be a contiguous " + type_name(type) + " vector of " + std::to_string(n) + " on " +
                       c.device.str());
  return t.data_ptr();
}
Tensor fresh(const Common& c, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(c.device));
}
// a tensor of the caller's has been written: torch's version of it goes up, so that autograd sees a saved one that has changed
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// an output given by the caller, or a new one
Tensor target(const Common& c, const char* name, PyObject* o, int64_t n, int64_t width) {
  if (o == Py_None) return fresh(c, {n, width}, c.type);
  const Tensor& t = tensor(c.what, name, o);
  if (t.dim() != 2 || t.size(0) != n) refuse(c.what, std::string(name) + " must have " + std::to_string(n) + " rows");
  return t;
}
Tensor scratch(const Common& c, size_t n) { return fresh(c, {(int64_t)std::max<size_t>(n, 1)}, at::kByte); }

// calls an entry point on the current stream of the device; its error code
template <typename F>
int run(const Common& c, F call) {
  const auto index = c.device.index();
  std::optional<c10::DeviceGuard> guard;
  if (c10::hip::current_device() != index) guard.emplace(c.device);
  return call((void*)c10::hip::getCurrentHIPStream(index).stream());
}
void checked(const Common& c, int rc) {
  if (!rc) return;
  PyObject* lib = PyImport_ImportModule("nmt_gan_amd._lib");
  PyObject* done = lib ? PyObject_CallMethod(lib, "check", "is", rc, c.what) : nullptr;
  Py_XDECREF(lib);
  Py_XDECREF(done);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, c.what);
  throw python_error();
}

// ---------------------------------------------------------------------------------------------- span attention
// o: q, k, v, lo, hi, heads, kv_heads, scale, cap, slopes, pos
Common span(const char* what, PyObject* const* o, nmtgan_span_args& a) {
  const Common c = common(what, "q", o[0]);
  const Tensor &q = THPVariable_Unpack(o[0]), &k = tensor(what, "k", o[1]), &v = tensor(what, "v", o[2]);
  const long heads = integer(what, "heads", o[5]), kv = o[6] == Py_None ? heads : integer(what, "kv_heads", o[6]);
  if (heads < 1 || kv < 1 || heads > (1 << 30) || heads % kv)
    refuse(what, "heads=" + std::to_string(heads) + " must be a multiple of kv_heads=" + std::to_string(kv));
  if (q.dim() != 2 || k.dim() != 2 || v.dim() != 2 || q.size(1) % heads) refuse(what, "q must be [rows, heads * dh] and k, v [keys, kv_heads * dh]");
  const int64_t dh = q.size(1) / heads, m = q.size(0), n = k.size(0);
  if (dh < 1 || dh % 8 || dh > 128) refuse(what, "the head width " + std::to_string(dh) + " must be a multiple of 8, at most 128");
  const double scale = number(what, "scale", o[7]), cap = number(what, "cap", o[8]);
  if (!std::isfinite((float)scale) || !std::isfinite((float)cap) || cap < 0) refuse(what, "scale and cap must be finite, cap >= 0");
  if (cap != 0.0 && (float)cap == 0.f) refuse(what, "cap is below the least float32 number and would read as no cap");
  if (m > INT32_MAX || n > INT32_MAX || v.size(0) != n)
    refuse(what, "k has " + std::to_string(n) + " rows, v " + std::to_string(v.size(0)));
  a = {};
  a.dtype = c.code; a.M = (int)m; a.N = (int)n; a.heads = (int)heads; a.kv_heads = (int)kv; a.dh = (int)dh;
  const Rows rq = rows(c, "q", q, heads * dh), rk = rows(c, "k", k, kv * dh), rv = rows(c, "v", v, kv * dh);
  a.q = rq.at; a.ldq = rq.ld; a.k = rk.at; a.ldk = rk.ld; a.v = rv.at; a.ldv = rv.ld;
  a.lo = (const int32_t*)vector(c, "lo", tensor(what, "lo", o[3]), m, at::kInt);
  a.hi = (const int32_t*)vector(c, "hi", tensor(what, "hi", o[4]), m, at::kInt);
  if (o[9] != Py_None) a.slopes = (const float*)vector(c, "slopes", tensor(what, "slopes", o[9]), heads, at::kFloat);
  if (o[10] != Py_None) a.pos = (const int32_t*)vector(c, "pos", tensor(what, "pos", o[10]), m, at::kInt);
  a.scale = (float)scale; a.cap = (float)cap;
  return c;
}
void need_args(Py_ssize_t have, Py_ssize_t want) {
  if (have == want) return;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, have);
  throw python_error();
}
PyObject* pair(Tensor a, Tensor b) {
  THPObjectPtr x(THPVariable_Wrap(std::move(a))), y(THPVariable_Wrap(std::move(b)));
  return x && y ? PyTuple_Pack(2, x.get(), y.get()) : nullptr;
}

// (span..., out) -> (out, lse)
PyObject* attn_span(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 12);
  nmtgan_span_args a;
  const Common c = span("attn_span", o, a);
  const int64_t width = (int64_t)a.heads * a.dh;
  Tensor out = target(c, "out", o[11], a.M, width), lse = fresh(c, {a.M, a.heads}, at::kFloat);
  const Rows ro = rows(c, "out", out, width);
  a.out = ro.at; a.ldo = ro.ld; a.lse = (float*)lse.data_ptr();
  checked(c, run(c, [&](void* st) { return entry.attn_span(&a, st); }));
  written(out);
  return pair(std::move(out), std::move(lse));
  END_HANDLE_TH_ERRORS
}
// (span..., max_keys, out) -> out
PyObject* attn_span_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 13);
  nmtgan_span_args a;
  const Common c = span("attn_span_step", o, a);
  const long keys = integer(c.what, "max_keys", o[11]);
  if (keys < 0 || keys > INT32_MAX) refuse(c.what, "max_keys=" + std::to_string(keys));
  const int64_t width = (int64_t)a.heads * a.dh;
  Tensor out = target(c, "out", o[12], a.M, width), ws;
  const Rows ro = rows(c, "out", out, width);
  a.out = ro.at; a.ldo = ro.ld;
  const size_t bytes = entry.attn_span_step_workspace_bytes(a.M, a.heads, a.kv_heads, a.dh, (int)keys);
  if (bytes) ws = scratch(c, bytes);
  checked(c, run(c, [&](void* st) { return entry.attn_span_step(&a, (int)keys, bytes ? ws.data_ptr() : nullptr, bytes, st); }));
  written(out);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}
// (span..., dout, out, lse, dq, dk, dv) -> (dq, dk, dv)
PyObject* attn_span_grads(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 17);
  nmtgan_span_args a;
  const Common c = span("attn_span_grads", o, a);
  if (c.type == at::kHalf) refuse(c.what, "bfloat16 or float32 (float16 gradients would underflow without loss scaling)");
  const int64_t wq = (int64_t)a.heads * a.dh, wk = (int64_t)a.kv_heads * a.dh;
  const Tensor &dout = tensor(c.what, "dout", o[11]), &out = tensor(c.what, "out", o[12]), &lse = tensor(c.what, "lse", o[13]);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("dout", dout), std::pair<const char*, const Tensor&>("out", out)})
    if (t.dim() != 2 || t.size(0) != a.M) refuse(c.what, std::string(name) + " must have " + std::to_string(a.M) + " rows");
  if (lse.dim() != 2 || lse.size(0) != a.M || lse.size(1) != a.heads || lse.scalar_type() != at::kFloat || lse.device() != c.device ||
      !lse.is_contiguous())
    refuse(c.what, "lse must be attn_span's [" + std::to_string(a.M) + ", " + std::to_string(a.heads) + "] float32 result");
  Tensor dq = target(c, "dq", o[14], a.M, wq), dk = target(c, "dk", o[15], a.N, wk), dv = target(c, "dv", o[16], a.N, wk);
  const Rows ro = rows(c, "out", out, wq), rd = rows(c, "dout", dout, wq), r1 = rows(c, "dq", dq, wq), r2 = rows(c, "dk", dk, wk),
             r3 = rows(c, "dv", dv, wk);
  a.out = ro.at; a.ldo = ro.ld; a.lse = (float*)lse.data_ptr();
  const nmtgan_span_grads g{rd.at, rd.ld, r1.at, r1.ld, r2.at, r2.ld, r3.at, r3.ld};
  const size_t bytes = entry.attn_span_grads_workspace_bytes(a.M, a.heads);
  const Tensor ws = scratch(c, bytes);
  checked(c, run(c, [&](void* st) { return entry.attn_span_grads(&a, &g, ws.data_ptr(), bytes, st); }));
  for (const Tensor* t : {&dq, &dk, &dv}) written(*t);
  THPObjectPtr x(THPVariable_Wrap(std::move(dq))), y(THPVariable_Wrap(std::move(dk))), z(THPVariable_Wrap(std::move(dv)));
  return x && y && z ? PyTuple_Pack(3, x.get(), y.get(), z.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- cross entropy
// o: h, w, labels, smoothing
Common xent(const char* what, PyObject* const* o, nmtgan_xent_args& a) {
  const Common c = common(what, "h", o[0]);
  const Tensor &h = THPVariable_Unpack(o[0]), &w = tensor(what, "w", o[1]);
  if (h.dim() != 2 || w.dim() != 2 || w.size(0) < 1 || h.size(1) < 1) refuse(what, "h must be [rows, d] and w [vocabulary, d]");
  const double smoothing = number(what, "smoothing", o[3]);
  if (!(smoothing >= 0.0 && (float)smoothing < 1.f) || (smoothing != 0.0 && w.size(0) < 2))
    refuse(what, "smoothing must be in [0, 1), and 0 for a vocabulary of one");
  if (h.size(1) * c.size % 16 || h.size(0) > INT32_MAX || w.size(0) > INT32_MAX || w.size(1) > INT32_MAX)
    refuse(what, "a row of h must be a multiple of 16 bytes");
  a = {};
  const Rows rh = rows(c, "h", h, h.size(1)), rw = rows(c, "w", w, h.size(1));
  a.dtype = c.code; a.M = (int)h.size(0); a.V = (int)w.size(0); a.d = (int)h.size(1);
  a.h = rh.at; a.ldh = rh.ld; a.w = rw.at; a.ldw = rw.ld;
  a.labels = (const int32_t*)vector(c, "labels", tensor(what, "labels", o[2]), a.M, at::kInt);
  a.smoothing = (float)smoothing;
  return c;
}
// (xent...) -> (loss, lse)
PyObject* linear_xent(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 4);
  nmtgan_xent_args a;
  const Common c = xent("linear_xent", o, a);
  Tensor loss = fresh(c, {a.M}, at::kFloat), lse = fresh(c, {a.M}, at::kFloat);
  const size_t bytes = entry.linear_xent_workspace_bytes(&a, 0);
  const Tensor ws = scratch(c, bytes);
  checked(c, run(c, [&](void* st) {
            return entry.linear_xent(&a, (float*)loss.data_ptr(), (float*)lse.data_ptr(), ws.data_ptr(), bytes, st);
          }));
  return pair(std::move(loss), std::move(lse));
  END_HANDLE_TH_ERRORS
}
// (xent..., lse, grad_row, dh, dw) -> (dh, dw)
PyObject* linear_xent_grads(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 8);
  nmtgan_xent_args a;
  const Common c = xent("linear_xent_grads", o, a);
  if (c.type == at::kHalf) refuse(c.what, "bfloat16 or float32 (float16 gradients would underflow without loss scaling)");
  const float* lse = (const float*)vector(c, "lse", tensor(c.what, "lse", o[4]), a.M, at::kFloat);
  const float* g = o[5] == Py_None ? nullptr : (const float*)vector(c, "grad_row", tensor(c.what, "grad_row", o[5]), a.M, at::kFloat);
  Tensor dh = target(c, "dh", o[6], a.M, a.d), dw = target(c, "dw", o[7], a.V, a.d);
  const Rows rh = rows(c, "dh", dh, a.d), rw = rows(c, "dw", dw, a.d);
  const size_t bytes = entry.linear_xent_workspace_bytes(&a, 1);
  const Tensor ws = scratch(c, bytes);
  checked(c, run(c, [&](void* st) {
            return entry.linear_xent_grads(&a, lse, g, rh.at, rh.ld, rw.at, rw.ld, ws.data_ptr(), bytes, st);
          }));
  written(dh);
  written(dw);
  return pair(std::move(dh), std::move(dw));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- global norm
int type_code(at::ScalarType s) { return s == at::kBFloat16 ? NMTGAN_BF16 : s == at::kHalf ? NMTGAN_F16 : s == at::kFloat ? NMTGAN_F32 : -1; }
// The list of o[0] (gradients) and o[1] (where their clipped values go), two Python lists, as the entry points take it.  Made
// anew by every call: a tensor may have been given other memory, another size or type since the last one.
Common refs_of(const char* what, PyObject* const* o, std::vector<nmtgan_grad_ref>& refs) {
  if (!PyList_Check(o[0]) || !PyList_Check(o[1])) refuse(what, "lists of tensors are needed");
  const Py_ssize_t count = PyList_GET_SIZE(o[0]);
  if (count == 0) refuse(what, "no tensors");
  if (PyList_GET_SIZE(o[1]) != count)
    refuse(what, std::to_string(count) + " gradients, " + std::to_string(PyList_GET_SIZE(o[1])) + " outputs");
  const Common c = common(what, "gradient", PyList_GET_ITEM(o[0], 0));
  refs.resize(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor& g = tensor(what, "every gradient", PyList_GET_ITEM(o[0], i));
    const Tensor& to = tensor(what, "every output", PyList_GET_ITEM(o[1], i));
    const bool other = !to.is_same(g);
    const int type = type_code(g.scalar_type()), to_type = other ? type_code(to.scalar_type()) : type;
    if (type < 0 || to_type < 0 || g.device() != c.device || !g.is_contiguous() || (other && (to.device() != c.device || !to.is_contiguous())))
      refuse(what, "tensor " + std::to_string(i) + " must be contiguous, floating and on " + c.device.str());
    const int64_t size = g.numel();
    if (other && (to.numel() != size || (to_type != type && to_type != NMTGAN_F32)))
      refuse(what, "output " + std::to_string(i) + " must have its gradient's size, and its type or float32");
    void* at = g.data_ptr();
    refs[i] = {at, other ? to.data_ptr() : at, size, type, to_type};
  }
  return c;
}
// (gradients, outputs): checks only
PyObject* check_list(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 2);
  std::vector<nmtgan_grad_ref> refs;
  refs_of("TensorList", o, refs);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (gradients, outputs, grad_scale, max_norm or None) -> norm
PyObject* global_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 4);
  const bool clip = o[3] != Py_None;
  const char* what = clip ? "clip_global_norm" : "global_norm";
  std::vector<nmtgan_grad_ref> refs;
  const Common c = refs_of(what, o, refs);
  const nmtgan_grad_ref* list = refs.data();
  const int count = (int)refs.size();
  const size_t bytes = entry.global_norm_workspace_bytes(count);
  const double scale = number(what, "grad_scale", o[2]), most = clip ? number(what, "max_norm", o[3]) : 1.0;
  if (!std::isfinite((float)scale)) refuse(what, "grad_scale=" + std::to_string(scale));
  if (!std::isfinite((float)most) || !((float)most > 0.f)) refuse(what, "max_norm=" + std::to_string(most));
  Tensor norm = fresh(c, {}, at::kFloat);
  const Tensor ws = scratch(c, bytes);
  float* to = (float*)norm.data_ptr();
  checked(c, run(c, [&](void* st) {
            return clip ? entry.clip_global_norm(list, count, (float)most, (float)scale, to, ws.data_ptr(), bytes, st)
                        : entry.global_norm(list, count, (float)scale, to, ws.data_ptr(), bytes, st);
          }));
  for (int i = 0; clip && i < count; ++i) written(THPVariable_Unpack(PyList_GET_ITEM(o[1], i)));
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

// ({name: address}) of every entry point above
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 1);
  auto set = [&](const char* name, auto& to) {
    PyObject* at = PyDict_GetItemString(o[0], name);
    void* p = at ? PyLong_AsVoidPtr(at) : nullptr;
    if (!p) refuse("bind", std::string(name) + " is missing");
    to = (std::decay_t<decltype(to)>)p;
  };
  set("nmtgan_attn_span", entry.attn_span);
  set("nmtgan_attn_span_step_workspace_bytes", entry.attn_span_step_workspace_bytes);
  set("nmtgan_attn_span_step", entry.attn_span_step);
  set("nmtgan_attn_span_grads_workspace_bytes", entry.attn_span_grads_workspace_bytes);
  set("nmtgan_attn_span_grads", entry.attn_span_grads);
  set("nmtgan_linear_xent_workspace_bytes", entry.linear_xent_workspace_bytes);
  set("nmtgan_linear_xent", entry.linear_xent);
  set("nmtgan_linear_xent_grads", entry.linear_xent_grads);
  set("nmtgan_global_norm_workspace_bytes", entry.global_norm_workspace_bytes);
  set("nmtgan_global_norm", entry.global_norm);
  set("nmtgan_clip_global_norm", entry.clip_global_norm);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {"attn_span", (PyCFunction)(void (*)())attn_span, METH_FASTCALL, nullptr},
    {"attn_span_step", (PyCFunction)(void (*)())attn_span_step, METH_FASTCALL, nullptr},
    {"attn_span_grads", (PyCFunction)(void (*)())attn_span_grads, METH_FASTCALL, nullptr},
    {"linear_xent", (PyCFunction)(void (*)())linear_xent, METH_FASTCALL, nullptr},
    {"linear_xent_grads", (PyCFunction)(void (*)())linear_xent_grads, METH_FASTCALL, nullptr},
    {"check_list", (PyCFunction)(void (*)())check_list, METH_FASTCALL, nullptr},
    {"global_norm", (PyCFunction)(void (*)())global_norm, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
