// The calls of the Python package from tensors to the C ABI, in native code.
//
// A decode or verify layer's kernel takes 3-20 us, and the Python form of a call (argument checks,
// views, output allocation, the stream lookup and a ctypes call of a dozen arguments) took 12-21 us of
// host time, so that small layers ran at the host's pace. Each function here takes the usual call as it
// is: plain contiguous, 16-byte aligned tensors of the right types and shapes on the current device.
// Anything else returns None, and the Python form, which handles every other case and raises every
// error, runs instead. A negative QMM4_ERR_* code of the library is returned as an int.
//
// Nothing is kept between calls: every property is read from the tensors on each call. The GIL is
// released around the library's call, as ctypes does.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "qmm4.h"
#include "qmm_cache.h"
#include "qmm_general.h"
#include "qmm_requests.h"

namespace {

decltype(&qmm4_affine_bf16) p_affine = nullptr;
decltype(&qmm4_gate_up_silu_bf16) p_gate_up = nullptr;
decltype(&qmm_affine_general_bf16) p_general = nullptr;
decltype(&qmm4_add_rms_norm_bf16) p_norm = nullptr;
decltype(&qmm4_add_rms_norm_qmm_bf16) p_norm_qmm = nullptr;
decltype(&qmm4_affine_lora_bf16) p_lora = nullptr;
decltype(&qmm4_qk_norm_rope_bf16) p_rope = nullptr;
decltype(&qmm4_sample_bf16) p_sample = nullptr;
decltype(&qmm4_sample_workspace) p_sample_workspace = nullptr;
decltype(&qmm4_cache_plan_words) p_plan_words = nullptr;
decltype(&qmm4_cache_step) p_cache_step = nullptr;
decltype(&qmm4_store_kv_bf16) p_store_kv = nullptr;
decltype(&qmm4_paged_workspace) p_paged_workspace = nullptr;
decltype(&qmm4_paged_attention_bf16) p_paged = nullptr;

// A plain tensor on a HIP device with data on an `align`-byte boundary, or null: no subclass, no wrapper of a
// transform or a mode, nothing whose storage is not its own.
const at::Tensor* strided(PyObject* o, size_t align) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  const c10::DispatchKeySet ks = t.key_set();
  if (ks.has(c10::DispatchKey::Python) || ks.has(c10::DispatchKey::FuncTorchBatched) ||
      ks.has(c10::DispatchKey::FuncTorchGradWrapper) || ks.has(c10::DispatchKey::Functionalize) ||
      ks.has(c10::DispatchKey::Conjugate) || ks.has(c10::DispatchKey::Negative) || ks.has(c10::DispatchKey::Batched))
    return nullptr;
  if (!t.has_storage() || t.numel() == 0) return nullptr;
  if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % align != 0) return nullptr;
  return &t;
}

// The same, contiguous.
const at::Tensor* plain(PyObject* o, size_t align) {
  const at::Tensor* t = strided(o, align);
  return t && t->is_contiguous() ? t : nullptr;
}

// Whether one of the inputs (or null) carries a tangent of forward mode (the Python form raises).
bool has_tangent(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t && t->_fw_grad(0).defined()) return true;
  return false;
}
// Whether a gradient of one of them is asked for, in either mode (the Python form raises).
bool wants_gradient(std::initializer_list<const at::Tensor*> ts) {
  if (has_tangent(ts)) return true;
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

// An index of one value per row: int32 or int64 of `lead` (a tensor's shape without its last `drop` dimensions).
bool is_index(const at::Tensor& t, const at::Tensor& x, int64_t drop) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) &&
         t.sizes() == x.sizes().slice(0, x.dim() - drop);
}
int index_bits(const at::Tensor& t) { return t.scalar_type() == at::kLong ? 64 : 32; }

bool same_current_device(const at::Tensor& x, std::initializer_list<const at::Tensor*> others) {
  const auto d = x.device();
  for (const at::Tensor* t : others)
    if (t->device() != d) return false;
  return d.index() == c10::hip::current_device() && !c10::impl::TorchDispatchModeTLS::any_modes_set();
}

void* stream_of(const at::Tensor& x) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
}

void* ptr(const at::Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }
// A new output's data, or null where a transform hands out a wrapper without storage of its own.
void* out_ptr(const at::Tensor& t) { return t.has_storage() && t.is_cuda() ? ptr(t) : nullptr; }

struct Weights {
  const uint32_t* w;
  const void *s, *b;
  Weights(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& biases)
      : w(static_cast<const uint32_t*>(ptr(codes))), s(ptr(scales)), b(ptr(biases)) {}
};

bool is_codes(const at::Tensor& w) { return w.dim() == 2 && (w.scalar_type() == at::kInt || w.scalar_type() == at::kUInt32); }
bool is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }

// A new tensor on the current device, without the dispatcher's rounds (at::empty takes 0.2 us more: 5.8 us a call of rope, 5.4 with this).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

at::Tensor empty_like_rows(const at::Tensor& x, int64_t n) {
  c10::SmallVector<int64_t, 8> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = n;
  return at::empty(sizes, x.options());
}

// w [n, k * bits / 32] with scales and biases [n, k / group] for x's last dimension k.
bool weights_match(const at::Tensor& w, const at::Tensor& s, const at::Tensor& b, int64_t k, int64_t group, int64_t bits) {
  return is_codes(w) && is_bf16(s) && is_bf16(b) && s.dim() == 2 && b.dim() == 2 && k % group == 0 &&
         w.size(1) * 32 == k * bits && s.size(0) == w.size(0) && b.size(0) == w.size(0) && s.size(1) == k / group &&
         b.size(1) == k / group;
}

// Whether something sees or rewrites torch's own operations (same_current_device declines for dispatch
// modes): the general path's library product is one of them, the kernel is not.
bool observed() {
  return at::impl::torch_function_mode_enabled() ||
         (at::autocast::is_autocast_enabled(at::kCUDA) && at::autocast::get_autocast_dtype(at::kCUDA) != at::kBFloat16);
}

PyObject* none() { Py_RETURN_NONE; }

// `expr` runs without the GIL: it touches no tensor and throws nothing (pointers are taken before).
#define CALL(rc, expr)   \
  Py_BEGIN_ALLOW_THREADS \
  rc = (expr);           \
  Py_END_ALLOW_THREADS

// qmm(x, w, scales, biases, group_size, bits, general): quantized_matmul of 4-bit groups of 64 on the
// packed kernels, or of any format on the general kernel when `general` is true (the caller's rule).
PyObject* qmm(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 7) return none();
  const at::Tensor *x = plain(a[0], 16), *w = plain(a[1], 16), *s = plain(a[2], 16), *b = plain(a[3], 16);
  if (!x || !w || !s || !b || !is_bf16(*x) || x->dim() < 1 || !same_current_device(*x, {w, s, b})) return none();
  const int64_t group = PyLong_AsLongLong(a[4]), bits = PyLong_AsLongLong(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const bool general = a[6] == Py_True;
  const int64_t k = x->sizes().back(), m = x->numel() / k, n = w->size(0);
  if (group <= 0 || bits <= 0 || !weights_match(*w, *s, *b, k, group, bits) || (general && observed())) return none();
  at::Tensor y = empty_like_rows(*x, n);
  const Weights q(*w, *s, *b);
  void *st = stream_of(*x), *xp = ptr(*x), *yp = out_ptr(y);
  if (!yp) return none();
  int rc;
  if (general) {
    CALL(rc, p_general(xp, q.w, q.s, q.b, yp, m, n, k, (int)group, (int)bits, st))
  } else {
    CALL(rc, p_affine(xp, q.w, q.s, q.b, yp, m, n, k, (int)group, (int)bits, 1, st))
  }
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// linear(x, w, scales, biases, w_ptr, scales_ptr, biases_ptr): a bound 4-bit layer; None as well when a
// tensor's data no longer lies where it was bound (the caller rebinds).
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 7) return none();
  const at::Tensor *x = plain(a[0], 16), *w = plain(a[1], 16), *s = plain(a[2], 16), *b = plain(a[3], 16);
  if (!x || !w || !s || !b || !is_bf16(*x) || x->dim() < 1 || !same_current_device(*x, {w, s, b})) return none();
  if (ptr(*w) != PyLong_AsVoidPtr(a[4]) || ptr(*s) != PyLong_AsVoidPtr(a[5]) || ptr(*b) != PyLong_AsVoidPtr(a[6]))
    return PyErr_Occurred() ? nullptr : none();
  const int64_t k = x->sizes().back(), m = x->numel() / k, n = w->size(0);
  if (!weights_match(*w, *s, *b, k, 64, 4)) return none();
  at::Tensor y = empty_like_rows(*x, n);
  const Weights q(*w, *s, *b);
  void *st = stream_of(*x), *xp = ptr(*x), *yp = out_ptr(y);
  if (!yp) return none();
  int rc;
  CALL(rc, p_affine(xp, q.w, q.s, q.b, yp, m, n, k, 64, 4, 1, st))
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// gate_up(x, w, scales, biases): gate_up_silu of 4-bit groups of 64.
PyObject* gate_up(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 4) return none();
  const at::Tensor *x = plain(a[0], 16), *w = plain(a[1], 16), *s = plain(a[2], 16), *b = plain(a[3], 16);
  if (!x || !w || !s || !b || !is_bf16(*x) || x->dim() < 1 || !same_current_device(*x, {w, s, b})) return none();
  const int64_t k = x->sizes().back(), m = x->numel() / k, n = w->size(0);
  if (n % 32 != 0 || !weights_match(*w, *s, *b, k, 64, 4)) return none();
  at::Tensor y = empty_like_rows(*x, n / 2);
  const Weights q(*w, *s, *b);
  void *st = stream_of(*x), *xp = ptr(*x), *yp = out_ptr(y);
  if (!yp) return none();
  int rc;
  CALL(rc, p_gate_up(xp, q.w, q.s, q.b, yp, m, n, k, 64, 4, 1, st))
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// x, r and the norm weight of add_rms_norm: bf16, x and r of one shape, weight of its last dimension.
bool norm_args(const at::Tensor* x, const at::Tensor* r, const at::Tensor* w) {
  return x && r && w && is_bf16(*x) && is_bf16(*r) && is_bf16(*w) && x->dim() >= 1 && x->sizes() == r->sizes() &&
         w->dim() == 1 && w->size(0) == x->sizes().back();
}

// norm(x, r, weight, eps): (h, n) of add_rms_norm.
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 4 || !PyFloat_Check(a[3])) return none();
  const at::Tensor *x = plain(a[0], 16), *r = plain(a[1], 16), *w = plain(a[2], 16);
  if (!norm_args(x, r, w) || !same_current_device(*x, {r, w})) return none();
  const int64_t d = x->sizes().back(), m = x->numel() / d;
  at::Tensor h = at::empty(x->sizes(), x->options()), n = at::empty(x->sizes(), x->options());
  void *st = stream_of(*x), *xp = ptr(*x), *rp = ptr(*r), *wp = ptr(*w), *hp = out_ptr(h), *np = out_ptr(n);
  if (!hp || !np) return none();
  const float eps = (float)PyFloat_AS_DOUBLE(a[3]);
  int rc;
  CALL(rc, p_norm(xp, rp, wp, hp, np, m, d, eps, st))
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(h)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(n)));
  return out;
  END_HANDLE_TH_ERRORS
}

// norm_qmm(x, r, weight, eps, w, scales, biases, silu_mul): (h, n, y) of add_rms_norm_qmm_.
PyObject* norm_qmm(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 8 || !PyFloat_Check(a[3])) return none();
  const at::Tensor *x = plain(a[0], 16), *r = plain(a[1], 16), *nw = plain(a[2], 16), *w = plain(a[4], 16),
                   *s = plain(a[5], 16), *b = plain(a[6], 16);
  if (!norm_args(x, r, nw) || !w || !s || !b || !same_current_device(*x, {r, nw, w, s, b})) return none();
  const bool silu = a[7] == Py_True;
  const int64_t k = x->sizes().back(), m = x->numel() / k, n = w->size(0);
  if ((silu && n % 32 != 0) || !weights_match(*w, *s, *b, k, 64, 4)) return none();
  at::Tensor h = at::empty(x->sizes(), x->options()), nn = at::empty(x->sizes(), x->options());
  at::Tensor y = empty_like_rows(*x, silu ? n / 2 : n);
  const Weights q(*w, *s, *b);
  void *st = stream_of(*x), *xp = ptr(*x), *rp = ptr(*r), *np = ptr(*nw);
  void *hp = out_ptr(h), *nnp = out_ptr(nn), *yp = out_ptr(y);
  if (!hp || !nnp || !yp) return none();
  const float eps = (float)PyFloat_AS_DOUBLE(a[3]);
  int rc;
  CALL(rc, p_norm_qmm(xp, rp, np, eps, hp, nnp, q.w, q.s, q.b, yp, m, n, k, 64, 4, 1,
                      silu ? QMM4_EPILOGUE_SILU_MUL : QMM4_EPILOGUE_NONE, st))
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(h)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(nn)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(y)));
  return out;
  END_HANDLE_TH_ERRORS
}

PyObject* pair(at::Tensor&& a, at::Tensor&& b) {
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(a)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(b)));
  return out;
}

// lora(x, w, scales, biases, lora_a, lora_b, lora_scale, adapters, group_size, bits): quantized_matmul_lora where one
// call of the library does it (the caller's rule).
PyObject* lora(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 10) return none();
  const at::Tensor *x = plain(a[0], 16), *w = plain(a[1], 16), *s = plain(a[2], 16), *b = plain(a[3], 16),
                   *la = plain(a[4], 16), *lb = plain(a[5], 16), *sc = plain(a[6], 4), *ids = plain(a[7], 4);
  if (!x || !w || !s || !b || !la || !lb || !sc || !ids || !is_bf16(*x) || x->dim() < 1 ||
      !same_current_device(*x, {w, s, b, la, lb, sc, ids}) || wants_gradient({x, s, b, la, lb, sc}))
    return none();
  const int64_t group = PyLong_AsLongLong(a[8]), bits = PyLong_AsLongLong(a[9]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t k = x->sizes().back(), m = x->numel() / k, n = w->size(0);
  if (group <= 0 || bits <= 0 || !weights_match(*w, *s, *b, k, group, bits)) return none();
  if (!is_bf16(*la) || !is_bf16(*lb) || la->dim() != 3 || lb->dim() != 3 || la->size(2) != k || lb->size(1) != n ||
      lb->size(0) != la->size(0) || lb->size(2) != la->size(1) || sc->scalar_type() != at::kFloat || sc->dim() != 1 ||
      sc->size(0) != la->size(0) || !is_index(*ids, *x, 1))
    return none();
  const int64_t count = la->size(0), rank = la->size(1);
  at::Tensor y = empty_like_rows(*x, n), ws = fresh({m, rank}, at::kInt, *x);
  const Weights q(*w, *s, *b);
  void *st = stream_of(*x), *xp = ptr(*x), *lap = ptr(*la), *lbp = ptr(*lb), *ip = ptr(*ids), *yp = out_ptr(y),
       *wp = out_ptr(ws);
  const float* sp = static_cast<const float*>(ptr(*sc));
  const int ib = index_bits(*ids);
  if (!yp || !wp) return none();
  int rc;
  CALL(rc, p_lora(xp, q.w, q.s, q.b, lap, lbp, sp, ip, ib, yp, wp, m, n, k, count, rank, (int)group, (int)bits, 1, st))
  return rc == 0 ? THPVariable_Wrap(std::move(y)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// Heads (..., H, D) as rows of heads: the row and head strides, where the leading dimensions are one run of rows and a
// head's values lie together, 16-byte aligned; the rows in *m.
bool heads(const at::Tensor& t, int64_t* m, int64_t* row, int64_t* head) {
  const int64_t n = t.dim(), d = t.size(n - 1);
  if (d > 1 && t.stride(n - 1) != 1) return false;
  *m = 1;
  *row = 0;
  for (int64_t i = n - 3; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (*m == 1) *row = t.stride(i);
    else if (t.stride(i) != *row * *m) return false;
    *m *= t.size(i);
  }
  *head = t.size(n - 2) > 1 ? t.stride(n - 2) : 0;
  return *row % 8 == 0 && *head % 8 == 0 && *row >= 0 && *head >= 0;
}

// rope(q, k, q_weight, k_weight, eps, positions, inv_freq, interleaved): (q', k') of qk_norm_rope.
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 8 || !PyFloat_Check(a[4])) return none();
  const at::Tensor *q = strided(a[0], 16), *k = strided(a[1], 16), *wq = plain(a[2], 16), *wk = plain(a[3], 16),
                   *pos = plain(a[5], 4), *inv = plain(a[6], 4);
  if (!q || !k || !wq || !wk || !pos || !inv || !is_bf16(*q) || !is_bf16(*k) || !is_bf16(*wq) || !is_bf16(*wk) ||
      q->dim() < 2 || k->dim() != q->dim() || !same_current_device(*q, {k, wq, wk, pos, inv}) || wants_gradient({q, k, inv}) ||
      has_tangent({wq, wk}))
    return none();
  const int64_t n = q->dim(), d = q->size(n - 1), p = inv->numel();
  if (q->sizes().slice(0, n - 2) != k->sizes().slice(0, n - 2) || k->size(n - 1) != d || wq->dim() != 1 || wk->dim() != 1 ||
      wq->size(0) != d || wk->size(0) != d || inv->dim() != 1 || 2 * p > d || !is_index(*pos, *q, 2) ||
      (inv->scalar_type() != at::kFloat && inv->scalar_type() != at::kDouble))
    return none();
  int64_t m, mk, qr, qh, kr, kh;
  if (!heads(*q, &m, &qr, &qh) || !heads(*k, &mk, &kr, &kh)) return none();
  at::Tensor qo = fresh(q->sizes(), at::kBFloat16, *q), ko = fresh(k->sizes(), at::kBFloat16, *k);
  void *st = stream_of(*q), *qp = ptr(*q), *kp = ptr(*k), *wqp = ptr(*wq), *wkp = ptr(*wk), *pp = ptr(*pos), *ip = ptr(*inv);
  void *qop = out_ptr(qo), *kop = out_ptr(ko);
  if (!qop || !kop) return none();
  const float eps = (float)PyFloat_AS_DOUBLE(a[4]);
  const int pb = index_bits(*pos), fb = inv->scalar_type() == at::kDouble ? 64 : 32, il = a[7] == Py_True;
  const int64_t hq = q->size(n - 2), hk = k->size(n - 2);
  int rc;
  CALL(rc, p_rope(qp, qr, qh, kp, kr, kh, wqp, wkp, eps, pp, pb, ip, fb, qop, kop, m, hq, hk, d, p, il, st))
  return rc == 0 ? pair(std::move(qo), std::move(ko)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// A setting of sample: a number (checked by the caller) or a tensor of one value per row. False: neither.
bool setting(PyObject* o, at::ScalarType type, const at::Tensor& logits, const at::Tensor** t, double* value) {
  *t = nullptr;
  if (THPVariable_Check(o)) {
    *t = plain(o, 4);
    return *t && (*t)->scalar_type() == type && (*t)->sizes() == logits.sizes().slice(0, logits.dim() - 1);
  }
  if (PyFloat_CheckExact(o)) *value = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *value = PyLong_AsDouble(o);
  else return false;
  return !PyErr_Occurred();
}

// sample(logits, uniform, temperature, top_k, top_p, min_p): (tokens, logprobs) of sample.
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 6) return none();
  const at::Tensor *l = strided(a[0], 2), *u = plain(a[1], 4);
  if (!l || !u || !is_bf16(*l) || l->dim() < 1 || u->scalar_type() != at::kFloat ||
      u->sizes() != l->sizes().slice(0, l->dim() - 1))
    return none();
  const int64_t n = l->dim(), v = l->size(n - 1), m = l->numel() / v;
  const int64_t stride = n == 1 ? v : l->stride(n - 2);
  if (n > 2 ? !l->is_contiguous() : (v > 1 && l->stride(n - 1) != 1) || (m > 1 && stride < v)) return none();
  const at::Tensor *t, *k, *p, *mp;
  double tv = 0, kv = 0, pv = 0, mv = 0;
  if (!setting(a[2], at::kFloat, *l, &t, &tv) || !setting(a[3], at::kInt, *l, &k, &kv) ||
      !setting(a[4], at::kFloat, *l, &p, &pv) || !setting(a[5], at::kFloat, *l, &mp, &mv)) {
    PyErr_Clear();
    return none();
  }
  if ((!t && !(tv >= 0 && tv <= 1e30)) || (!k && !(kv >= 0 && kv < 2147483648.0)) || (!p && !(pv > 0 && pv <= 1)) ||
      (!mp && !(mv >= 0 && mv <= 1)))
    return none();  // (out of range: the Python form raises)
  if (wants_gradient({l, u, t, p, mp})) return none();
  for (const at::Tensor* x : {u, t, k, p, mp})
    if (x && x->device() != l->device()) return none();
  if (!same_current_device(*l, {u})) return none();
  const int64_t bytes = p_sample_workspace(m, v);
  if (bytes < 0) return PyLong_FromLong((long)bytes);
  const auto lead = l->sizes().slice(0, n - 1);
  at::Tensor tokens = fresh(lead, at::kLong, *l), logprobs = fresh(lead, at::kFloat, *l);
  at::Tensor ws = fresh({bytes}, at::kByte, *l);
  void *tp = out_ptr(tokens), *pp = out_ptr(logprobs), *wp = out_ptr(ws), *st = stream_of(*l), *lp = ptr(*l);
  if (!tp || !pp || !wp) return none();
  auto f = [](const at::Tensor* x) { return x ? static_cast<const float*>(ptr(*x)) : nullptr; };
  const float *up = f(u), *t_p = f(t), *p_p = f(p), *m_p = f(mp);
  const int32_t* k_p = k ? static_cast<const int32_t*>(ptr(*k)) : nullptr;
  int rc;
  CALL(rc, p_sample(lp, m, v, stride, up, t_p, (float)tv, k_p, (int32_t)kv, p_p, (float)pv, m_p, (float)mv,
                    static_cast<int64_t*>(tp), static_cast<float*>(pp), wp, st))
  return rc == 0 ? pair(std::move(tokens), std::move(logprobs)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// A tensor of `type` and `sizes`.
bool is_table(const at::Tensor& t, at::ScalarType type, at::IntArrayRef sizes) {
  return t.scalar_type() == type && t.sizes() == sizes;
}

// Integers from..from + N - 1 of a call's arguments. False: not all are integers.
template <int N>
bool integers(PyObject* const* a, int from, int64_t (&out)[N]) {
  for (int i = 0; i < N; ++i) {
    if (!PyLong_CheckExact(a[from + i])) return false;
    out[i] = PyLong_AsLongLong(a[from + i]);
    if (out[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  }
  return true;
}

// An optional tensor: null where the argument is None. False: neither.
bool optional(PyObject* o, size_t align, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || (*t = plain(o, align));
}

// cache_step(lengths, block_table, free_pages, free_count, rows, total, page_size, heads, kv_heads, head_dim, base, keep,
// max_rows): (slots, positions, request, plan) of step_tables_.
PyObject* cache_step(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 13) return none();
  const at::Tensor *len = plain(a[0], 4), *tab = plain(a[1], 4), *fp = plain(a[2], 4), *fc = plain(a[3], 4), *rows = plain(a[4], 4);
  const at::Tensor *base, *keep;
  int64_t v[5], most[1];  // total, page_size, heads, kv_heads, head_dim; max_rows
  if (!len || !tab || !fp || !fc || !rows || !integers(a, 5, v) || !optional(a[10], 4, &base) || !optional(a[11], 1, &keep) ||
      !integers(a, 12, most) || len->dim() != 1 || tab->dim() != 2 || fp->dim() != 1)
    return none();
  const int64_t r = len->size(0), capacity = tab->size(1), pages = fp->size(0), total = v[0];
  if (total < 0 || !is_table(*len, at::kInt, {r}) || !is_table(*tab, at::kInt, {r, capacity}) || !is_table(*fp, at::kInt, {pages}) ||
      !is_table(*fc, at::kInt, {1}) || !is_table(*rows, at::kInt, {r}) || (base && !is_table(*base, at::kInt, {r})) ||
      (keep && !is_table(*keep, at::kBool, {total})) ||
      (v[4] != 64 && v[4] != 96 && v[4] != 128 && v[4] != 192 && v[4] != 256))
    return none();
  for (const at::Tensor* t : {base, keep})
    if (t && t->device() != len->device()) return none();
  if (!same_current_device(*len, {tab, fp, fc, rows})) return none();
  const int64_t words = p_plan_words(r, v[2], v[3], v[4], most[0]);
  if (words < 0 || total > (keep ? QMM4_CACHE_MAX_KEEP : QMM4_CACHE_MAX_ROWS)) return none();  // (the Python form raises)
  at::Tensor slots = fresh({total}, at::kInt, *len), positions = fresh({total}, at::kInt, *len),
             request = fresh({total}, at::kInt, *len), plan;
  if (!keep) plan = fresh({words}, at::kInt, *len);
  auto i32 = [](const at::Tensor* t) { return t ? static_cast<int32_t*>(ptr(*t)) : nullptr; };
  auto out = [](const at::Tensor& t) { return static_cast<int32_t*>(out_ptr(t)); };
  int32_t *sp = out(slots), *pp = out(positions), *rp = out(request), *plp = keep ? nullptr : out(plan);
  if ((total > 0 && (!sp || !pp || !rp)) || (!keep && !plp)) return none();
  int32_t *lenp = i32(len), *tabp = i32(tab), *fpp = i32(fp), *fcp = i32(fc), *rowsp = i32(rows), *basep = i32(base);
  const uint8_t* keepp = keep ? static_cast<const uint8_t*>(ptr(*keep)) : nullptr;
  void* st = stream_of(*len);
  int rc;
  CALL(rc, p_cache_step(lenp, tabp, fpp, fcp, rowsp, basep, keepp, sp, pp, rp, plp, r, capacity, pages, total, most[0], v[1],
                        v[2], v[3], v[4], st))
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject* o = PyTuple_New(4);
  if (!o) return nullptr;
  PyTuple_SET_ITEM(o, 0, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(o, 1, THPVariable_Wrap(std::move(positions)));
  PyTuple_SET_ITEM(o, 2, THPVariable_Wrap(std::move(request)));
  PyTuple_SET_ITEM(o, 3, keep ? none() : THPVariable_Wrap(std::move(plan)));
  return o;
  END_HANDLE_TH_ERRORS
}

// A layer's cache (keys, values, key_scales, value_scales): a KVCache of these arguments.
struct Cache {
  const at::Tensor *keys, *values, *ks, *vs;
  int64_t pages, heads, dim, page;
  int bits;
  bool read(PyObject* const* a) {
    keys = plain(a[0], 16);
    values = plain(a[1], 16);
    if (!keys || !values || !optional(a[2], 16, &ks) || !optional(a[3], 16, &vs) || keys->dim() != 5) return false;
    const bool codes = keys->scalar_type() == at::kChar;
    if (!codes && !is_bf16(*keys)) return false;
    bits = codes ? 8 : 16;
    const int64_t e = codes ? 16 : 8;
    pages = keys->size(0);
    heads = keys->size(1);
    dim = keys->size(2) * e;
    page = keys->size(3);
    if (keys->size(4) != e || page % e != 0 || codes != (ks != nullptr) || codes != (vs != nullptr) ||
        !is_table(*values, keys->scalar_type(), {pages, heads, page / e, dim, e}))
      return false;
    for (const at::Tensor* t : {ks, vs})
      if (t && (!is_table(*t, at::kFloat, {pages, heads, page}) || t->device() != keys->device())) return false;
    return !wants_gradient({keys, values, ks, vs});
  }
};

// store_kv(k, v, keys, values, key_scales, value_scales, slots): store_kv_ (0).
PyObject* store_kv(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 7) return none();
  const at::Tensor *k = strided(a[0], 16), *v = strided(a[1], 16), *slots = plain(a[6], 4);
  Cache c;
  if (!k || !v || !slots || !c.read(a + 2) || !is_bf16(*k) || !is_bf16(*v) || k->dim() != 3 || v->sizes() != k->sizes() ||
      k->size(1) != c.heads || k->size(2) != c.dim || !is_table(*slots, at::kInt, {k->size(0)}) ||
      !same_current_device(*k, {v, slots, c.keys, c.values}) || wants_gradient({k, v}))
    return none();
  int64_t m, mv, kr, kh, vr, vh;
  if (!heads(*k, &m, &kr, &kh) || !heads(*v, &mv, &vr, &vh)) return none();
  void *st = stream_of(*k), *kp = ptr(*k), *vp = ptr(*v), *keys = ptr(*c.keys), *values = ptr(*c.values);
  const int32_t* sp = static_cast<const int32_t*>(ptr(*slots));
  float *ks = c.ks ? static_cast<float*>(ptr(*c.ks)) : nullptr, *vs = c.vs ? static_cast<float*>(ptr(*c.vs)) : nullptr;
  int rc;
  CALL(rc, p_store_kv(kp, kr, kh, vp, vr, vh, sp, keys, values, ks, vs, m, c.heads, c.dim, c.pages, c.page, c.bits, st))
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// paged(q, keys, values, key_scales, value_scales, block_table, request, plan, heads, kv_heads, head_dim, max_rows, page_size,
// scale, ancestors, gate): paged_attention's output. Without q (None): True where a call with the step's rows would be made.
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t na) {
  HANDLE_TH_ERRORS
  if (na != 16 || !PyFloat_CheckExact(a[13])) return none();
  const bool ask = a[0] == Py_None;
  const at::Tensor *q = ask ? nullptr : strided(a[0], 16), *tab = plain(a[5], 4), *req = plain(a[6], 4), *plan = plain(a[7], 4), *anc;
  const at::Tensor* gate = a[15] == Py_None ? nullptr : strided(a[15], 16);
  Cache c;
  int64_t v[5];  // heads, kv_heads, head_dim, max_rows, page_size
  if ((!q && !ask) || !tab || !req || !plan || (a[15] != Py_None && !gate) || !c.read(a + 1) || !optional(a[14], 8, &anc) ||
      !integers(a, 8, v) || (q && (!is_bf16(*q) || q->dim() != 3)) || tab->dim() != 2 || req->dim() != 1)
    return none();
  const int64_t m = req->size(0), r = tab->size(0), capacity = tab->size(1);
  if (v[1] != c.heads || v[2] != c.dim || v[4] != c.page || !is_table(*tab, at::kInt, {r, capacity}) ||
      req->scalar_type() != at::kInt || plan->scalar_type() != at::kInt || (anc && !is_table(*anc, at::kLong, {m})) ||
      !same_current_device(*req, {tab, plan, c.keys, c.values}) || (anc && anc->device() != req->device()))
    return none();
  if (plan->dim() != 1 || plan->size(0) != p_plan_words(r, v[0], v[1], v[2], v[3])) return none();
  if (ask) {
    if (!std::isfinite((float)PyFloat_AS_DOUBLE(a[13])) || (m > 0 && (c.pages == 0 || capacity == 0))) return none();
    Py_RETURN_TRUE;
  }
  if (q->size(0) != m || q->size(1) != v[0] || q->size(2) != c.dim || q->device() != req->device() ||
      (gate && (!is_bf16(*gate) || gate->sizes() != q->sizes() || gate->device() != q->device())) || wants_gradient({q, gate}))
    return none();
  int64_t mq, qr, qh, gr = 0, gh = 0;
  if (!heads(*q, &mq, &qr, &qh) || (gate && !heads(*gate, &mq, &gr, &gh))) return none();
  const int64_t bytes = p_paged_workspace(m, r, v[0], v[1], v[2], v[3]);
  if (bytes < 0) return PyLong_FromLong((long)bytes);
  at::Tensor out = fresh(q->sizes(), at::kBFloat16, *q), ws = fresh({bytes}, at::kByte, *q);
  void *op = out_ptr(out), *wp = out_ptr(ws), *st = stream_of(*q), *qp = ptr(*q), *keys = ptr(*c.keys), *values = ptr(*c.values),
       *gp = gate ? ptr(*gate) : nullptr;
  if (!op || !wp) return none();
  const float *ks = c.ks ? static_cast<const float*>(ptr(*c.ks)) : nullptr,
              *vs = c.vs ? static_cast<const float*>(ptr(*c.vs)) : nullptr;
  const int32_t *tabp = static_cast<const int32_t*>(ptr(*tab)), *reqp = static_cast<const int32_t*>(ptr(*req)),
                *planp = static_cast<const int32_t*>(ptr(*plan));
  const int64_t* ancp = anc ? static_cast<const int64_t*>(ptr(*anc)) : nullptr;
  const float scale = (float)PyFloat_AS_DOUBLE(a[13]);
  int rc;
  CALL(rc, p_paged(qp, qr, qh, keys, values, ks, vs, tabp, reqp, planp, ancp, gp, gr, gh, op, wp, scale, m, r, v[0], v[1], v[2],
                   c.pages, c.page, capacity, v[3], c.bits, st))
  return rc == 0 ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// bind(affine, gate_up, general, norm, norm_qmm, lora, rope, sample, sample_workspace, cache_plan_words, cache_step, store_kv,
// paged_workspace, paged_attention): the addresses of the loaded library's functions.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t na) {
  constexpr int kFunctions = 14;
  if (na != kFunctions) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kFunctions);
    return nullptr;
  }
  void* p[kFunctions];
  for (int i = 0; i < kFunctions; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function address");
      return nullptr;
    }
  }
  p_affine = reinterpret_cast<decltype(p_affine)>(p[0]);
  p_gate_up = reinterpret_cast<decltype(p_gate_up)>(p[1]);
  p_general = reinterpret_cast<decltype(p_general)>(p[2]);
  p_norm = reinterpret_cast<decltype(p_norm)>(p[3]);
  p_norm_qmm = reinterpret_cast<decltype(p_norm_qmm)>(p[4]);
  p_lora = reinterpret_cast<decltype(p_lora)>(p[5]);
  p_rope = reinterpret_cast<decltype(p_rope)>(p[6]);
  p_sample = reinterpret_cast<decltype(p_sample)>(p[7]);
  p_sample_workspace = reinterpret_cast<decltype(p_sample_workspace)>(p[8]);
  p_plan_words = reinterpret_cast<decltype(p_plan_words)>(p[9]);
  p_cache_step = reinterpret_cast<decltype(p_cache_step)>(p[10]);
  p_store_kv = reinterpret_cast<decltype(p_store_kv)>(p[11]);
  p_paged_workspace = reinterpret_cast<decltype(p_paged_workspace)>(p[12]);
  p_paged = reinterpret_cast<decltype(p_paged)>(p[13]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&bind)), METH_FASTCALL, nullptr},
    {"qmm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&qmm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&linear)), METH_FASTCALL, nullptr},
    {"gate_up", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&gate_up)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&norm)), METH_FASTCALL, nullptr},
    {"norm_qmm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&norm_qmm)), METH_FASTCALL, nullptr},
    {"lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&lora)), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&rope)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&sample)), METH_FASTCALL, nullptr},
    {"cache_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&cache_step)), METH_FASTCALL, nullptr},
    {"store_kv", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&store_kv)), METH_FASTCALL, nullptr},
    {"paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&paged)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
  PyObject* m = PyModule_Create(&module);
  // The torch this was built for (the loader refuses another: ATen's layouts are not stable).
  if (m && PyModule_AddStringConstant(m, "TORCH_VERSION", QMM4_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
