// The per-layer operators' way from Python to the C ABI (wnw_amd/_callpath.so).
//
// A decode step calls the attention once per layer; at a minute of audio the
// device needs ~10 us for it, and checking nine tensors, taking their pointers
// and converting ~20 arguments in Python took 13.7 us (now 5.1, 3.4 of them the
// launch: 30 layers of 2,586 rows 425 -> 293 us).  The functions here do
// the same for a call in its plain form: ordinary device tensors, contiguous,
// of the types and shapes the operator documents.  For any other call they
// return None and launch nothing, and the Python operator checks, copies
// or refuses as it always does, so no message or conversion is repeated here.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

#include "../../include/wnw_amd.h"

namespace {

PyObject* g_stream = nullptr;     // (device index) -> raw stream
PyObject* g_workspace = nullptr;  // (device index, stream, n_seg, group, head_dim) -> buffer tensor
PyObject* g_score_ws = nullptr;   // (device index, stream, items, heads) -> buffer tensor
PyObject* g_paged_ws = nullptr;   // (device index, stream, n_seg, bytes) -> buffer tensor, its counters zero
PyObject* g_check = nullptr;      // (status, what): raises

// A plain tensor in device memory: no subclass, and no wrapper of a
// transform (vmap, grad levels, functionalisation) around the data.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
  constexpr c10::DispatchKeySet wrapped(
      {c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
       c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::Conjugate,
       c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  if (t.key_set().has_any(wrapped)) return nullptr;
  return &t;
}
const at::Tensor* vec(PyObject* o, at::ScalarType type, int64_t n) {  // contiguous, n elements
  const at::Tensor* t = plain(o);
  return t && t->scalar_type() == type && t->numel() == n && t->is_contiguous() ? t : nullptr;
}
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? WNW_F32 : t == at::kHalf ? WNW_F16 : t == at::kBFloat16 ? WNW_BF16 : -1;
}
// [rows, d] with contiguous rows (rows > 0)
bool row_major(const at::Tensor& t, int64_t d) {
  return t.dim() == 2 && t.size(0) > 0 && t.size(1) == d && t.stride(1) == 1 && t.stride(0) == d;
}
bool number(PyObject* o, double* x) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  *x = PyFloat_AsDouble(o);
  if (*x != -1.0 || !PyErr_Occurred()) return true;
  PyErr_Clear();  // beyond the type's range: the general path's to judge
  return false;
}
bool whole(PyObject* o, int64_t* x) {
  if (!PyLong_CheckExact(o)) return false;
  *x = PyLong_AsLongLong(o);
  if (*x != -1 || !PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

struct Ref {  // an owned reference
  PyObject* o;
  explicit Ref(PyObject* x) : o(x) {}
  ~Ref() { Py_XDECREF(o); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

// The current raw stream of a device, false with an exception set.
bool stream_of(int64_t index, PyObject** stream_obj, void** stream) {
  Ref idx(PyLong_FromLongLong(index));
  if (!idx.o) return false;
  *stream_obj = PyObject_CallOneArg(g_stream, idx.o);
  if (!*stream_obj) return false;
  *stream = PyLong_AsVoidPtr(*stream_obj);
  return !PyErr_Occurred();
}
const at::Tensor* buffer(const Ref& r) {
  if (!r.o) return nullptr;
  if (!THPVariable_Check(r.o)) {
    PyErr_SetString(PyExc_TypeError, "the workspace callback must return a tensor");
    return nullptr;
  }
  return &THPVariable_Unpack(r.o);
}
// Raises for a failed launch.
PyObject* failed(int rc, const char* what) {
  Ref r(PyObject_CallFunction(g_check, "is", rc, what));
  if (r.o) PyErr_SetString(PyExc_RuntimeError, what);
  return nullptr;
}

PyObject* attn_impl(PyObject* const* a) {
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
  if (!q || !k || !v || q->dim() != 3 || !q->is_contiguous()) Py_RETURN_NONE;
  const int64_t n = q->size(0), g = q->size(1), d = q->size(2);
  const int dt = dtype_code(q->scalar_type());
  if (n < 1 || dt < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
      !row_major(*k, d) || !row_major(*v, d) || k->size(0) != v->size(0))
    Py_RETURN_NONE;
  const at::Tensor* cu = vec(a[3], at::kInt, n + 1);
  double scale = 0;
  if (!cu || !number(a[4], &scale)) Py_RETURN_NONE;
  const at::Tensor* base = nullptr;
  if (a[5] != Py_None && !(base = vec(a[5], at::kLong, n))) Py_RETURN_NONE;
  int64_t rows = k->size(0);
  if (a[6] == Py_None ? base != nullptr : !whole(a[6], &rows)) Py_RETURN_NONE;
  const at::Tensor *nk = nullptr, *nv = nullptr, *cu_new = nullptr, *cap = nullptr;
  if (a[8] != Py_None) {
    if (!base || !PyTuple_CheckExact(a[8]) || PyTuple_GET_SIZE(a[8]) != 4) Py_RETURN_NONE;
    nk = vec(PyTuple_GET_ITEM(a[8], 0), q->scalar_type(), n * d);
    nv = vec(PyTuple_GET_ITEM(a[8], 1), q->scalar_type(), n * d);
    cu_new = vec(PyTuple_GET_ITEM(a[8], 2), at::kInt, n + 1);
    cap = vec(PyTuple_GET_ITEM(a[8], 3), at::kInt, n);
    if (!nk || !nv || !cu_new || !cap || nk->dim() != 2 || nv->dim() != 2 || nk->size(0) != n || nv->size(0) != n ||
        cu_new->data_ptr() == cu->data_ptr())
      Py_RETURN_NONE;
  }
  const int64_t dev = q->device().index();
  at::Tensor out;
  Ref given(nullptr);
  if (a[7] != Py_None) {
    const at::Tensor* o = plain(a[7]);
    if (!o) Py_RETURN_NONE;
    out = *o;
    given.o = Py_NewRef(a[7]);
  } else {
    out = at::empty({n, g, d}, q->options().requires_grad(false));
  }
  PyObject* so = nullptr;
  void* stream = nullptr;
  const bool has_stream = stream_of(dev, &so, &stream);
  Ref stream_ref(so);
  if (!has_stream) return nullptr;
  Ref ws(PyObject_CallFunction(g_workspace, "LOLLL", (long long)dev, so, (long long)n, (long long)g, (long long)d));
  const at::Tensor* buf = buffer(ws);
  if (!buf) return nullptr;
  void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr(), *op = out.data_ptr(), *wp = buf->data_ptr();
  const int64_t wbytes = buf->numel(), kv_rows = k->size(0);
  const int32_t* cup = cu->const_data_ptr<int32_t>();
  const int64_t* bp = base ? base->const_data_ptr<int64_t>() : nullptr;
  const char* what = nk ? "decode_attn_append" : "decode_attn";
  void *nkp = nk ? nk->data_ptr() : nullptr, *nvp = nv ? nv->data_ptr() : nullptr;
  int32_t* cnp = cu_new ? cu_new->data_ptr<int32_t>() : nullptr;
  const int32_t* cpp = cap ? cap->const_data_ptr<int32_t>() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (nkp)
    rc = wnw_decode_attn_append(qp, kp, vp, nkp, nvp, cup, cnp, bp, cpp, n, g, d, rows, kv_rows, (float)scale, dt, op, wp,
                                wbytes, stream);
  else
    rc = wnw_decode_attn(qp, kp, vp, cup, bp, n, g, d, rows, kv_rows, (float)scale, dt, op, wp, wbytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, what);
  if (given.o) return Py_NewRef(given.o);
  return THPVariable_Wrap(std::move(out));
}

PyObject* score_impl(PyObject* const* a) {
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]);
  if (!q || !k || q->dim() != 3 || !q->is_contiguous()) Py_RETURN_NONE;
  const int64_t n = q->size(0), h = q->size(1), d = q->size(2);
  const int dt = dtype_code(q->scalar_type());
  if (n < 1 || h < 1 || dt < 0 || k->scalar_type() != q->scalar_type() || !row_major(*k, d)) Py_RETURN_NONE;
  const at::Tensor* idx[4];
  for (int i = 0; i < 4; ++i)
    if (!(idx[i] = vec(a[2 + i], at::kInt, n))) Py_RETURN_NONE;
  const at::Tensor *acc = plain(a[6]), *off = plain(a[7]);
  if (!acc || acc->scalar_type() != at::kFloat || !acc->is_contiguous() || !off || off->scalar_type() != at::kInt ||
      !off->is_contiguous() || off->numel() < n + 1)
    Py_RETURN_NONE;
  int64_t max_audio = 0;
  if (!whole(a[8], &max_audio) || max_audio <= 0) Py_RETURN_NONE;
  double scale = 0;
  if (!number(a[9], &scale)) Py_RETURN_NONE;
  const int64_t dev = q->device().index();
  PyObject* so = nullptr;
  void* stream = nullptr;
  const bool has_stream = stream_of(dev, &so, &stream);
  Ref stream_ref(so);
  if (!has_stream) return nullptr;
  Ref ws(PyObject_CallFunction(g_score_ws, "LOLL", (long long)dev, so, (long long)n, (long long)h));
  const at::Tensor* buf = buffer(ws);
  if (!buf) return nullptr;
  void *qp = q->data_ptr(), *kp = k->data_ptr(), *wp = buf->data_ptr();
  const int32_t* ip[4];
  for (int i = 0; i < 4; ++i) ip[i] = idx[i]->const_data_ptr<int32_t>();
  float* ap = acc->data_ptr<float>();
  const int32_t* fp = off->const_data_ptr<int32_t>();
  const int64_t k_rows = k->size(0), alen = acc->numel(), wbytes = buf->numel();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_fused_score_accumulate(qp, kp, ip[0], ip[1], ip[2], ip[3], ap, fp, n, h, d, k_rows, alen, max_audio,
                                  (float)scale, dt, wp, wbytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "fused_score_accumulate");
  Py_RETURN_TRUE;
}

// The paged cache's operators.  Their tensors may be on another device than
// the current one, and a call that would need a gradient (or has a tangent), or
// that may be traced, is left to the general path's refusal.
bool needs_grad(const at::Tensor* t) {
  return t && ((c10::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined());
}
bool watched() {
  return c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer) || c10::impl::TorchDispatchModeTLS::any_modes_set();
}

bool paged_cache(PyObject* const* a, PyObject* ks, PyObject* vs, const at::Tensor& q, wnw_paged_cache* c,
                 const int32_t** seg_len) {
  const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *table = plain(a[2]), *len = plain(a[3]);
  if (watched() || !k || !v || !table || !len || k->dim() != 3 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type())
    return false;
  const at::ScalarType dt = k->scalar_type();
  const bool q8 = dt == at::kFloat8_e4m3fn;
  if (!q8 && dt != q.scalar_type()) return false;
  const int64_t P = k->size(0), R = k->size(1), D = k->size(2);
  if (P < 1 || R < 1 || k->stride(2) != 1 || v->stride(2) != 1 || k->stride(1) != D || v->stride(1) != D) return false;
  if (table->dim() != 2 || table->scalar_type() != at::kInt || (table->size(1) > 1 && table->stride(1) != 1)) return false;
  const int64_t N = table->size(0), M = table->size(1);
  if (N < 1 || len->scalar_type() != at::kInt || len->dim() != 1 || len->size(0) != N || !len->is_contiguous()) return false;
  const at::Tensor* sc[2] = {nullptr, nullptr};
  PyObject* const so[2] = {ks, vs};
  for (int i = 0; i < 2; ++i) {
    if (!q8) {
      if (so[i] != Py_None) return false;
      continue;
    }
    if (!(sc[i] = vec(so[i], at::kFloat, P)) || sc[i]->dim() != 1 || sc[i]->device() != q.device()) return false;
  }
  const at::Tensor* const all[] = {k, v, table, len, sc[0], sc[1]};
  for (const at::Tensor* t : all)
    if (t && (t->device() != q.device() || needs_grad(t))) return false;
  c->k_pages = k->data_ptr();
  c->v_pages = v->data_ptr();
  c->k_scale = sc[0] ? sc[0]->data_ptr<float>() : nullptr;
  c->v_scale = sc[1] ? sc[1]->data_ptr<float>() : nullptr;
  c->page_table = table->const_data_ptr<int32_t>();
  c->n_seg = N;
  c->n_pages = P;
  c->max_blocks = M;
  c->page_rows = R;
  c->head_dim = D;
  c->k_stride = P > 1 ? k->stride(0) : R * D;
  c->v_stride = P > 1 ? v->stride(0) : R * D;
  c->table_stride = N > 1 ? table->stride(0) : M;
  c->page_dtype = q8 ? WNW_E4M3 : dtype_code(dt);
  *seg_len = len->const_data_ptr<int32_t>();
  return true;
}
// wnw_init once per device, with that device current: not for the first time in a graph's capture, if the caller has
// made any call before it
bool ready(int64_t dev) {
  static uint64_t done = 0;  // under the GIL
  if (dev < 0 || dev >= 64) return wnw_init() == WNW_OK;
  if (!(done >> dev & 1) && wnw_init() == WNW_OK) done |= 1ull << dev;
  return done >> dev & 1;
}
// [tokens, heads, dim] that the kernels take as it lies
bool heads(const at::Tensor& t, int64_t dim) {
  if (t.dim() != 3 || t.size(2) != dim || t.size(0) < 1 || t.size(1) < 1 || t.stride(2) != 1 ||
      (uintptr_t)t.const_data_ptr() % 16 != 0)
    return false;
  for (int i = 0; i < 2; ++i)
    if (t.stride(i) < 0 || t.stride(i) % 8 != 0) return false;
  return true;
}
bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool usable(const at::Tensor* t, const at::Tensor& q) { return t && t->device() == q.device() && !needs_grad(t); }
// cu_tokens [B + 1] and the most tokens of a sample (None: all)
bool tokens_of(PyObject* cu_obj, PyObject* most_obj, const at::Tensor& q, int64_t n_seg, const int32_t** cu, int64_t* samples,
               int64_t* most) {
  const at::Tensor* t = plain(cu_obj);
  if (!usable(t, q) || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) < 2 || !t->is_contiguous()) return false;
  *samples = t->size(0) - 1;
  *most = q.size(0);
  int64_t given = 0;
  if (most_obj != Py_None) {
    if (!whole(most_obj, &given) || given < 1) return false;
    *most = std::min(*most, given);
  }
  *cu = t->const_data_ptr<int32_t>();
  return n_seg % *samples == 0;
}
// Where the result goes: the tensor given, or a new one
bool result(PyObject* given, const at::Tensor& q, at::Tensor* out) {
  if (given == Py_None) {
    *out = at::empty(q.sizes(), q.options().requires_grad(false));
    return true;
  }
  const at::Tensor* o = plain(given);
  if (!usable(o, q) || o->scalar_type() != q.scalar_type() || o->sizes() != q.sizes() || !heads(*o, q.size(2))) return false;
  *out = *o;
  return true;
}

// A window and sinks: int32 [n_seg] tensors, or numbers (sinks: None, for none).
struct View {
  const int32_t *window = nullptr, *sinks = nullptr;
  int64_t window_all = 0, sinks_all = 0;
};
bool view_of(PyObject* window, PyObject* sinks, const at::Tensor& q, int64_t n_seg, View* y) {
  PyObject* const o[2] = {window, sinks};
  const int32_t** p[2] = {&y->window, &y->sinks};
  int64_t* all[2] = {&y->window_all, &y->sinks_all};
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && o[i] == Py_None) continue;
    if (whole(o[i], all[i])) {
      if (*all[i] < 0) return false;
      continue;
    }
    const at::Tensor* t = vec(o[i], at::kInt, n_seg);
    if (!usable(t, q) || t->dim() != 1) return false;
    *p[i] = t->const_data_ptr<int32_t>();
  }
  return true;
}

// (q, k_pages, v_pages, page_table, seg_len, scale, k_scale, v_scale, out), WIN: and (window, sinks)
template <bool WIN>
PyObject* paged_decode_impl(PyObject* const* a) {
  const at::Tensor* q = plain(a[0]);
  wnw_paged_cache c;
  const int32_t* len;
  double scale = 0;
  at::Tensor out;
  if (!q || !half_type(*q) || needs_grad(q) || q->dim() != 3 || !q->is_contiguous() ||
      !paged_cache(a + 1, a[6], a[7], *q, &c, &len) || q->size(0) != c.n_seg || !heads(*q, c.head_dim) || q->size(1) > 16 ||
      !number(a[5], &scale) || !(scale > 0) || !std::isfinite(scale) || !result(a[8], *q, &out) || !out.is_contiguous())
    Py_RETURN_NONE;
  View y;
  if (WIN && !view_of(a[9], a[10], *q, c.n_seg, &y)) Py_RETURN_NONE;
  const int64_t dev = q->device().index(), g = q->size(1);
  const c10::DeviceGuard guard(q->device());
  if (!ready(dev)) Py_RETURN_NONE;
  PyObject* so = nullptr;
  void* stream = nullptr;
  const bool has_stream = stream_of(dev, &so, &stream);
  Ref stream_ref(so);
  if (!has_stream) return nullptr;
  const int64_t need = wnw_paged_decode_workspace_bytes(c.n_seg, g, c.head_dim);
  if (need < 0) Py_RETURN_NONE;  // the general path says why
  Ref ws(PyObject_CallFunction(g_paged_ws, "LOLL", (long long)dev, so, (long long)c.n_seg, (long long)need));
  const at::Tensor* buf = buffer(ws);
  if (!buf) return nullptr;
  void *qp = q->data_ptr(), *op = out.data_ptr(), *wp = buf->data_ptr();
  const int64_t bytes = buf->numel();
  const int dt = dtype_code(q->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = WIN ? wnw_paged_decode_attn_window(&c, len, qp, op, g, y.window, y.window_all, y.sinks, y.sinks_all, (float)scale, dt, wp,
                                          bytes, stream)
           : wnw_paged_decode_attn(&c, len, qp, op, g, (float)scale, dt, wp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_decode_attn");
  return a[8] != Py_None ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(out));
}

// (q, k_pages, v_pages, page_table, seg_len, cu_tokens, scale, max_tokens, k_scale, v_scale, out), WIN: and (window, sinks)
template <bool WIN>
PyObject* paged_prompt_impl(PyObject* const* a) {
  const at::Tensor* q = plain(a[0]);
  wnw_paged_cache c;
  const int32_t *len, *cu;
  int64_t samples = 0, most = 0;
  double scale = 0;
  at::Tensor out;
  if (!q || !half_type(*q) || needs_grad(q) || !paged_cache(a + 1, a[8], a[9], *q, &c, &len) || !heads(*q, c.head_dim) ||
      !tokens_of(a[5], a[7], *q, c.n_seg, &cu, &samples, &most) || q->size(1) % (c.n_seg / samples) != 0 ||
      !number(a[6], &scale) || !(scale > 0) || !std::isfinite(scale) || !result(a[10], *q, &out))
    Py_RETURN_NONE;
  View y;
  if (WIN && !view_of(a[11], a[12], *q, c.n_seg, &y)) Py_RETURN_NONE;
  const int64_t dev = q->device().index(), g = q->size(1) / (c.n_seg / samples);
  const c10::DeviceGuard guard(q->device());
  if (!ready(dev)) Py_RETURN_NONE;
  PyObject* so = nullptr;
  void* stream = nullptr;
  const bool has_stream = stream_of(dev, &so, &stream);
  Ref stream_ref(so);
  if (!has_stream) return nullptr;
  const int64_t need = WIN ? wnw_paged_prompt_window_workspace_bytes(&c, g, most, y.window, y.window_all, y.sinks, y.sinks_all)
                           : wnw_paged_prompt_workspace_bytes(&c, g, most);
  if (need < 0) Py_RETURN_NONE;  // the general path says why
  at::Tensor own;
  Ref ws(g * most <= 16 ? PyObject_CallFunction(g_paged_ws, "LOLL", (long long)dev, so, (long long)c.n_seg, (long long)need)
                        : Py_NewRef(Py_None));
  void* wp = nullptr;
  if (ws.o != Py_None) {
    const at::Tensor* buf = buffer(ws);
    if (!buf) return nullptr;
    wp = buf->data_ptr();
  } else if (need > 0) {
    own = at::empty({need}, q->options().dtype(at::kByte).requires_grad(false));
    wp = own.data_ptr();
  }
  void *qp = q->data_ptr(), *op = out.data_ptr();
  const int64_t strides[4] = {q->stride(0), q->stride(1), out.stride(0), out.stride(1)}, tokens = q->size(0);
  const int dt = dtype_code(q->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = WIN ? wnw_paged_prompt_attn_window(&c, len, qp, op, strides, tokens, samples, g, cu, most, y.window, y.window_all, y.sinks,
                                          y.sinks_all, (float)scale, dt, wp, need, stream)
           : wnw_paged_prompt_attn(&c, len, qp, op, strides, tokens, samples, g, cu, most, (float)scale, dt, wp, need, stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_prompt_attn");
  return a[10] != Py_None ? Py_NewRef(a[10]) : THPVariable_Wrap(std::move(out));
}

// (k, v, k_pages, v_pages, page_table, seg_len, q, positions, inv_freq, sections, interleaved, cu_tokens, max_tokens, k_scale,
// v_scale)
PyObject* paged_append_impl(PyObject* const* a) {
  const at::Tensor *k = plain(a[0]), *v = plain(a[1]);
  wnw_paged_cache c;
  const int32_t *len, *cu = nullptr;
  if (!k || !v || !half_type(*k) || needs_grad(k) || !usable(v, *k) || v->scalar_type() != k->scalar_type() ||
      !paged_cache(a + 2, a[13], a[14], *k, &c, &len) || !heads(*k, c.head_dim) || !heads(*v, c.head_dim) ||
      v->sizes() != k->sizes())
    Py_RETURN_NONE;
  const int64_t T = k->size(0), H = k->size(1);
  int64_t samples = T, most = 1;
  if (a[11] != Py_None ? !tokens_of(a[11], a[12], *k, c.n_seg, &cu, &samples, &most) : a[12] != Py_None) Py_RETURN_NONE;
  if (c.n_seg != samples * H) Py_RETURN_NONE;
  const at::Tensor *q = nullptr, *pos = nullptr, *freq = nullptr;
  int64_t g = 1, rot = 0, pos_stride = 0, secs[4] = {0, 0, 0, 0};
  int n_secs = 0;
  if (a[6] != Py_None) {
    q = plain(a[6]);
    if (!usable(q, *k) || q->scalar_type() != k->scalar_type() || !heads(*q, c.head_dim) || q->size(0) != T ||
        q->size(1) % H != 0)
      Py_RETURN_NONE;
    g = q->size(1) / H;
  }
  if (a[7] != Py_None) {
    pos = plain(a[7]);
    freq = plain(a[8]);
    if (!usable(pos, *k) || !usable(freq, *k) || freq->dim() != 1 || !freq->is_contiguous() ||
        (freq->scalar_type() != at::kDouble && freq->scalar_type() != at::kFloat) ||
        (pos->scalar_type() != at::kLong && pos->scalar_type() != at::kInt) || !pos->is_contiguous())
      Py_RETURN_NONE;
    rot = 2 * freq->numel();
    if (a[9] == Py_None) {
      n_secs = 1;
      secs[0] = rot / 2;
    } else {
      if (!PyList_CheckExact(a[9]) && !PyTuple_CheckExact(a[9])) Py_RETURN_NONE;
      const Py_ssize_t n = PySequence_Fast_GET_SIZE(a[9]);
      if (n < 1 || n > 4) Py_RETURN_NONE;
      for (Py_ssize_t i = 0; i < n; ++i)
        if (!whole(PySequence_Fast_GET_ITEM(a[9], i), &secs[i]) || secs[i] < 0 || secs[i] > rot / 2) Py_RETURN_NONE;
      n_secs = (int)n;
    }
    if (rot % 16 != 0 || rot < 16 || rot > c.head_dim || secs[0] + secs[1] + secs[2] + secs[3] != rot / 2) Py_RETURN_NONE;
    const bool flat = pos->dim() == 1 && n_secs == 1 && pos->size(0) == T;
    if (!flat && !(pos->dim() == 2 && pos->size(0) == n_secs && pos->size(1) == T)) Py_RETURN_NONE;
    pos_stride = T;
  } else if (a[8] != Py_None || a[9] != Py_None) {
    Py_RETURN_NONE;
  }
  const int interleaved = PyObject_IsTrue(a[10]);
  if (interleaved < 0) return nullptr;
  const c10::DeviceGuard guard(k->device());
  if (!ready(k->device().index())) Py_RETURN_NONE;
  at::Tensor q_out, new_len = at::empty({c.n_seg}, k->options().dtype(at::kInt).requires_grad(false));
  if (q && pos) q_out = at::empty(q->sizes(), q->options().requires_grad(false));
  PyObject* so = nullptr;
  void* stream = nullptr;
  const bool has_stream = stream_of(k->device().index(), &so, &stream);
  Ref stream_ref(so);
  if (!has_stream) return nullptr;
  const at::Tensor& qs = q_out.defined() ? *q : *k;
  const int64_t strides[6] = {qs.stride(0), qs.stride(1), k->stride(0), k->stride(1), v->stride(0), v->stride(1)};
  const int32_t sections[4] = {(int32_t)secs[0], (int32_t)secs[1], (int32_t)secs[2], (int32_t)secs[3]};
  int32_t* nl = new_len.data_ptr<int32_t>();
  void *qp = q_out.defined() ? q->data_ptr() : nullptr, *qo = q_out.defined() ? q_out.data_ptr() : nullptr;
  void *kp = k->data_ptr(), *vp = v->data_ptr(), *pp = pos ? pos->data_ptr() : nullptr, *fp = pos ? freq->data_ptr() : nullptr;
  const int pos_bits = pos ? 8 * (int)pos->element_size() : 0, freq_bits = pos ? 8 * (int)freq->element_size() : 0;
  const int dt = dtype_code(k->scalar_type());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_paged_append(&c, len, nl, qp, kp, vp, qo, strides, T, samples, g, cu, most, pp, pos_bits, pos_stride, fp, freq_bits,
                        rot, sections, n_secs, interleaved, dt, stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_append");
  Ref first(q_out.defined() ? THPVariable_Wrap(std::move(q_out)) : Py_NewRef(a[6]));
  Ref second(THPVariable_Wrap(std::move(new_len)));
  return first.o && second.o ? PyTuple_Pack(2, first.o, second.o) : nullptr;
}

// The current stream and device of a call on t's device; false: leave it to the general path, or (stream) an exception.
struct Call {
  const c10::DeviceGuard guard;
  PyObject* so = nullptr;
  void* stream = nullptr;
  bool ok = false, has_stream = false;
  explicit Call(const at::Tensor& t) : guard(t.device()) {
    ok = ready(t.device().index());
    if (ok) has_stream = stream_of(t.device().index(), &so, &stream);
  }
  ~Call() { Py_XDECREF(so); }
};
at::Tensor like(const at::Tensor& t, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, t.options().dtype(type).requires_grad(false));
}

// A pool's table and counts, and (len) its segments' lengths
struct Pool {
  const at::Tensor *table, *refs, *len = nullptr;
  int64_t N, M, P, stride;
};
bool pool_of(PyObject* table, PyObject* refs, PyObject* len, Pool* p) {
  p->table = plain(table);
  p->refs = plain(refs);
  if (watched() || !p->table || !usable(p->refs, *p->table) || p->table->dim() != 2 || p->table->scalar_type() != at::kInt ||
      p->refs->scalar_type() != at::kInt || p->refs->dim() != 1 || !p->refs->is_contiguous())
    return false;
  p->N = p->table->size(0);
  p->M = p->table->size(1);
  p->P = p->refs->size(0);
  if (p->N < 1 || p->M < 1 || p->P < 1 || p->table->stride(1) != 1) return false;
  p->stride = p->N > 1 ? p->table->stride(0) : p->M;
  if (!len) return true;
  p->len = vec(len, at::kInt, p->N);
  return usable(p->len, *p->table) && p->len->dim() == 1;
}
// Where a pool's new state goes: the two tensors given, or new ones
bool pool_out(PyObject* out, const Pool& p, at::Tensor* table, at::Tensor* refs) {
  if (out == Py_None) {
    *table = like(*p.table, {p.N, p.M}, at::kInt);
    *refs = like(*p.table, {p.P}, at::kInt);
    return true;
  }
  if (!PyTuple_CheckExact(out) || PyTuple_GET_SIZE(out) != 2) return false;
  Pool o;
  if (!pool_of(PyTuple_GET_ITEM(out, 0), PyTuple_GET_ITEM(out, 1), nullptr, &o) || o.table->device() != p.table->device() ||
      o.N != p.N || o.M != p.M || o.P != p.P || o.stride < o.M)
    return false;
  *table = *o.table;
  *refs = *o.refs;
  return true;
}
PyObject* wrapped(PyObject* given, at::Tensor&& t) { return given ? Py_NewRef(given) : THPVariable_Wrap(std::move(t)); }

// (page_table, seg_len, page_refs, parents, page_rows, kv_heads)
PyObject* paged_fork_impl(PyObject* const* a) {
  Pool p;
  int64_t rows, heads;
  const at::Tensor* parents = plain(a[3]);
  if (!pool_of(a[0], a[2], a[1], &p) || !usable(parents, *p.table) || parents->scalar_type() != at::kInt || parents->dim() != 1 ||
      !parents->is_contiguous() || !whole(a[4], &rows) || !whole(a[5], &heads) || heads < 1 || p.N % heads != 0 ||
      parents->size(0) < 1)
    Py_RETURN_NONE;
  const int64_t n_new = parents->size(0), S = n_new * heads;
  const int64_t need = wnw_pages_workspace_bytes(std::max(p.N, S), p.N / heads, p.P);
  if (need < 0) Py_RETURN_NONE;
  Call call(*p.table);
  if (!call.ok) Py_RETURN_NONE;
  if (!call.has_stream) return nullptr;
  at::Tensor table = like(*p.table, {S, p.M}, at::kInt), len = like(*p.table, {S}, at::kInt), refs = like(*p.table, {p.P}, at::kInt);
  at::Tensor copies = like(*p.table, {S, 3}, at::kInt), ws = like(*p.table, {need}, at::kByte);
  const int32_t *t = p.table->const_data_ptr<int32_t>(), *l = p.len->const_data_ptr<int32_t>(), *r = p.refs->const_data_ptr<int32_t>();
  const int32_t* pa = parents->const_data_ptr<int32_t>();
  int32_t *nt = table.data_ptr<int32_t>(), *nl = len.data_ptr<int32_t>(), *nr = refs.data_ptr<int32_t>(), *cp = copies.data_ptr<int32_t>();
  void* w = ws.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_paged_fork(t, p.stride, l, r, pa, p.N / heads, n_new, heads, p.M, p.P, rows, nt, p.M, nl, nr, cp, w, need, call.stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_fork");
  Ref o0(THPVariable_Wrap(std::move(table))), o1(THPVariable_Wrap(std::move(len))), o2(THPVariable_Wrap(std::move(refs))),
      o3(THPVariable_Wrap(std::move(copies)));
  return o0.o && o1.o && o2.o && o3.o ? PyTuple_Pack(4, o0.o, o1.o, o2.o, o3.o) : nullptr;
}

// (page_table, seg_len, page_refs, page_rows, tokens, cu_tokens, window, sinks, out)
PyObject* paged_reserve_impl(PyObject* const* a) {
  Pool p;
  int64_t rows, tokens;
  if (!pool_of(a[0], a[2], a[1], &p) || !whole(a[3], &rows) || !whole(a[4], &tokens) || tokens < 0) Py_RETURN_NONE;
  const int32_t* cu = nullptr;
  int64_t samples = p.N;
  if (a[5] != Py_None) {
    const at::Tensor* t = plain(a[5]);
    if (!usable(t, *p.table) || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) < 2 || !t->is_contiguous()) Py_RETURN_NONE;
    samples = t->size(0) - 1;
    if (p.N % samples != 0) Py_RETURN_NONE;
    cu = t->const_data_ptr<int32_t>();
  }
  View y;
  y.window_all = -1;
  if (a[6] == Py_None ? a[7] != Py_None : !view_of(a[6], a[7], *p.table, p.N, &y)) Py_RETURN_NONE;
  const int64_t need = wnw_pages_workspace_bytes(p.N, samples, p.P);
  if (need < 0) Py_RETURN_NONE;
  Call call(*p.table);
  if (!call.ok) Py_RETURN_NONE;
  if (!call.has_stream) return nullptr;
  at::Tensor table, refs;
  if (!pool_out(a[8], p, &table, &refs)) Py_RETURN_NONE;
  at::Tensor ws = like(*p.table, {need}, at::kByte);
  const int32_t *t = p.table->const_data_ptr<int32_t>(), *l = p.len->const_data_ptr<int32_t>(), *r = p.refs->const_data_ptr<int32_t>();
  int32_t *nt = table.data_ptr<int32_t>(), *nr = refs.data_ptr<int32_t>();
  const int64_t ns = p.N > 1 ? table.stride(0) : p.M;
  void* w = ws.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_paged_reserve(t, p.stride, l, r, p.N, samples, p.M, p.P, rows, cu, tokens, y.window, y.window_all, y.sinks, y.sinks_all, nt,
                         ns, nr, w, need, call.stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_reserve");
  const bool given = a[8] != Py_None;
  Ref o0(wrapped(given ? PyTuple_GET_ITEM(a[8], 0) : nullptr, std::move(table))),
      o1(wrapped(given ? PyTuple_GET_ITEM(a[8], 1) : nullptr, std::move(refs)));
  return o0.o && o1.o ? PyTuple_Pack(2, o0.o, o1.o) : nullptr;
}

// (page_table, page_refs, page_rows, out)
PyObject* paged_compact_impl(PyObject* const* a) {
  Pool p;
  int64_t rows;
  if (!pool_of(a[0], a[1], nullptr, &p) || !whole(a[2], &rows)) Py_RETURN_NONE;
  const int64_t need = wnw_pages_workspace_bytes(p.N, 0, p.P);
  if (need < 0) Py_RETURN_NONE;
  Call call(*p.table);
  if (!call.ok) Py_RETURN_NONE;
  if (!call.has_stream) return nullptr;
  at::Tensor table, refs;
  if (!pool_out(a[3], p, &table, &refs)) Py_RETURN_NONE;
  at::Tensor moves = like(*p.table, {p.P / 2, 3}, at::kInt), used = like(*p.table, {1}, at::kInt), ws = like(*p.table, {need}, at::kByte);
  const int32_t *t = p.table->const_data_ptr<int32_t>(), *r = p.refs->const_data_ptr<int32_t>();
  int32_t *nt = table.data_ptr<int32_t>(), *nr = refs.data_ptr<int32_t>(), *mv = moves.data_ptr<int32_t>(), *us = used.data_ptr<int32_t>();
  const int64_t ns = p.N > 1 ? table.stride(0) : p.M;
  void* w = ws.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_paged_compact(t, p.stride, r, p.N, p.M, p.P, rows, nt, ns, nr, mv, us, w, need, call.stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_compact");
  const bool given = a[3] != Py_None;
  Ref o0(wrapped(given ? PyTuple_GET_ITEM(a[3], 0) : nullptr, std::move(table))),
      o1(wrapped(given ? PyTuple_GET_ITEM(a[3], 1) : nullptr, std::move(refs))), o2(THPVariable_Wrap(std::move(moves))),
      o3(THPVariable_Wrap(std::move(used)));
  return o0.o && o1.o && o2.o && o3.o ? PyTuple_Pack(4, o0.o, o1.o, o2.o, o3.o) : nullptr;
}

// (k_pages, v_pages, copies, k_scale, v_scale)
PyObject* paged_copy_impl(PyObject* const* a) {
  const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *copies = plain(a[2]);
  if (watched() || !k || needs_grad(k) || !usable(v, *k) || !usable(copies, *k) || k->dim() != 3 || k->sizes() != v->sizes() ||
      k->scalar_type() != v->scalar_type())
    Py_RETURN_NONE;
  const at::ScalarType dt = k->scalar_type();
  const bool q8 = dt == at::kFloat8_e4m3fn;
  const int64_t P = k->size(0), R = k->size(1), D = k->size(2);
  if ((!q8 && !half_type(*k)) || P < 1 || k->stride(2) != 1 || v->stride(2) != 1 || k->stride(1) != D || v->stride(1) != D ||
      copies->scalar_type() != at::kInt || copies->dim() != 2 || copies->size(1) != 3 || !copies->is_contiguous())
    Py_RETURN_NONE;
  const at::Tensor* sc[2] = {nullptr, nullptr};
  for (int i = 0; i < 2; ++i) {
    if (q8 ? !usable(sc[i] = vec(a[3 + i], at::kFloat, P), *k) || sc[i]->dim() != 1 : a[3 + i] != Py_None) Py_RETURN_NONE;
  }
  wnw_paged_cache c = {};
  c.k_pages = k->data_ptr();
  c.v_pages = v->data_ptr();
  c.k_scale = q8 ? sc[0]->data_ptr<float>() : nullptr;
  c.v_scale = q8 ? sc[1]->data_ptr<float>() : nullptr;
  c.n_pages = P;
  c.page_rows = R;
  c.head_dim = D;
  c.k_stride = P > 1 ? k->stride(0) : R * D;
  c.v_stride = P > 1 ? v->stride(0) : R * D;
  c.page_dtype = q8 ? WNW_E4M3 : dtype_code(dt);
  Call call(*k);
  if (!call.ok) Py_RETURN_NONE;
  if (!call.has_stream) return nullptr;
  const int32_t* cp = copies->const_data_ptr<int32_t>();
  const int64_t n = copies->size(0);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_paged_copy(&c, cp, n, call.stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "paged_copy");
  Py_RETURN_TRUE;
}

// (logits, scores, k, done, end)
PyObject* beam_select_impl(PyObject* const* a) {
  const at::Tensor *x = plain(a[0]), *s = plain(a[1]), *done = nullptr;
  if (watched() || !x || needs_grad(x) || !usable(s, *x) || x->dim() != 3 || x->stride(2) != 1) Py_RETURN_NONE;
  const int64_t B = x->size(0), W = x->size(1), V = x->size(2);
  const int dt = dtype_code(x->scalar_type());
  int64_t k = W, end = 0;
  if (dt < 0 || B < 1 || s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != B || s->size(1) != W || !s->is_contiguous() ||
      (a[2] != Py_None && !whole(a[2], &k)) || k < 1 || k > 64 || !whole(a[4], &end))
    Py_RETURN_NONE;
  if (a[3] != Py_None) {
    done = plain(a[3]);
    if (!usable(done, *x) || done->scalar_type() != at::kBool || done->dim() != 2 || done->size(0) != B || done->size(1) != W ||
        !done->is_contiguous())
      Py_RETURN_NONE;
  }
  const int64_t need = wnw_beam_workspace_bytes(B, W, V, dt);
  if (need < 0) Py_RETURN_NONE;
  Call call(*x);
  if (!call.ok) Py_RETURN_NONE;
  if (!call.has_stream) return nullptr;
  at::Tensor out = like(*x, {B, k}, at::kFloat), parents = like(*x, {B, k}, at::kInt), tokens = like(*x, {B, k}, at::kLong);
  at::Tensor ws = like(*x, {need}, at::kByte);
  const int64_t strides[2] = {x->stride(0), x->stride(1)};
  const void* xp = x->const_data_ptr();
  const float* sp = s->const_data_ptr<float>();
  const uint8_t* dp = done ? (const uint8_t*)done->const_data_ptr() : nullptr;
  float* op = out.data_ptr<float>();
  int32_t* pp = parents.data_ptr<int32_t>();
  int64_t* tp = tokens.data_ptr<int64_t>();
  void* w = ws.data_ptr();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = wnw_beam_select(xp, strides, B, W, V, sp, dp, end, k, dt, op, pp, tp, w, need, call.stream);
  Py_END_ALLOW_THREADS
  if (rc != WNW_OK) return failed(rc, "beam_select");
  Ref o0(THPVariable_Wrap(std::move(out))), o1(THPVariable_Wrap(std::move(parents))), o2(THPVariable_Wrap(std::move(tokens)));
  return o0.o && o1.o && o2.o ? PyTuple_Pack(3, o0.o, o1.o, o2.o) : nullptr;
}

// No C++ exception leaves an entry: such a call takes the general path.
template <PyObject* (*f)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  if (!g_check) {
    PyErr_SetString(PyExc_RuntimeError, "setup() has not been called");
    return nullptr;
  }
  try {
    return f(args);
  } catch (const std::exception&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

PyObject* setup(PyObject*, PyObject* args) {
  PyObject *s, *w, *sw, *pw, *c;
  if (!PyArg_ParseTuple(args, "OOOOO", &s, &w, &sw, &pw, &c)) return nullptr;
  PyObject** dst[5] = {&g_stream, &g_workspace, &g_score_ws, &g_paged_ws, &g_check};
  PyObject* src[5] = {s, w, sw, pw, c};
  for (int i = 0; i < 5; ++i) {
    PyObject* old = *dst[i];
    *dst[i] = Py_NewRef(src[i]);
    Py_XDECREF(old);
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"setup", setup, METH_VARARGS, "setup(raw_stream, workspace, score_workspace, paged_workspace, check)"},
    {"attn", (PyCFunction)(void (*)(void))entry<attn_impl, 9>, METH_FASTCALL,
     "attn(q, k, v, cu, scale, seg_base, total_rows, out, append) -> out, or None: not the plain form"},
    {"score", (PyCFunction)(void (*)(void))entry<score_impl, 10>, METH_FASTCALL,
     "score(q, k, starts, ends, audio_starts, audio_ends, acc, offsets, max_audio, scale) -> True, or None: not the "
     "plain form"},
    {"paged_decode", (PyCFunction)(void (*)(void))entry<paged_decode_impl<false>, 9>, METH_FASTCALL,
     "paged_decode(q, k_pages, v_pages, page_table, seg_len, scale, k_scale, v_scale, out) -> out, or None: not the plain "
     "form"},
    {"paged_prompt", (PyCFunction)(void (*)(void))entry<paged_prompt_impl<false>, 11>, METH_FASTCALL,
     "paged_prompt(q, k_pages, v_pages, page_table, seg_len, cu_tokens, scale, max_tokens, k_scale, v_scale, out) -> out, or "
     "None: not the plain form"},
    {"paged_decode_window", (PyCFunction)(void (*)(void))entry<paged_decode_impl<true>, 11>, METH_FASTCALL,
     "paged_decode_window(..., out, window, sinks): paged_decode through a window"},
    {"paged_prompt_window", (PyCFunction)(void (*)(void))entry<paged_prompt_impl<true>, 13>, METH_FASTCALL,
     "paged_prompt_window(..., out, window, sinks): paged_prompt through a window"},
    {"paged_append", (PyCFunction)(void (*)(void))entry<paged_append_impl, 15>, METH_FASTCALL,
     "paged_append(k, v, k_pages, v_pages, page_table, seg_len, q, positions, inv_freq, sections, interleaved, cu_tokens, "
     "max_tokens, k_scale, v_scale) -> (q rotated, new lengths), or None: not the plain form"},
    {"paged_fork", (PyCFunction)(void (*)(void))entry<paged_fork_impl, 6>, METH_FASTCALL,
     "paged_fork(page_table, seg_len, page_refs, parents, page_rows, kv_heads) -> (table, lengths, counts, copies), or None: not "
     "the plain form"},
    {"paged_reserve", (PyCFunction)(void (*)(void))entry<paged_reserve_impl, 9>, METH_FASTCALL,
     "paged_reserve(page_table, seg_len, page_refs, page_rows, tokens, cu_tokens, window, sinks, out) -> (table, counts), or None: "
     "not the plain form"},
    {"paged_compact", (PyCFunction)(void (*)(void))entry<paged_compact_impl, 4>, METH_FASTCALL,
     "paged_compact(page_table, page_refs, page_rows, out) -> (table, counts, moves, used), or None: not the plain form"},
    {"paged_copy", (PyCFunction)(void (*)(void))entry<paged_copy_impl, 5>, METH_FASTCALL,
     "paged_copy(k_pages, v_pages, copies, k_scale, v_scale) -> True, or None: not the plain form"},
    {"beam_select", (PyCFunction)(void (*)(void))entry<beam_select_impl, 5>, METH_FASTCALL,
     "beam_select(logits, scores, k, done, end) -> (scores, parents, tokens), or None: not the plain form"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_callpath", "Plain calls of the per-layer operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__callpath() { return PyModule_Create(&module); }
