// Native host path of the fused steps' Python entry points: argument checks,
// output allocation and the C-ABI call of step.speculative_step,
// paged.speculative_step, paged.speculative_signed_step, paged.exact,
// paged.extend, paged.attention and paged.shared_attention.
//
// A small step's kernel takes 5 us and its call from Python took 26 on the
// host: about 6 us of checks, 10 of allocations, 4 of ctypes conversions and
// the current stream, 4 of launch.  Done here the same call takes a third of
// that.  A call that does not pass every check below, or whose
// arguments are not plain strided tensors (subclasses, wrappers of transforms,
// active modes), returns None, and the Python code runs it as before, with its
// own messages; nothing is kept between calls but the C entry points'
// addresses and which devices were prepared.
#include <Python.h>

#include <cmath>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/strict_topk.h"

namespace {

struct Entry {
  decltype(&stk_step_supported) step_supported;
  decltype(&stk_step_workspace_bytes) step_workspace;
  decltype(&stk_speculative_step) step;
  decltype(&stk_paged_workspace_bytes) paged_workspace;
  decltype(&stk_paged_step) paged_step;
  decltype(&stk_paged_signed_step) paged_signed;
  decltype(&stk_paged_extend) extend;
  decltype(&stk_paged_attention_workspace_bytes) attention_workspace;
  decltype(&stk_paged_attention) attention;
  decltype(&stk_paged_shared_workspace_bytes) shared_workspace;
  decltype(&stk_paged_shared_attention) shared;
} g_entry;
constexpr int kEntries = sizeof(Entry) / sizeof(void*);
bool g_bound = false;
uint64_t g_prepared = 0;   // bit per device whose step memory was looked up

const c10::DispatchKeySet kWrapped({c10::DispatchKey::FuncTorchBatched,
                                    c10::DispatchKey::FuncTorchGradWrapper,
                                    c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                    c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
                                    c10::DispatchKey::ZeroTensor,
                                    c10::DispatchKey::NestedTensor});

// A plain tensor on a GPU, or null.
const at::Tensor* plain_strided(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided ||
      t.key_set().has_any(kWrapped) || t.unsafeGetTensorImpl()->has_symbolic_sizes_strides())
    return nullptr;
  return &t;
}

// A plain contiguous tensor on a GPU, or null.
const at::Tensor* plain(PyObject* o) {
  const at::Tensor* t = plain_strided(o);
  return t && t->is_contiguous() ? t : nullptr;
}

bool no_modes() {
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !at::impl::torch_function_mode_enabled();
}

int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? 1 : (t.scalar_type() == at::kBFloat16 ? 2 : -1);
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

bool small(const at::Tensor& t) {
  for (int64_t s : t.sizes())
    if (s < 1 || s > 0x7fffffff) return false;
  return true;
}

// topk as a C int when it is a plain Python int in range
bool plain_int(PyObject* o, long lo, long hi, int* out) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long v = PyLong_AsLongAndOverflow(o, &over);
  if (over || v < lo || v > hi) return false;
  *out = (int)v;
  return true;
}

bool plain_float(PyObject* o, double* out) {
  if (PyFloat_CheckExact(o)) *out = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *out = PyLong_AsDouble(o);
  else return false;
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

PyObject* pack(std::initializer_list<const at::Tensor*> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : ts) {
    PyObject* o;
    if (t->defined()) {
      o = THPVariable_Wrap(*t);
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// A C++ exception (a tensor kind the checks do not know, memory that ran out;
// all of them before anything is launched) means None: the Python code then
// meets the same and raises torch's own.
template <typename F>
PyObject* checked(F f) {
  try {
    return f();
  } catch (const std::exception&) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
}

// (q, k, v, lo, hi, predicted, topk, union): (selected, m, l, u, out), an error
// code, or None
PyObject* step_impl(PyObject* const* a, Py_ssize_t n) {
  if (!g_bound || n != 8 || !no_modes()) Py_RETURN_NONE;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = plain(a[i]))) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &lo = *t[3], &hi = *t[4], &p = *t[5];
  if (q.dim() != 2 || k.dim() != 4 || lo.dim() != 3 || p.dim() != 2 || !small(q) || !small(k) ||
      !small(p) || v.sizes() != k.sizes() || hi.sizes() != lo.sizes())
    Py_RETURN_NONE;
  const int64_t hq = q.size(0), d = q.size(1), hkv = k.size(0), nb = k.size(1), b = k.size(2);
  const int64_t sp = p.size(1);
  const int dt = dtype_code(q);
  if (dt < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.size(3) != d || hq % hkv || p.size(0) != hq || p.scalar_type() != at::kInt ||
      lo.size(0) != hkv || lo.size(1) != nb || lo.size(2) != d ||
      hi.scalar_type() != lo.scalar_type() ||
      (lo.scalar_type() != at::kFloat && lo.scalar_type() != q.scalar_type()))
    Py_RETURN_NONE;
  const auto dev = q.device();
  for (int i = 1; i < 6; ++i)
    if (t[i]->device() != dev) Py_RETURN_NONE;
  for (int i = 0; i < 5; ++i)
    if (!aligned(*t[i])) Py_RETURN_NONE;
  int topk;
  const int uni = PyObject_IsTrue(a[7]);
  if (uni < 0) return nullptr;
  if (dev.index() < 0 || dev.index() > 63 || !(g_prepared >> dev.index() & 1) ||
      !plain_int(a[6], 1, nb, &topk) ||
      !g_entry.step_supported(dt, (int)hq, (int)hkv, (int)nb, (int)b, (int)d, topk, (int)sp, 0))
    Py_RETURN_NONE;
  const auto f = q.options().dtype(at::kFloat).requires_grad(false);
  const at::Tensor sel = at::empty({hq, topk}, f.dtype(at::kInt));
  const at::Tensor m = at::empty({hq, sp}, f), l = at::empty({hq, sp}, f);
  const at::Tensor u = at::empty({hq, sp, d}, f), out = at::empty({hq, d}, f);
  const size_t bytes = g_entry.step_workspace((int)hq, (int)hkv, (int)nb, (int)d, topk);
  const at::Tensor ws = at::empty({(int64_t)(bytes ? bytes : 1)}, f.dtype(at::kByte));
  void* st = stream_of(q);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_entry.step(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, (int)hq, (int)hkv, (int)nb,
                    (int)b, (int)d, lo.data_ptr(), hi.data_ptr(),
                    lo.scalar_type() == at::kFloat ? 0 : dt, topk, p.data_ptr(), 0, (int)sp, uni,
                    sel.data_ptr<int32_t>(), m.data_ptr<float>(), l.data_ptr<float>(),
                    u.data_ptr<float>(), out.data_ptr<float>(), ws.data_ptr(), bytes, st);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  return pack({&sel, &m, &l, &u, &out});
}

// (q, k_pages, v_pages, lo, hi, table, nblocks, ntokens or None, predicted or
// None, topk, mode, tau, min_remaining, cancellation, eps): mode 0 saved (or no
// prediction), 1 union, 2 signed saved, 3 signed hybrid.
// Returns (selected, m, l, u, out[, fallback, remaining, approx, extra, pos,
// total]), an error code, or None.
PyObject* paged_impl(PyObject* const* a, Py_ssize_t n) {
  if (!g_bound || n != 15 || !no_modes()) Py_RETURN_NONE;
  const at::Tensor* t[9] = {};
  for (int i = 0; i < 9; ++i) {
    if (i >= 7 && a[i] == Py_None) continue;
    if (!(t[i] = plain(a[i]))) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &lo = *t[3], &hi = *t[4], &tab = *t[5],
                   &nbk = *t[6];
  if (q.dim() != 3 || k.dim() != 3 || lo.dim() != 2 || tab.dim() != 3 || nbk.dim() != 1 ||
      !small(q) || !small(k) || !small(tab) || v.sizes() != k.sizes() ||
      hi.sizes() != lo.sizes())
    Py_RETURN_NONE;
  const int64_t r = q.size(0), hq = q.size(1), d = q.size(2), pages = k.size(0), b = k.size(1);
  const int64_t hkv = tab.size(1), width = tab.size(2);
  const int dt = dtype_code(q);
  if (dt < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.size(2) != d || lo.size(0) != pages || lo.size(1) != d || tab.size(0) != r || hq % hkv ||
      nbk.size(0) != r || tab.scalar_type() != at::kInt || nbk.scalar_type() != at::kInt ||
      hi.scalar_type() != lo.scalar_type() ||
      (lo.scalar_type() != at::kFloat && lo.scalar_type() != q.scalar_type()))
    Py_RETURN_NONE;
  if (t[7] && (t[7]->dim() != 1 || t[7]->size(0) != r || t[7]->scalar_type() != at::kInt))
    Py_RETURN_NONE;
  if (t[8] && (t[8]->dim() != 3 || !small(*t[8]) || t[8]->size(0) != r || t[8]->size(1) != hq ||
               t[8]->scalar_type() != at::kInt))
    Py_RETURN_NONE;
  const auto dev = q.device();
  for (int i = 1; i < 9; ++i)
    if (t[i] && t[i]->device() != dev) Py_RETURN_NONE;
  int topk, mode;
  double tau, minr, tol, eps;
  if (!plain_int(a[9], 1, 256, &topk) || !plain_int(a[10], 0, 3, &mode) ||
      !plain_float(a[11], &tau) || !plain_float(a[12], &minr) || !plain_float(a[13], &tol) ||
      !plain_float(a[14], &eps) || !(tau >= 0 && tau <= 1) || !(eps >= 0 && eps <= 1) ||
      (mode >= 2 && !t[8]))
    Py_RETURN_NONE;
  const int64_t sp = t[8] ? t[8]->size(2) : 0;
  const auto f = q.options().dtype(at::kFloat).requires_grad(false);
  const at::Tensor sel = at::empty({r, hq, topk}, f.dtype(at::kInt));
  at::Tensor m, l, u;
  if (sp) {
    m = at::empty({r, hq, sp}, f);
    l = at::empty({r, hq, sp}, f);
    u = at::empty({r, hq, sp, d}, f);
  }
  const at::Tensor out = at::empty({r, hq, d}, f);
  const size_t bytes = g_entry.paged_workspace((int)r, (int)hq, (int)width);
  const at::Tensor ws = at::empty({(int64_t)(bytes ? bytes : 1)}, f.dtype(at::kByte));
  auto fp = [](const at::Tensor& x) { return x.defined() ? x.data_ptr<float>() : nullptr; };
  const int32_t* nt = t[7] ? t[7]->data_ptr<int32_t>() : nullptr;
  const int32_t* p = t[8] ? t[8]->data_ptr<int32_t>() : nullptr;
  const int lb = lo.scalar_type() == at::kFloat ? 0 : dt;
  void* st = stream_of(q);
  int rc;
  if (mode < 2) {
    Py_BEGIN_ALLOW_THREADS
    rc = g_entry.paged_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, (int)r, (int)hq,
                            (int)hkv, (int)width, (int)b, (int)d, (int)pages, lo.data_ptr(),
                            hi.data_ptr(), lb, tab.data_ptr<int32_t>(),
                            nbk.data_ptr<int32_t>(), nt, topk, p, (int)sp, mode,
                            sel.data_ptr<int32_t>(), fp(m), fp(l), fp(u),
                            out.data_ptr<float>(), ws.data_ptr(), bytes, st);
    Py_END_ALLOW_THREADS
    if (rc) return PyLong_FromLong(rc);
    return pack({&sel, &m, &l, &u, &out});
  }
  const at::Tensor bad = at::empty({r, hq}, f.dtype(at::kBool)), rem = at::empty({r, hq}, f);
  at::Tensor approx, extra;
  if (eps > 0) {
    approx = at::empty({r, hq}, f.dtype(at::kBool));
    extra = at::empty({r, hq}, f);
  }
  const at::Tensor pos = at::empty({r, hq}, f.dtype(at::kInt));
  const at::Tensor tot = at::empty({r, hq}, f.dtype(at::kInt));
  Py_BEGIN_ALLOW_THREADS
  rc = g_entry.paged_signed(
      q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, (int)r, (int)hq, (int)hkv, (int)width,
      (int)b, (int)d, (int)pages, lo.data_ptr(), hi.data_ptr(), lb, tab.data_ptr<int32_t>(),
      nbk.data_ptr<int32_t>(), nt, topk, p, (int)sp, mode == 3, (float)tau, (float)minr,
      (float)tol, (float)eps, sel.data_ptr<int32_t>(), fp(m), fp(l), fp(u),
      out.data_ptr<float>(), static_cast<uint8_t*>(bad.data_ptr()), rem.data_ptr<float>(),
      approx.defined() ? static_cast<uint8_t*>(approx.data_ptr()) : nullptr, fp(extra),
      pos.data_ptr<int32_t>(), tot.data_ptr<int32_t>(), ws.data_ptr(), bytes, st);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  return pack({&sel, &m, &l, &u, &out, &bad, &rem, &approx, &extra, &pos, &tot});
}

// The page pool of the dense operators: a[0..3 + bounds * 2) are K pages, V pages[,
// lo, hi], table, nblocks; then ntokens or None.
struct Pool {
  const at::Tensor *k, *v, *lo, *hi, *table, *nblocks, *ntokens;
  int64_t pages, b, d, r, hkv, width;
  int dt;
};

bool int_vector(const at::Tensor& t, int64_t n) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n;
}

bool on(const at::Tensor* t, const at::Device& d) { return !t || t->device() == d; }

bool pool_of(PyObject* const* a, bool bounds, Pool* p) {
  const at::Tensor* t[7] = {};
  const int n = bounds ? 6 : 4;
  for (int i = 0; i < n; ++i)
    if (!(t[i] = plain(a[i]))) return false;
  if (a[n] != Py_None && !(t[6] = plain(a[n]))) return false;
  p->k = t[0];
  p->v = t[1];
  p->lo = bounds ? t[2] : nullptr;
  p->hi = bounds ? t[3] : nullptr;
  p->table = t[n - 2];
  p->nblocks = t[n - 1];
  p->ntokens = t[6];
  const at::Tensor &k = *p->k, &tab = *p->table;
  p->dt = dtype_code(k);
  if (p->dt < 0 || k.dim() != 3 || !small(k) || p->v->sizes() != k.sizes() ||
      p->v->scalar_type() != k.scalar_type() || tab.dim() != 3 || !small(tab) ||
      tab.scalar_type() != at::kInt)
    return false;
  p->pages = k.size(0);
  p->b = k.size(1);
  p->d = k.size(2);
  p->r = tab.size(0);
  p->hkv = tab.size(1);
  p->width = tab.size(2);
  if (!int_vector(*p->nblocks, p->r) || (p->ntokens && !int_vector(*p->ntokens, p->r)))
    return false;
  const auto dev = k.device();
  if (dev.index() != c10::hip::current_device()) return false;
  for (const at::Tensor* x : {p->v, p->lo, p->hi, p->table, p->nblocks, p->ntokens})
    if (!on(x, dev)) return false;
  if (!bounds) return true;
  const at::Tensor &lo = *p->lo, &hi = *p->hi;
  return lo.dim() == 2 && lo.size(0) == p->pages && lo.size(1) == p->d &&
         hi.sizes() == lo.sizes() && hi.scalar_type() == lo.scalar_type() &&
         (lo.scalar_type() == at::kFloat || lo.scalar_type() == k.scalar_type());
}

// Rows [T, heads, D] of the pool's type, contiguous within a token; *stride
// from one token to the next.
const at::Tensor* tokens_of(PyObject* o, const Pool& p, int64_t heads, int64_t* stride) {
  const at::Tensor* t = plain_strided(o);
  if (!t || t->dim() != 3 || !small(*t) || t->size(2) != p.d ||
      (heads > 0 && t->size(1) != heads) || t->scalar_type() != p.k->scalar_type() ||
      t->device() != p.k->device())
    return nullptr;
  const int64_t n = t->size(0), h = t->size(1);
  if (t->stride(2) != 1 || (h > 1 && t->stride(1) != p.d) ||
      (n > 1 && (t->stride(0) < h * p.d || t->stride(0) % 8)))
    return nullptr;
  *stride = n > 1 ? t->stride(0) : h * p.d;
  return t;
}

bool disjoint(const at::Tensor& a, const at::Tensor* b) {
  if (!b) return true;
  const char* x = static_cast<const char*>(a.data_ptr());
  const char* y = static_cast<const char*>(b->data_ptr());
  return x + a.nbytes() <= y || y + b->nbytes() <= x;
}

const int32_t* ip(const at::Tensor* t) { return t ? t->data_ptr<int32_t>() : nullptr; }

// (k_pages, v_pages, lo, hi, table, nblocks, ntokens or None, k_new, v_new,
// starts, positions, cos, sin, q or None, interleaved): (rotated q or None,),
// an error code, or None.  cos and sin may be None.
PyObject* extend_impl(PyObject* const* a, Py_ssize_t n) {
  Pool p;
  if (!g_bound || n != 15 || !no_modes() || !pool_of(a, true, &p)) Py_RETURN_NONE;
  int64_t ks, vs, qs = 0;
  const at::Tensor* k = tokens_of(a[7], p, p.hkv, &ks);
  const at::Tensor* v = tokens_of(a[8], p, p.hkv, &vs);
  const at::Tensor *st = plain(a[9]), *pos = plain(a[10]);
  if (!k || !v || k->size(0) != v->size(0) || !st || !pos || !int_vector(*st, p.r + 1) ||
      !int_vector(*pos, p.r))
    Py_RETURN_NONE;
  const at::Tensor *co = nullptr, *si = nullptr, *q = nullptr;
  const auto dev = p.k->device();
  int64_t rows = 0, rot = 0, hq = 0;
  if (a[11] != Py_None || a[12] != Py_None) {
    co = plain(a[11]);
    si = plain(a[12]);
    if (!co || !si || co->dim() != 2 || !small(*co) || si->sizes() != co->sizes() ||
        co->scalar_type() != at::kFloat || si->scalar_type() != at::kFloat)
      Py_RETURN_NONE;
    rows = co->size(0);
    rot = 2 * co->size(1);
  }
  if (rot > p.d) Py_RETURN_NONE;
  const int64_t t = k->size(0);
  if (a[13] != Py_None) {
    if (!co || !(q = tokens_of(a[13], p, 0, &qs)) || q->size(0) != t) Py_RETURN_NONE;
    hq = q->size(1);
  }
  for (const at::Tensor* x : {st, pos, co, si})
    if (!on(x, dev)) Py_RETURN_NONE;
  if (!disjoint(*pos, p.ntokens) || !disjoint(*pos, p.nblocks)) Py_RETURN_NONE;
  const int inter = PyObject_IsTrue(a[14]);
  if (inter < 0) return nullptr;
  at::Tensor out;
  if (q) out = at::empty({t, hq, p.d}, p.k->options().requires_grad(false));
  void* stream = stream_of(*p.k);
  const int lb = p.lo->scalar_type() == at::kFloat ? 0 : p.dt;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_entry.extend(k->data_ptr(), ks, v->data_ptr(), vs, q ? q->data_ptr() : nullptr, qs,
                      q ? out.data_ptr() : nullptr, p.dt, (int)t, (int)p.r, (int)hq, (int)p.hkv,
                      (int)p.width, (int)p.b, (int)p.d, (int)p.pages, ip(st), ip(pos),
                      co ? co->data_ptr<float>() : nullptr, si ? si->data_ptr<float>() : nullptr,
                      (int)rows, (int)rot, inter, p.k->data_ptr(), p.v->data_ptr(),
                      p.lo->data_ptr(), p.hi->data_ptr(), lb, ip(p.table),
                      p.nblocks->data_ptr<int32_t>(),
                      p.ntokens ? p.ntokens->data_ptr<int32_t>() : nullptr, stream);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  return pack({&out});
}

// (k_pages, v_pages, table, nblocks, ntokens or None, q, starts, groups, shared, scale,
// softcap, slopes, window, prefix, first, out): starts, groups and shared, scale,
// slopes, prefix, first and out may be None.  Returns the output, an error code, or None.
PyObject* attention_impl(PyObject* const* a, Py_ssize_t n) {
  Pool p;
  if (!g_bound || n != 16 || !no_modes() || !pool_of(a, false, &p)) Py_RETURN_NONE;
  int64_t qs;
  const at::Tensor* q = tokens_of(a[5], p, 0, &qs);
  if (!q || q->size(1) % p.hkv) Py_RETURN_NONE;
  const int64_t t = q->size(0), hq = q->size(1);
  const at::Tensor* o[8] = {};                 // starts, groups, shared, slopes, prefix, first, out
  const int at_[7] = {6, 7, 8, 11, 13, 14, 15};
  for (int i = 0; i < 7; ++i)
    if (a[at_[i]] != Py_None && (!(o[i] = plain(a[at_[i]])) || !on(o[i], p.k->device())))
      Py_RETURN_NONE;
  const at::Tensor *st = o[0], *gr = o[1], *sh = o[2], *slo = o[3], *pre = o[4], *fir = o[5];
  double scale = 1.0 / std::sqrt((double)p.d), cap;
  int window;
  if ((a[9] != Py_None && !plain_float(a[9], &scale)) || !plain_float(a[10], &cap) ||
      !plain_int(a[12], 0, 0x7fffffff, &window) || !(scale > 0) || !(scale <= 1e30) ||
      !(cap >= 0) || !(cap <= 4096))
    Py_RETURN_NONE;
  if ((st && !int_vector(*st, p.r + 1)) || (!st && t != p.r) || (pre && !int_vector(*pre, p.r)) ||
      (fir && !int_vector(*fir, t)) ||
      (slo && (slo->scalar_type() != at::kFloat || slo->dim() != 1 || slo->size(0) != hq)))
    Py_RETURN_NONE;
  int64_t ng = 0;
  if (gr || sh) {
    if (!gr || !sh || st || pre || gr->dim() != 1) Py_RETURN_NONE;
    ng = gr->size(0) - 1;
    if (ng < 1 || ng > p.r || !int_vector(*gr, ng + 1) || !int_vector(*sh, ng)) Py_RETURN_NONE;
  }
  if (o[6] && (o[6]->sizes() != q->sizes() || o[6]->scalar_type() != q->scalar_type()))
    Py_RETURN_NONE;
  const auto opt = q->options().requires_grad(false);
  const at::Tensor out = o[6] ? *o[6] : at::empty({t, hq, p.d}, opt);
  const size_t bytes =
      ng ? g_entry.shared_workspace((int)p.r, (int)ng, (int)hq, (int)p.hkv, (int)p.width, (int)p.b,
                                    (int)p.d)
         : g_entry.attention_workspace((int)t, (int)p.r, (int)hq, (int)p.hkv, (int)p.width,
                                       (int)p.b, (int)p.d, st != nullptr);
  const at::Tensor ws = at::empty({(int64_t)(bytes ? bytes : 1)}, opt.dtype(at::kByte));
  void* stream = stream_of(*q);
  const float* slopes = slo ? slo->data_ptr<float>() : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (ng)
    rc = g_entry.shared(q->data_ptr(), qs, p.dt, (int)p.r, (int)hq, (int)p.hkv, (int)p.width,
                        (int)p.b, (int)p.d, (int)p.pages, p.k->data_ptr(), p.v->data_ptr(),
                        ip(p.table), ip(p.nblocks), ip(p.ntokens), ip(gr), ip(sh), (int)ng,
                        (float)scale, (float)cap, slopes, window, ip(fir), out.data_ptr(),
                        ws.data_ptr(), bytes, stream);
  else
    rc = g_entry.attention(q->data_ptr(), qs, p.dt, (int)t, (int)p.r, (int)hq, (int)p.hkv,
                           (int)p.width, (int)p.b, (int)p.d, (int)p.pages, p.k->data_ptr(),
                           p.v->data_ptr(), ip(p.table), ip(p.nblocks), ip(p.ntokens), ip(st),
                           (float)scale, (float)cap, slopes, window, ip(pre), ip(fir),
                           out.data_ptr(), o[6] == nullptr, ws.data_ptr(), bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  if (o[6]) {
    Py_INCREF(a[15]);
    return a[15];
  }
  return THPVariable_Wrap(out);
}

PyObject* paged_extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked([&] { return extend_impl(a, n); });
}

PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked([&] { return attention_impl(a, n); });
}

PyObject* speculative_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked([&] { return step_impl(a, n); });
}

PyObject* paged_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return checked([&] { return paged_impl(a, n); });
}

// bind(...): the addresses of Entry's C entry points, in its order
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != kEntries) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kEntries);
    return nullptr;
  }
  void* p[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  memcpy(&g_entry, p, sizeof(g_entry));
  g_bound = true;
  Py_RETURN_NONE;
}

PyObject* prepared(PyObject*, PyObject* o) {
  int idx;
  if (plain_int(o, 0, 63, &idx)) g_prepared |= 1ull << idx;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"speculative_step", (PyCFunction)(void (*)())speculative_step, METH_FASTCALL, nullptr},
    {"paged_step", (PyCFunction)(void (*)())paged_step, METH_FASTCALL, nullptr},
    {"paged_extend", (PyCFunction)(void (*)())paged_extend, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)())paged_attention, METH_FASTCALL, nullptr},
    {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
    {"prepared", (PyCFunction)prepared, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch that the module was built for
PyMODINIT_FUNC PyInit__host(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "torch_version", STK_TORCH_VERSION)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
