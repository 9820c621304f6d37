// native.cpp -- the host side of the attention block's calls: checks the
// tensors, allocates results and fills the argument blocks of
// include/ubridge_hip.h.
//
// A decode step calls these operators a few times a layer, at sizes where the
// kernels take 5 to 15 us; reading shapes, strides and types of six tensors
// from Python took 8 to 10 us a call, here about 1 us.  Every refusal is a ValueError, as in
// the Python modules; a nonzero status of the C entry is returned as an int, for
// the caller to raise.  Compute stays behind the C ABI, whose entry points
// attention.py, rope.py, kvcache.py and int8.py hand over (bind) from the library
// they have loaded.
#include <Python.h>
#include <cfloat>
#include <cmath>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ubridge_hip.h"

namespace {

struct {
  decltype(&ubridge_paged_decode) decode;
  decltype(&ubridge_rope) rope;
  decltype(&ubridge_rope_append) append;
  decltype(&ubridge_int8_linear) linear;
  decltype(&ubridge_kv_free) free;
  decltype(&ubridge_kv_fork) fork;
  decltype(&ubridge_kv_compact) compact;
} fn;

#define REFUSE(...)                             \
  do {                                          \
    PyErr_Format(PyExc_ValueError, __VA_ARGS__); \
    return nullptr;                             \
  } while (0)

typedef const at::Tensor* Ten;

// A tensor on the device, or null (None, if `maybe`); false: refused.
bool device_tensor(PyObject* o, Ten& t, bool maybe = false) {
  t = nullptr;
  if (o == Py_None && maybe) return true;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "expected a tensor, not %s", Py_TYPE(o)->tp_name);
    return false;
  }
  t = &THPVariable_Unpack(o);
  if (!t->is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "ubridge_amd ops take device tensors");
    return false;
  }
  return true;
}

// 0 f32, 1 f16, 2 bf16, 3 e4m3, else -1
int code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    case at::kFloat8_e4m3fn: return 3;
    default: return -1;
  }
}
bool dense(const at::Tensor& t) { return t.is_contiguous(); }
bool last1(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
// f32 [n], contiguous
bool vec(Ten t, int64_t n) {
  return !t || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && dense(*t));
}
template <class T = float>
const T* ptr(Ten t) { return t ? (const T*)t->data_ptr() : nullptr; }

at::Tensor result(at::IntArrayRef sizes, const at::Tensor& like) { return at::empty(sizes, like.options().requires_grad(false)); }
at::Tensor result(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType t) {
  return at::empty(sizes, like.options().requires_grad(false).dtype(t));
}
// whether the memory of two tensors meets (strides are never negative)
bool meet(const at::Tensor& x, const at::Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  auto end = [](const at::Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); i++) n += (t.size(i) - 1) * t.stride(i);
    return (const char*)t.data_ptr() + n * t.element_size();
  };
  return (const char*)x.data_ptr() < end(y) && (const char*)y.data_ptr() < end(x);
}
bool fits(int64_t x) { return x >= 0 && x <= 0x7fffffff; }

// args: count and place checks
struct Args {
  PyObject* const* a;
  void* p(int i) const { return PyLong_AsVoidPtr(a[i]); }
  long n(int i) const { return PyLong_AsLong(a[i]); }
  double f(int i) const { return PyFloat_AsDouble(a[i]); }
};
#define COUNT(n_)                                                                                     \
  if (nargs != n_) {                                                                                  \
    PyErr_Format(PyExc_TypeError, "%d arguments expected", n_);                                       \
    return nullptr;                                                                                   \
  }

PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(7)
  const Args A{args};
  fn.decode = (decltype(fn.decode))A.p(0);
  fn.rope = (decltype(fn.rope))A.p(1);
  fn.append = (decltype(fn.append))A.p(2);
  fn.linear = (decltype(fn.linear))A.p(3);
  fn.free = (decltype(fn.free))A.p(4);
  fn.fork = (decltype(fn.fork))A.p(5);
  fn.compact = (decltype(fn.compact))A.p(6);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// q, k_pages, v_pages, tables, lens, scale | None, softcap, window, slopes,
// k_scale, v_scale, out, return_lse, stream
PyObject* py_decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(14)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten q, k, v, tables, lens, slopes, ks, vs, out;
  if (!device_tensor(args[0], q) || !device_tensor(args[1], k) || !device_tensor(args[2], v) ||
      !device_tensor(args[3], tables) || !device_tensor(args[4], lens) || !device_tensor(args[8], slopes, true) ||
      !device_tensor(args[9], ks, true) || !device_tensor(args[10], vs, true) || !device_tensor(args[11], out, true))
    return nullptr;
  const int dt = code(*q), ct = code(*k);
  if ((dt != 1 && dt != 2) || (ct != dt && ct != 3) || code(*v) != ct)
    REFUSE("paged_decode takes f16 or bf16 queries and pages of that type or e4m3");
  if (q->dim() != 3 || k->dim() != 4 || v->sizes() != k->sizes())
    REFUSE("paged_decode: q [B, Hq, D], k_pages and v_pages [P, Hkv, S, D]");
  const int64_t B = q->size(0), Hq = q->size(1), D = q->size(2);
  const int64_t P = k->size(0), Hkv = k->size(1), S = k->size(2);
  if (k->size(3) != D || D % 8 || D <= 0 || D > 256)
    REFUSE("paged_decode: heads of %ld and %ld (one multiple of 8, at most 256)", D, k->size(3));
  if (Hkv == 0 || Hq % Hkv || S == 0)
    REFUSE("paged_decode: %ld query heads over %ld kv heads, %ld slots a page", Hq, Hkv, S);
  if (tables->scalar_type() != at::kInt || tables->dim() != 2 || tables->size(0) != B)
    REFUSE("paged_decode: tables must be int32 [%ld, width]", B);
  if (lens->scalar_type() != at::kInt || lens->dim() != 1 || lens->size(0) != B || !dense(*lens))
    REFUSE("paged_decode: lens must be contiguous int32 [%ld]", B);
  const int64_t width = tables->size(1);
  if (!last1(*q) || !last1(*k) || !last1(*v) || !last1(*tables))
    REFUSE("paged_decode: the last dim of q, pages and tables must be contiguous");
  if (!fits(B) || !fits(Hq) || !fits(P) || !fits(S) || !fits(width)) REFUSE("paged_decode: sizes of 32 bits");
  const double cap = A.f(6), scale = args[5] == Py_None ? 1.0 / std::sqrt((double)D) : A.f(5);
  const long window = A.n(7);
  if (PyErr_Occurred()) return nullptr;
  const float fcap = (float)cap;
  if (window < 0 || !(cap == 0 || (fcap >= FLT_MIN && fcap <= FLT_MAX)))
    REFUSE("paged_decode: window=%ld (at least 0), softcap (0, or a float32 above it)", window);
  if (!vec(slopes, Hq)) REFUSE("paged_decode: slopes must be contiguous float32 [%ld]", Hq);
  if (!vec(ks, Hkv) || !vec(vs, Hkv)) REFUSE("paged_decode: k_scale and v_scale must be contiguous float32 [%ld]", Hkv);
  if (out && (out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type() || !dense(*out)))
    REFUSE("paged_decode: out must be contiguous, of q's type and shape");
  if (out && (meet(*out, *q) || meet(*out, *k) || meet(*out, *v))) REFUSE("paged_decode: out overlaps an input");
  const bool with_lse = PyObject_IsTrue(args[12]);
  at::Tensor o = out ? *out : result({B, Hq, D}, *q), l;
  if (with_lse) l = result({B, Hq}, *q, at::kFloat);
  UbridgePagedDecodeArgs p = {};
  p.q = q->data_ptr(), p.out = o.data_ptr(), p.lse = with_lse ? (float*)l.data_ptr() : nullptr;
  p.k_pages = k->data_ptr(), p.v_pages = v->data_ptr();
  p.tables = ptr<int32_t>(tables), p.lens = ptr<int32_t>(lens);
  p.slopes = ptr(slopes), p.k_scale = ptr(ks), p.v_scale = ptr(vs);
  p.q_sb = q->stride(0), p.q_sh = q->stride(1);
  p.k_sp = k->stride(0), p.k_sh = k->stride(1), p.k_ss = k->stride(2);
  p.v_sp = v->stride(0), p.v_sh = v->stride(1), p.v_ss = v->stride(2);
  p.table_stride = tables->stride(0);
  p.B = B, p.Hq = Hq, p.Hkv = Hkv, p.D = D, p.S = S, p.P = P, p.width = width;
  p.window = window > 0x7fffffff ? 0x7fffffff : (int)window;
  p.dtype = dt, p.cache_dtype = ct, p.scale = (float)scale, p.softcap = fcap;
  void* stream = A.p(13);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.decode(&p, stream)) return PyLong_FromLong(rc);
  PyObject* po = THPVariable_Wrap(std::move(o));
  return with_lse ? Py_BuildValue("[NN]", po, THPVariable_Wrap(std::move(l))) : po;
  END_HANDLE_TH_ERRORS
}

// a Rope's turns per position, f64 [rot / 2]
bool turn_list(Ten t, int rot) {
  if (rot >= 0 && t->scalar_type() == at::kDouble && t->dim() == 1 && t->size(0) == rot / 2 && dense(*t)) return true;
  PyErr_Format(PyExc_ValueError, "rope: turns must be contiguous float64 [%d]", rot / 2);
  return false;
}
// x [T, H, D] with its last dim contiguous
bool heads(const char* name, const at::Tensor& x, int64_t T, int64_t D) {
  if (x.dim() != 3 || x.size(0) != T || x.size(2) != D) {
    PyErr_Format(PyExc_ValueError, "rope: %s must be [%ld, heads, %ld]", name, T, D);
    return false;
  }
  if (!last1(x)) {
    PyErr_Format(PyExc_ValueError, "rope: the last dim of %s must be contiguous", name);
    return false;
  }
  return true;
}
bool position_list(Ten t, int64_t T, UbridgeRopeArgs& p) {
  if (t->dim() != 1 || t->size(0) != T || (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) || !dense(*t)) {
    PyErr_Format(PyExc_ValueError, "rope: positions must be contiguous int32 or int64 [%ld]", T);
    return false;
  }
  p.positions = t->data_ptr();
  p.pos64 = t->scalar_type() == at::kLong;
  return true;
}

// q, k | None, positions, turns, rot, interleaved, factor, inverse, stream
PyObject* py_rope(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(9)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten q, k, pos, turns;
  if (!device_tensor(args[0], q) || !device_tensor(args[1], k, true) || !device_tensor(args[2], pos) ||
      !device_tensor(args[3], turns))
    return nullptr;
  const int dt = code(*q);
  if (dt < 0 || dt > 2 || (k && k->scalar_type() != q->scalar_type()))
    REFUSE("rope takes f32, f16 or bf16 q and k of one type");
  UbridgeRopeArgs p = {};
  p.rot = (int)A.n(4);
  if (q->dim() != 3 || p.rot > q->size(2)) REFUSE("rope: q must be [T, heads, D] with D >= rot=%d", p.rot);
  const int64_t T = q->size(0), Hq = q->size(1), D = q->size(2), Hkv = k ? k->size(k->dim() == 3 ? 1 : 0) : 0;
  if (!heads("q", *q, T, D) || (k && !heads("k", *k, T, D)) || !position_list(pos, T, p) || !turn_list(turns, p.rot))
    return nullptr;
  if (!fits(T) || !fits(Hq) || !fits(Hkv) || !fits(D)) REFUSE("rope: sizes of 32 bits");
  at::Tensor qo = result({T, Hq, D}, *q), ko;
  p.q = q->data_ptr(), p.q_out = qo.data_ptr(), p.turns = ptr<double>(turns);
  p.q_st = q->stride(0), p.q_sh = q->stride(1);
  if (k) {
    ko = result({T, Hkv, D}, *q);
    p.k = k->data_ptr(), p.k_out = ko.data_ptr(), p.k_st = k->stride(0), p.k_sh = k->stride(1);
  }
  p.T = T, p.Hq = Hq, p.Hkv = Hkv, p.D = D;
  p.interleaved = PyObject_IsTrue(args[5]), p.factor = (float)A.f(6), p.inverse = PyObject_IsTrue(args[7]);
  p.dtype = p.cache_dtype = dt, p.S = 1;
  void* stream = A.p(8);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.rope(&p, stream)) return PyLong_FromLong(rc);
  PyObject* po = THPVariable_Wrap(std::move(qo));
  if (k) return Py_BuildValue("[NN]", po, THPVariable_Wrap(std::move(ko)));
  return Py_BuildValue("[NO]", po, Py_None);
  END_HANDLE_TH_ERRORS
}

// kv [L, 2, P, H, S, D], layer, k_scale, v_scale, q, k, v, slots, positions, turns
// | None, rot, interleaved, factor, stream
PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(14)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten kv, ks, vs, q, k, v, slots, pos, turns;
  const bool turned = args[9] != Py_None;
  if (!device_tensor(args[0], kv) || !device_tensor(args[2], ks, true) || !device_tensor(args[3], vs, true) ||
      !device_tensor(args[4], q, !turned) || !device_tensor(args[5], k) || !device_tensor(args[6], v) ||
      !device_tensor(args[7], slots) || !device_tensor(args[8], pos, true) || !device_tensor(args[9], turns, true))
    return nullptr;
  const long layer = A.n(1);
  if (kv->dim() != 6 || kv->size(1) != 2 || !dense(*kv) || !vec(ks, kv->size(3)) || !vec(vs, kv->size(3)))
    REFUSE("PagedCache.append: kv [L, 2, P, H, S, D], scales float32 [H], all contiguous");
  const int64_t L = kv->size(0), P = kv->size(2), H = kv->size(3), S = kv->size(4), D = kv->size(5);
  const int dt = code(*k), ct = code(*kv);
  if (dt < 0 || dt > 2 || v->scalar_type() != k->scalar_type() || (ct != dt && ct != 3))
    REFUSE("PagedCache.append: k and v of one type, that of the pages or into e4m3 pages");
  if (layer < 0 || layer >= L) REFUSE("PagedCache.append: layer %ld of %ld", layer, L);
  if (turned != (pos != nullptr)) REFUSE("PagedCache.append: rope and positions go together");
  const int64_t T = k->dim() == 3 ? k->size(0) : 0;
  if (k->dim() != 3 || k->size(1) != H || k->size(2) != D || v->sizes() != k->sizes())
    REFUSE("PagedCache.append: k and v must be [T, %ld, %ld]", H, D);
  if (slots->dim() != 1 || slots->size(0) != T || slots->scalar_type() != at::kLong || !dense(*slots))
    REFUSE("PagedCache.append: slots must be contiguous int64 [%ld]", T);
  if (!heads("k", *k, T, D) || !heads("v", *v, T, D)) return nullptr;
  if (!fits(T) || !fits(P) || !fits(S) || !fits(H) || !fits(D)) REFUSE("PagedCache.append: sizes of 32 bits");
  UbridgeRopeArgs p = {};
  at::Tensor qo;
  p.S = S, p.P = P, p.T = T, p.Hkv = H, p.D = D, p.dtype = dt, p.cache_dtype = ct, p.factor = 1.f;
  if (turned) {
    p.rot = (int)A.n(10);
    if (q->scalar_type() != k->scalar_type()) REFUSE("PagedCache.append: q and k of one type");
    if (p.rot > D) REFUSE("PagedCache.append: rot=%d of heads of %ld", p.rot, D);
    if (!heads("q", *q, T, D) || !position_list(pos, T, p) || !turn_list(turns, p.rot)) return nullptr;
    if (!fits(q->size(1))) REFUSE("PagedCache.append: sizes of 32 bits");
    p.Hq = q->size(1);
    qo = result({T, q->size(1), D}, *q);
    p.q = q->data_ptr(), p.q_out = qo.data_ptr(), p.q_st = q->stride(0), p.q_sh = q->stride(1);
    p.turns = ptr<double>(turns), p.interleaved = PyObject_IsTrue(args[11]), p.factor = (float)A.f(12);
  }
  p.page_stride = H * S * D;
  char* base = (char*)kv->data_ptr() + 2 * layer * P * p.page_stride * kv->element_size();
  p.k_pages = base, p.v_pages = base + P * p.page_stride * kv->element_size();
  p.k = k->data_ptr(), p.k_st = k->stride(0), p.k_sh = k->stride(1);
  p.v = v->data_ptr(), p.v_st = v->stride(0), p.v_sh = v->stride(1);
  p.slots = ptr<int64_t>(slots), p.k_scale = ptr(ks), p.v_scale = ptr(vs);
  void* stream = A.p(13);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.append(&p, stream)) return PyLong_FromLong(rc);
  if (turned) return THPVariable_Wrap(std::move(qo));
  Py_INCREF(args[4]);
  return args[4];
  END_HANDLE_TH_ERRORS
}

// x, w [N, ld], w_scale, bias | None, K, out | None, stream
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(7)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten x, w, sw, b, out;
  if (!device_tensor(args[0], x) || !device_tensor(args[1], w) || !device_tensor(args[2], sw) ||
      !device_tensor(args[3], b, true))
    return nullptr;
  const long K = A.n(4);
  if (w->scalar_type() != at::kChar || w->dim() != 2 || !dense(*w) || K <= 0 || w->size(1) < K || !vec(sw, w->size(0)) ||
      !vec(b, w->size(0)))
    REFUSE("int8.Linear: weight int8 [N, >= %ld], w_scale and bias float32 [N], all contiguous", K);
  const int dt = code(*x);
  if (dt < 0 || dt > 2 || x->dim() == 0 || x->size(-1) != K)
    REFUSE("int8.Linear takes f32, f16 or bf16 activations [..., %ld]", K);
  const int64_t M = x->numel() / K, N = w->size(0), ld = w->size(1);
  if (!fits(M)) REFUSE("int8.Linear: %ld rows", M);
  c10::SmallVector<int64_t, 4> sizes(x->sizes().begin(), x->sizes().end());
  sizes.back() = N;
  if (!THPVariable_Check(args[5]) && args[5] != Py_None) REFUSE("int8.Linear: out must be a tensor");
  out = args[5] == Py_None ? nullptr : &THPVariable_Unpack(args[5]);
  if (out && (!out->is_cuda() || out->scalar_type() != x->scalar_type() || out->sizes() != at::IntArrayRef(sizes) || !dense(*out)))
    REFUSE("int8.Linear: out must be contiguous, of x's type, [..., %ld]", N);
  if (out && meet(*out, *x)) REFUSE("int8.Linear: out overlaps x");
  at::Tensor y = out ? *out : result(sizes, *x), xc;
  const void* xp = x->data_ptr();
  if (!dense(*x)) {
    xc = x->contiguous();
    xp = xc.data_ptr();
  }
  void* stream = A.p(6);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.linear(xp, dt, (const int8_t*)w->data_ptr(), ptr(sw), ptr(b), y.data_ptr(), M, K, N, ld, stream))
    return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// The pool of a cache, whose two tensors are kv [L, 2, P, H, S, D] and meta [refs P
// | lens rows | tables rows x width]; false: refused.  (From the tensors at every
// call: addresses kept from another would outlive a copy of the cache.)
bool pool(PyObject* okv, PyObject* ometa, int64_t rows, int64_t width, UbridgeKvPool& p) {
  Ten kv, meta;
  if (!device_tensor(okv, kv) || !device_tensor(ometa, meta)) return false;
  if (kv->dim() != 6 || kv->size(1) != 2 || !dense(*kv) || !fits(rows) || !fits(width) || !fits(kv->size(0)) ||
      !fits(kv->size(2)) || !fits(kv->size(4)) || meta->scalar_type() != at::kInt || meta->dim() != 1 ||
      meta->size(0) != kv->size(2) + rows + rows * width || !dense(*meta)) {
    PyErr_SetString(PyExc_ValueError, "PagedCache: kv [L, 2, P, H, S, D] and meta int32 [P + rows + rows * width], contiguous");
    return false;
  }
  p = {};
  p.L = kv->size(0), p.P = kv->size(2), p.S = kv->size(4), p.rows = rows, p.width = width;
  p.kv = kv->data_ptr(), p.page_bytes = kv->size(3) * kv->size(4) * kv->size(5) * kv->element_size();
  p.refs = (int32_t*)meta->data_ptr(), p.lens = p.refs + p.P, p.tables = p.lens + rows;
  return true;
}
bool row_list(const char* name, const at::Tensor& t) {
  if (t.dim() == 1 && t.scalar_type() == at::kInt && dense(t) && fits(t.size(0))) return true;
  PyErr_Format(PyExc_ValueError, "PagedCache: %s must be contiguous int32 [n]", name);
  return false;
}

// kv, meta, the pool's rows, width, rows to free, stream
PyObject* py_free(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(6)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten rows;
  UbridgeKvPool p;
  if (!pool(args[0], args[1], A.n(2), A.n(3), p) || !device_tensor(args[4], rows) || !row_list("rows", *rows))
    return nullptr;
  void* stream = A.p(5);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.free(&p, ptr<int32_t>(rows), (int)rows->size(0), stream)) return PyLong_FromLong(rc);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// kv, meta, rows, width, src, dst, stream
PyObject* py_fork(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(7)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten src, dst;
  UbridgeKvPool p;
  if (!pool(args[0], args[1], A.n(2), A.n(3), p) || !device_tensor(args[4], src) || !device_tensor(args[5], dst) ||
      !row_list("src", *src) || !row_list("dst", *dst))
    return nullptr;
  const int64_t n = src->size(0);
  if (dst->size(0) != n || n > 65535)
    REFUSE("PagedCache.fork: %ld prompts, %ld samples (as many, at most 65535)", n, dst->size(0));
  at::Tensor pages = result({n}, *src);
  void* stream = A.p(6);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.fork(&p, ptr<int32_t>(src), ptr<int32_t>(dst), (int)n, (int32_t*)pages.data_ptr(), stream))
    return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(pages));
  END_HANDLE_TH_ERRORS
}

// kv, meta, rows, width, stream
PyObject* py_compact(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(5)
  HANDLE_TH_ERRORS
  const Args A{args};
  UbridgeKvPool p;
  if (!pool(args[0], args[1], A.n(2), A.n(3), p)) return nullptr;
  at::Tensor n = result({}, THPVariable_Unpack(args[1]));
  void* stream = A.p(4);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.compact(&p, (int32_t*)n.data_ptr(), stream)) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(n));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())py_bind, METH_FASTCALL, "the C entry points, as addresses"},
    {"paged_decode", (PyCFunction)(void (*)())py_decode, METH_FASTCALL, nullptr},
    {"rope", (PyCFunction)(void (*)())py_rope, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void (*)())py_append, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)())py_linear, METH_FASTCALL, nullptr},
    {"free", (PyCFunction)(void (*)())py_free, METH_FASTCALL, nullptr},
    {"fork", (PyCFunction)(void (*)())py_fork, METH_FASTCALL, nullptr},
    {"compact", (PyCFunction)(void (*)())py_compact, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module_def); }
