// native.cpp -- the host side of the attention block's calls and of the norm and
// feed-forward half: checks the tensors, allocates results and fills the argument
// blocks of include/ubridge_hip.h.
//
// A decode step calls these operators a few times a layer, at sizes where the
// kernels take 5 to 15 us; reading shapes, strides and types of six tensors
// from Python took 8 to 10 us a call, here about 1 us.  Every refusal is a ValueError, as in
// the Python modules; a nonzero status of the C entry is returned as an int, for
// the caller to raise.  Compute stays behind the C ABI, whose entry points
// native.py hands over (bind) from the library that it has loaded.
#include <Python.h>
#include <cfloat>
#include <cmath>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

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
  decltype(&ubridge_int8_linear_codes) linear_codes;
  decltype(&ubridge_rms_norm) norm;
  decltype(&ubridge_rms_norm_grad) norm_grad;
  decltype(&ubridge_mx_quantize) mx_quantize;
  decltype(&ubridge_mx_dequantize) mx_dequantize;
  decltype(&ubridge_mx_pack) mx_pack;
  decltype(&ubridge_mx_linear) mx_linear;
  decltype(&ubridge_moe_decode) moe_decode;
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
// After a caller's tensor (or null) has been written: graphs that saved it notice.
void written(Ten t) {
  if (t && !t->is_inference()) torch::autograd::impl::bump_version(*t);
}
bool records(Ten t) { return t && at::GradMode::is_enabled() && t->requires_grad(); }
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
  COUNT(15)
  const Args A{args};
  fn.decode = (decltype(fn.decode))A.p(0);
  fn.rope = (decltype(fn.rope))A.p(1);
  fn.append = (decltype(fn.append))A.p(2);
  fn.linear = (decltype(fn.linear))A.p(3);
  fn.free = (decltype(fn.free))A.p(4);
  fn.fork = (decltype(fn.fork))A.p(5);
  fn.compact = (decltype(fn.compact))A.p(6);
  fn.linear_codes = (decltype(fn.linear_codes))A.p(7);
  fn.norm = (decltype(fn.norm))A.p(8);
  fn.norm_grad = (decltype(fn.norm_grad))A.p(9);
  fn.mx_quantize = (decltype(fn.mx_quantize))A.p(10);
  fn.mx_dequantize = (decltype(fn.mx_dequantize))A.p(11);
  fn.mx_pack = (decltype(fn.mx_pack))A.p(12);
  fn.mx_linear = (decltype(fn.mx_linear))A.p(13);
  fn.moe_decode = (decltype(fn.moe_decode))A.p(14);
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
  written(out);
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
  written(out);
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

// ------------------------------------------- norm and feed-forward half
// Tensors of one call lie on one device.
bool together(const char* name, std::initializer_list<Ten> ts) {
  Ten first = nullptr;
  for (Ten t : ts) {
    if (!t) continue;
    if (!first) first = t;
    if (t->device() != first->device()) {
      PyErr_Format(PyExc_ValueError, "%s: tensors on several devices", name);
      return false;
    }
  }
  return true;
}
// Whether a gradient is asked for that the operator does not have: of an input that
// records, or one with a tangent (forward mode).  Refused: a result without it would be
// silently cut off.
bool without_gradient(const char* name, std::initializer_list<Ten> ts) {
  const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (Ten t : ts)
    if (records(t) || (t && forward && t->_fw_grad(/*level=*/0).defined())) {
      PyErr_Format(PyExc_ValueError, "%s: no gradient, and an input asks for one (detach it, or call under no_grad)", name);
      return false;
    }
  return true;
}
// None, or a tensor (anything else refused)
bool optional(PyObject* o, Ten& t) { return device_tensor(o, t, true); }
// a tuple of them, None for one that is not there
PyObject* tuple_of(std::initializer_list<at::Tensor*> ts) {
  PyObject* l = PyTuple_New(ts.size());
  Py_ssize_t i = 0;
  for (at::Tensor* t : ts) {
    PyObject* o = t->defined() ? THPVariable_Wrap(std::move(*t)) : (Py_INCREF(Py_None), Py_None);
    if (!l || !o) {
      Py_XDECREF(l), Py_XDECREF(o);
      return nullptr;
    }
    PyTuple_SET_ITEM(l, i++, o);
  }
  return l;
}
int64_t padded(int64_t c) { return (c + 127) / 128 * 128; }
c10::SmallVector<int64_t, 5> ended(const at::Tensor& x, int64_t last) {
  c10::SmallVector<int64_t, 5> s(x.sizes().begin(), x.sizes().end());
  s.back() = last;
  return s;
}
bool same(const at::Tensor& a, const at::Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes();
}

// x [..., C], w [C], residual | None, residual_out | None, eps, out (0 as x, 1 int8, 2
// e4m3, 3 fp4 blocks, 4 fp8 blocks), stream -> y, or (y, scale), (y, h), (y, scale, h);
// None where a gradient is asked for (refused with quant or residual_out)
PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(7)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten x, w, res, ho;
  if (!device_tensor(args[0], x) || !device_tensor(args[1], w) || !optional(args[2], res) || !optional(args[3], ho)) return nullptr;
  const int dt = code(*x), wt = code(*w);
  if (dt < 0 || dt > 2 || (wt != dt && wt != 0)) REFUSE("rms_norm takes f32, f16 or bf16 rows and a gain of that type or f32");
  if (x->dim() == 0 || w->dim() != 1 || w->size(0) != x->size(-1) || !dense(*w)) REFUSE("rms_norm: x [..., C], gain contiguous [C]");
  const int64_t C = x->size(-1), R = C ? x->numel() / C : 0;
  if (C == 0 || C * x->element_size() > 65536) REFUSE("rms_norm: rows of %ld (1 element to 64 KiB)", C);
  if (R >= 1 << 22) REFUSE("rms_norm: %ld rows", R);
  if (res && !same(*res, *x)) REFUSE("rms_norm: residual must be of x's type and shape");
  if (ho && (!res || !same(*ho, *x) || !dense(*ho))) REFUSE("rms_norm: residual_out goes with residual, contiguous, of x's type and shape");
  if (!together("rms_norm", {x, w, res, ho})) return nullptr;
  if (records(x) || records(w) || records(res) || records(ho)) {
    if (A.n(5) || ho) REFUSE("rms_norm: no gradient with quant or residual_out");
    Py_RETURN_NONE;
  }
  const double eps = A.f(4);
  const int out = (int)A.n(5);
  if (PyErr_Occurred()) return nullptr;
  if (!(eps >= 0 && eps <= 3.4e38)) REFUSE("rms_norm: eps must be a float32 of at least 0");
  at::Tensor xc = dense(*x) ? *x : x->contiguous(), rc, h, y, scale;
  if (res) {
    rc = dense(*res) ? *res : res->contiguous();
    h = ho ? *ho : result(x->sizes(), *x);
    // (each element is read ahead of its store by the thread that stores it)
    auto clash = [&](const at::Tensor& t) { return meet(h, t) && h.data_ptr() != t.data_ptr(); };
    if (clash(*x) || clash(*res) || meet(h, *w)) REFUSE("rms_norm: residual_out overlaps an input in part");
  }
  if (out == 0) {
    y = result(x->sizes(), *x);
  } else if (out <= 2) {
    y = result(x->sizes(), *x, out == 1 ? at::kChar : at::kByte);
    scale = result(x->sizes().slice(0, x->dim() - 1), *x, at::kFloat);
  } else {
    y = result(ended(*x, padded(C) / (out == 3 ? 2 : 1)), *x, at::kByte);
    scale = result(ended(*x, padded(C) / 32), *x, at::kByte);
  }
  UbridgeRmsNormArgs p = {};
  p.x = xc.data_ptr(), p.w = w->data_ptr(), p.y = y.data_ptr(), p.eps = eps;
  p.residual = res ? rc.data_ptr() : nullptr, p.h = res ? h.data_ptr() : nullptr;
  p.scale = out ? scale.data_ptr() : nullptr;
  p.R = R, p.C = C, p.dtype = dt, p.w_dtype = wt, p.out = out;
  void* stream = A.p(6);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc2 = fn.norm(&p, stream)) return PyLong_FromLong(rc2);
  written(ho);
  if (out && res) return tuple_of({&y, &scale, &h});
  if (out || res) return tuple_of({&y, out ? &scale : &h});
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// Whether one of the tensors (or None) is a leaf whose gradient is accumulated on the
// default stream, by a graph that lives already: a backward pass that is being captured
// would wait for that stream, which ends the capture and with it the process.
PyObject* py_default_stream_leaf(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < nargs; i++) {
    Ten t;
    if (!optional(args[i], t)) return nullptr;
    if (!t || !t->requires_grad() || t->grad_fn()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && stream->id() == 0) Py_RETURN_TRUE;
  }
  Py_RETURN_FALSE;
  END_HANDLE_TH_ERRORS
}

// h [..., C], w, dy, dh | None, eps, whether dx, whether dw, stream -> (dx | None, dw | None)
PyObject* py_norm_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(8)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten h, w, dy, dh;
  if (!device_tensor(args[0], h) || !device_tensor(args[1], w) || !device_tensor(args[2], dy) || !optional(args[3], dh)) return nullptr;
  const int dt = code(*h), wt = code(*w);
  const int64_t C = h->dim() ? h->size(-1) : 0, R = C ? h->numel() / C : 0;
  if (dt < 0 || dt > 2 || (wt != dt && wt != 0) || C == 0 || C * h->element_size() > 65536 || R >= 1 << 22 || w->dim() != 1 ||
      w->size(0) != C || !dense(*w) || !dense(*h) || !same(*dy, *h) || (dh && !same(*dh, *h)))
    REFUSE("rms_norm's gradient: h, dy and dh [..., C] of one type and shape, gain [C]");
  if (!together("rms_norm's gradient", {h, w, dy, dh})) return nullptr;
  at::Tensor dyc = dense(*dy) ? *dy : dy->contiguous(), dhc, dx, dw;
  if (dh) dhc = dense(*dh) ? *dh : dh->contiguous();
  if (PyObject_IsTrue(args[5])) dx = result(h->sizes(), *h);
  if (PyObject_IsTrue(args[6])) dw = result(w->sizes(), *w);
  UbridgeRmsNormGradArgs p = {};
  p.h = h->data_ptr(), p.w = w->data_ptr(), p.dy = dyc.data_ptr(), p.dh = dh ? dhc.data_ptr() : nullptr;
  p.dx = dx.defined() ? dx.data_ptr() : nullptr, p.dw = dw.defined() ? dw.data_ptr() : nullptr;
  p.eps = A.f(4), p.R = R, p.C = C, p.dtype = dt, p.w_dtype = wt;
  void* stream = A.p(7);
  if (PyErr_Occurred()) return nullptr;
  // (without rows dx has no memory, and there is nothing to run but dw's zeros)
  if ((p.dx && R) || p.dw)
    if (const int rc = fn.norm_grad(&p, stream)) return PyLong_FromLong(rc);
  return tuple_of({&dx, &dw});
  END_HANDLE_TH_ERRORS
}

// x [..., C], format (4, 8), stream -> (codes, scales)
PyObject* py_mx_quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(3)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten x;
  if (!device_tensor(args[0], x)) return nullptr;
  const int dt = code(*x), f = (int)A.n(1);
  if (dt < 0 || dt > 2 || x->dim() == 0 || x->size(-1) == 0) REFUSE("mx.quantize takes f32, f16 or bf16 [..., C]");
  if (!without_gradient("mx.quantize", {x})) return nullptr;
  const int64_t C = x->size(-1), R = x->numel() / C;
  if (!fits(R) || C > 1 << 30 || R * (C + 127) > 1ll << 33) REFUSE("mx.quantize: %ld rows of %ld", R, C);
  at::Tensor xc = dense(*x) ? *x : x->contiguous();
  at::Tensor q = result(ended(*x, padded(C) * f / 8), *x, at::kByte), s = result(ended(*x, padded(C) / 32), *x, at::kByte);
  void* stream = A.p(2);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.mx_quantize(xc.data_ptr(), dt, q.data_ptr(), s.data_ptr(), R, C, f, stream)) return PyLong_FromLong(rc);
  return tuple_of({&q, &s});
  END_HANDLE_TH_ERRORS
}

// codes and scales of rows of K elements; false: refused
bool block_rows(const char* name, Ten q, Ten s, int64_t K, int f) {
  if (K > 0 && K <= 1 << 30 && q->dim() > 0 && s->dim() == q->dim() && q->scalar_type() == at::kByte && s->scalar_type() == at::kByte &&
      q->size(-1) == padded(K) * f / 8 && s->size(-1) == padded(K) / 32 &&
      q->sizes().slice(0, q->dim() - 1) == s->sizes().slice(0, s->dim() - 1) && dense(*q) && dense(*s) &&
      ((uintptr_t)q->data_ptr() & 15) == 0 && ((uintptr_t)s->data_ptr() & 3) == 0)
    return true;
  PyErr_Format(PyExc_ValueError, "%s: codes uint8 [..., %ld] and scales uint8 [..., %ld] of rows of %ld, contiguous, aligned to 16 and 4 bytes",
               name, padded(K) * f / 8, padded(K) / 32, K);
  return false;
}

at::ScalarType type_of(int dt) { return dt == 0 ? at::kFloat : dt == 1 ? at::kHalf : at::kBFloat16; }

// codes, scales, C, type code, format, stream -> values [..., C]
PyObject* py_mx_dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(6)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten q, s;
  if (!device_tensor(args[0], q) || !device_tensor(args[1], s)) return nullptr;
  const int64_t C = A.n(2);
  const int dt = (int)A.n(3), f = (int)A.n(4);
  if (PyErr_Occurred() || !block_rows("mx.dequantize", q, s, C, f) || !together("mx.dequantize", {q, s})) return nullptr;
  const int64_t R = q->numel() / q->size(-1);
  if (!fits(R) || R * (C + 127) > 1ll << 33) REFUSE("mx.dequantize: %ld rows of %ld", R, C);
  at::Tensor y = result(ended(*q, C), *q, type_of(dt));
  void* stream = A.p(5);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.mx_dequantize(q->data_ptr(), s->data_ptr(), y.data_ptr(), dt, R, C, f, stream)) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// codes [N, ld / 2], scales [N, ld / 32], K, stream -> (w, w_scales)
PyObject* py_mx_pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(4)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten q, s;
  if (!device_tensor(args[0], q) || !device_tensor(args[1], s)) return nullptr;
  const int64_t K = A.n(2);
  if (PyErr_Occurred() || !block_rows("mx.Linear", q, s, K, 4) || !together("mx.Linear", {q, s})) return nullptr;
  const int64_t N = q->size(0), N16 = (N + 15) / 16 * 16;
  if (q->dim() != 2 || !fits(N) || K > 131072) REFUSE("mx.Linear: weight [N, K=%ld] (1..131072)", K);
  at::Tensor w = result({N16, padded(K) / 2}, *q), ws = result({N16, padded(K) / 32}, *q);
  void* stream = A.p(3);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.mx_pack(q->data_ptr(), s->data_ptr(), w.data_ptr(), ws.data_ptr(), N, K, stream)) return PyLong_FromLong(rc);
  return tuple_of({&w, &ws});
  END_HANDLE_TH_ERRORS
}

// first (x [..., K], or codes), scales | None, w, w_scales, bias | None, K, N, format,
// type code (of y, with codes), out | None, whether one product, stream
PyObject* py_mx_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(12)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten x, s, w, ws, b, out;
  if (!device_tensor(args[0], x) || !optional(args[1], s) || !device_tensor(args[2], w) || !device_tensor(args[3], ws) ||
      !optional(args[4], b) || !optional(args[9], out))
    return nullptr;
  const int64_t K = A.n(5), N = A.n(6);
  const int f = (int)A.n(7);
  int dt = (int)A.n(8);
  if (PyErr_Occurred()) return nullptr;
  if (s) {
    if (!block_rows("mx.Linear", x, s, K, f)) return nullptr;
  } else {
    dt = code(*x);
    if (dt < 0 || dt > 2 || x->dim() == 0 || x->size(-1) != K) REFUSE("mx.Linear takes f32, f16 or bf16 activations [..., %ld]", K);
  }
  const int64_t N16 = (N + 15) / 16 * 16;
  if (w->scalar_type() != at::kByte || ws->scalar_type() != at::kByte || !dense(*w) || !dense(*ws) || w->numel() != N16 * padded(K) / 2 ||
      ws->numel() != N16 * padded(K) / 32 || !vec(b, N))
    REFUSE("mx.Linear: weight as mx.Linear laid it out, bias contiguous float32 [%ld]", N);
  if (!together("mx.Linear", {x, s, w, ws, b, out})) return nullptr;
  const int64_t M = x->numel() / x->size(-1);
  if (M >= 1 << 22 || M * N >= 1ll << 38 || (M + 15) * (K + 127) > 1ll << 33) REFUSE("mx.Linear: %ld rows of %ld to %ld", M, K, N);
  const auto sizes = ended(*x, N);
  if (out && (out->scalar_type() != type_of(dt) || out->sizes() != at::IntArrayRef(sizes) || !dense(*out)))
    REFUSE("mx.Linear: out must be contiguous, of y's type, [..., %ld]", N);
  if (!without_gradient("mx.Linear", {x, b, out})) return nullptr;
  if (out && (meet(*out, *x) || (s && meet(*out, *s)) || meet(*out, *w) || meet(*out, *ws) || (b && meet(*out, *b))))
    REFUSE("mx.Linear: out overlaps an input");
  at::Tensor y = out ? *out : result(sizes, *x, type_of(dt)), xc = dense(*x) ? *x : x->contiguous();
  UbridgeMxLinearArgs p = {};
  if (s) p.codes = xc.data_ptr(), p.scales = s->data_ptr();
  else p.x = xc.data_ptr();
  p.w = w->data_ptr(), p.w_scales = ws->data_ptr(), p.bias = ptr(b), p.y = y.data_ptr();
  p.M = M, p.K = K, p.N = N, p.dtype = dt, p.format = f, p.one_product = PyObject_IsTrue(args[10]);
  void* stream = A.p(11);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.mx_linear(&p, stream)) return PyLong_FromLong(rc);
  written(out);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// codes int8 [..., ld], scales [...], w [N, ld], w_scale, bias | None, K, type code, out |
// None, stream
PyObject* py_linear_codes(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(9)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten q, s, w, sw, b, out;
  if (!device_tensor(args[0], q) || !device_tensor(args[1], s) || !device_tensor(args[2], w) || !device_tensor(args[3], sw) ||
      !optional(args[4], b) || !optional(args[7], out))
    return nullptr;
  const int64_t K = A.n(5);
  const int dt = (int)A.n(6);
  if (PyErr_Occurred()) return nullptr;
  if (w->scalar_type() != at::kChar || w->dim() != 2 || !dense(*w) || K <= 0 || w->size(1) < K || !vec(sw, w->size(0)) ||
      !vec(b, w->size(0)))
    REFUSE("int8.Linear: weight int8 [N, >= %ld], w_scale and bias float32 [N], all contiguous", K);
  const int64_t N = w->size(0), ld = w->size(1);
  if (q->scalar_type() != at::kChar || q->dim() == 0 || q->size(-1) != ld || !dense(*q) || ((uintptr_t)q->data_ptr() & 15) ||
      s->scalar_type() != at::kFloat || s->sizes() != q->sizes().slice(0, q->dim() - 1) || !dense(*s))
    REFUSE("int8.Linear: codes int8 [..., %ld], aligned to 16 bytes, and scales float32 [...], contiguous", ld);
  if (!together("int8.Linear", {q, s, w, sw, b, out})) return nullptr;
  const int64_t M = q->numel() / ld;
  if (!fits(M)) REFUSE("int8.Linear: %ld rows", M);
  const auto sizes = ended(*q, N);
  if (out && (out->scalar_type() != type_of(dt) || out->sizes() != at::IntArrayRef(sizes) || !dense(*out)))
    REFUSE("int8.Linear: out must be contiguous, of y's type, [..., %ld]", N);
  if (!without_gradient("int8.Linear", {s, sw, b, out})) return nullptr;
  if (out && (meet(*out, *q) || meet(*out, *s) || meet(*out, *w) || meet(*out, *sw) || (b && meet(*out, *b))))
    REFUSE("int8.Linear: out overlaps an input");
  at::Tensor y = out ? *out : result(sizes, *q, type_of(dt));
  void* stream = A.p(8);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.linear_codes((const int8_t*)q->data_ptr(), ptr(s), (const int8_t*)w->data_ptr(), ptr(sw), ptr(b), y.data_ptr(), dt, M,
                                     K, N, ld, stream))
    return PyLong_FromLong(rc);
  written(out);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// x [T, H], logits [T, E], w13, s13 | None, w2, s2 | None, k, renormalize, stream
PyObject* py_moe_decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  COUNT(9)
  HANDLE_TH_ERRORS
  const Args A{args};
  Ten x, lg, w13, s13, w2, s2;
  if (!device_tensor(args[0], x) || !device_tensor(args[1], lg) || !device_tensor(args[2], w13) || !optional(args[3], s13) ||
      !device_tensor(args[4], w2) || !optional(args[5], s2))
    return nullptr;
  const long k = A.n(6);
  if (PyErr_Occurred()) return nullptr;
  const int dt = code(*x), lt = code(*lg);
  if ((dt != 1 && dt != 2) || lt < 0 || lt > 2) REFUSE("FusedMoE.decode takes f16 or bf16 rows and f32, f16 or bf16 logits");
  if (x->dim() != 2 || lg->dim() != 2 || w13->dim() != 3 || w2->dim() != 3) REFUSE("FusedMoE.decode: x [T, H], logits [T, E], w13 [E, 2 I, H], w2 [E, H, I]");
  const int64_t T = x->size(0), H = x->size(1), E = w13->size(0), I = w2->size(2);
  if (lg->size(0) != T || lg->size(1) != E || w13->size(1) != 2 * I || w13->size(2) != H || w2->size(0) != E || w2->size(1) != H)
    REFUSE("FusedMoE.decode: x [%ld, %ld], logits [%ld, %ld], w13 [%ld, %ld, %ld], w2 [%ld, %ld, %ld] do not fit", T, H, lg->size(0),
           lg->size(1), E, w13->size(1), w13->size(2), w2->size(0), w2->size(1), I);
  const bool q8 = w13->scalar_type() == at::kChar;
  if (w2->scalar_type() != w13->scalar_type() || (!q8 && w13->scalar_type() != x->scalar_type()))
    REFUSE("FusedMoE.decode: experts are both int8 or both in the activations' dtype");
  if (q8 != (s13 != nullptr) || q8 != (s2 != nullptr)) REFUSE("FusedMoE.decode: int8 experts, and they alone, have scales");
  if (q8 && (s13->scalar_type() != x->scalar_type() || s2->scalar_type() != x->scalar_type() || s13->numel() != E * 2 * I ||
             s2->numel() != E * H || !dense(*s13) || !dense(*s2)))
    REFUSE("FusedMoE.decode: scales of x's type, [E, 2 I] and [E, H], contiguous");
  if (!dense(*w13) || !dense(*w2)) REFUSE("FusedMoE.decode: experts must be contiguous");
  if (T > 16 || k < 1 || k > 16 || k > E || E > 1024 || H == 0 || I == 0 || H % 32 || I % 32 || H > 1 << 20 || I > 1 << 20)
    REFUSE("FusedMoE.decode: T=%ld (at most 16), topk=%ld (1..16, at most E), E=%ld (at most 1024), H=%ld and I=%ld (multiples of 32)", T, k,
           E, H, I);
  if (!together("FusedMoE.decode", {x, lg, w13, s13, w2, s2})) return nullptr;
  if (!without_gradient("FusedMoE.decode", {x, lg, w13, s13, w2, s2})) return nullptr;
  auto whole = [](const at::Tensor& t, int align) { return dense(t) && ((uintptr_t)t.data_ptr() & (align - 1)) == 0; };
  at::Tensor xc = *x, lc = dense(*lg) ? *lg : lg->contiguous();
  if (!whole(xc, 16)) xc = xc.clone(at::MemoryFormat::Contiguous);
  if (!whole(*w13, 16) || !whole(*w2, 16)) REFUSE("FusedMoE.decode: experts not 16-byte aligned");
  at::Tensor y = result({T, H}, *x);
  UbridgeMoeDecodeArgs p = {};
  p.x = xc.data_ptr(), p.logits = lc.data_ptr(), p.w13 = w13->data_ptr(), p.w2 = w2->data_ptr(), p.y = y.data_ptr();
  p.s13 = q8 ? s13->data_ptr() : nullptr, p.s2 = q8 ? s2->data_ptr() : nullptr;
  p.T = T, p.E = E, p.k = k, p.H = H, p.I = I, p.dtype = dt, p.logits_dtype = lt, p.renormalize = PyObject_IsTrue(args[7]);
  void* stream = A.p(8);
  if (PyErr_Occurred()) return nullptr;
  if (const int rc = fn.moe_decode(&p, stream)) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(y));
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
    {"linear_codes", (PyCFunction)(void (*)())py_linear_codes, METH_FASTCALL, nullptr},
    {"norm", (PyCFunction)(void (*)())py_norm, METH_FASTCALL, nullptr},
    {"default_stream_leaf", (PyCFunction)(void (*)())py_default_stream_leaf, METH_FASTCALL, nullptr},
    {"norm_grad", (PyCFunction)(void (*)())py_norm_grad, METH_FASTCALL, nullptr},
    {"mx_quantize", (PyCFunction)(void (*)())py_mx_quantize, METH_FASTCALL, nullptr},
    {"mx_dequantize", (PyCFunction)(void (*)())py_mx_dequantize, METH_FASTCALL, nullptr},
    {"mx_pack", (PyCFunction)(void (*)())py_mx_pack, METH_FASTCALL, nullptr},
    {"mx_linear", (PyCFunction)(void (*)())py_mx_linear, METH_FASTCALL, nullptr},
    {"moe_decode", (PyCFunction)(void (*)())py_moe_decode, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module_def); }
