// Host side of the row ops' Python entry points: the argument checks and the C-ABI call of ops.gpu_adam,
// gpu_ops.init_rows and gpu_ops.replay_rows in one native call, and of the operators in logprobs, norms, gradnorm, int8 and sampling, for
// the arguments a training loop passes (plain contiguous GPU tensors of the expected types on the current device).
// Everything else -- other types, strides or devices, arenas in host memory, wrapped tensors, errors -- is answered with NOT_TAKEN, and the Python path then
// converts, raises or runs as it always has, so the two accept and refuse the same calls.
//
// Why: at a few hundred rows a call is host time.  The Python checks and ctypes conversions of gpu_adam took 3.7 of its
// 7.5 us (600 rows of width 32), those of replay_rows 8 of 13.5 (5,000 rows); the calls here take 4.1 and 6.0 us.
//
// The library's entry points are handed over by address (bind), so this module calls the library that ctypes loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstring>
#include <vector>

#include <ATen/ops/empty.h>
#include <c10/core/DefaultDtype.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/elara_amd.h"

namespace {

using adam_scalars_t = decltype(&elr_adam_scalars);
using adam_rows_t = decltype(&elr_adam_rows);
using init_rows_t = decltype(&elr_init_rows);
using replay_rows_t = decltype(&elr_replay_rows);
adam_scalars_t f_scalars = nullptr;
adam_rows_t f_adam = nullptr;
init_rows_t f_init = nullptr;
replay_rows_t f_replay = nullptr;

constexpr int kNotTaken = -1000;

PyObject* not_taken() { return PyLong_FromLong(kNotTaken); }

// A plain dense GPU tensor: no subclass, no functorch or functional wrapper, no lazy negation or conjugation, strided
// and contiguous.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
  constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::Python,
                                         c10::DispatchKey::Negative, c10::DispatchKey::Conjugate,
                                         c10::DispatchKey::ZeroTensor});
  if (t.key_set().has_any(wrapped) || !t.is_contiguous()) return nullptr;
  return &t;
}

bool real(PyObject* o, double& v) {
  v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool integer(PyObject* o, int64_t& v) {   // an int that fits (anything else is the Python path's to convert)
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  v = PyLong_AsLongLongAndOverflow(o, &over);
  return !over;
}

// Other Python threads run while torch allocates and the library launches, as they do through torch and ctypes.  (The
// caller's frame keeps the arguments alive.)
struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  NoGil() = default;
  NoGil(const NoGil&) = delete;
  ~NoGil() { PyEval_RestoreThread(s); }
};

// The current stream of the current device, if that is t's device.
bool stream_on(const at::Tensor& t, void*& st) {
  const auto s = c10::hip::getCurrentHIPStream();   // of the current device
  if (s.device_index() != t.device().index()) return false;
  st = s.stream();
  return true;
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d;
  if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return nullptr;
  f_scalars = reinterpret_cast<adam_scalars_t>(a);
  f_adam = reinterpret_cast<adam_rows_t>(b);
  f_init = reinterpret_cast<init_rows_t>(c);
  f_replay = reinterpret_cast<replay_rows_t>(d);
  Py_RETURN_NONE;
}

// adam(pool, slots, grad, lr, b1, b2, eps, step) -> return code, or NOT_TAKEN
PyObject* adam(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 8 || !f_adam) return not_taken();
  const at::Tensor *pool = plain(a[0]), *slots = plain(a[1]), *grad = plain(a[2]);
  double lr, b1, b2, eps;
  int64_t step;
  if (!pool || !slots || !grad || !real(a[3], lr) || !real(a[4], b1) || !real(a[5], b2) || !real(a[6], eps) ||
      !integer(a[7], step))
    return not_taken();
  const auto it = slots->scalar_type();
  if (pool->scalar_type() != at::kFloat || pool->dim() != 3 || pool->size(1) != 3 ||
      (it != at::kInt && it != at::kLong) || grad->scalar_type() != at::kFloat || slots->device() != pool->device() ||
      grad->device() != pool->device())
    return not_taken();
  const int64_t n = slots->numel(), D = pool->size(2);
  if (n == 0 || D == 0 || grad->numel() != n * D) return not_taken();
  int rc = kNotTaken;
  try {
    NoGil g;
    void* st;
    if (stream_on(*pool, st)) {
      float sc[8];
      f_scalars(lr, b1, b2, eps, step, sc);
      rc = f_adam(static_cast<float*>(pool->data_ptr()), pool->size(0), slots->data_ptr(), it == at::kLong,
                  static_cast<const float*>(grad->data_ptr()), n, D, sc, st);
    }
  } catch (const std::exception&) {   // torch's own error comes from the Python path
    return not_taken();
  }
  return PyLong_FromLong(rc);
}

// The result [n, 3, D] on rows' device, as torch.empty(n, 3, D, device=...) makes it with the default type float32.
bool new_states(const at::Tensor& rows, int64_t D, at::Tensor& out) {
  if (c10::get_default_dtype_as_scalartype() != at::kFloat) return false;
  out = at::empty({rows.numel(), 3, D}, at::TensorOptions().dtype(at::kFloat).device(rows.device()));
  return true;
}

// init(rows, D, seed, bound) -> (return code, out), or NOT_TAKEN
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 4 || !f_init) return not_taken();
  const at::Tensor* rows = plain(a[0]);
  int64_t D, seed;
  double bound;
  if (!rows || rows->scalar_type() != at::kLong || !integer(a[1], D) || D < 1 || !integer(a[2], seed) ||
      !real(a[3], bound) || rows->numel() == 0)
    return not_taken();
  try {
    at::Tensor out;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*rows, st) && new_states(*rows, D, out))
        rc = f_init(static_cast<float*>(out.data_ptr()), static_cast<const int64_t*>(rows->data_ptr()),
                    rows->numel(), D, static_cast<uint32_t>(seed), static_cast<float>(bound), st);
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(out));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// replay(rows, logs, offs, steps, cnt, D, K, seed, bound, table, recip) -> (return code, out), or NOT_TAKEN
PyObject* replay(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 11 || !f_replay) return not_taken();
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i)
    if (!(t[i] = plain(a[i]))) return not_taken();
  const at::Tensor *table = plain(a[9]), *recip = plain(a[10]);
  const at::Tensor &rows = *t[0], &logs = *t[1], &offs = *t[2], &steps = *t[3], &cnt = *t[4];
  int64_t D, K, seed;
  double bound;
  if (!table || !recip || !integer(a[5], D) || D < 1 || !integer(a[6], K) || K < 1 || K > 8 || !integer(a[7], seed) ||
      !real(a[8], bound))
    return not_taken();
  const int64_t n = rows.numel();
  if (rows.scalar_type() != at::kLong || logs.scalar_type() != at::kFloat || offs.scalar_type() != at::kLong ||
      steps.scalar_type() != at::kInt || cnt.scalar_type() != at::kInt || table->scalar_type() != at::kFloat ||
      recip->scalar_type() != at::kDouble || n == 0 || offs.numel() != n || cnt.numel() != n ||
      steps.numel() != n * K || logs.numel() % D || table->dim() != 2 || table->size(1) != 8 || recip->dim() != 2 ||
      recip->size(0) != table->size(0) || recip->size(1) != 2)
    return not_taken();
  for (const at::Tensor* x : {&logs, &offs, &steps, &cnt, table, recip})
    if (x->device() != rows.device()) return not_taken();
  try {
    at::Tensor out;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(rows, st) && new_states(rows, D, out))
        rc = f_replay(static_cast<float*>(out.data_ptr()), static_cast<const int64_t*>(rows.data_ptr()),
                      static_cast<const float*>(logs.data_ptr()), logs.numel() / D,
                      static_cast<const int64_t*>(offs.data_ptr()), static_cast<const int32_t*>(steps.data_ptr()),
                      static_cast<const int32_t*>(cnt.data_ptr()), n, D, static_cast<int>(K),
                      static_cast<uint32_t>(seed), static_cast<float>(bound),
                      static_cast<const float*>(table->data_ptr()), static_cast<const double*>(recip->data_ptr()),
                      table->size(0), st);
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(out));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// ---- logprobs, norms, gradnorm

decltype(&elr_token_logprobs_scratch_bytes) f_lp_bytes = nullptr;
decltype(&elr_token_logprobs) f_lp = nullptr;
decltype(&elr_token_logprobs_backward) f_lp_back = nullptr;
decltype(&elr_rms_norm) f_norm = nullptr;
decltype(&elr_rms_norm_backward_scratch_bytes) f_norm_bytes = nullptr;
decltype(&elr_rms_norm_backward) f_norm_back = nullptr;
decltype(&elr_grad_norm_scratch_bytes) f_grad_bytes = nullptr;
decltype(&elr_grad_norm) f_grad_norm = nullptr;
decltype(&elr_clip_grad_norm) f_clip = nullptr;

template <class F>
void set_address(F& f, unsigned long long a) {
  f = reinterpret_cast<F>(a);
}

PyObject* bind_ops(PyObject*, PyObject* args) {
  unsigned long long a[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7, a + 8)) return nullptr;
  set_address(f_lp_bytes, a[0]), set_address(f_lp, a[1]), set_address(f_lp_back, a[2]);
  set_address(f_norm, a[3]), set_address(f_norm_bytes, a[4]), set_address(f_norm_back, a[5]);
  set_address(f_grad_bytes, a[6]), set_address(f_grad_norm, a[7]), set_address(f_clip, a[8]);
  Py_RETURN_NONE;
}

int elem_type(const at::Tensor& t) {   // ELR_F32, ELR_F16, ELR_BF16, or -1
  switch (t.scalar_type()) {
    case at::kFloat: return ELR_F32;
    case at::kHalf: return ELR_F16;
    case at::kBFloat16: return ELR_BF16;
    default: return -1;
  }
}

// None (sets t to nullptr) or a plain tensor; false: anything else.
bool maybe(PyObject* o, const at::Tensor*& t) {
  t = nullptr;
  return o == Py_None || (t = plain(o)) != nullptr;
}

at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

// The scratch of a call (8-byte elements), undefined for none.
at::Tensor scratch_on(const at::Tensor& like, int64_t bytes) {
  return bytes > 0 ? empty_on(like, {(bytes + 7) / 8}, at::kDouble) : at::Tensor();
}
void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* floats(const at::Tensor* t) { return t ? static_cast<const float*>(t->data_ptr()) : nullptr; }

PyObject* wrap_or_none(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// A tensor's bytes.
struct Range {
  uintptr_t begin, end;
  bool out;
};
Range range_of(const at::Tensor& t, bool out) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + static_cast<uintptr_t>(t.numel() * t.element_size()), out};
}
// Whether an output meets another range (inputs may meet one another).
bool meet(std::vector<Range>& r) {
  const auto before = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
  uintptr_t out_end = 0, end = 0;
  for (const Range& x : r) {
    if (x.begin < (x.out ? end : out_end)) return true;
    end = std::max(end, x.end);
    if (x.out) out_end = std::max(out_end, x.end);
  }
  return false;
}

// logprobs(logits, tokens, k) -> (return code, logprob, lse, entropy, top_logprob, top_id), or NOT_TAKEN
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 3 || !f_lp) return not_taken();
  const at::Tensor *x = plain(a[0]), *tok = plain(a[1]);
  int64_t k;
  if (!x || !tok || !integer(a[2], k) || x->dim() < 1 || x->numel() == 0) return not_taken();
  const int type = elem_type(*x);
  const auto it = tok->scalar_type();
  const int64_t V = x->size(-1), n = x->numel() / V;
  if (type < 0 || (it != at::kInt && it != at::kLong) || tok->device() != x->device() ||
      tok->sizes() != x->sizes().slice(0, x->dim() - 1) || k < 0 || k > V || k > ELR_TOPK_MAX)
    return not_taken();
  try {
    at::Tensor lp, id, lse, ent, val;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x, st)) {
        std::vector<int64_t> shape(tok->sizes().begin(), tok->sizes().end());
        val = empty_on(*x, shape, at::kFloat), lse = empty_on(*x, shape, at::kFloat);
        ent = empty_on(*x, shape, at::kFloat);
        if (k) {
          shape.push_back(k);
          lp = empty_on(*x, shape, at::kFloat), id = empty_on(*x, shape, at::kLong);
        }
        const int64_t bytes = f_lp_bytes(n, V, static_cast<int>(k));
        const at::Tensor scratch = scratch_on(*x, bytes);
        rc = f_lp(x->data_ptr(), type, n, V, V, tok->data_ptr(), it == at::kLong, static_cast<int>(k),
                  static_cast<float*>(val.data_ptr()), static_cast<float*>(lse.data_ptr()),
                  static_cast<float*>(ent.data_ptr()), static_cast<float*>(data_or_null(lp)),
                  static_cast<int64_t*>(data_or_null(id)), data_or_null(scratch), bytes, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iNNNNN)", rc, THPVariable_Wrap(val), THPVariable_Wrap(lse), THPVariable_Wrap(ent),
                         wrap_or_none(lp), wrap_or_none(id));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// logprobs_back(logits, tokens, lse, entropy, d_logprob, d_entropy, d_lse, out) -> (return code, out), or NOT_TAKEN
PyObject* logprobs_back(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 8 || !f_lp_back) return not_taken();
  const at::Tensor *x = plain(a[0]), *tok = plain(a[1]), *lse = plain(a[2]), *r[4], *out;
  for (int i = 0; i < 4; ++i)
    if (!maybe(a[3 + i], r[i])) return not_taken();
  if (!x || !tok || !lse || !maybe(a[7], out) || x->dim() < 1 || x->numel() == 0) return not_taken();
  const int type = elem_type(*x);
  const auto it = tok->scalar_type();
  const int64_t V = x->size(-1), n = x->numel() / V;
  if (type < 0 || (it != at::kInt && it != at::kLong) || tok->device() != x->device() ||
      tok->sizes() != x->sizes().slice(0, x->dim() - 1) || (r[2] && !r[0]))
    return not_taken();
  for (const at::Tensor* t : {lse, r[0], r[1], r[2], r[3]})
    if (t && (t->scalar_type() != at::kFloat || t->device() != x->device() || t->sizes() != tok->sizes()))
      return not_taken();
  if (out && (out->scalar_type() != x->scalar_type() || out->device() != x->device() || out->sizes() != x->sizes()))
    return not_taken();
  if (out && out->data_ptr() != x->data_ptr()) {
    std::vector<Range> ranges{range_of(*x, false), range_of(*out, true)};
    if (meet(ranges)) return not_taken();
  }
  try {
    at::Tensor made;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x, st)) {
        if (!out) made = empty_on(*x, x->sizes(), x->scalar_type());
        rc = f_lp_back(x->data_ptr(), type, n, V, V, tok->data_ptr(), it == at::kLong, floats(lse),
                       r[2] ? floats(r[0]) : nullptr, floats(r[1]), floats(r[2]), floats(r[3]),
                       out ? out->data_ptr() : made.data_ptr(), V, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    if (!out) return Py_BuildValue("(iN)", rc, THPVariable_Wrap(made));
    return Py_BuildValue("(iO)", rc, a[7]);
  } catch (const std::exception&) {
    return not_taken();
  }
}

// A weight of D elements for inputs of type `like` (None: ones); its type in `type`.
bool weight_ok(const at::Tensor* w, const at::Tensor& like, int64_t D, int& type) {
  type = elem_type(w ? *w : like);
  return !w || ((w->scalar_type() == like.scalar_type() || w->scalar_type() == at::kFloat) && w->dim() == 1 &&
                w->size(0) == D && w->device() == like.device());
}

// norm(x, weight, eps, residual, fp8, group) -> (return code, y, scale, h, rstd), or NOT_TAKEN
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 6 || !f_norm) return not_taken();
  const at::Tensor *x = plain(a[0]), *w, *r;
  double eps;
  int64_t fp8, group;
  if (!x || !maybe(a[1], w) || !real(a[2], eps) || !maybe(a[3], r) || !integer(a[4], fp8) || !integer(a[5], group) ||
      x->dim() < 1 || x->numel() == 0)
    return not_taken();
  const int type = elem_type(*x);
  const int64_t D = x->size(-1), n = x->numel() / D;
  int wt, rt = type;
  if (type < 0 || group < 0 || !weight_ok(w, *x, D, wt)) return not_taken();
  if (r) {
    rt = elem_type(*r);
    if (r->sizes() != x->sizes() || r->device() != x->device() || (rt != type && rt != ELR_F32)) return not_taken();
  }
  try {
    at::Tensor y, scale, h, rstd;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x, st)) {
        std::vector<int64_t> lead(x->sizes().begin(), x->sizes().end() - 1);
        y = empty_on(*x, x->sizes(), fp8 ? at::kFloat8_e4m3fn : x->scalar_type());
        rstd = empty_on(*x, lead, at::kFloat);
        if (r) h = empty_on(*x, x->sizes(), r->scalar_type());
        if (fp8) {
          lead.push_back(group ? D / group : 1);
          scale = empty_on(*x, lead, at::kFloat);
        }
        rc = f_norm(x->data_ptr(), type, n, D, D, r ? r->data_ptr() : nullptr, rt, D, w ? w->data_ptr() : nullptr, wt,
                    static_cast<float>(eps), y.data_ptr(), fp8 != 0, group, static_cast<float*>(data_or_null(scale)),
                    data_or_null(h), static_cast<float*>(rstd.data_ptr()), st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    PyObject* ho = r ? THPVariable_Wrap(h) : (Py_INCREF(a[0]), a[0]);
    return Py_BuildValue("(iNNNN)", rc, THPVariable_Wrap(y), wrap_or_none(scale), ho, THPVariable_Wrap(rstd));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// norm_back(dy, h, weight, rstd, dh, need_dweight) -> (return code, dx, dweight), or NOT_TAKEN
PyObject* norm_back(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 6 || !f_norm_back) return not_taken();
  const at::Tensor *dy = plain(a[0]), *h = plain(a[1]), *w, *rstd = plain(a[3]), *dh;
  int64_t need;
  if (!dy || !h || !rstd || !maybe(a[2], w) || !maybe(a[4], dh) || !integer(a[5], need) || dy->dim() < 1 ||
      dy->numel() == 0)
    return not_taken();
  const int type = elem_type(*dy), ht = elem_type(*h);
  const int64_t D = dy->size(-1), n = dy->numel() / D;
  int wt;
  if (type < 0 || (ht != type && ht != ELR_F32) || h->sizes() != dy->sizes() || h->device() != dy->device() ||
      !weight_ok(w, *dy, D, wt) || rstd->scalar_type() != at::kFloat || rstd->device() != dy->device() ||
      rstd->sizes() != dy->sizes().slice(0, dy->dim() - 1))
    return not_taken();
  if (dh && (dh->sizes() != h->sizes() || dh->scalar_type() != h->scalar_type() || dh->device() != h->device()))
    return not_taken();
  try {
    at::Tensor dx, dw;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*dy, st)) {
        dx = empty_on(*dy, h->sizes(), h->scalar_type());
        at::Tensor scratch;
        int64_t bytes = 0;
        if (need) {
          dw = empty_on(*dy, {D}, at::kFloat);
          bytes = f_norm_bytes(n, D, type);
          scratch = scratch_on(*dy, bytes);
        }
        rc = f_norm_back(dy->data_ptr(), type, n, D, D, h->data_ptr(), ht, D, dh ? dh->data_ptr() : nullptr, D,
                         w ? w->data_ptr() : nullptr, wt, floats(rstd), dx.data_ptr(),
                         static_cast<float*>(data_or_null(dw)), data_or_null(scratch), bytes, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(dx), wrap_or_none(dw));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// A reference given back at the end of its block, with the GIL.
struct Held {
  PyObject* o;
  explicit Held(PyObject* p) : o(p) {}
  Held(const Held&) = delete;
  ~Held() { Py_XDECREF(o); }
};

// clip(grads, out or None, kind, max_norm or None, eps) -> (return code, norm), or NOT_TAKEN; max_norm None: the norm alone
PyObject* clip(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 5 || !f_clip) return not_taken();
  if (!(PyList_CheckExact(a[0]) || PyTuple_CheckExact(a[0])) ||
      !(a[1] == Py_None || PyList_CheckExact(a[1]) || PyTuple_CheckExact(a[1])))
    return not_taken();
  int64_t kind;
  double max_norm = 0, eps = 0;
  const bool scale = a[3] != Py_None;
  if (!integer(a[2], kind) || (scale && (!real(a[3], max_norm) || !real(a[4], eps)))) return not_taken();
  // Tuples of its own: another thread may change the caller's lists while this one launches without the GIL, and the tensors
  // have to outlive that.
  const bool outs = a[1] != Py_None;
  const Held ins(PySequence_Tuple(a[0])), to_outs(outs ? PySequence_Tuple(a[1]) : nullptr);
  if (!ins.o || (outs && !to_outs.o)) {
    PyErr_Clear();
    return not_taken();
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(ins.o);
  if (n == 0 || (outs && PyTuple_GET_SIZE(to_outs.o) != n)) return not_taken();
  try {
    std::vector<elr_grad> list(static_cast<size_t>(n));
    std::vector<Range> ranges;      // of what a call that scales reads and writes; in place: once
    if (scale) ranges.reserve(static_cast<size_t>(outs ? 2 * n : n));
    const at::Tensor* first = nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* to = PyTuple_GET_ITEM(ins.o, i);
      PyObject* oo = outs ? PyTuple_GET_ITEM(to_outs.o, i) : to;
      const at::Tensor *t = plain(to), *o = oo == to ? t : plain(oo);
      if (!t || !o) return not_taken();
      if (!first) first = t;
      const int type = elem_type(*t), ot = elem_type(*o);
      if (type < 0 || (ot != type && ot != ELR_F32) || t->device() != first->device() || o->device() != first->device() ||
          (o != t && o->sizes() != t->sizes()))
        return not_taken();
      const int64_t m = t->numel();
      list[static_cast<size_t>(i)] = elr_grad{t->data_ptr(), o->data_ptr(), 1, m, m, 1, m, 1, type, ot};
      if (!scale || m == 0) continue;
      ranges.push_back(range_of(*o, true));
      if (o->data_ptr() != t->data_ptr() || ot != type) ranges.push_back(range_of(*t, false));
    }
    if (meet(ranges)) return not_taken();
    at::Tensor norm;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*first, st)) {
        norm = empty_on(*first, {}, at::kFloat);
        const int64_t bytes = f_grad_bytes(list.data(), n);
        const at::Tensor scratch = scratch_on(*first, bytes);
        float* np = static_cast<float*>(norm.data_ptr());
        rc = scale ? f_clip(list.data(), n, static_cast<int>(kind), static_cast<float>(max_norm),
                            static_cast<float>(eps), np, data_or_null(scratch), bytes, st)
                   : f_grad_norm(list.data(), n, static_cast<int>(kind), np, data_or_null(scratch), bytes, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(norm));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// ---- int8, sampling

decltype(&elr_quantize_int8) f_quantize = nullptr;
decltype(&elr_dequantize_int8) f_dequantize = nullptr;
decltype(&elr_int8_linear) f_linear = nullptr;
decltype(&elr_int8_weight_grad_scratch_bytes) f_wgrad_bytes = nullptr;
decltype(&elr_int8_weight_grad) f_wgrad = nullptr;
decltype(&elr_rms_norm_backward_int8) f_norm_back8 = nullptr;
decltype(&elr_sample_tokens) f_sample = nullptr;

PyObject* bind_int8(PyObject*, PyObject* args) {
  unsigned long long a[7];
  if (!PyArg_ParseTuple(args, "KKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6)) return nullptr;
  set_address(f_quantize, a[0]), set_address(f_dequantize, a[1]), set_address(f_linear, a[2]);
  set_address(f_wgrad_bytes, a[3]), set_address(f_wgrad, a[4]);
  set_address(f_norm_back8, a[5]), set_address(f_sample, a[6]);
  Py_RETURN_NONE;
}

bool group_ok(int64_t g) { return g == 0 || g == 32 || g == 64 || g == 128 || g == 256; }
int64_t groups_of(int64_t D, int64_t g) { return g ? (D + g - 1) / g : 1; }

// The three parts of an Int8Rows (q, scale, group), with a scale for each of a row's groups.
struct Rows8 {
  const at::Tensor *q = nullptr, *scale = nullptr;
  int64_t group = 0, n = 0, D = 0;
  bool take(PyObject* qo, PyObject* so, PyObject* go) {
    if (!(q = plain(qo)) || !(scale = plain(so)) || !integer(go, group) || !group_ok(group) || q->scalar_type() != at::kChar ||
        q->dim() < 1 || q->numel() == 0 || scale->scalar_type() != at::kFloat || scale->device() != q->device() ||
        scale->dim() != q->dim())
      return false;
    const int64_t d = q->dim() - 1;
    D = q->size(d), n = q->numel() / D;
    return scale->size(d) == groups_of(D, group) && scale->sizes().slice(0, d) == q->sizes().slice(0, d);
  }
  const int8_t* data() const { return static_cast<const int8_t*>(q->data_ptr()); }
};

at::ScalarType scalar_type_of(int64_t elem) {
  return elem == ELR_F32 ? at::kFloat : elem == ELR_F16 ? at::kHalf : at::kBFloat16;
}

// quantize(x, group, pow2) -> (return code, q, scale), or NOT_TAKEN
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 3 || !f_quantize) return not_taken();
  const at::Tensor* x = plain(a[0]);
  int64_t group, pow2;
  if (!x || !integer(a[1], group) || !integer(a[2], pow2) || x->dim() < 1 || x->numel() == 0 || !group_ok(group))
    return not_taken();
  const int type = elem_type(*x);
  const int64_t D = x->size(-1), n = x->numel() / D;
  if (type < 0) return not_taken();
  try {
    at::Tensor q, scale;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x, st)) {
        std::vector<int64_t> shape(x->sizes().begin(), x->sizes().end());
        q = empty_on(*x, shape, at::kChar);
        shape.back() = groups_of(D, group);
        scale = empty_on(*x, shape, at::kFloat);
        rc = f_quantize(x->data_ptr(), type, n, D, D, group, pow2 != 0, static_cast<int8_t*>(q.data_ptr()),
                        static_cast<float*>(scale.data_ptr()), st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(q), THPVariable_Wrap(scale));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// dequantize(q, scale, group, type) -> (return code, x), or NOT_TAKEN
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 4 || !f_dequantize) return not_taken();
  Rows8 r;
  int64_t type;
  if (!r.take(a[0], a[1], a[2]) || !integer(a[3], type) || type < 0) return not_taken();
  try {
    at::Tensor x;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*r.q, st)) {
        x = empty_on(*r.q, r.q->sizes(), scalar_type_of(type));
        rc = f_dequantize(r.data(), r.n, r.D, r.D, r.group, floats(r.scale), x.data_ptr(), static_cast<int>(type), st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(x));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// linear(x.q, x.scale, x.group, w.q, w.scale, w.group, type) -> (return code, y), or NOT_TAKEN
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 7 || !f_linear) return not_taken();
  Rows8 x, w;
  int64_t type;
  if (!x.take(a[0], a[1], a[2]) || !w.take(a[3], a[4], a[5]) || !integer(a[6], type) || type < 0 || x.group || w.group ||
      w.q->dim() != 2 || w.D != x.D || w.q->device() != x.q->device() || x.D >= int64_t(1) << 17)
    return not_taken();
  try {
    at::Tensor y;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x.q, st)) {
        std::vector<int64_t> shape(x.q->sizes().begin(), x.q->sizes().end());
        shape.back() = w.n;
        y = empty_on(*x.q, shape, scalar_type_of(type));
        rc = f_linear(x.data(), x.n, x.D, x.D, floats(x.scale), w.data(), w.n, w.D, floats(w.scale), y.data_ptr(),
                      static_cast<int>(type), st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(y));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// weight_grad(dy, x.q, x.scale, x.group, transposed) -> (return code, dw), or NOT_TAKEN
PyObject* weight_grad(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 5 || !f_wgrad) return not_taken();
  const at::Tensor* dy = plain(a[0]);
  Rows8 x;
  int64_t transposed;
  if (!dy || !x.take(a[1], a[2], a[3]) || !integer(a[4], transposed) || dy->dim() != x.q->dim() || dy->numel() == 0 ||
      dy->device() != x.q->device())
    return not_taken();
  const int64_t d = dy->dim() - 1, N = dy->size(d);
  const int type = elem_type(*dy);
  if (type < 0 || dy->sizes().slice(0, d) != x.q->sizes().slice(0, d)) return not_taken();
  try {
    at::Tensor dw;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*dy, st)) {
        dw = empty_on(*dy, transposed ? at::IntArrayRef{x.D, N} : at::IntArrayRef{N, x.D}, at::kFloat);
        const int64_t bytes = f_wgrad_bytes(x.n, N, x.D, type);
        const at::Tensor scratch = scratch_on(*dy, bytes);
        rc = f_wgrad(dy->data_ptr(), type, x.n, N, N, x.data(), x.D, x.D, x.group, floats(x.scale),
                     static_cast<float*>(dw.data_ptr()), transposed != 0, data_or_null(scratch), bytes, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iN)", rc, THPVariable_Wrap(dw));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// norm_back_int8(dy, h.q, h.scale, h.group, weight, rstd, dh, need_dweight) -> (return code, dx, dweight), or NOT_TAKEN
PyObject* norm_back_int8(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 8 || !f_norm_back8) return not_taken();
  const at::Tensor *dy = plain(a[0]), *w, *rstd = plain(a[5]), *dh;
  Rows8 h;
  int64_t need;
  if (!dy || !h.take(a[1], a[2], a[3]) || !maybe(a[4], w) || !rstd || !maybe(a[6], dh) || !integer(a[7], need) ||
      dy->sizes() != h.q->sizes() || dy->device() != h.q->device())
    return not_taken();
  const int type = elem_type(*dy);
  int wt, xt = type;
  if (type < 0 || !weight_ok(w, *dy, h.D, wt) || rstd->scalar_type() != at::kFloat || rstd->device() != dy->device() ||
      rstd->sizes() != dy->sizes().slice(0, dy->dim() - 1))
    return not_taken();
  if (dh) {
    xt = elem_type(*dh);
    if (dh->sizes() != dy->sizes() || dh->device() != dy->device() || (xt != type && xt != ELR_F32)) return not_taken();
  }
  try {
    at::Tensor dx, dw;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*dy, st)) {
        dx = empty_on(*dy, dy->sizes(), scalar_type_of(xt));
        at::Tensor scratch;
        int64_t bytes = 0;
        if (need) {
          dw = empty_on(*dy, {h.D}, at::kFloat);
          bytes = f_norm_bytes(h.n, h.D, type);
          scratch = scratch_on(*dy, bytes);
        }
        rc = f_norm_back8(dy->data_ptr(), type, h.n, h.D, h.D, h.data(), h.D, h.group, floats(h.scale),
                          dh ? dh->data_ptr() : nullptr, xt, h.D, w ? w->data_ptr() : nullptr, wt, floats(rstd), dx.data_ptr(),
                          static_cast<float*>(data_or_null(dw)), data_or_null(scratch), bytes, st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(dx), wrap_or_none(dw));
  } catch (const std::exception&) {
    return not_taken();
  }
}

// A setting: a number in [low, high], or a plain fp32 tensor of u's shape and device.
bool setting(PyObject* o, const at::Tensor& u, double low, double high, double& v, const at::Tensor*& rows) {
  v = 0, rows = nullptr;
  if (PyFloat_CheckExact(o) || PyLong_CheckExact(o)) return real(o, v) && v >= low && v <= high;
  rows = plain(o);
  return rows && rows->scalar_type() == at::kFloat && rows->device() == u.device() && rows->sizes() == u.sizes();
}

// sample(logits, u, temperature, top_k, top_p, min_p) -> (return code, token, logprob), or NOT_TAKEN
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t na) {
  if (na != 6 || !f_sample) return not_taken();
  const at::Tensor *x = plain(a[0]), *u = plain(a[1]), *temps, *ks = nullptr, *ps, *mps;
  if (!x || !u || x->dim() < 1 || x->numel() == 0 || u->scalar_type() != at::kFloat || u->device() != x->device() ||
      u->sizes() != x->sizes().slice(0, x->dim() - 1))
    return not_taken();
  double temp, p, mp;
  int64_t k = 0;
  const int type = elem_type(*x);
  if (type < 0 || !setting(a[2], *u, 0, 1.7e308, temp, temps) || !setting(a[4], *u, 0, 1, p, ps) ||
      !setting(a[5], *u, 0, 1, mp, mps))
    return not_taken();
  if (PyLong_CheckExact(a[3])) {
    if (!integer(a[3], k) || k < 0) return not_taken();
  } else if (!(ks = plain(a[3])) || (ks->scalar_type() != at::kInt && ks->scalar_type() != at::kLong) ||
             ks->device() != x->device() || ks->sizes() != u->sizes()) {
    return not_taken();
  }
  try {
    at::Tensor token, logprob;
    int rc = kNotTaken;
    {
      NoGil g;
      void* st;
      if (stream_on(*x, st)) {
        token = empty_on(*x, u->sizes(), at::kLong), logprob = empty_on(*x, u->sizes(), at::kFloat);
        const int64_t V = x->size(-1);
        rc = f_sample(x->data_ptr(), type, x->numel() / V, V, V, floats(u), temp, floats(temps), k, ks ? ks->data_ptr() : nullptr,
                      ks && ks->scalar_type() == at::kLong, p, floats(ps), mp, floats(mps),
                      static_cast<int64_t*>(token.data_ptr()), static_cast<float*>(logprob.data_ptr()), st);
      }
    }
    if (rc == kNotTaken) return not_taken();
    return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(token), THPVariable_Wrap(logprob));
  } catch (const std::exception&) {
    return not_taken();
  }
}

#define ELR_STR1(x) #x
#define ELR_STR(x) ELR_STR1(x)
#define ELR_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "Addresses of the library's entry points."},
                         {"adam", ELR_FAST(adam), METH_FASTCALL, "elr_adam_rows with gpu_adam's checks."},
                         {"init", ELR_FAST(init), METH_FASTCALL, "elr_init_rows into a new tensor."},
                         {"replay", ELR_FAST(replay), METH_FASTCALL, "elr_replay_rows into a new tensor."},
                         {"bind_ops", bind_ops, METH_VARARGS, "Addresses of the operators' entry points."},
                         {"logprobs", ELR_FAST(logprobs), METH_FASTCALL, "elr_token_logprobs into new tensors."},
                         {"logprobs_back", ELR_FAST(logprobs_back), METH_FASTCALL, "elr_token_logprobs_backward."},
                         {"norm", ELR_FAST(norm), METH_FASTCALL, "elr_rms_norm into new tensors."},
                         {"norm_back", ELR_FAST(norm_back), METH_FASTCALL, "elr_rms_norm_backward into new tensors."},
                         {"clip", ELR_FAST(clip), METH_FASTCALL, "elr_clip_grad_norm or elr_grad_norm."},
                         {"bind_int8", bind_int8, METH_VARARGS, "Addresses of the entry points of int8 and sampling."},
                         {"quantize", ELR_FAST(quantize), METH_FASTCALL, "elr_quantize_int8 into new tensors."},
                         {"dequantize", ELR_FAST(dequantize), METH_FASTCALL, "elr_dequantize_int8 into a new tensor."},
                         {"linear", ELR_FAST(linear), METH_FASTCALL, "elr_int8_linear into a new tensor."},
                         {"weight_grad", ELR_FAST(weight_grad), METH_FASTCALL, "elr_int8_weight_grad into a new tensor."},
                         {"norm_back_int8", ELR_FAST(norm_back_int8), METH_FASTCALL, "elr_rms_norm_backward_int8."},
                         {"sample", ELR_FAST(sample), METH_FASTCALL, "elr_sample_tokens into new tensors."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// The file's name carries neither version, and another Python's or torch's objects are laid out differently: the former is
// refused here, the latter by the caller (elara_amd/_lib.py: host), both before any tensor is touched.
PyMODINIT_FUNC PyInit__hostcall() {
  constexpr const char built[] = ELR_STR(PY_MAJOR_VERSION) "." ELR_STR(PY_MINOR_VERSION) ".";
  if (std::strncmp(Py_GetVersion(), built, sizeof built - 1) != 0) {
    PyErr_Format(PyExc_ImportError, "_hostcall was built for Python %sx", built);
    return nullptr;
  }
  PyObject* m = PyModule_Create(&module);
  if (m) {
    PyModule_AddIntConstant(m, "NOT_TAKEN", kNotTaken);
    PyModule_AddStringConstant(m, "TORCH", ELR_TORCH_VERSION);
  }
  return m;
}
