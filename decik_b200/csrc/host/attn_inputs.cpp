// The attention-input operators of decik_b200/ops.py (counter-based dropout, LoRA down projections under
// it, head norms with rotation, rotation by several axes) as functions of torch tensors: the checks
// of their arguments, their outputs and workspaces, and the call of the C ABI, on the tensors' device
// and its current stream. They are called once a layer and token in serving, where the host's time is
// the time: checking, allocating and calling through ctypes from Python took 10 to 30 us a call beside
// kernels of 2 to 3 us.
//
// A CPython extension module; each function takes its arguments by position (ops.py has the names, the
// defaults and the documentation) and raises RuntimeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>

#include "decik_b200.h"

namespace {

using at::Tensor;

[[noreturn]] void fail(const char* what, const std::string& why) {
  throw std::runtime_error(std::string("decik_b200 ") + what + ": " + why);
}

void check(int rc, const char* what) {
  if (rc != DECIK_OK)
    throw std::runtime_error(std::string("decik_b200 ") + what + " failed (status " + std::to_string(rc) +
                             "): " + decik_last_error());
}

// ---- arguments ----
struct Args {
  const char* what;
  PyObject* const* v;
  Args(const char* w, PyObject* const* args, Py_ssize_t got, Py_ssize_t want) : what(w), v(args) {
    if (got != want) fail(what, std::to_string(got) + " arguments instead of " + std::to_string(want));
  }
  const Tensor& tensor(int i) const {
    if (!THPVariable_Check(v[i])) fail(what, "argument " + std::to_string(i) + " is not a tensor");
    return THPVariable_Unpack(v[i]);
  }
  const Tensor* maybe(int i) const { return v[i] == Py_None ? nullptr : &tensor(i); }
  double number(int i) const {
    const double d = PyFloat_AsDouble(v[i]);
    if (d == -1.0 && PyErr_Occurred()) throw python_error();
    return d;
  }
  int64_t integer(int i) const {
    const long long n = PyLong_AsLongLong(v[i]);
    if (n == -1 && PyErr_Occurred()) throw python_error();
    return n;
  }
};

int code(const char* what, at::ScalarType t) {
  if (t == at::kHalf) return DECIK_F16;
  if (t == at::kBFloat16) return DECIK_BF16;
  if (t == at::kFloat) return DECIK_F32;
  fail(what, std::string("unsupported dtype ") + c10::toString(t));
}

// The one CUDA device of all tensors, made current, and its stream.
struct Place {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  Place(const char* what, std::initializer_list<const Tensor*> ts) {
    const Tensor* first = nullptr;
    for (const Tensor* t : ts) {
      if (t == nullptr) continue;
      if (first == nullptr) first = t;
      if (!t->is_cuda() || t->device() != first->device())
        fail(what, "tensors must be on one CUDA device (no CPU fallback)");
    }
    guard.set_device(first->device());
    stream = c10::cuda::getCurrentCUDAStream(first->device().index()).stream();
  }
};

Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType t) { return at::empty(size, like.options().dtype(t)); }
Tensor empty(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options()); }
void* ptr(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// the row stride of a 2-D tensor; of a single row its width
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

PyObject* wrap(std::initializer_list<Tensor> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (out == nullptr) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

// ---- queries and keys ----
struct View {
  int64_t tok, heads, dim;
  decik_tensor3 v;
};
// a [T, H, D] view (with swap [H, T, D]); the stride of a dimension of one element does not matter
View view(const char* what, const Tensor& t, bool swap = false) {
  if (t.dim() != 3) fail(what, "expected a 3-D tensor");
  if (t.stride(2) != 1 && t.size(2) > 1) fail(what, "[T, H, D] views need contiguous D");
  const int a = swap ? 1 : 0, b = 1 - a;
  return {t.size(a), t.size(b), t.size(2),
          {t.data_ptr(), t.size(a) > 1 ? t.stride(a) : 0, t.size(b) > 1 ? t.stride(b) : 0}};
}
decik_tensor3_mut out_view(const Tensor& t, int64_t tok_stride, int64_t head_stride) {
  return {t.data_ptr(), tok_stride, head_stride};
}

struct Heads {
  View q, k;
  decik_tensor3 lora;
  int64_t T;
  int Hq, Hk, D;
};
Heads heads(const char* what, const Tensor& q, const Tensor& k, const Tensor* lora, const Tensor* wq,
            const Tensor* wk) {
  if (q.dim() != 3 || k.dim() != 3 || q.size(0) != k.size(0) || q.size(2) != k.size(2) ||
      q.scalar_type() != k.scalar_type())
    fail(what, "q [T, Hq, D] and k [T, Hk, D] of one dtype");
  Heads h{view(what, q), view(what, k), {nullptr, 0, 0}, q.size(0), static_cast<int>(q.size(1)),
          static_cast<int>(k.size(1)), static_cast<int>(q.size(2))};
  if (lora != nullptr) {
    if (lora->sizes() != q.sizes() || lora->scalar_type() != q.scalar_type()) fail(what, "q_lora must be like q");
    h.lora = view(what, *lora).v;
  }
  if ((wq == nullptr) != (wk == nullptr)) fail(what, "norm weights for both queries and keys, or for neither");
  if (wq != nullptr && !(wq->dim() == 1 && wk->dim() == 1 && wq->size(0) == h.D && wk->size(0) == h.D &&
                         wq->scalar_type() == wk->scalar_type() && wq->is_contiguous() && wk->is_contiguous()))
    fail(what, "norm weights must be contiguous [head_dim] of one dtype");
  return h;
}

int tables(const char* what, const Tensor& cos, const Tensor& sin, int64_t T) {
  if (!(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(0) == T && cos.scalar_type() == at::kFloat &&
        sin.scalar_type() == at::kFloat && cos.is_contiguous() && sin.is_contiguous()))
    fail(what, "cos and sin must be contiguous fp32 [T, rotary_dim]");
  return static_cast<int>(cos.size(1));
}

struct Axes {
  Tensor positions, inv_freq;  // as they are passed
  int pos_dtype, n_axes, R;
  int64_t ld_pos;
  const uint8_t* axis_of;
  const float* inv_freq_ptr() const { return static_cast<const float*>(inv_freq.data_ptr()); }
};
// axis_of: bytes, the axis of each frequency; n_axes sections
Axes axes(const Args& a, int i_pos, int i_inv, int i_map, int i_axes, int64_t T) {
  char* map = nullptr;
  Py_ssize_t n = 0;
  if (PyBytes_AsStringAndSize(a.v[i_map], &map, &n) != 0) throw python_error();
  Axes x;
  x.n_axes = static_cast<int>(a.integer(i_axes));
  x.positions = a.tensor(i_pos);
  if (x.positions.dim() == 1) x.positions = x.positions.unsqueeze(0);
  const at::ScalarType t = x.positions.scalar_type();
  if ((t != at::kLong && t != at::kInt) || x.positions.dim() != 2 || x.positions.size(0) != x.n_axes ||
      x.positions.size(1) != T)
    fail(a.what, "positions must be int64 or int32 [axes, T], an axis for each section");
  if ((x.positions.stride(1) != 1 && T > 1) || (x.n_axes > 1 && x.positions.stride(0) < T))
    x.positions = x.positions.contiguous();
  x.pos_dtype = t == at::kInt ? 1 : 0;
  x.ld_pos = ld(x.positions);
  const Tensor& inv = a.tensor(i_inv);
  if (inv.scalar_type() != at::kFloat || inv.dim() != 1 || inv.size(0) != n || !inv.is_contiguous())
    fail(a.what, "inv_freq must be contiguous fp32 [sum(sections)]");
  // a slice of a longer table may start anywhere; the kernels read 16-byte pieces
  x.inv_freq = reinterpret_cast<uintptr_t>(inv.data_ptr()) % 16 == 0 ? inv : inv.clone();
  x.axis_of = reinterpret_cast<const uint8_t*>(map);
  x.R = static_cast<int>(2 * n);
  return x;
}

struct Grads {
  View q, k;
};
Grads grads(const char* what, const Tensor& gq, const Tensor& gk, int64_t Hq, int64_t Hk, int64_t T, int64_t D,
            at::ScalarType t) {
  if (gq.dim() != 3 || gk.dim() != 3) fail(what, "grad_q [Hq, T, D] and grad_k [Hk, T, D]");
  Grads g{view(what, gq, true), view(what, gk, true)};
  if (g.q.heads != Hq || g.k.heads != Hk || g.q.tok != T || g.k.tok != T || g.q.dim != D || g.k.dim != D ||
      gq.scalar_type() != t || gk.scalar_type() != t)
    fail(what, "grad_q [Hq, T, D] and grad_k [Hk, T, D] of the inputs' dtype");
  return g;
}

struct HeadOuts {
  Tensor dq, dk, dwq, dwk, ws;
};
HeadOuts head_outs(const Tensor& like, int64_t T, int64_t Hq, int64_t Hk, int64_t D, bool norm) {
  HeadOuts o{empty({T, Hq, D}, like), empty({T, Hk, D}, like), {}, {}, {}};
  if (norm) {
    o.dwq = empty({D}, like, at::kFloat);
    o.dwk = empty({D}, like, at::kFloat);
    o.ws = empty({decik_qk_norm_rope_bwd_workspace(static_cast<int>(D))}, like, at::kByte);
  }
  return o;
}

// q, k, q_weight, k_weight, eps, cos, sin, q_lora
PyObject* qk_norm_rope_fwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("qk_norm_rope_fwd", v, n, 8);
  const Tensor &q = a.tensor(0), &k = a.tensor(1), &wq = a.tensor(2), &wk = a.tensor(3), &cos = a.tensor(5),
               &sin = a.tensor(6);
  const Tensor* lora = a.maybe(7);
  const Place at(a.what, {&q, &k, &wq, &wk, &cos, &sin, lora});
  const Heads h = heads(a.what, q, k, lora, &wq, &wk);
  const int R = tables(a.what, cos, sin, h.T);
  const Tensor oq = empty({h.Hq, h.T, h.D}, q), ok = empty({h.Hk, h.T, h.D}, q);
  check(decik_qk_norm_rope_fwd(h.q.v, h.lora, h.k.v, wq.data_ptr(), wk.data_ptr(), code(a.what, wq.scalar_type()),
                               static_cast<float>(a.number(4)), static_cast<const float*>(cos.data_ptr()),
                               static_cast<const float*>(sin.data_ptr()), out_view(oq, h.D, h.T * h.D),
                               out_view(ok, h.D, h.T * h.D), h.T, h.Hq, h.Hk, h.D, R, code(a.what, q.scalar_type()),
                               at.stream),
        a.what);
  return wrap({oq, ok});
  END_HANDLE_TH_ERRORS
}

// grad_q, grad_k, q, k, q_weight, k_weight, eps, cos, sin, q_lora
PyObject* qk_norm_rope_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("qk_norm_rope_bwd", v, n, 10);
  const Tensor &gq = a.tensor(0), &gk = a.tensor(1), &q = a.tensor(2), &k = a.tensor(3), &wq = a.tensor(4),
               &wk = a.tensor(5), &cos = a.tensor(7), &sin = a.tensor(8);
  const Tensor* lora = a.maybe(9);
  const Place at(a.what, {&gq, &gk, &q, &k, &wq, &wk, &cos, &sin, lora});
  const Heads h = heads(a.what, q, k, lora, &wq, &wk);
  const int R = tables(a.what, cos, sin, h.T);
  const Grads g = grads(a.what, gq, gk, h.Hq, h.Hk, h.T, h.D, q.scalar_type());
  const HeadOuts o = head_outs(q, h.T, h.Hq, h.Hk, h.D, true);
  check(decik_qk_norm_rope_bwd(g.q.v, g.k.v, h.q.v, h.lora, h.k.v, wq.data_ptr(), wk.data_ptr(),
                               code(a.what, wq.scalar_type()), static_cast<float>(a.number(6)),
                               static_cast<const float*>(cos.data_ptr()), static_cast<const float*>(sin.data_ptr()),
                               out_view(o.dq, int64_t(h.Hq) * h.D, h.D), out_view(o.dk, int64_t(h.Hk) * h.D, h.D),
                               static_cast<float*>(o.dwq.data_ptr()), static_cast<float*>(o.dwk.data_ptr()), h.T, h.Hq,
                               h.Hk, h.D, R, code(a.what, q.scalar_type()), o.ws.data_ptr(), at.stream),
        a.what);
  return wrap({o.dq, o.dk, o.dwq, o.dwk});
  END_HANDLE_TH_ERRORS
}

// q, k, positions, inv_freq, axis_of, n_axes, q_weight, k_weight, eps, q_lora
PyObject* rope_axes_fwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("rope_axes_fwd", v, n, 10);
  const Tensor &q = a.tensor(0), &k = a.tensor(1), &pos = a.tensor(2), &inv = a.tensor(3);
  const Tensor *wq = a.maybe(6), *wk = a.maybe(7), *lora = a.maybe(9);
  const Place at(a.what, {&q, &k, &pos, &inv, wq, wk, lora});
  const Heads h = heads(a.what, q, k, lora, wq, wk);
  const Axes x = axes(a, 2, 3, 4, 5, h.T);
  const Tensor oq = empty({h.Hq, h.T, h.D}, q), ok = empty({h.Hk, h.T, h.D}, q);
  check(decik_rope_axes_fwd(h.q.v, h.lora, h.k.v, ptr(wq), ptr(wk),
                            wq == nullptr ? DECIK_F32 : code(a.what, wq->scalar_type()),
                            static_cast<float>(a.number(8)), x.positions.data_ptr(), x.pos_dtype, x.ld_pos, x.n_axes,
                            x.inv_freq_ptr(), x.axis_of, out_view(oq, h.D, h.T * h.D), out_view(ok, h.D, h.T * h.D),
                            h.T, h.Hq, h.Hk, h.D, x.R, code(a.what, q.scalar_type()), at.stream),
        a.what);
  return wrap({oq, ok});
  END_HANDLE_TH_ERRORS
}

// grad_q, grad_k, positions, inv_freq, axis_of, n_axes, q, k, q_weight, k_weight, eps, q_lora
PyObject* rope_axes_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("rope_axes_bwd", v, n, 12);
  const Tensor &gq = a.tensor(0), &gk = a.tensor(1), &pos = a.tensor(2), &inv = a.tensor(3);
  const Tensor *q = a.maybe(6), *k = a.maybe(7), *wq = a.maybe(8), *wk = a.maybe(9), *lora = a.maybe(11);
  const Place at(a.what, {&gq, &gk, &pos, &inv, q, k, wq, wk, lora});
  const bool norm = wq != nullptr || wk != nullptr;
  Heads h{};
  if (norm) {
    if (q == nullptr || k == nullptr) fail(a.what, "the backward of the norms needs the forward's q and k");
    h = heads(a.what, *q, *k, lora, wq, wk);
  } else {
    if (gq.dim() != 3 || gk.dim() != 3) fail(a.what, "grad_q [Hq, T, D] and grad_k [Hk, T, D]");
    h.T = gq.size(1), h.D = static_cast<int>(gq.size(2));
    h.Hq = static_cast<int>(gq.size(0)), h.Hk = static_cast<int>(gk.size(0));
  }
  const Axes x = axes(a, 2, 3, 4, 5, h.T);
  const Grads g = grads(a.what, gq, gk, h.Hq, h.Hk, h.T, h.D, norm ? q->scalar_type() : gq.scalar_type());
  const HeadOuts o = head_outs(gq, h.T, h.Hq, h.Hk, h.D, norm);
  check(decik_rope_axes_bwd(g.q.v, g.k.v, h.q.v, h.lora, h.k.v, ptr(wq), ptr(wk),
                            norm ? code(a.what, wq->scalar_type()) : DECIK_F32, static_cast<float>(a.number(10)),
                            x.positions.data_ptr(), x.pos_dtype, x.ld_pos, x.n_axes, x.inv_freq_ptr(), x.axis_of,
                            out_view(o.dq, int64_t(h.Hq) * h.D, h.D), out_view(o.dk, int64_t(h.Hk) * h.D, h.D),
                            norm ? static_cast<float*>(o.dwq.data_ptr()) : nullptr,
                            norm ? static_cast<float*>(o.dwk.data_ptr()) : nullptr, h.T, h.Hq, h.Hk, h.D, x.R,
                            code(a.what, gq.scalar_type()), norm ? o.ws.data_ptr() : nullptr, at.stream),
        a.what);
  if (norm) return wrap({o.dq, o.dk, o.dwq, o.dwk});
  return wrap({o.dq, o.dk});
  END_HANDLE_TH_ERRORS
}

// ---- dropout ----
const int64_t* state(const char* what, const Tensor& rng) {
  if (rng.scalar_type() != at::kLong || rng.dim() != 1 || rng.size(0) != 2 || !rng.is_contiguous())
    fail(what, "rng must be int64 [2] (seed, offset)");
  return static_cast<const int64_t*>(rng.data_ptr());
}

// x, p, rng, stream, residual, like: the result's dtype where there is no residual, as a tensor of it, or None
PyObject* dropout(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("dropout", v, n, 6);
  const Tensor &x = a.tensor(0), &rng = a.tensor(2);
  const Tensor* residual = a.maybe(4);
  const Place at(a.what, {&x, &rng, residual});
  const int64_t* st = state(a.what, rng);
  at::ScalarType t = x.scalar_type();
  if (v[5] != Py_None) {
    if (!THPDtype_Check(v[5])) fail(a.what, "out_dtype is not a dtype");
    t = reinterpret_cast<THPDtype*>(v[5])->scalar_type;
  }
  if (residual != nullptr) {
    if (residual->sizes() != x.sizes() || (v[5] != Py_None && t != residual->scalar_type()))
      fail(a.what, "residual must be like x, and gives the result its dtype");
    t = residual->scalar_type();
  }
  const Tensor xc = x.contiguous(), rc = residual == nullptr ? Tensor() : residual->contiguous();
  const Tensor out = empty(x.sizes(), x, t);
  check(decik_dropout(xc.data_ptr(), code(a.what, x.scalar_type()), residual == nullptr ? nullptr : rc.data_ptr(),
                      out.data_ptr(), code(a.what, t), x.numel(), a.number(1), st, a.integer(3), at.stream),
        a.what);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// rank of a [n_branch * rank, width]
int rank_of(const char* what, const Tensor& a, int64_t n_branch, int64_t width) {
  if (a.dim() != 2 || a.size(1) != width || (a.stride(1) != 1 && width > 1) || n_branch < 1 || n_branch > 2 ||
      a.size(0) % n_branch != 0)
    fail(what, "a must be [branches * rank, width] with a p for each of 1 or 2 branches");
  return static_cast<int>(a.size(0) / n_branch);
}

// x, a, n_branch, p0, p1, rng, stream, u_cols (0: the branches' alone)
PyObject* lora_down_dropout(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("lora_down_dropout", v, n, 8);
  const Tensor &x = a.tensor(0), &w = a.tensor(1), &rng = a.tensor(5);
  const Place at(a.what, {&x, &w, &rng});
  const int64_t* st = state(a.what, rng);
  if (x.dim() != 2 || (x.scalar_type() != at::kFloat && x.scalar_type() != w.scalar_type()))
    fail(a.what, "x must be [T, width], fp32 or of a's dtype");
  const Tensor xc = x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
  const int64_t T = x.size(0), W = x.size(1), nb = a.integer(2);
  const int rank = rank_of(a.what, w, nb, W);
  const int64_t u_cols = a.integer(7) ? a.integer(7) : nb * rank;
  if (u_cols < nb * rank || u_cols > 65536) fail(a.what, "u_cols smaller than the branches' columns");
  const bool cast = x.scalar_type() != w.scalar_type();
  const Tensor x16 = cast ? empty({T, W}, w) : xc, u = empty({T, u_cols}, w);
  check(decik_lora_down_dropout(xc.data_ptr(), code(a.what, x.scalar_type()), ld(xc), w.data_ptr(), ld(w),
                                cast ? x16.data_ptr() : nullptr, W, u.data_ptr(), u_cols, static_cast<int>(u_cols), T,
                                static_cast<int>(W), rank, static_cast<int>(nb), a.number(3), a.number(4), st,
                                a.integer(6), code(a.what, w.scalar_type()), at.stream),
        a.what);
  return wrap({x16, u});
  END_HANDLE_TH_ERRORS
}

// du, x16, a, n_branch, p0, p1, rng, stream, addend, out
PyObject* lora_down_dropout_bwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a("lora_down_dropout_bwd", v, n, 10);
  const Tensor &du = a.tensor(0), &x16 = a.tensor(1), &w = a.tensor(2), &rng = a.tensor(6);
  const Tensor *addend = a.maybe(8), *out = a.maybe(9);
  const Place at(a.what, {&du, &x16, &w, &rng, addend, out});
  const int64_t* st = state(a.what, rng);
  if (x16.dim() != 2 || (x16.stride(1) != 1 && x16.size(1) > 1) || x16.scalar_type() != w.scalar_type())
    fail(a.what, "x16 must be [T, width] of a's dtype with contiguous rows");
  const int64_t T = x16.size(0), W = x16.size(1), nb = a.integer(3);
  const int rank = rank_of(a.what, w, nb, W);
  if (du.dim() != 2 || du.size(0) != T || du.size(1) != nb * rank || du.scalar_type() != w.scalar_type() ||
      (du.stride(1) != 1 && du.size(1) > 1))
    fail(a.what, "du must be [T, branches * rank] of a's dtype with contiguous rows");
  for (const Tensor* t : {addend, out})
    if (t != nullptr && (t->sizes() != x16.sizes() || t->scalar_type() != at::kFloat || (t->stride(1) != 1 && W > 1)))
      fail(a.what, "addend and out must be fp32 [T, width] with contiguous rows");
  const Tensor dx = out != nullptr ? *out : empty({T, W}, x16, at::kFloat), da = empty({nb * rank, W}, x16, at::kFloat);
  const Tensor ws = empty({decik_lora_down_dropout_bwd_workspace(T, static_cast<int>(W), rank, static_cast<int>(nb))},
                          x16, at::kByte);
  check(decik_lora_down_dropout_bwd(du.data_ptr(), ld(du), x16.data_ptr(), ld(x16), w.data_ptr(), ld(w),
                                    static_cast<const float*>(ptr(addend)), addend == nullptr ? 0 : ld(*addend),
                                    static_cast<float*>(dx.data_ptr()), ld(dx), static_cast<float*>(da.data_ptr()), T,
                                    static_cast<int>(W), rank, static_cast<int>(nb), a.number(4), a.number(5), st,
                                    a.integer(7), code(a.what, w.scalar_type()), ws.data_ptr(), at.stream),
        a.what);
  return wrap({dx, da});
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
#define DECIK_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
    DECIK_METHOD(qk_norm_rope_fwd),  DECIK_METHOD(qk_norm_rope_bwd), DECIK_METHOD(rope_axes_fwd),
    DECIK_METHOD(rope_axes_bwd),     DECIK_METHOD(dropout),          DECIK_METHOD(lora_down_dropout),
    DECIK_METHOD(lora_down_dropout_bwd), {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_attn_inputs", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attn_inputs(void) {
  PyObject* m = PyModule_Create(&kModule);
  // the torch it was built against: another one's tensors are not these
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", DECIK_TORCH_VERSION) != 0) return nullptr;
  return m;
}
