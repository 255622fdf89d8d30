// fast.cpp — a short way from Python to the C ABI for the training operators.
//
// ops.py checks and lays out its arguments in Python and converts them with
// ctypes: 37 us a call with one launch, 41 to 60 us with two. The functions here
// do the same for calls that need nothing done: every tensor on one GPU, of the
// right shape and type, laid out as the kernels read it. They allocate the
// outputs and call the library's entry point: 5 and 10 us. Anything else (a
// tensor to copy, an argument to refuse, a device without its status word) gives
// None, and ops.py goes the long way, which copies, refuses with a message, or
// launches.
//
// The entry points' addresses come from ops.py (bind), so that there is one
// loaded library, whichever was loaded.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/sinkattn.h"

namespace {

struct Library {
  decltype(&sa_bsattn_bwd) bsattn_bwd = nullptr;
  decltype(&sa_bsattn_bwd_workspace_size) bsattn_bwd_ws = nullptr;
  decltype(&sa_qk_norm_rope_bwd) norm_bwd = nullptr;
  decltype(&sa_qk_norm_rope_bwd_workspace_size) norm_bwd_ws = nullptr;
  decltype(&sa_qk_head_norm_rope) head = nullptr;
  decltype(&sa_qk_head_norm_rope_bwd) head_bwd = nullptr;
  decltype(&sa_qk_head_norm_rope_bwd_workspace_size) head_bwd_ws = nullptr;
} lib;
constexpr int kDevices = 64;
int32_t* g_status[kDevices] = {};

// An argument that is a tensor, or None.
struct Arg {
  const at::Tensor* t = nullptr;
  bool ok = true;  // a tensor or None
  explicit Arg(PyObject* o) {
    if (o == Py_None) return;
    if (THPVariable_Check(o)) t = &THPVariable_Unpack(o);
    else ok = false;
  }
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  const at::Tensor& operator*() const { return *t; }
  void* ptr() const { return t == nullptr ? nullptr : t->data_ptr(); }
};

bool on(const Arg& a, int dev) { return a.ok && (!a || (a->is_cuda() && a->get_device() == dev)); }

// Whole 16-byte vectors along every dimension that is stepped along.
bool vectors(const at::Tensor& t) {
  const int64_t n = 16 / t.element_size();
  if (t.dim() == 0 || t.stride(-1) != 1 || (uintptr_t)t.data_ptr() % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % n != 0) return false;
  return true;
}

// An output may not be expanded, a workspace is one run of bytes.
bool output(const Arg& a) {
  if (!a) return true;
  for (int64_t i = 0; i < a->dim(); ++i)
    if (a->size(i) > 1 && a->stride(i) == 0) return false;
  return true;
}

// ops.py refuses an output that begins where a tensor does that is still read.
bool apart(const Arg& out, std::initializer_list<const Arg*> others) {
  for (const Arg* o : others)
    if (out && *o && out.ptr() == o->ptr()) return false;
  return true;
}

bool workspace(const Arg& a) { return !a || a->is_contiguous(); }

struct Strides {
  int64_t s[4] = {8, 8, 8, 1};
  explicit Strides(const at::Tensor& t) {
    for (int i = 0; i < 3; ++i)
      if (t.size(i) > 1) s[i] = t.stride(i);
  }
  Strides() = default;
};

int dtype_of(at::ScalarType t) {
  return t == at::kBFloat16 ? SA_DTYPE_BF16 : t == at::kHalf ? SA_DTYPE_FP16
         : t == at::kFloat  ? SA_DTYPE_FP32 : -1;
}

bool same(const at::Tensor& a, const at::Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes();
}

bool flat(const at::Tensor& t) { return t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0; }

// Fresh contiguous memory, past the dispatcher (0.25 us less than at::empty).
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return fresh({(int64_t)n}, at::kByte, like);
}

bool number(PyObject* o, double& x) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  x = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

// The library's calls wait where the launch queue is full, so they run without
// the interpreter lock.
template <typename F>
int without_gil(F&& f) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}

// A tuple of results, or the library's return code for ops.py to raise.
PyObject* finish(int rc, const std::initializer_list<at::Tensor>& out) {
  if (rc != SA_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New((Py_ssize_t)out.size());
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const auto& t : out) {
    PyObject* o = wrap(t);
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// ---- attention backward: (dout, q, k, v, out, lse, block_mask, scale or None,
// head_mask_type, dlse, dq, dk, dv, workspace) ---------------------------------
PyObject* bsattn_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 || lib.bsattn_bwd == nullptr) return none();
  const Arg dout(a[0]), q(a[1]), k(a[2]), v(a[3]), out(a[4]), lse(a[5]), mask(a[6]), hmt(a[8]),
      dlse(a[9]), dq(a[10]), dk(a[11]), dv(a[12]), ws(a[13]);
  if (!q || !q->is_cuda() || q->dim() != 4 || !k || k->dim() != 4 || !dout || !v || !out || !lse ||
      !mask)
    return none();
  const int dev = q->get_device();
  for (const Arg* t : {&dout, &k, &v, &out, &lse, &mask, &hmt, &dlse, &dq, &dk, &dv, &ws})
    if (!on(*t, dev)) return none();
  if (dev >= kDevices || g_status[dev] == nullptr) return none();
  const int64_t B = q->size(0), H = q->size(1), Sq = q->size(2), Sk = k->size(2);
  if (q->scalar_type() != at::kBFloat16 || q->size(3) != 128 || k->size(0) != B ||
      k->size(1) != H || k->size(3) != 128 || !same(*dout, *q) || !same(*out, *q) ||
      k->scalar_type() != at::kBFloat16 || !same(*v, *k) || (dq && !same(*dq, *q)) ||
      (dk && !same(*dk, *k)) || (dv && !same(*dv, *k)) || Sq < 1 || Sk < 1 || Sq > 131072 ||
      Sk > 131072)
    return none();
  for (const Arg* t : {&dout, &q, &k, &v, &out, &dq, &dk, &dv})
    if (*t && !vectors(**t)) return none();
  if (!output(dq) || !output(dk) || !output(dv) || !workspace(ws)) return none();
  if (!apart(dq, {&dout, &q, &k, &v, &out, &dk, &dv}) ||
      !apart(dk, {&dout, &q, &k, &v, &out, &dv}) || !apart(dv, {&dout, &q, &k, &v, &out}))
    return none();
  for (const Arg* t : {&lse, &dlse})
    if (*t && ((*t)->scalar_type() != at::kFloat || (*t)->dim() != 3 || (*t)->size(0) != B ||
               (*t)->size(1) != H || (*t)->size(2) != Sq || !(*t)->is_contiguous()))
      return none();
  const int64_t nq = (Sq + 127) / 128, nk = (Sk + 127) / 128;
  if (mask->dim() != 4 || (mask->size(0) != 1 && mask->size(0) != B) || mask->size(2) != nq ||
      mask->size(3) != nk ||
      (mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte))
    return none();
  if (hmt && (hmt->scalar_type() != at::kInt || hmt->numel() != H || !hmt->is_contiguous()))
    return none();
  double scale = -1.0;
  if (a[7] != Py_None && !number(a[7], scale)) return none();

  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  // each gradient by default [B,S,H,D]-contiguous, viewed [B,H,S,D]
  const auto grad = [&](const Arg& given, int64_t S) {
    return given ? *given
                 : at::Tensor(at::detail::empty_strided_cuda(
                       {B, H, S, 128}, {S * H * 128, 128, H * 128, 1}, at::kBFloat16, q->device()));
  };
  const at::Tensor gq = grad(dq, Sq), gk = grad(dk, Sk), gv = grad(dv, Sk);
  const at::Tensor w = ws ? *ws : bytes(lib.bsattn_bwd_ws((int)B, (int)H, (int)Sq, (int)Sk), *q);
  const int64_t ms[4] = {mask->size(0) == 1 ? 0 : mask->stride(0), mask->stride(1),
                         mask->stride(2), mask->stride(3)};
  const Strides sd(*dout), sq(*q), sk(*k), sv(*v), so(*out), tq(gq), tk(gk), tv(gv);
  const int rc = without_gil([&] {
    return lib.bsattn_bwd(
        dout.ptr(), q.ptr(), k.ptr(), v.ptr(), out.ptr(), sd.s, sq.s, sk.s, sv.s, so.s,
        (const float*)lse.ptr(), (const float*)dlse.ptr(), (int)B, (int)H, (int)Sq, (int)Sk, 128,
        (const uint8_t*)mask.ptr(), ms, (int)mask->size(1), (const int32_t*)hmt.ptr(), (float)scale,
        gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), tq.s, tk.s, tv.s, w.data_ptr(),
        (size_t)w.nbytes(), g_status[dev], c10::cuda::getCurrentCUDAStream(dev).stream());
  });
  return finish(rc, {gq, gk, gv});
  END_HANDLE_TH_ERRORS
}

// The stride at which the B * S rows of [B, S, hidden] lie; -1 if there is none.
int64_t row_stride(const at::Tensor& t) {
  const int64_t B = t.size(0), S = t.size(1);
  if (t.stride(2) != 1 || (uintptr_t)t.data_ptr() % 16 != 0) return -1;
  const int64_t st = B * S == 1                                       ? t.size(2)
                     : S == 1                                         ? t.stride(0)
                     : B == 1 || t.stride(0) == S * t.stride(1) ? t.stride(1)
                                                                      : -1;
  return st % 8 == 0 ? st : -1;
}

// ---- hidden-wide norm gradient: (dq_out, dk_out, q, k, head_dim, eps, w_q,
// w_k, cos, sin, dq, dk, workspace) ---------------------------------------------
PyObject* qk_norm_rope_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || lib.norm_bwd == nullptr) return none();
  const Arg dqo(a[0]), dko(a[1]), q(a[2]), k(a[3]), wq(a[6]), wk(a[7]), cos(a[8]), sin(a[9]),
      dq(a[10]), dk(a[11]), ws(a[12]);
  if (!q || !q->is_cuda() || q->dim() != 3 || !dqo || !dko || !k || q->numel() == 0) return none();
  const int dev = q->get_device();
  for (const Arg* t : {&dqo, &dko, &k, &wq, &wk, &cos, &sin, &dq, &dk, &ws})
    if (!on(*t, dev)) return none();
  if (dev >= kDevices || g_status[dev] == nullptr) return none();
  double eps, hd;
  if (!number(a[5], eps) || !PyLong_Check(a[4]) || !number(a[4], hd)) return none();
  const int64_t B = q->size(0), S = q->size(1), hidden = q->size(2);
  if (q->scalar_type() != at::kBFloat16 || B * S > 0x7fffffff || hidden > 4096 || hd < 8 ||
      hd > hidden)
    return none();
  for (const Arg* t : {&dqo, &dko, &k, &dq, &dk})
    if (*t && !same(**t, *q)) return none();
  const Arg* rows[6] = {&dqo, &dko, &q, &k, &dq, &dk};
  int64_t st[6];
  for (int i = 0; i < 6; ++i) {
    st[i] = *rows[i] ? row_stride(**rows[i]) : hidden;
    if (st[i] < 0) return none();
  }
  if (!output(dq) || !output(dk) || !workspace(ws)) return none();
  if (!apart(dq, {&k, &dko, &dk}) || !apart(dk, {&q, &dqo})) return none();
  if (bool(wq) != bool(wk) || bool(cos) != bool(sin)) return none();
  if (wq && (wq->dim() != 1 || wq->size(0) != hidden || !same(*wk, *wq) || !flat(*wq) ||
             !flat(*wk) ||
             (wq->scalar_type() != at::kBFloat16 && wq->scalar_type() != at::kFloat)))
    return none();
  const int D = (int)hd;
  if (cos && (cos->scalar_type() != at::kFloat || cos->dim() != 2 || cos->size(0) != S ||
              cos->size(1) != D / 2 || !same(*sin, *cos) || !flat(*cos) || !flat(*sin)))
    return none();

  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  const at::Tensor gq = dq ? *dq : fresh(q->sizes(), at::kBFloat16, *q);
  const at::Tensor gk = dk ? *dk : fresh(q->sizes(), at::kBFloat16, *q);
  at::Tensor w, gwq, gwk;
  if (wq) {
    gwq = fresh({hidden}, at::kFloat, *q);
    gwk = fresh({hidden}, at::kFloat, *q);
    w = ws ? *ws : bytes(lib.norm_bwd_ws((int)hidden), *q);
  }
  const int rc = without_gil([&] {
    return lib.norm_bwd(
        dqo.ptr(), dko.ptr(), st[0], st[1], q.ptr(), k.ptr(), st[2], st[3], (int)(B * S), (int)S,
        (int)hidden, D, wq.ptr(), wk.ptr(), wq && wq->scalar_type() == at::kBFloat16, (float)eps,
        (const float*)cos.ptr(), (const float*)sin.ptr(), cos ? D / 2 : 0, gq.data_ptr(),
        gk.data_ptr(), st[4], st[5], wq ? gwq.data_ptr<float>() : nullptr,
        wq ? gwk.data_ptr<float>() : nullptr, wq ? w.data_ptr() : nullptr,
        wq ? (size_t)w.nbytes() : 0, g_status[dev], c10::cuda::getCurrentCUDAStream(dev).stream());
  });
  return finish(rc, {gq, gk, gwq, gwk});
  END_HANDLE_TH_ERRORS
}

// ---- per-head norm and its gradient --------------------------------------------
// What both check: q, k, eps, w_q, w_k, cos, sin, positions, interleaved.
struct Head {
  Arg q, k, wq, wk, cos, sin, pos;
  double eps = 0;
  int inter = 0, dev = 0, B = 0, S = 0, Hq = 0, Hk = 0, D = 0, dtype = 0, wdtype = SA_DTYPE_FP32;
  int rows = 0, rot = 0, pos64 = 0;
  int64_t fs = 0, pst[2] = {0, 0};
  bool ok = false;

  explicit Head(PyObject* const* a)
      : q(a[0]), k(a[1]), wq(a[3]), wk(a[4]), cos(a[5]), sin(a[6]), pos(a[7]) {
    if (!q || !q->is_cuda() || q->dim() != 4 || !number(a[2], eps) || !PyBool_Check(a[8])) return;
    inter = a[8] == Py_True;
    dev = q->get_device();
    for (const Arg* t : {&k, &wq, &wk, &cos, &sin, &pos})
      if (!on(*t, dev)) return;
    dtype = dtype_of(q->scalar_type());
    if (dev >= kDevices || g_status[dev] == nullptr || dtype < 0 || q->numel() == 0 ||
        q->size(0) * q->size(1) > 0x7fffffff || q->size(2) > 8192 || q->size(3) > 256)
      return;
    B = (int)q->size(0); S = (int)q->size(1); Hq = (int)q->size(2); D = (int)q->size(3);
    if (!vectors(*q)) return;
    if (k) {
      if (k->dim() != 4 || k->scalar_type() != q->scalar_type() || k->size(0) != B ||
          k->size(1) != S || k->size(3) != D || k->size(2) < 1 || k->size(2) > 8192 ||
          !vectors(*k))
        return;
      Hk = (int)k->size(2);
    }
    if (bool(wq) != (bool(wk) || (!k && wq)) || (wk && !k)) return;
    for (const Arg* t : {&wq, &wk})
      if (*t && ((*t)->dim() != 1 || (*t)->size(0) != D || !flat(**t) ||
                 (*t)->scalar_type() != wq->scalar_type()))
        return;
    if (wq) wdtype = dtype_of(wq->scalar_type());
    if (wdtype < 0 || bool(cos) != bool(sin)) return;
    if (cos) {
      if (cos->dim() != 2 || cos->size(0) < 1 || cos->scalar_type() != at::kFloat || !same(*sin, *cos) ||
          !vectors(*cos) || !vectors(*sin) || cos->size(0) > 0x7fffffff || cos->size(1) > 128)
        return;
      rows = (int)cos->size(0);
      rot = 2 * (int)cos->size(1);
      fs = rows > 1 ? cos->stride(0) : (rot / 2 + 3) / 4 * 4;
      if (rows > 1 && (sin->stride(0) != fs || fs < rot / 2)) return;
    }
    if (pos) {
      pos64 = pos->scalar_type() == at::kLong;
      if ((!pos64 && pos->scalar_type() != at::kInt) || !cos || pos->dim() < 1 || pos->dim() > 2 ||
          pos->size(-1) != S || (pos->dim() == 2 && pos->size(0) != B))
        return;
      pst[0] = pos->dim() == 2 ? pos->stride(0) : 0;
      pst[1] = pos->stride(-1);
    }
    ok = true;
  }
};

bool fits(const Arg& t, const Arg& like) {
  return t.ok && (!t || (like && t->is_cuda() && t->get_device() == like->get_device() &&
                         same(*t, *like) && vectors(*t)));
}

at::Tensor result(const Arg& given, const Arg& like) {
  if (given) return *given;
  return like ? fresh(like->sizes(), like->scalar_type(), *like) : at::Tensor();
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// (q, k, eps, w_q, w_k, cos, sin, positions, interleaved, out_q, out_k)
PyObject* qk_head_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || lib.head == nullptr) return none();
  const Head h(a);
  const Arg oq(a[9]), ok(a[10]);
  if (!h.ok || !fits(oq, h.q) || !fits(ok, h.k) || !output(oq) || !output(ok) ||
      !apart(oq, {&h.k, &ok}) || !apart(ok, {&h.q}))
    return none();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)h.dev);
  const at::Tensor rq = result(oq, h.q), rk = result(ok, h.k);
  const Strides sq(*h.q), sk = h.k ? Strides(*h.k) : Strides(), tq(rq),
                tk = h.k ? Strides(rk) : Strides();
  const int rc = without_gil([&] {
    return lib.head(
        h.q.ptr(), h.k.ptr(), sq.s, sk.s, h.B, h.S, h.Hq, h.Hk, h.D, h.dtype, h.wq.ptr(), h.wk.ptr(),
        h.wdtype, (float)h.eps, (const float*)h.cos.ptr(), (const float*)h.sin.ptr(), h.fs, h.rows,
        h.rot, h.inter, h.pos.ptr(), h.pos64, h.pst, ptr(rq), ptr(rk), tq.s, tk.s, g_status[h.dev],
        c10::cuda::getCurrentCUDAStream(h.dev).stream());
  });
  return finish(rc, {rq, rk});
  END_HANDLE_TH_ERRORS
}

// (q, k, eps, w_q, w_k, cos, sin, positions, interleaved, dq_out, dk_out, dq, dk,
// workspace)
PyObject* qk_head_norm_rope_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 || lib.head_bwd == nullptr) return none();
  const Head h(a);
  const Arg uq(a[9]), uk(a[10]), dq(a[11]), dk(a[12]), ws(a[13]);
  if (!h.ok || !uq || bool(uk) != bool(h.k) || !fits(uq, h.q) || !fits(uk, h.k) ||
      !fits(dq, h.q) || !fits(dk, h.k) || !output(dq) || !output(dk) || !on(ws, h.dev) ||
      !workspace(ws) || !apart(dq, {&h.k, &uk, &dk}) || !apart(dk, {&h.q, &uq}))
    return none();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)h.dev);
  const at::Tensor rq = result(dq, h.q), rk = result(dk, h.k);
  at::Tensor w, gwq, gwk;
  if (h.wq) {
    gwq = fresh({h.D}, at::kFloat, *h.q);
    if (h.k) gwk = fresh({h.D}, at::kFloat, *h.q);
    w = ws ? *ws : bytes(lib.head_bwd_ws(h.D), *h.q);
  }
  const Strides sq(*h.q), sk = h.k ? Strides(*h.k) : Strides(), tq(rq),
                tk = h.k ? Strides(rk) : Strides(), vq(*uq), vk = h.k ? Strides(*uk) : Strides();
  const int rc = without_gil([&] {
    return lib.head_bwd(
        uq.ptr(), uk.ptr(), vq.s, vk.s, h.q.ptr(), h.k.ptr(), sq.s, sk.s, h.B, h.S, h.Hq, h.Hk, h.D,
        h.dtype, h.wq.ptr(), h.wk.ptr(), h.wdtype, (float)h.eps, (const float*)h.cos.ptr(),
        (const float*)h.sin.ptr(), h.fs, h.rows, h.rot, h.inter, h.pos.ptr(), h.pos64, h.pst,
        ptr(rq), ptr(rk), tq.s, tk.s, (float*)ptr(gwq), (float*)ptr(gwk), ptr(w),
        w.defined() ? (size_t)w.nbytes() : 0, g_status[h.dev],
        c10::cuda::getCurrentCUDAStream(h.dev).stream());
  });
  return finish(rc, {rq, rk, gwq, gwk});
  END_HANDLE_TH_ERRORS
}

// bind(addresses in the order of Library's members)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes seven addresses");
    return nullptr;
  }
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib.bsattn_bwd = reinterpret_cast<decltype(lib.bsattn_bwd)>(p[0]);
  lib.bsattn_bwd_ws = reinterpret_cast<decltype(lib.bsattn_bwd_ws)>(p[1]);
  lib.norm_bwd = reinterpret_cast<decltype(lib.norm_bwd)>(p[2]);
  lib.norm_bwd_ws = reinterpret_cast<decltype(lib.norm_bwd_ws)>(p[3]);
  lib.head = reinterpret_cast<decltype(lib.head)>(p[4]);
  lib.head_bwd = reinterpret_cast<decltype(lib.head_bwd)>(p[5]);
  lib.head_bwd_ws = reinterpret_cast<decltype(lib.head_bwd_ws)>(p[6]);
  Py_RETURN_NONE;
}

// set_status(device index, address): where kernels on a device report failures
PyObject* set_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "set_status takes a device index and an address");
    return nullptr;
  }
  const long dev = PyLong_AsLong(a[0]);
  void* p = PyLong_AsVoidPtr(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if (dev >= 0 && dev < kDevices) g_status[dev] = static_cast<int32_t*>(p);
  Py_RETURN_NONE;
}

#define SA_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {SA_METHOD(bsattn_bwd),        SA_METHOD(qk_norm_rope_bwd),
                         SA_METHOD(qk_head_norm_rope), SA_METHOD(qk_head_norm_rope_bwd),
                         SA_METHOD(bind),              SA_METHOD(set_status),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
