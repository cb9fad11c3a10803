// torch binding of the attention layer's operators: checks the tensors, allocates outputs and
// workspaces from torch's allocator and calls the C ABI (include/b200attn.h) on the current
// stream of the tensors' device.  A decoding step's kernels take a few microseconds, so the
// host side of a call counts: measured on the B200 host, a single-token qk_norm_rope through
// ctypes and Python checks took 23.5 us a call, through this file 6.1 us.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <optional>

#include "b200attn.h"

namespace {

// A failed call, raised as benchmark_b200._lib.B200Error.
struct Failed {
  b200_status status;
};

void check(b200_status st) {
  if (st != B200_OK) throw Failed{st};
}

PyObject* raise_failed(b200_status st) {
  PyObject* lib = PyImport_ImportModule("benchmark_b200._lib");
  if (!lib) return nullptr;
  PyObject* type = PyObject_GetAttrString(lib, "B200Error");
  Py_DECREF(lib);
  if (!type) return nullptr;
  PyObject* e = PyObject_CallFunction(type, "is", static_cast<int>(st), b200_last_error());
  if (e) PyErr_SetObject(type, e);
  Py_XDECREF(e);
  Py_DECREF(type);
  return nullptr;
}

// Positional arguments by place; None is an absent tensor.
struct Args {
  PyObject* const* v;
  const at::Tensor& tensor(int i, const char* name) const {
    TORCH_CHECK_TYPE(THPVariable_Check(v[i]), name, ": expected a tensor");
    return THPVariable_Unpack(v[i]);
  }
  std::optional<at::Tensor> maybe(int i, const char* name) const {
    if (v[i] == Py_None) return std::nullopt;
    return tensor(i, name);
  }
  double real(int i) const {
    const double x = PyFloat_AsDouble(v[i]);
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
  }
  // A whole number, held to int's range (a window may be as large as the caller likes).
  int whole(int i) const {
    int over = 0;
    const long x = PyLong_AsLongAndOverflow(v[i], &over);
    if (x == -1 && !over && PyErr_Occurred()) throw python_error();
    if (over > 0 || x > INT_MAX) return INT_MAX;
    if (over < 0 || x < INT_MIN) return INT_MIN;
    return static_cast<int>(x);
  }
  bool truth(int i) const {
    const int x = PyObject_IsTrue(v[i]);
    if (x < 0) throw python_error();
    return x != 0;
  }
};

int dim(int64_t n) {
  TORCH_CHECK_VALUE(n <= INT_MAX, "an axis of ", n, " elements is too long");
  return static_cast<int>(n);
}

// The first tensor gives the device of a call.
struct Call {
  c10::Device device;
  c10::cuda::OptionalCUDAGuard guard;
  b200_stream_t stream;
  explicit Call(const at::Tensor& t) : device(t.device()) {
    TORCH_CHECK_VALUE(device.is_cuda(), "expected CUDA tensors");
    guard.set_device(device);
    stream = reinterpret_cast<b200_stream_t>(
        c10::cuda::getCurrentCUDAStream(device.index()).stream());
  }
  b200_tensor view(const at::Tensor& t, at::IntArrayRef shape, const char* name) const {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.device() == device, name,
                      ": expected a bf16 tensor on ", device);
    TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected shape ", shape, ", got ", t.sizes());
    TORCH_CHECK_VALUE(t.stride(3) == 1, name, ": the last axis must be contiguous");
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
  }
  // [H, S, D] as [1, H, S, D].
  b200_tensor view3(const at::Tensor& t, at::IntArrayRef shape, const char* name) const {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.device() == device, name,
                      ": expected a bf16 tensor on ", device);
    TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected shape ", shape, ", got ", t.sizes());
    TORCH_CHECK_VALUE(t.stride(2) == 1, name, ": the last axis must be contiguous");
    return {t.data_ptr(), 0, t.stride(0), t.stride(1)};
  }
  void* flat(const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape,
             const char* name) const {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == device && t.sizes() == shape &&
                          t.is_contiguous(),
                      name, ": expected a contiguous ", type, " tensor of shape ", shape, " on ",
                      device);
    return t.data_ptr();
  }
  void* flat(const std::optional<at::Tensor>& t, at::ScalarType type, at::IntArrayRef shape,
             const char* name) const {
    return t ? flat(*t, type, shape, name) : nullptr;
  }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type = at::kBFloat16) const {
    return at::empty(shape, at::TensorOptions().dtype(type).device(device));
  }
  at::Tensor given_or_empty(const std::optional<at::Tensor>& t, at::IntArrayRef shape) const {
    return t ? *t : empty(shape);
  }
  // n bytes that the stream's later work may reuse once this call's kernels are done.
  at::Tensor workspace(size_t n) const {
    return n == 0 ? at::Tensor() : empty({static_cast<int64_t>(n)}, at::kByte);
  }
};

void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

template <typename F>
b200_status unlocked(F&& f) {
  b200_status st;
  Py_BEGIN_ALLOW_THREADS;
  st = f();
  Py_END_ALLOW_THREADS;
  return st;
}

template <typename... T>
PyObject* tuple_of(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t)), ...);
  return r;
}

struct Sizes {
  int B, H, S, D;
  explicit Sizes(const at::Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 4, name, ": expected [B, H, S, D], got ", t.sizes());
    B = dim(t.size(0));
    H = dim(t.size(1));
    S = dim(t.size(2));
    D = dim(t.size(3));
  }
};

// What qk_norm_rope and its backward share: q, k, weights, frequencies, positions.
struct Rope {
  Sizes q_size, k_size;
  at::DimVector qs, ks;
  b200_tensor q, k;
  void *wq, *wk;
  int w_f32, rot;
  const float* freq;
  const int32_t* pos;
  int64_t pos_sb;
  Rope(const Call& c, const Args& a, int at0)
      : q_size(a.tensor(at0, "q"), "q"), k_size(a.tensor(at0 + 1, "k"), "k") {
    const at::Tensor &qt = a.tensor(at0, "q"), &kt = a.tensor(at0 + 1, "k"),
                     &wqt = a.tensor(at0 + 2, "q_weight"), &wkt = a.tensor(at0 + 3, "k_weight"),
                     &f = a.tensor(at0 + 4, "inv_freq"), &p = a.tensor(at0 + 5, "positions");
    const int64_t B = q_size.B, S = q_size.S, D = q_size.D;
    qs = {B, q_size.H, S, D};
    ks = {B, k_size.H, S, D};
    q = c.view(qt, qs, "q");
    k = c.view(kt, ks, "k");
    const at::ScalarType w = wqt.scalar_type() == at::kFloat ? at::kFloat : at::kBFloat16;
    w_f32 = w == at::kFloat;
    wq = c.flat(wqt, w, {D}, "q_weight");
    wk = c.flat(wkt, w, {D}, "k_weight");
    freq = static_cast<const float*>(c.flat(f, at::kFloat, {f.numel()}, "inv_freq"));
    rot = dim(2 * f.numel());
    const bool shared = p.dim() == 1;
    TORCH_CHECK_VALUE(p.scalar_type() == at::kInt && p.device() == c.device &&
                          (shared ? p.size(0) == S
                                  : p.dim() == 2 && p.size(0) == B && p.size(1) == S) &&
                          (S == 1 || p.stride(-1) == 1),
                      "positions: expected int32 [", S, "] or [", B, ", ", S, "] on ", c.device,
                      ", contiguous along the tokens");
    pos = p.data_ptr<int32_t>();
    pos_sb = shared || B == 1 ? 0 : p.stride(0);
  }
};

PyObject* qk_norm_rope_(const Args& a) {
  const Call c(a.tensor(0, "q"));
  const Rope r(c, a, 0);
  const at::Tensor qo = c.given_or_empty(a.maybe(8, "q_out"), r.qs);
  const at::Tensor ko = c.given_or_empty(a.maybe(9, "k_out"), r.ks);
  const b200_tensor qv = c.view(qo, r.qs, "q_out"), kv = c.view(ko, r.ks, "k_out");
  const float eps = static_cast<float>(a.real(6));
  const int interleaved = a.truth(7);
  check(unlocked([&] {
    return qk_norm_rope(&r.q, &r.k, r.wq, r.wk, r.w_f32, r.freq, r.rot, interleaved, r.pos,
                        r.pos_sb, eps, &qv, &kv, r.q_size.B, r.q_size.S, r.q_size.H, r.k_size.H,
                        r.q_size.D, c.stream);
  }));
  return tuple_of(qo, ko);
}

PyObject* qk_norm_rope_bwd_(const Args& a) {
  const Call c(a.tensor(2, "q"));
  const Rope r(c, a, 2);
  const b200_tensor gq = c.view(a.tensor(0, "dq_out"), r.qs, "dq_out");
  const b200_tensor gk = c.view(a.tensor(1, "dk_out"), r.ks, "dk_out");
  const at::Tensor dq = c.given_or_empty(a.maybe(10, "dq"), r.qs);
  const at::Tensor dk = c.given_or_empty(a.maybe(11, "dk"), r.ks);
  const b200_tensor qv = c.view(dq, r.qs, "dq"), kv = c.view(dk, r.ks, "dk");
  const int64_t D = r.q_size.D;
  const at::Tensor dwq = c.empty({D}, at::kFloat), dwk = c.empty({D}, at::kFloat);
  const float eps = static_cast<float>(a.real(8));
  const int interleaved = a.truth(9);
  size_t n = 0;
  check(qk_norm_rope_bwd_workspace(r.q_size.B, r.q_size.S, r.q_size.D, &n));
  const at::Tensor ws = c.workspace(n);
  check(unlocked([&] {
    return qk_norm_rope_bwd(&gq, &gk, &r.q, &r.k, r.wq, r.wk, r.w_f32, r.freq, r.rot, interleaved,
                            r.pos, r.pos_sb, eps, &qv, &kv, static_cast<float*>(dwq.data_ptr()),
                            static_cast<float*>(dwk.data_ptr()), r.q_size.B, r.q_size.S,
                            r.q_size.H, r.k_size.H, r.q_size.D, pointer(ws), n, c.stream);
  }));
  return tuple_of(dq, dk, dwq, dwk);
}

PyObject* attention_window_fwd_(const Args& a) {
  const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &v = a.tensor(2, "v");
  const Call c(q);
  const Sizes s(q, "q"), t(k, "k");
  const at::DimVector qs{s.B, s.H, s.S, s.D}, ks{s.B, t.H, t.S, s.D};
  const int window = a.whole(3), sinks = a.whole(4);
  const auto kv_len = a.maybe(5, "kv_len"), lse = a.maybe(8, "lse");
  const at::Tensor out = c.given_or_empty(a.maybe(6, "out"), qs);
  const b200_tensor qv = c.view(q, qs, "q"), kv = c.view(k, ks, "k"), vv = c.view(v, ks, "v"),
                    ov = c.view(out, qs, "out");
  const auto* len = static_cast<const int32_t*>(c.flat(kv_len, at::kInt, {s.B}, "kv_len"));
  auto* lse_p = static_cast<float*>(c.flat(lse, at::kFloat, {s.B, s.H, s.S}, "lse"));
  const float scale = static_cast<float>(a.real(7));
  size_t n = 0;
  check(attention_window_fwd_workspace(s.B, s.H, t.H, s.S, t.S, s.D, window, sinks, &n));
  const at::Tensor ws = c.workspace(n);
  check(unlocked([&] {
    return attention_window_fwd(&qv, &kv, &vv, &ov, lse_p, len, s.B, s.H, t.H, s.S, t.S, s.D,
                                window, sinks, scale, pointer(ws), n, c.stream);
  }));
  return THPVariable_Wrap(out);
}

PyObject* attention_window_bwd_(const Args& a) {
  const at::Tensor &q = a.tensor(1, "q"), &k = a.tensor(2, "k"), &lse = a.tensor(5, "lse");
  const Call c(q);
  const Sizes s(q, "q"), t(k, "k");
  const at::DimVector qs{s.B, s.H, s.S, s.D}, ks{s.B, t.H, t.S, s.D};
  const int window = a.whole(6), sinks = a.whole(7);
  const auto kv_len = a.maybe(8, "kv_len");
  const at::Tensor dq = c.given_or_empty(a.maybe(10, "dq"), qs);
  const at::Tensor dk = c.given_or_empty(a.maybe(11, "dk"), ks);
  const at::Tensor dv = c.given_or_empty(a.maybe(12, "dv"), ks);
  const b200_tensor gv = c.view(a.tensor(0, "dout"), qs, "dout"), qv = c.view(q, qs, "q"),
                    kv = c.view(k, ks, "k"), vv = c.view(a.tensor(3, "v"), ks, "v"),
                    ov = c.view(a.tensor(4, "o"), qs, "o"), dqv = c.view(dq, qs, "dq"),
                    dkv = c.view(dk, ks, "dk"), dvv = c.view(dv, ks, "dv");
  const auto* lse_p = static_cast<const float*>(c.flat(lse, at::kFloat, {s.B, s.H, s.S}, "lse"));
  const auto* len = static_cast<const int32_t*>(c.flat(kv_len, at::kInt, {s.B}, "kv_len"));
  const float scale = static_cast<float>(a.real(9));
  size_t n = 0;
  check(attention_window_bwd_workspace(s.B, s.H, t.H, s.S, t.S, s.D, window, sinks, &n));
  const at::Tensor ws = c.workspace(n);
  check(unlocked([&] {
    return attention_window_bwd(&gv, &qv, &kv, &vv, &ov, lse_p, &dqv, &dkv, &dvv, len, s.B, s.H,
                                t.H, s.S, t.S, s.D, window, sinks, scale, pointer(ws), n,
                                c.stream);
  }));
  return tuple_of(dq, dk, dv);
}

PyObject* attention_shared_prefix_(const Args& a) {
  const at::Tensor &q = a.tensor(0, "q"), &kp = a.tensor(1, "k_prefix"),
                   &vp = a.tensor(2, "v_prefix"), &k = a.tensor(3, "k"), &v = a.tensor(4, "v");
  const Call c(q);
  const Sizes s(q, "q"), t(k, "k");
  TORCH_CHECK_VALUE(kp.dim() == 3, "k_prefix: expected [H, P, D], got ", kp.sizes());
  const int P = dim(kp.size(1));
  const at::DimVector qs{s.B, s.H, s.S, s.D}, ks{s.B, t.H, t.S, s.D}, ps{t.H, P, s.D};
  const auto kv_len = a.maybe(5, "kv_len");
  const at::Tensor out = c.given_or_empty(a.maybe(6, "out"), qs);
  const b200_tensor qv = c.view(q, qs, "q"), kpv = c.view3(kp, ps, "k_prefix"),
                    vpv = c.view3(vp, ps, "v_prefix"), kv = c.view(k, ks, "k"),
                    vv = c.view(v, ks, "v"), ov = c.view(out, qs, "out");
  const auto* len = static_cast<const int32_t*>(c.flat(kv_len, at::kInt, {s.B}, "kv_len"));
  const float scale = static_cast<float>(a.real(7));
  size_t n = 0;
  check(attention_shared_prefix_workspace(s.B, s.H, t.H, s.S, P, t.S, s.D, &n));
  const at::Tensor ws = c.workspace(n);
  check(unlocked([&] {
    return attention_shared_prefix(&qv, &kpv, &vpv, &kv, &vv, &ov, len, s.B, s.H, t.H, s.S, P,
                                   t.S, s.D, scale, pointer(ws), n, c.stream);
  }));
  return THPVariable_Wrap(out);
}

template <PyObject* (*kBody)(const Args&), int kCount>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == kCount, "expected ", kCount, " arguments, got ", n);
  try {
    return kBody(Args{args});
  } catch (const Failed& f) {
    return raise_failed(f.status);
  }
  END_HANDLE_TH_ERRORS
}

#define B200_METHOD(name, count)                                                      \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<name##_, count>)), \
   METH_FASTCALL, nullptr}

PyMethodDef methods[] = {B200_METHOD(qk_norm_rope, 10),
                         B200_METHOD(qk_norm_rope_bwd, 12),
                         B200_METHOD(attention_window_fwd, 9),
                         B200_METHOD(attention_window_bwd, 13),
                         B200_METHOD(attention_shared_prefix, 8),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
