// The host side of the entry points' common case, as a CPython module (warpy_kernels_b200/_host.so).
//
// A call of an entry point costs 20-70 us of interpreter time when its checks, its output
// tensors and its argument block are made in Python, which is more than the kernels of a small problem take.  Here
// the same work takes 3-6 us: arguments are read from the vectorcall array, outputs come from the caching allocator
// without going through the dispatcher, and the C ABI entry point is called with the GIL released.
//
// Every function returns None for anything but the plain, valid case (a wrong shape or dtype, a tensor that needs a
// copy, an unknown option): the Python function of the same name then does the call, copies and raises as documented.
// So this file repeats conditions, never messages.  The kernels are reached through the C ABI of libwarpy_b200.so,
// whose addresses _lib.py hands over (bind()), so that another build of that library can be used.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>
#include <cstring>
#include <exception>
#include <map>
#include <string>
#include <unordered_map>
#include <utility>

#include "../../../include/warpy_b200.h"

namespace {

// ---- the C ABI --------------------------------------------------------------------------------------------------
struct Abi {
  int (*device_arch)(int);
  const char* (*error_string)(int);
  int (*attn_fwd_fp8)(const wk_attn_fwd_args*, void*);
  int (*attn_fwd_bf16)(const wk_attn_fwd_args*, void*);
  int64_t (*attn_fwd_workspace_bytes)(int, int, int);
  int (*attn_bwd_fp8)(const wk_attn_bwd_args*, void*);
  int (*attn_bwd_bf16)(const wk_attn_bwd_args*, void*);
  int64_t (*attn_bwd_fp8_workspace_bytes)(int, int, int);
  int64_t (*attn_bwd_bf16_workspace_bytes)(int, int, int);
  int (*gemm_16bit)(const wk_gemm16_args*, void*);
  int (*gemm_mxfp8)(const wk_gemm_mx_args*, void*);
  int64_t (*gemm_mxfp8_workspace_bytes)(int, int, int);
  int (*quantize_mx)(const void*, int, int64_t, int64_t, int64_t, void*, void*, void*);
  int (*rope)(const wk_rope_args*, void*);
  int64_t (*qk_norm_rope_bwd_workspace_bytes)(int);
  int (*qk_norm_rope_bwd)(const wk_rope_args*, void*);
  int64_t (*attn_prefix_workspace_bytes)(int, int, int, int, int, int, int);
  int (*attn_prefix)(const wk_attn_prefix_args*, void*);
} abi;
bool bound = false;

const struct {
  const char* name;
  void** slot;
} kSymbols[] = {
    {"wk_device_arch", reinterpret_cast<void**>(&abi.device_arch)},
    {"wk_error_string", reinterpret_cast<void**>(&abi.error_string)},
    {"wk_attn_fwd_fp8", reinterpret_cast<void**>(&abi.attn_fwd_fp8)},
    {"wk_attn_fwd_bf16", reinterpret_cast<void**>(&abi.attn_fwd_bf16)},
    {"wk_attn_fwd_workspace_bytes", reinterpret_cast<void**>(&abi.attn_fwd_workspace_bytes)},
    {"wk_attn_bwd_fp8", reinterpret_cast<void**>(&abi.attn_bwd_fp8)},
    {"wk_attn_bwd_bf16", reinterpret_cast<void**>(&abi.attn_bwd_bf16)},
    {"wk_attn_bwd_fp8_workspace_bytes", reinterpret_cast<void**>(&abi.attn_bwd_fp8_workspace_bytes)},
    {"wk_attn_bwd_bf16_workspace_bytes", reinterpret_cast<void**>(&abi.attn_bwd_bf16_workspace_bytes)},
    {"wk_gemm_16bit", reinterpret_cast<void**>(&abi.gemm_16bit)},
    {"wk_gemm_mxfp8", reinterpret_cast<void**>(&abi.gemm_mxfp8)},
    {"wk_gemm_mxfp8_workspace_bytes", reinterpret_cast<void**>(&abi.gemm_mxfp8_workspace_bytes)},
    {"wk_quantize_mx", reinterpret_cast<void**>(&abi.quantize_mx)},
    {"wk_rope", reinterpret_cast<void**>(&abi.rope)},
    {"wk_qk_norm_rope_bwd_workspace_bytes", reinterpret_cast<void**>(&abi.qk_norm_rope_bwd_workspace_bytes)},
    {"wk_qk_norm_rope_bwd", reinterpret_cast<void**>(&abi.qk_norm_rope_bwd)},
    {"wk_attn_fwd_shared_prefix_workspace_bytes", reinterpret_cast<void**>(&abi.attn_prefix_workspace_bytes)},
    {"wk_attn_fwd_shared_prefix", reinterpret_cast<void**>(&abi.attn_prefix)},
};

constexpr int kMaxDevices = 64;
constexpr int kArch = 100;

// Whether the library has kernels for CUDA device `dev` (asked once per device).
bool device_ok(int dev) {
  static signed char known[kMaxDevices] = {};  // 0 not asked, 1 yes; guarded by the GIL
  if (dev < 0 || dev >= kMaxDevices) return false;
  if (!known[dev] && abi.device_arch(dev) == kArch) known[dev] = 1;
  return known[dev] == 1;
}

// ---- arguments --------------------------------------------------------------------------------------------------
// The values of a fixed list of parameter names, from the positional and keyword arguments of a vectorcall.
template <int N>
struct Params {
  std::array<PyObject*, N> v{};

  // False if an argument is not in the list (the Python function decides what that means).
  bool read(const std::array<PyObject*, N>& names, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    if (nargs > N) return false;
    for (Py_ssize_t i = 0; i < nargs; ++i) v[i] = args[i];
    const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    for (Py_ssize_t j = 0; j < nkw; ++j) {
      PyObject* key = PyTuple_GET_ITEM(kwnames, j);
      int at = -1;
      for (int i = 0; i < N && at < 0; ++i)  // keyword names of a call site are interned: the pointers are equal
        if (names[i] == key) at = i;
      for (int i = 0; i < N && at < 0; ++i)
        if (PyUnicode_Compare(names[i], key) == 0) at = i;
      if (at < 0 || v[at]) return false;
      v[at] = args[nargs + j];
    }
    return true;
  }
  bool given(int i) const { return v[i] && v[i] != Py_None; }
  // A truth value, `fallback` where the argument is absent. False if the argument has none (a tensor of several
  // elements): the Python function asks it again and raises.
  bool flag(int i, bool fallback, bool& out) const {
    const int t = v[i] ? PyObject_IsTrue(v[i]) : fallback;
    if (t < 0) PyErr_Clear();
    out = t > 0;
    return t >= 0;
  }
};

template <int N>
std::array<PyObject*, N> interned(const std::array<const char*, N>& names) {
  std::array<PyObject*, N> out{};
  for (int i = 0; i < N; ++i) out[i] = PyUnicode_InternFromString(names[i]);
  return out;
}

const at::Tensor* tensor_of(PyObject* o) {
  return o && THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

PyObject* declined() { Py_RETURN_NONE; }

PyObject* failed(int code, const char* what) {
  PyErr_Format(code == WK_E_ARG ? PyExc_ValueError : PyExc_RuntimeError,
               code == WK_E_ARG ? "%s: %s" : "%s: %s (code %d)", what, abi.error_string(code), code);
  return nullptr;
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, dev, std::nullopt));
}
at::Tensor empty_strided(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType dtype, const at::Device& dev) {
  return at::Tensor(at::detail::empty_strided_cuda(sizes, strides, dtype, dev));
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Gives up the GIL for as long as it lives; an exception on the way out takes it back too.
struct GilReleased {
  PyThreadState* state = PyEval_SaveThread();
  ~GilReleased() { PyEval_RestoreThread(state); }
};

// Calls fn(stream) on the current stream of `dev` with that device current and the GIL released.
template <class F>
int on_device(int dev, F fn) {
  const GilReleased gil;
  const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)));
  return fn(static_cast<void*>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream()));
}

// ---- attention --------------------------------------------------------------------------------------------------
// Zeroed scratch for the forward's block flags, one per (device, stream): the kernels hand it back zeroed, so the
// calls that follow one another on a stream share it.  Torch has a fixed number of streams per device, which bounds
// the table; a buffer only ever grows.  Graphs may be replayed beside one another and beside other calls, whatever stream
// they were captured on: a capture has a buffer of its own, in its graph's memory, whose zeros are part of the graph.  The
// table keeps it as long as calls of that capture may come.  Guarded by the GIL.
at::Tensor& block_flags(int dev, void* stream, int64_t nbytes) {
  struct Buffers {
    at::Tensor eager, captured;
    unsigned long long capture = 0;
  };
  static auto* table = new std::map<std::pair<int, void*>, Buffers>();  // outlives the interpreter's teardown
  Buffers& b = (*table)[{dev, stream}];
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &capture) != cudaSuccess) {
    cudaGetLastError();  // whatever it is, the launch will tell
    status = cudaStreamCaptureStatusNone;
  }
  const bool capturing = status == cudaStreamCaptureStatusActive;
  if (capturing && b.capture != capture) b.captured = at::Tensor(), b.capture = capture;
  at::Tensor& buf = capturing ? b.captured : b.eager;
  if (!buf.defined() || buf.numel() < nbytes)
    buf = at::zeros({std::max<int64_t>(nbytes, 1 << 16)},
                    at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)));
  return buf;
}

struct AttnShape {
  int64_t B, Hq, Hkv, Nq, Nk, d;
  bool fp8;
  at::Device dev{at::kCPU};
};

// TMA reads a tensor where it is: last stride 1, the others multiples of 16 elements, 16-byte aligned base.
bool tma_direct(const at::Tensor& t) {
  return t.stride(3) == 1 && t.stride(0) % 16 == 0 && t.stride(1) % 16 == 0 && t.stride(2) % 16 == 0 &&
         aligned(t.data_ptr(), 16);
}

bool attn_shape(const at::Tensor* q, const at::Tensor* k, const at::Tensor* v, AttnShape& s) {
  if (!q || !k || !v || q->dim() != 4 || k->dim() != 4 || v->dim() != 4) return false;
  const at::ScalarType t = q->scalar_type();
  s.fp8 = t == at::kFloat8_e4m3fn;
  if ((!s.fp8 && t != at::kBFloat16) || k->scalar_type() != t || v->scalar_type() != t) return false;
  s.dev = q->device();
  if (!s.dev.is_cuda() || k->device() != s.dev || v->device() != s.dev || !device_ok(s.dev.index())) return false;
  s.B = q->size(0), s.Hq = q->size(1), s.Nq = q->size(2), s.d = q->size(3);
  s.Hkv = k->size(1), s.Nk = k->size(2);
  if (k->sizes() != v->sizes() || k->size(0) != s.B || k->size(3) != s.d || (s.d != 64 && s.d != 128)) return false;
  if (s.B < 1 || s.Hkv < 1 || s.Nq < 1 || s.Nk < 1 || s.Hq % s.Hkv || s.Nq > INT32_MAX / 2 || s.Nk > INT32_MAX / 2)
    return false;
  return tma_direct(*q) && tma_direct(*k) && tma_direct(*v);
}

// A [B, Hkv] contiguous float32 descale on the inputs' device.
bool descale(PyObject* o, const AttnShape& s, const float*& out) {
  const at::Tensor* t = tensor_of(o);
  if (!t || t->dim() != 2 || t->size(0) != s.B || t->size(1) != s.Hkv || t->scalar_type() != at::kFloat ||
      t->device() != s.dev || !t->is_contiguous())
    return false;
  out = t->const_data_ptr<float>();
  return true;
}

bool softmax_scale_of(PyObject* o, int64_t d, float& out) {
  if (!o || o == Py_None) {
    out = static_cast<float>(1.0 / std::sqrt(static_cast<double>(d)));
    return true;
  }
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  const double x = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  out = static_cast<float>(x);
  return x > 0.0;
}

void put_strides(int64_t (&dst)[3], const at::Tensor& t) {
  for (int i = 0; i < 3; ++i) dst[i] = t.stride(i);
}

PyObject* attn_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, K, V, QD, KD, VD, CAUSAL, SCALE, STAGES, PIPE, BLOCK_N, BLOCK_M, WARP_ROWS, CTAS, LOCAL, LPT, TMA, OUT,
         LSE, USED, NATURAL, SPEC, SPLIT, COUNT };
  static const auto names = interned<COUNT>(
      {"q", "k", "v", "q_descale", "k_descale", "v_descale", "causal", "softmax_scale", "num_stages", "pipelined",
       "block_n", "block_m", "warp_rows", "ctas_per_sm", "tile_local", "lpt", "tma", "out", "return_lse", "seqused_k",
       "lse_natural", "warp_spec", "split_kv"});
  Params<COUNT> p;
  AttnShape s;
  if (!bound || !p.read(names, args, nargs, kwnames)) return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *k = tensor_of(p.v[K]), *v = tensor_of(p.v[V]);
  if (!attn_shape(q, k, v, s)) return declined();
  wk_attn_fwd_args a = {};
  if (s.fp8) {
    if (!descale(p.v[QD], s, a.q_descale) || !descale(p.v[KD], s, a.k_descale) || !descale(p.v[VD], s, a.v_descale))
      return declined();
  } else if (p.given(QD) || p.given(KD) || p.given(VD)) {
    return declined();
  }
  if (!softmax_scale_of(p.v[SCALE], s.d, a.softmax_scale)) return declined();
  bool with_lse, causal, natural;
  if (!p.flag(LSE, true, with_lse) || !p.flag(CAUSAL, false, causal) || !p.flag(NATURAL, false, natural))
    return declined();
  if (p.given(CTAS)) {
    const long n = PyLong_Check(p.v[CTAS]) ? PyLong_AsLong(p.v[CTAS]) : 0;
    if (n == -1) PyErr_Clear();  // beyond a long
    if (n != 1 && n != 2) return declined();
    a.ctas_per_sm = static_cast<int32_t>(n);
  }
  if (p.given(USED)) {
    const at::Tensor* used = tensor_of(p.v[USED]);
    if (!used || used->dim() != 1 || used->size(0) != s.B || used->scalar_type() != at::kInt ||
        used->device() != s.dev || !used->is_contiguous())
      return declined();
    a.seqused_k = used->const_data_ptr<int32_t>();
  }
  at::Tensor out;
  if (p.given(OUT)) {
    const at::Tensor* o = tensor_of(p.v[OUT]);
    if (!o || o->dim() != 4 || o->sizes() != q->sizes() || o->scalar_type() != at::kBFloat16 || o->device() != s.dev ||
        o->stride(3) != 1 || o->stride(0) % 8 || o->stride(1) % 8 || o->stride(2) % 8 || !aligned(o->data_ptr(), 16))
      return declined();
    out = *o;
  } else if (q->is_non_overlapping_and_dense()) {
    out = empty_strided(q->sizes(), q->strides(), at::kBFloat16, s.dev);  // the memory layout of q
  } else {
    out = at::empty_like(*q, q->options().dtype(at::kBFloat16));
  }
  a.q = q->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr(), a.out = out.data_ptr();
  put_strides(a.q_strides, *q), put_strides(a.k_strides, *k), put_strides(a.v_strides, *v);
  put_strides(a.out_strides, out);
  at::Tensor lse, pmax;
  if (with_lse) {
    const int64_t nq_pad = (s.Nq + 127) / 128 * 128;  // rows of lse and pmax start every nq_pad entries
    const std::array<int64_t, 3> sizes = {s.B, s.Hq, s.Nq}, strides = {s.Hq * nq_pad, nq_pad, 1};
    lse = empty_strided(sizes, strides, at::kFloat, s.dev);
    pmax = empty_strided(sizes, strides, at::kFloat, s.dev);
    a.lse = lse.mutable_data_ptr<float>(), a.pmax = pmax.mutable_data_ptr<float>();
    a.lse_strides[0] = strides[0], a.lse_strides[1] = strides[1];
    a.write_lse = 1;
  }
  a.B = s.B, a.Hq = s.Hq, a.Hkv = s.Hkv, a.Nq = s.Nq, a.Nk = s.Nk, a.d = s.d;
  a.causal = causal, a.lse_natural = natural;
  a.workspace_bytes = abi.attn_fwd_workspace_bytes(a.B, a.Hq, a.Nq);
  void* stream = c10::cuda::getCurrentCUDAStream(s.dev.index()).stream();
  a.workspace = block_flags(s.dev.index(), stream, a.workspace_bytes).data_ptr();
  const int code = on_device(s.dev.index(), [&](void* st) { return (s.fp8 ? abi.attn_fwd_fp8 : abi.attn_fwd_bf16)(&a, st); });
  if (code) return failed(code, "attn_fwd");
  PyObject* o = p.given(OUT) ? Py_NewRef(p.v[OUT]) : THPVariable_Wrap(std::move(out));
  PyObject* l = with_lse ? THPVariable_Wrap(std::move(lse)) : Py_NewRef(Py_None);
  PyObject* m = with_lse ? THPVariable_Wrap(std::move(pmax)) : Py_NewRef(Py_None);
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, o), PyTuple_SET_ITEM(r, 1, l), PyTuple_SET_ITEM(r, 2, m);
  return r;
}

// bf16 with last stride 1: out and dout of the FP8 backward go through 8-byte loads, dout of the BF16 one through TMA.
bool bf16_rows(const at::Tensor* t, const at::Tensor& q, int64_t stride_unit, uintptr_t base_unit) {
  return t && t->dim() == 4 && t->sizes() == q.sizes() && t->scalar_type() == at::kBFloat16 &&
         t->device() == q.device() && t->stride(3) == 1 && t->stride(0) % stride_unit == 0 &&
         t->stride(1) % stride_unit == 0 && t->stride(2) % stride_unit == 0 && aligned(t->data_ptr(), base_unit);
}

PyObject* attn_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, K, V, OUT, LSE, PMAX, DOUT, QD, KD, VD, CAUSAL, SCALE, STAGES, BULK, INTER, DET, BLOCK_M, MAJOR, USED, ONE,
         COUNT };
  static const auto names = interned<COUNT>(
      {"q", "k", "v", "out", "lse", "pmax", "dout", "q_descale", "k_descale", "v_descale", "causal", "softmax_scale",
       "num_stages", "dq_bulk", "dq_interleave", "deterministic", "block_m", "kb_major", "seqused_k", "one_barrier"});
  Params<COUNT> p;
  AttnShape s;
  if (!bound || !p.read(names, args, nargs, kwnames) || p.given(USED)) return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *k = tensor_of(p.v[K]), *v = tensor_of(p.v[V]);
  const at::Tensor *out = tensor_of(p.v[OUT]), *dout = tensor_of(p.v[DOUT]);
  const at::Tensor *lse = tensor_of(p.v[LSE]), *pmax = tensor_of(p.v[PMAX]);
  if (!attn_shape(q, k, v, s)) return declined();
  wk_attn_bwd_args a = {};
  if (s.fp8) {
    if (!descale(p.v[QD], s, a.q_descale) || !descale(p.v[KD], s, a.k_descale) || !descale(p.v[VD], s, a.v_descale))
      return declined();
  } else if (p.given(QD) || p.given(KD) || p.given(VD)) {
    return declined();
  }
  if (!bf16_rows(out, *q, 4, 8) || !bf16_rows(dout, *q, s.fp8 ? 4 : 16, s.fp8 ? 8 : 16)) return declined();
  const std::array<int64_t, 3> rows = {s.B, s.Hq, s.Nq};
  if (!lse || !pmax || lse->sizes() != at::IntArrayRef(rows) || pmax->sizes() != at::IntArrayRef(rows) ||
      lse->scalar_type() != at::kFloat || lse->device() != s.dev || lse->stride(2) != 1)
    return declined();
  bool causal;
  if (!softmax_scale_of(p.v[SCALE], s.d, a.softmax_scale) || !p.flag(CAUSAL, false, causal)) return declined();
  at::Tensor dq = empty({s.B, s.Hq, s.Nq, s.d}, at::kBFloat16, s.dev);
  at::Tensor dk = empty({s.B, s.Hkv, s.Nk, s.d}, at::kBFloat16, s.dev);
  at::Tensor dv = empty({s.B, s.Hkv, s.Nk, s.d}, at::kBFloat16, s.dev);
  a.workspace_bytes = (s.fp8 ? abi.attn_bwd_fp8_workspace_bytes : abi.attn_bwd_bf16_workspace_bytes)(s.B, s.Hq, s.Nq);
  at::Tensor workspace = empty({a.workspace_bytes}, at::kByte, s.dev);
  a.q = q->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr(), a.out = out->data_ptr(), a.dout = dout->data_ptr();
  a.lse = lse->const_data_ptr<float>();
  a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr(), a.workspace = workspace.data_ptr();
  put_strides(a.q_strides, *q), put_strides(a.k_strides, *k), put_strides(a.v_strides, *v);
  put_strides(a.out_strides, *out), put_strides(a.dout_strides, *dout);
  a.lse_strides[0] = lse->stride(0), a.lse_strides[1] = lse->stride(1);
  a.B = s.B, a.Hq = s.Hq, a.Hkv = s.Hkv, a.Nq = s.Nq, a.Nk = s.Nk, a.d = s.d;
  a.causal = causal;
  const int code = on_device(s.dev.index(), [&](void* st) { return (s.fp8 ? abi.attn_bwd_fp8 : abi.attn_bwd_bf16)(&a, st); });
  if (code) return failed(code, "attn_bwd");
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(dq)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(dk)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(dv)));
  return r;
}

// ---- GEMM -------------------------------------------------------------------------------------------------------
bool small_int(PyObject* o, long& out) {
  if (!PyLong_CheckExact(o)) return false;  // no bool
  out = PyLong_AsLong(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return out >= 1 && out <= (1 << 20);
}

// A float32 scale of one element or of `size` (then contiguous, aligned for the kernels' vector loads).
bool gemm_scale(PyObject* o, int64_t size, const at::Device& dev, uintptr_t unit, const float*& ptr, int32_t& vec) {
  const at::Tensor* t = tensor_of(o);
  if (!t || t->scalar_type() != at::kFloat || t->device() != dev) return false;
  const int64_t n = t->numel();
  if (n != 1 && n != size) return false;
  vec = n > 1 && size > 1;
  if (n > 1 && (!t->is_contiguous() || !aligned(t->data_ptr(), unit))) return false;
  ptr = t->const_data_ptr<float>();
  return true;
}

bool mx_scale(PyObject* o, int64_t rows, int64_t k, const at::Device& dev, const void*& ptr) {
  const at::Tensor* t = tensor_of(o);
  if (!t || t->scalar_type() != at::kByte || t->dim() != 2 || t->size(0) != rows || t->size(1) != k / 32 ||
      t->device() != dev || !t->is_contiguous() || !aligned(t->data_ptr(), 4))
    return false;
  ptr = t->data_ptr();
  return true;
}

PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { A, B, OUT, BK, STAGES, GROUP_M, MIN_BLOCKS, BN, FRAG, TMA, SPEC, PERSIST, MAXNREG, SA, SB, OUT_DTYPE, ACT,
         STORE_PRE, PRE, A_TRANS, B_TRANS, ACCUM, SA_MX, OUT_MX, SB_MX, PAIR, COUNT };
  static const auto names = interned<COUNT>(
      {"a", "b", "out", "bk", "stages", "group_m", "min_blocks", "bn", "frag_pipe", "tma", "warp_spec", "persistent",
       "setmaxnreg", "scale_a", "scale_b", "out_dtype", "act", "store_pre", "pre", "a_trans", "b_trans", "accum",
       "a_scale_mx", "out_mx", "b_scale_mx", "cta_pair"});
  Params<COUNT> p;
  if (!bound || !p.read(names, args, nargs, kwnames)) return declined();
  const at::Tensor *a = tensor_of(p.v[A]), *b = tensor_of(p.v[B]);
  if (!a || !b || a->dim() != 2 || b->dim() != 2) return declined();
  const at::ScalarType dt = a->scalar_type();
  const bool fp8 = dt == at::kFloat8_e4m3fn;
  if ((!fp8 && dt != at::kBFloat16 && dt != at::kHalf) || b->scalar_type() != dt) return declined();
  const at::Device dev = a->device();
  if (!dev.is_cuda() || b->device() != dev || !device_ok(dev.index())) return declined();
  if (!a->is_contiguous() || !b->is_contiguous() || !aligned(a->data_ptr(), 16) || !aligned(b->data_ptr(), 16))
    return declined();
  bool a_trans, b_trans, store_pre, accum, out_mx, pair;
  if (!p.flag(A_TRANS, false, a_trans) || !p.flag(B_TRANS, false, b_trans) || !p.flag(STORE_PRE, false, store_pre) ||
      !p.flag(ACCUM, false, accum) || !p.flag(OUT_MX, false, out_mx) || !p.flag(PAIR, false, pair))
    return declined();
  const int64_t m = a->size(a_trans ? 1 : 0), k = a->size(a_trans ? 0 : 1);
  const int64_t n = b->size(b_trans ? 1 : 0), kb = b->size(b_trans ? 0 : 1);
  if (kb != k || ((a_trans || b_trans) && fp8) || m < 1 || n < 1 || k < 1) return declined();
  if (m > INT32_MAX / 2 || n > INT32_MAX / 2 || k > INT32_MAX / 2) return declined();
  long bk = fp8 ? 128 : 64, bn = 128, group_m = 0;
  if (p.given(BK) && !small_int(p.v[BK], bk)) return declined();
  if (p.v[BN] && (!small_int(p.v[BN], bn) || (bn != 128 && bn != 256))) return declined();
  if (p.given(GROUP_M) && !small_int(p.v[GROUP_M], group_m)) return declined();
  if (m % 128 || n % bn || k % bk || k % (fp8 ? 128 : 64)) return declined();
  int act = 0;
  if (p.v[ACT]) {
    if (!PyUnicode_Check(p.v[ACT])) return declined();
    if (PyUnicode_CompareWithASCIIString(p.v[ACT], "gelu") == 0)
      act = 1;
    else if (PyUnicode_CompareWithASCIIString(p.v[ACT], "dgelu") == 0)
      act = 2;
    else if (PyUnicode_GET_LENGTH(p.v[ACT]) != 0)
      return declined();
  }
  if ((store_pre && act != 1) || (accum && !p.given(OUT))) return declined();
  at::ScalarType odt = dt;
  at::Tensor out;
  if (p.given(OUT)) {
    const at::Tensor* o = tensor_of(p.v[OUT]);
    if (!o || o->dim() != 2 || o->size(0) != m || o->size(1) != n || !o->is_contiguous() || o->device() != dev ||
        !aligned(o->data_ptr(), 16))
      return declined();
    odt = o->scalar_type();
    out = *o;
  } else if (fp8) {
    odt = at::kBFloat16;
    if (p.v[OUT_DTYPE]) {
      if (!THPDtype_Check(p.v[OUT_DTYPE])) return declined();
      odt = reinterpret_cast<THPDtype*>(p.v[OUT_DTYPE])->scalar_type;
    }
  }
  if ((odt != at::kBFloat16 && odt != at::kHalf) || (!fp8 && odt != dt)) return declined();
  const float *scale_a = nullptr, *scale_b = nullptr;
  int32_t row_scale = 0, col_scale = 0;
  if (p.given(SA) && !gemm_scale(p.v[SA], m, dev, 8, scale_a, row_scale)) return declined();
  if (p.given(SB) && !gemm_scale(p.v[SB], n, dev, 16, scale_b, col_scale)) return declined();
  if (!fp8) {  // one-element scales apply to fp8 inputs only
    if (!row_scale) scale_a = nullptr;
    if (!col_scale) scale_b = nullptr;
  }
  const void *sa_mx = nullptr, *sb_mx = nullptr, *pre_in = nullptr;
  if ((p.given(SA_MX) || p.given(SB_MX)) && !fp8) return declined();
  if (p.given(SA_MX) && !mx_scale(p.v[SA_MX], m, k, dev, sa_mx)) return declined();
  if (p.given(SB_MX) && !mx_scale(p.v[SB_MX], n, k, dev, sb_mx)) return declined();
  if (act == 2) {
    const at::Tensor* pre = tensor_of(p.v[PRE]);
    if (!pre || pre->dim() != 2 || pre->size(0) != m || pre->size(1) != n || pre->scalar_type() != odt ||
        pre->device() != dev || !pre->is_contiguous() || !aligned(pre->data_ptr(), 16))
      return declined();
    pre_in = pre->data_ptr();
  }
  int cta_pair = 0;
  if (p.given(PAIR)) cta_pair = pair ? 1 : 2;

  if (!out.defined()) out = empty({m, n}, odt, dev);
  at::Tensor pre_out, q_mx, s_mx, workspace;
  if (store_pre) pre_out = empty({m, n}, odt, dev);
  if (out_mx) {
    q_mx = empty({m, n}, at::kFloat8_e4m3fn, dev);
    s_mx = empty({m, n / 32}, at::kByte, dev);
  }
  auto fill = [&](auto& g) {
    g.a = a->data_ptr(), g.b = b->data_ptr(), g.out = out.data_ptr();
    g.m = m, g.n = n, g.k = k;
    g.scale_a = scale_a, g.scale_b = scale_b, g.scale_a_rows = row_scale, g.scale_b_cols = col_scale;
    g.accum = accum, g.act = act;
    g.pre_out = store_pre ? pre_out.data_ptr() : nullptr, g.pre_in = pre_in;
    g.q_mx = out_mx ? q_mx.data_ptr() : nullptr, g.s_mx = out_mx ? s_mx.data_ptr() : nullptr;
    g.cta_pair = cta_pair, g.group_m = static_cast<int32_t>(group_m);
  };
  int code;
  if (fp8) {
    wk_gemm_mx_args g = {};
    fill(g);
    g.a_scale_mx = sa_mx, g.b_scale_mx = sb_mx;
    g.out_f16 = odt == at::kHalf;
    g.workspace_bytes = abi.gemm_mxfp8_workspace_bytes(g.m, g.n, g.k);
    workspace = empty({g.workspace_bytes}, at::kByte, dev);
    g.workspace = workspace.data_ptr();
    code = on_device(dev.index(), [&](void* st) { return abi.gemm_mxfp8(&g, st); });
  } else {
    wk_gemm16_args g = {};
    fill(g);
    g.f16 = dt == at::kHalf, g.a_trans = a_trans, g.b_trans = b_trans;
    code = on_device(dev.index(), [&](void* st) { return abi.gemm_16bit(&g, st); });
  }
  if (code) return failed(code, fp8 ? "gemm (fp8)" : "gemm (16-bit)");
  PyObject* o = p.given(OUT) ? Py_NewRef(p.v[OUT]) : THPVariable_Wrap(std::move(out));
  if (act != 1 && !out_mx) return o;
  PyObject* r = PyTuple_New(1 + (act == 1) + 2 * out_mx);
  Py_ssize_t at = 0;
  PyTuple_SET_ITEM(r, at++, o);
  if (act == 1) PyTuple_SET_ITEM(r, at++, store_pre ? THPVariable_Wrap(std::move(pre_out)) : Py_NewRef(Py_None));
  if (out_mx) {
    PyTuple_SET_ITEM(r, at++, THPVariable_Wrap(std::move(q_mx)));
    PyTuple_SET_ITEM(r, at++, THPVariable_Wrap(std::move(s_mx)));
  }
  return r;
}

PyObject* quantize_mx(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { X, Q, S, COUNT };
  static const auto names = interned<COUNT>({"x", "q", "s"});
  Params<COUNT> p;
  if (!bound || !p.read(names, args, nargs, kwnames)) return declined();
  const at::Tensor* x = tensor_of(p.v[X]);
  if (!x || x->dim() != 2 || (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kFloat)) return declined();
  const at::Device dev = x->device();
  const int64_t m = x->size(0), k = x->size(1);
  if (!dev.is_cuda() || !device_ok(dev.index()) || m < 1 || k < 32 || k % 32 || x->stride(1) != 1 ||
      (m > 1 && x->stride(0) % 8))
    return declined();
  at::Tensor q, s;
  if (p.given(Q)) {
    const at::Tensor* t = tensor_of(p.v[Q]);
    if (!t || t->sizes() != x->sizes() || t->scalar_type() != at::kFloat8_e4m3fn || !t->is_contiguous() ||
        t->device() != dev)
      return declined();
    q = *t;
  }
  if (p.given(S)) {
    const at::Tensor* t = tensor_of(p.v[S]);
    if (!t || t->dim() != 2 || t->size(0) != m || t->size(1) != k / 32 || t->scalar_type() != at::kByte ||
        !t->is_contiguous() || t->device() != dev)
      return declined();
    s = *t;
  }
  if (!q.defined()) q = empty({m, k}, at::kFloat8_e4m3fn, dev);
  if (!s.defined()) s = empty({m, k / 32}, at::kByte, dev);
  const int dtype = x->scalar_type() == at::kBFloat16 ? WK_BF16 : WK_F32;
  const int64_t ld = m > 1 ? x->stride(0) : std::max<int64_t>(k, 8);
  const int code = on_device(dev.index(), [&](void* st) {
    return abi.quantize_mx(x->data_ptr(), dtype, m, k, ld, q.data_ptr(), s.data_ptr(), st);
  });
  if (code) return failed(code, "quantize_mx");
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, p.given(Q) ? Py_NewRef(p.v[Q]) : THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(r, 1, p.given(S) ? Py_NewRef(p.v[S]) : THPVariable_Wrap(std::move(s)));
  return r;
}

// ---- rotation of queries and keys -------------------------------------------------------------------------------
int rope_dtype(at::ScalarType t) {
  return t == at::kBFloat16 ? WK_BF16 : t == at::kHalf ? WK_F16 : t == at::kFloat ? WK_F32 : -1;
}

// [B, H, N, d] rows the kernels can address: last stride 1, base and other strides multiples of `unit` bytes.
bool rope_rows(const at::Tensor& t, int64_t unit) {
  const int64_t size = t.element_size();
  for (int i = 0; i < 3; ++i)
    if (t.stride(i) * size % unit) return false;
  return t.stride(3) == 1 && aligned(t.data_ptr(), unit);
}

// No two elements share memory: every stride spans what the smaller ones reach.
bool apart(const at::Tensor& t) {
  int64_t span = 1, last = 0;
  for (;;) {  // the dimensions by their strides, smallest first
    int next = -1, equal = 0;
    for (int i = 0; i < 4; ++i) {
      if (t.size(i) <= 1 || t.stride(i) <= last) continue;
      if (next < 0 || t.stride(i) < t.stride(next)) next = i, equal = 0;
      else if (t.stride(i) == t.stride(next)) ++equal;
    }
    for (int i = 0; i < 4; ++i) equal += t.size(i) > 1 && t.stride(i) <= 0;
    if (equal) return false;
    if (next < 0) return true;
    if (t.stride(next) < span) return false;
    last = t.stride(next);
    span = last * t.size(next);
  }
}

// Whether two tensors of four dimensions share a byte; also true where that takes long to tell.  As `overlap` of
// utils/__init__.py, where the method stands.
struct Overlap {
  int64_t stride[8], most[8], rest[9];  // terms of the sum: stride, number of values less one; what the later ones reach
  int terms = 0, steps = 4096;
  int64_t target;
  void add(const at::Tensor& t, bool back) {
    const int64_t size = t.element_size();
    for (int i = 0; i < 4; ++i) {
      const int64_t st = t.stride(i) * size, n = t.size(i) - 1;
      if (!n || !st) continue;
      if (back) target += st * n;
      int at = 0;
      while (at < terms && stride[at] > st) ++at;
      if (at == terms || stride[at] != st) {
        for (int j = terms++; j > at; --j) stride[j] = stride[j - 1], most[j] = most[j - 1];
        stride[at] = st, most[at] = 0;
      }
      most[at] += n;
    }
  }
  bool reached(int i, int64_t low, int64_t high) {
    if (--steps < 0) return true;
    if (i == terms) return low <= 0 && 0 <= high;
    const int64_t need = low - rest[i + 1], first = need > 0 ? (need + stride[i] - 1) / stride[i] : 0;
    const int64_t last = high < 0 ? -1 : std::min(most[i], high / stride[i]);
    for (int64_t x = first; x <= last; ++x)
      if (reached(i + 1, low - x * stride[i], high - x * stride[i])) return true;
    return false;
  }
  Overlap(const at::Tensor& a, const at::Tensor& b)
      : target(static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr())) {
    add(a, false), add(b, true);
    rest[terms] = 0;
    for (int i = terms - 1; i >= 0; --i) rest[i] = rest[i + 1] + stride[i] * most[i];
  }
};
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  Overlap o(a, b);
  return o.reached(0, o.target - static_cast<int64_t>(a.element_size()) + 1, o.target + static_cast<int64_t>(b.element_size()) - 1);
}

// The position axis of every pair, two bits each, and the number of axes (0: positions have no axis).
bool rope_axes(PyObject* sections, bool cycle, int64_t pairs, uint64_t (&words)[4], int64_t& axes) {
  axes = 0;
  if (!sections || sections == Py_None) return true;
  if (!PyTuple_Check(sections)) return false;
  axes = PyTuple_GET_SIZE(sections);
  if (axes < 1 || axes > 4) return false;
  long n[4] = {}, sum = 0;
  for (int a = 0; a < axes; ++a) {
    PyObject* o = PyTuple_GET_ITEM(sections, a);
    if (!PyLong_CheckExact(o)) return false;
    n[a] = PyLong_AsLong(o);
    if (n[a] < 0 || n[a] > pairs) {
      PyErr_Clear();
      return false;
    }
    sum += n[a];
    if (cycle && a && n[a] && a + axes * (n[a] - 1) >= pairs) return false;
  }
  if (sum != pairs) return false;
  int a = 0;
  for (int64_t j = 0, used = 0; j < pairs; ++j) {
    uint64_t axis;
    if (cycle) {
      axis = j < axes * n[j % axes] ? j % axes : 0;
    } else {
      while (used == n[a]) ++a, used = 0;
      axis = a, ++used;
    }
    words[j / 32] |= axis << (2 * (j % 32));
  }
  return true;
}

// What all rotation calls share: q, k, positions, inv_freq and how pairs are formed.
bool rope_inputs(const at::Tensor* q, PyObject* k_obj, const at::Tensor* k, const at::Tensor* pos, const at::Tensor* freq,
                 PyObject* sections, bool cycle, bool interleaved, wk_rope_args& a) {
  if (!q || !pos || !freq || (!k && k_obj != Py_None) || q->dim() != 4) return false;
  a.dtype = rope_dtype(q->scalar_type());
  const at::Device dev = q->device();
  if (a.dtype < 0 || !dev.is_cuda() || !device_ok(dev.index()) || !rope_rows(*q, 16)) return false;
  const int64_t B = q->size(0), Hq = q->size(1), N = q->size(2), d = q->size(3);
  if (B < 1 || Hq < 1 || N < 1 || B > INT32_MAX / 4 / N || Hq > (1 << 18) || d % 16 || d < 32 || d > 256) return false;
  if (k && (k->dim() != 4 || k->size(0) != B || k->size(1) < 1 || k->size(1) > (1 << 18) || k->size(2) != N || k->size(3) != d ||
            k->scalar_type() != q->scalar_type() || k->device() != dev || !rope_rows(*k, 16)))
    return false;
  const at::ScalarType ft = freq->scalar_type(), pt = pos->scalar_type();
  if (freq->dim() != 1 || (ft != at::kFloat && ft != at::kDouble) || freq->device() != dev || !freq->is_contiguous())
    return false;
  const int64_t pairs = freq->size(0);
  int64_t axes;
  if (pairs < 8 || pairs % 8 || 2 * pairs > d || !rope_axes(sections, cycle, pairs, a.axis_map, axes)) return false;
  if ((pt != at::kInt && pt != at::kLong) || pos->device() != dev) return false;
  const int lead = axes ? 1 : 0;
  const int64_t dims = pos->dim() - lead;
  if (dims < 1 || dims > 2 || (lead && pos->size(0) != axes) || pos->size(-1) != N || (dims == 2 && pos->size(lead) != B))
    return false;
  a.position_strides[0] = lead ? pos->stride(0) : 0;
  a.position_strides[1] = dims == 2 ? pos->stride(lead) : 0;
  a.position_strides[2] = pos->stride(-1);
  a.positions = pos->data_ptr(), a.inv_freq = freq->data_ptr();
  a.position_int64 = pt == at::kLong, a.inv_freq_f64 = ft == at::kDouble;
  a.interleaved = interleaved;
  a.q = q->data_ptr(), a.k = k ? k->data_ptr() : nullptr;
  put_strides(a.q_strides, *q);
  if (k) put_strides(a.k_strides, *k);
  a.B = B, a.N = N, a.Hq = Hq, a.Hk = k ? k->size(1) : 0, a.d = d, a.rot = 2 * pairs;
  return true;
}

bool rope_weights(PyObject* q_obj, PyObject* k_obj, PyObject* eps, const at::Tensor* q, const at::Tensor* k, wk_rope_args& a) {
  const at::Tensor *wq = tensor_of(q_obj), *wk = tensor_of(k_obj);
  if (!wq || (k && !wk)) return false;
  for (const at::Tensor* w : {wq, k ? wk : wq})
    if (w->dim() != 1 || w->size(0) != a.d || w->scalar_type() != wq->scalar_type() || w->device() != q->device() ||
        !w->is_contiguous() || !aligned(w->data_ptr(), 16))
      return false;
  a.w_dtype = rope_dtype(wq->scalar_type());
  if (a.w_dtype < 0) return false;
  a.q_weight = wq->data_ptr(), a.k_weight = k ? wk->data_ptr() : nullptr;
  double e = 1e-6;
  if (eps) {
    if (!PyFloat_Check(eps)) return false;
    e = PyFloat_AS_DOUBLE(eps);
  }
  a.eps = static_cast<float>(e);
  return e >= 0.0;
}

at::Tensor like(const at::Tensor& x, at::ScalarType dtype) {  // the memory layout of x
  if (x.is_non_overlapping_and_dense()) return empty_strided(x.sizes(), x.strides(), dtype, x.device());
  return at::empty_like(x, x.options().dtype(dtype));
}

PyObject* pair_of(PyObject* a, PyObject* b) {
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, a), PyTuple_SET_ITEM(r, 1, b);
  return r;
}

PyObject* rope_forward(const at::Tensor* q, const at::Tensor* k, PyObject* q_out, PyObject* k_out,
                       PyObject* q_descale, PyObject* k_descale, wk_rope_args& a, const char* what) {
  auto given = [](PyObject* o) { return o && o != Py_None; };
  const bool fp8 = given(q_descale);
  if (given(k_descale) != (fp8 && k) || (!k && given(k_out))) return declined();
  const at::ScalarType dtype = fp8 ? at::kFloat8_e4m3fn : q->scalar_type();
  if (fp8) {
    const at::Tensor *sq = tensor_of(q_descale), *sk = k ? tensor_of(k_descale) : sq;
    for (const at::Tensor* s : {sq, sk})
      if (!s || s->dim() != 2 || s->size(0) != a.B || s->size(1) < 1 || s->size(1) != sq->size(1) ||
          s->scalar_type() != at::kFloat || s->device() != q->device() || !s->is_contiguous())
        return declined();
    a.Hkv = static_cast<int32_t>(sq->size(1));
    if (a.Hq % a.Hkv || (k && a.Hk != a.Hkv)) return declined();
    a.q_descale = sq->const_data_ptr<float>(), a.k_descale = k ? sk->const_data_ptr<float>() : nullptr;
  }
  at::Tensor outs[2];
  for (int i = 0; i < 2; ++i) {
    const at::Tensor* x = i ? k : q;
    PyObject* o = i ? k_out : q_out;
    if (!x) continue;
    if (given(o)) {
      const at::Tensor* t = tensor_of(o);
      if (!t || t->dim() != 4 || t->sizes() != x->sizes() || t->scalar_type() != dtype || t->device() != x->device() ||
          !rope_rows(*t, fp8 ? 8 : 16) || !apart(*t))
        return declined();
      const bool same = t->data_ptr() == x->data_ptr() && t->strides() == x->strides() && dtype == x->scalar_type();
      const at::Tensor* other = i ? q : k;
      if ((!same && overlap(*t, *x)) || (other && overlap(*t, *other)) || (i && outs[0].defined() && overlap(*t, outs[0])))
        return declined();
      outs[i] = *t;
    }
  }
  for (int i = 0; i < 2; ++i)
    if ((i ? k : q) && !outs[i].defined()) outs[i] = like(i ? *k : *q, dtype);
  a.q_out = outs[0].data_ptr();
  put_strides(a.q_out_strides, outs[0]);
  if (k) {
    a.k_out = outs[1].data_ptr();
    put_strides(a.k_out_strides, outs[1]);
  }
  const int code = on_device(q->device().index(), [&](void* st) { return abi.rope(&a, st); });
  if (code) return failed(code, what);
  return pair_of(given(q_out) ? Py_NewRef(q_out) : THPVariable_Wrap(std::move(outs[0])),
                 !k ? Py_NewRef(Py_None) : given(k_out) ? Py_NewRef(k_out) : THPVariable_Wrap(std::move(outs[1])));
}

PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, K, POS, FREQ, SECTIONS, CYCLE, INTER, INVERSE, Q_OUT, K_OUT, QD, KD, COUNT };
  static const auto names = interned<COUNT>({"q", "k", "positions", "inv_freq", "sections", "cycle", "interleaved", "inverse",
                                             "q_out", "k_out", "q_descale", "k_descale"});
  Params<COUNT> p;
  bool cycle, interleaved, inverse;
  if (!bound || !p.read(names, args, nargs, kwnames) || !p.flag(CYCLE, false, cycle) ||
      !p.flag(INTER, false, interleaved) || !p.flag(INVERSE, false, inverse))
    return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *k = tensor_of(p.v[K]);
  wk_rope_args a = {};
  if (!rope_inputs(q, p.v[K], k, tensor_of(p.v[POS]), tensor_of(p.v[FREQ]), p.v[SECTIONS], cycle, interleaved, a))
    return declined();
  a.inverse = inverse;
  return rope_forward(q, k, p.v[Q_OUT], p.v[K_OUT], p.v[QD], p.v[KD], a, "rope");
}

PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, K, WQ, WK, POS, FREQ, EPS, SECTIONS, CYCLE, INTER, Q_OUT, K_OUT, QD, KD, COUNT };
  static const auto names = interned<COUNT>({"q", "k", "q_weight", "k_weight", "positions", "inv_freq", "eps", "sections",
                                             "cycle", "interleaved", "q_out", "k_out", "q_descale", "k_descale"});
  Params<COUNT> p;
  bool cycle, interleaved;
  if (!bound || !p.read(names, args, nargs, kwnames) || !p.flag(CYCLE, false, cycle) || !p.flag(INTER, false, interleaved))
    return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *k = tensor_of(p.v[K]);
  wk_rope_args a = {};
  if (!rope_inputs(q, p.v[K], k, tensor_of(p.v[POS]), tensor_of(p.v[FREQ]), p.v[SECTIONS], cycle, interleaved, a) ||
      !rope_weights(p.v[WQ], p.v[WK], p.v[EPS], q, k, a))
    return declined();
  return rope_forward(q, k, p.v[Q_OUT], p.v[K_OUT], p.v[QD], p.v[KD], a, "qk_norm_rope");
}

PyObject* qk_norm_rope_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { DQ, DK, Q, K, WQ, WK, POS, FREQ, EPS, SECTIONS, CYCLE, INTER, COUNT };
  static const auto names = interned<COUNT>({"dq_out", "dk_out", "q", "k", "q_weight", "k_weight", "positions", "inv_freq",
                                             "eps", "sections", "cycle", "interleaved"});
  Params<COUNT> p;
  bool cycle, interleaved;
  if (!bound || !p.read(names, args, nargs, kwnames) || !p.flag(CYCLE, false, cycle) || !p.flag(INTER, false, interleaved))
    return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *k = tensor_of(p.v[K]), *dq = tensor_of(p.v[DQ]), *dk = tensor_of(p.v[DK]);
  wk_rope_args a = {};
  if (!rope_inputs(q, p.v[K], k, tensor_of(p.v[POS]), tensor_of(p.v[FREQ]), p.v[SECTIONS], cycle, interleaved, a) ||
      !rope_weights(p.v[WQ], p.v[WK], p.v[EPS], q, k, a))
    return declined();
  auto grad_ok = [](const at::Tensor* g, const at::Tensor& x) {
    return g && g->dim() == 4 && g->sizes() == x.sizes() && g->scalar_type() == x.scalar_type() && g->device() == x.device() &&
           rope_rows(*g, 16);
  };
  if (!grad_ok(dq, *q) || (k ? !grad_ok(dk, *k) : p.v[DK] != Py_None)) return declined();
  const at::Device dev = q->device();
  const at::ScalarType wt = tensor_of(p.v[WQ])->scalar_type();
  at::Tensor gq = like(*q, q->scalar_type()), gwq = empty({a.d}, wt, dev), gk, gwk;
  a.dq_out = dq->data_ptr(), a.q_out = gq.data_ptr(), a.dq_weight = gwq.data_ptr();
  put_strides(a.dq_out_strides, *dq), put_strides(a.q_out_strides, gq);
  if (k) {
    gk = like(*k, k->scalar_type()), gwk = empty({a.d}, wt, dev);
    a.dk_out = dk->data_ptr(), a.k_out = gk.data_ptr(), a.dk_weight = gwk.data_ptr();
    put_strides(a.dk_out_strides, *dk), put_strides(a.k_out_strides, gk);
  }
  {
    const c10::cuda::OptionalCUDAGuard guard(dev);
    a.workspace_bytes = abi.qk_norm_rope_bwd_workspace_bytes(a.d);
  }
  at::Tensor workspace = empty({a.workspace_bytes}, at::kByte, dev);
  a.workspace = workspace.data_ptr();
  const int code = on_device(dev.index(), [&](void* st) { return abi.qk_norm_rope_bwd(&a, st); });
  if (code) return failed(code, "qk_norm_rope_bwd");
  PyObject* r = PyTuple_New(4);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(gq)));
  PyTuple_SET_ITEM(r, 1, k ? THPVariable_Wrap(std::move(gk)) : Py_NewRef(Py_None));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(gwq)));
  PyTuple_SET_ITEM(r, 3, k ? THPVariable_Wrap(std::move(gwk)) : Py_NewRef(Py_None));
  return r;
}

PyObject* attn_fwd_shared_prefix(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, KP, VP, K, V, QD, KD, VD, KPD, VPD, CAUSAL, SCALE, OUT, LSE, USED, NATURAL, COUNT };
  static const auto names = interned<COUNT>({"q", "k_prefix", "v_prefix", "k", "v", "q_descale", "k_descale", "v_descale",
                                             "k_prefix_descale", "v_prefix_descale", "causal", "softmax_scale", "out",
                                             "return_lse", "seqused_k", "lse_natural"});
  Params<COUNT> p;
  AttnShape s, prefix;
  if (!bound || !p.read(names, args, nargs, kwnames)) return declined();
  const at::Tensor *q = tensor_of(p.v[Q]), *kp = tensor_of(p.v[KP]), *vp = tensor_of(p.v[VP]);
  const at::Tensor *k = tensor_of(p.v[K]), *v = tensor_of(p.v[V]);
  if (!attn_shape(q, k, v, s) || !kp || !vp || kp->dim() != 4 || kp->sizes() != vp->sizes() || kp->size(0) != 1 ||
      kp->size(1) != s.Hkv || kp->size(3) != s.d || kp->size(2) < 1 || kp->size(2) > INT32_MAX / 2)
    return declined();
  for (const at::Tensor* x : {kp, vp})
    if (x->scalar_type() != q->scalar_type() || x->device() != s.dev || !tma_direct(*x)) return declined();
  for (const at::Tensor* x : {q, kp, vp, k, v})
    if (x->stride(0) < 1 || x->stride(1) < 1 || x->stride(2) < 1) return declined();
  prefix = s, prefix.B = 1;
  wk_attn_prefix_args a = {};
  if (s.fp8) {
    if (!descale(p.v[QD], s, a.q_descale) || !descale(p.v[KD], s, a.k_descale) || !descale(p.v[VD], s, a.v_descale) ||
        !descale(p.v[KPD], prefix, a.k_prefix_descale) || !descale(p.v[VPD], prefix, a.v_prefix_descale))
      return declined();
  } else if (p.given(QD) || p.given(KD) || p.given(VD) || p.given(KPD) || p.given(VPD)) {
    return declined();
  }
  bool with_lse, causal, natural;
  if (!softmax_scale_of(p.v[SCALE], s.d, a.softmax_scale) || !p.flag(LSE, true, with_lse) ||
      !p.flag(CAUSAL, false, causal) || !p.flag(NATURAL, false, natural))
    return declined();
  if (p.given(USED)) {
    const at::Tensor* used = tensor_of(p.v[USED]);
    if (!used || used->dim() != 1 || used->size(0) != s.B || used->scalar_type() != at::kInt || used->device() != s.dev ||
        !used->is_contiguous())
      return declined();
    a.seqused_k = used->const_data_ptr<int32_t>();
  }
  {
    const c10::cuda::OptionalCUDAGuard guard(s.dev);
    a.workspace_bytes = abi.attn_prefix_workspace_bytes(s.B, s.Hq, s.Hkv, s.Nq, kp->size(2), s.Nk, s.d);
  }
  if (!a.workspace_bytes) return declined();
  at::Tensor out, lse;
  if (p.given(OUT)) {
    const at::Tensor* o = tensor_of(p.v[OUT]);
    if (!o || o->dim() != 4 || o->sizes() != q->sizes() || o->scalar_type() != at::kBFloat16 || o->device() != s.dev ||
        o->stride(3) != 1 || !aligned(o->data_ptr(), 8))
      return declined();
    for (int i = 0; i < 3; ++i)
      if (o->stride(i) < 1 || o->stride(i) % 4) return declined();
    if (!apart(*o)) return declined();
    for (const at::Tensor* x : {q, kp, vp, k, v}) {
      const bool same = x == q && o->data_ptr() == q->data_ptr() && o->strides() == q->strides() && !s.fp8;
      if (!same && overlap(*o, *x)) return declined();
    }
    out = *o;
  } else {
    out = like(*q, at::kBFloat16);
  }
  at::Tensor workspace = empty({a.workspace_bytes}, at::kByte, s.dev);
  if (with_lse) {
    lse = empty({s.B, s.Hq, s.Nq}, at::kFloat, s.dev);
    a.lse = lse.mutable_data_ptr<float>();
    a.lse_strides[0] = s.Hq * s.Nq, a.lse_strides[1] = s.Nq;
  }
  a.q = q->data_ptr(), a.k_prefix = kp->data_ptr(), a.v_prefix = vp->data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr();
  a.out = out.data_ptr(), a.workspace = workspace.data_ptr();
  put_strides(a.q_strides, *q), put_strides(a.k_prefix_strides, *kp), put_strides(a.v_prefix_strides, *vp);
  put_strides(a.k_strides, *k), put_strides(a.v_strides, *v), put_strides(a.out_strides, out);
  a.B = s.B, a.Hq = s.Hq, a.Hkv = s.Hkv, a.Nq = s.Nq, a.P = kp->size(2), a.S = s.Nk, a.d = s.d;
  a.fp8 = s.fp8, a.causal = causal, a.lse_natural = natural;
  const int code = on_device(s.dev.index(), [&](void* st) { return abi.attn_prefix(&a, st); });
  if (code) return failed(code, "attn_fwd_shared_prefix");
  return pair_of(p.given(OUT) ? Py_NewRef(p.v[OUT]) : THPVariable_Wrap(std::move(out)),
                 with_lse ? THPVariable_Wrap(std::move(lse)) : Py_NewRef(Py_None));
}

// ---- prepared launches --------------------------------------------------------------------------------------------
// launch(entry, args, device) -> code: calls the C ABI function at address `entry` with the argument block at address
// `args` on the current stream of the device.
PyObject* launch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "launch(entry, args, device)");
    return nullptr;
  }
  void* entry = PyLong_AsVoidPtr(args[0]);
  void* block = PyLong_AsVoidPtr(args[1]);
  const long dev = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  return PyLong_FromLong(on_device(static_cast<int>(dev), [&](void* st) {
    return reinterpret_cast<int (*)(const void*, void*)>(entry)(block, st);
  }));
}

// block_flags(device, nbytes) -> tensor: the forward's flag scratch of the device's current stream.
PyObject* py_block_flags(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "block_flags(device, nbytes)");
    return nullptr;
  }
  const long dev = PyLong_AsLong(args[0]);
  const long long nbytes = PyLong_AsLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  return THPVariable_Wrap(
      block_flags(static_cast<int>(dev), c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(), nbytes));
}

// bind({name: address}): the C ABI functions of the loaded library.
PyObject* bind(PyObject*, PyObject* table) {
  if (!PyDict_Check(table)) {
    PyErr_SetString(PyExc_TypeError, "bind() takes a dict of addresses");
    return nullptr;
  }
  for (const auto& sym : kSymbols) {
    PyObject* o = PyDict_GetItemString(table, sym.name);
    void* ptr = o ? PyLong_AsVoidPtr(o) : nullptr;
    if (!ptr) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s is missing", sym.name);
      return nullptr;
    }
    *sym.slot = ptr;
  }
  bound = true;
  Py_RETURN_NONE;
}

// A C++ exception (an allocation that failed, a CUDA error) becomes the Python exception torch raises for it.
template <class F>
PyObject* guard(F call) {
  try {
    return call();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_Clear();
    PyErr_SetString(type ? type : PyExc_MemoryError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guard([&] { return F(self, args, nargs, kwnames); });
}
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded_plain(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  return guard([&] { return F(self, args, nargs); });
}

template <auto F>
PyCFunction as_method() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef methods[] = {
    {"attn_fwd", as_method<guarded<attn_fwd>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"attn_bwd", as_method<guarded<attn_bwd>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"gemm", as_method<guarded<gemm>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"quantize_mx", as_method<guarded<quantize_mx>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"rope", as_method<guarded<rope>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"qk_norm_rope", as_method<guarded<qk_norm_rope>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"qk_norm_rope_bwd", as_method<guarded<qk_norm_rope_bwd>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"attn_fwd_shared_prefix", as_method<guarded<attn_fwd_shared_prefix>>(), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"launch", as_method<guarded_plain<launch>>(), METH_FASTCALL, nullptr},
    {"block_flags", as_method<guarded_plain<py_block_flags>>(), METH_FASTCALL, nullptr},
    {"bind", bind, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
