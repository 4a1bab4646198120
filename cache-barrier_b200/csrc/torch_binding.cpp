// Native torch layer of the decoder-layer operators: checks tensors, allocates
// what the caller did not give, and calls the C ABI (include/cb200.h) on the
// tensors' device and torch's current stream.
//
// These calls run once per layer and token, and their kernels take a few
// microseconds; reading a tensor's shape, strides and type through Python and
// packing ctypes arguments took 11 to 18 us a call, here the whole call takes
// about 4 us, most of it the launch.
//
// The C functions' addresses come from the ctypes binding (init), so this module
// and the Python layer share one loaded library. Workspaces belong to the Python
// pool, which registers them here (set_workspace).
#include <ATen/ATen.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>
#include <unordered_map>
#include <vector>

#include "cb200.h"

namespace {

struct Api {
  decltype(&cb_add_rmsnorm_quant) add_rmsnorm_quant;
  decltype(&cb_quant_act_fp8_block) quant_act_fp8_block;
  decltype(&cb_fp8_block_gemm) fp8_block_gemm;
  decltype(&cb_fp8_block_gemm_dynamic) fp8_block_gemm_dynamic;
  decltype(&cb_paged_kv_append) paged_kv_append;
  decltype(&cb_paged_decode_attention) paged_decode_attention;
  decltype(&cb_workspace_bytes) workspace_bytes;
  decltype(&cb_stream_capture_id) stream_capture_id;
} api;
PyObject* py_check = nullptr;      // _lib.check(name, code): raises
PyObject* py_workspace = nullptr;  // (bytes, device index): makes the pool register a workspace of that size

// A Python exception is set: unwinds to the entry, which returns null.
struct Raised {};

[[noreturn]] void refuse(const std::string& message) {
  PyErr_SetString(PyExc_ValueError, message.c_str());
  throw Raised{};
}

void done(const char* name, int code) {
  if (code == CB_OK) return;
  PyObject* r = PyObject_CallFunction(py_check, "si", name, code);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed (cb_status %d)", name, code);
  throw Raised{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

// An optional tensor: null for None.
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

c10::Device gpu_of(const at::Tensor& t) {
  const c10::Device d = t.device();
  if (!d.is_cuda()) refuse("all tensors must be CUDA tensors (the kernels run only on the GPU)");
  return d;
}

template <typename... Ts>
void one_device(c10::Device d, const Ts*... ts) {
  const at::Tensor* all[] = {ts...};
  for (const at::Tensor* t : all)
    if (t && t->device() != d) refuse("all tensors must be on one device: all CUDA tensors, got " + t->device().str() + " and " + d.str());
}

int act_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return CB_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return CB_DTYPE_F16;
  refuse(std::string(name) + " must be float16 or bfloat16");
}

int float_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return CB_DTYPE_F32;
  if (t.scalar_type() == at::kBFloat16) return CB_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return CB_DTYPE_F16;
  refuse(std::string(name) + " must be float16, bfloat16 or float32");
}

bool is_fp8(const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte; }
bool inner(const at::Tensor& t) { return t.dim() > 0 && (t.stride(-1) == 1 || t.size(-1) <= 1); }
bool same_shape(const at::Tensor& a, const at::Tensor& b) { return a.sizes() == b.sizes(); }
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
float* fptr(const at::Tensor* t) { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }
int64_t groups(int64_t n) { return (n + 127) / 128; }

cb_stream_t current_stream(c10::Device d) {
  return reinterpret_cast<cb_stream_t>(c10::cuda::getCurrentCUDAStream(d.index()).stream());
}

// ---- workspaces ---------------------------------------------------------------
struct Key {
  int device;
  uint64_t stream, capture;  // capture: 0 outside a capture
  bool operator==(const Key& o) const { return device == o.device && stream == o.stream && capture == o.capture; }
};
struct KeyHash {
  size_t operator()(const Key& k) const { return std::hash<uint64_t>()((k.stream + k.capture * 0x9e3779b97f4a7c15ull) * 64 + k.device); }
};
struct Buffer {
  void* p;
  size_t bytes;
};
std::unordered_map<Key, Buffer, KeyHash> workspaces;

// The pool's workspace of the device, the stream and the capture that it is in, of at
// least `need` bytes.
Buffer workspace(c10::Device d, cb_stream_t stream, size_t need) {
  const Key key{d.index(), reinterpret_cast<uint64_t>(stream), api.stream_capture_id(stream)};
  auto it = workspaces.find(key);
  if (it == workspaces.end() || it->second.bytes < need) {
    PyObject* r = PyObject_CallFunction(py_workspace, "ni", static_cast<Py_ssize_t>(need), static_cast<int>(d.index()));
    if (!r) throw Raised{};
    Py_DECREF(r);
    it = workspaces.find(key);
    if (it == workspaces.end() || it->second.bytes < need) {
      PyErr_SetString(PyExc_RuntimeError, "the workspace pool registered no workspace");
      throw Raised{};
    }
  }
  return it->second;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* same(PyObject* given, const at::Tensor& t) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return wrap(t);
}

void count(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    throw Raised{};
  }
}

// ---- residual RMSNorm ---------------------------------------------------------
// (x, weight, eps, residual, mode, q, s, h) -> (q, s, h)
PyObject* add_rmsnorm_quant(PyObject* const* a, Py_ssize_t n) {
  count(n, 8);
  const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "weight");
  const double eps = PyFloat_AsDouble(a[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw Raised{};
  const at::Tensor* res = maybe(a[3], "residual");
  const char* mode_name = PyUnicode_Check(a[4]) ? PyUnicode_AsUTF8(a[4]) : "";
  const std::string mode_str = mode_name ? mode_name : "";
  int mode;
  if (mode_str == "int8") mode = CB_NORM_INT8;
  else if (mode_str == "fp8") mode = CB_NORM_FP8;
  else if (mode_str == "fp8_block") mode = CB_NORM_FP8_BLOCK;
  else refuse("mode must be one of ['fp8', 'fp8_block', 'int8']");
  const at::Tensor *q = maybe(a[5], "q"), *s = maybe(a[6], "s"), *h = maybe(a[7], "h");
  const c10::Device d = gpu_of(x);
  one_device(d, &w, res, q, s, h);
  if (x.dim() != 2 || !inner(x)) refuse("x must be [rows, H], contiguous along H");
  const int code = act_code(x, "x");
  const int64_t rows = x.size(0), H = x.size(1);
  if (w.dim() != 1 || w.size(0) != H || !inner(w)) refuse("weight must be a contiguous [H] tensor");
  if (res && (!same_shape(*res, x) || res->scalar_type() != x.scalar_type() || !inner(*res))) refuse("residual must be like x");
  if (!res && h) refuse("h is the sum with the residual: give one");
  if (h && (!same_shape(*h, x) || h->scalar_type() != x.scalar_type() || !inner(*h))) refuse("h must be like x");
  const at::ScalarType qt = mode == CB_NORM_INT8 ? at::kChar : at::kFloat8_e4m3fn;
  if (q && (!same_shape(*q, x) || q->scalar_type() != qt || !inner(*q)))
    refuse(mode == CB_NORM_INT8 ? "q must be int8 [rows, H], contiguous along H" : "q must be float8_e4m3fn [rows, H], contiguous along H");
  const bool block = mode == CB_NORM_FP8_BLOCK;
  if (s) {
    if (block && (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != rows || s->size(1) != groups(H) || !inner(*s)))
      refuse("s must be fp32 [rows, ceil(H / 128)], contiguous along the blocks");
    if (!block && (s->scalar_type() != at::kFloat || s->dim() != 1 || s->size(0) != rows)) refuse("s must be fp32 [rows]");
  }
  const c10::cuda::CUDAGuard guard(d);
  at::Tensor qn, sn, hn;
  if (!q) q = &(qn = at::empty({rows, H}, x.options().dtype(qt)));
  if (!s) s = &(sn = block ? at::empty({rows, groups(H)}, x.options().dtype(at::kFloat)) : at::empty({rows}, x.options().dtype(at::kFloat)));
  if (res && !h) h = &(hn = at::empty({rows, H}, x.options()));
  done("cb_add_rmsnorm_quant",
       api.add_rmsnorm_quant(x.data_ptr(), ptr(res), code, w.data_ptr(), float_code(w, "weight"), static_cast<float>(eps), rows, H,
                             x.stride(0), res ? res->stride(0) : 0, mode, q->data_ptr(), q->stride(0), fptr(s), s->stride(0), ptr(h),
                             h ? h->stride(0) : 0, current_stream(d)));
  PyObject* out = PyTuple_New(3);
  if (!out) throw Raised{};
  PyTuple_SET_ITEM(out, 0, same(a[5], *q));
  PyTuple_SET_ITEM(out, 1, same(a[6], *s));
  if (h) {
    PyTuple_SET_ITEM(out, 2, same(a[7], *h));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 2, Py_None);
  }
  return out;
}

// ---- block quantizer ----------------------------------------------------------
// q and s of a block-quantized a ([M, K] or [B, M, K]): checked, or allocated in qn and sn
void block_outputs(const at::Tensor& a, const at::Tensor*& q, const at::Tensor*& s, at::Tensor& qn, at::Tensor& sn) {
  const int64_t kb = groups(a.size(-1));
  if (q && (!same_shape(*q, a) || !is_fp8(*q) || !inner(*q))) refuse("q must be float8_e4m3fn like a, contiguous along K");
  if (s) {
    bool ok = s->dim() == a.dim() && s->scalar_type() == at::kFloat && inner(*s) && s->size(-1) == kb;
    for (int64_t i = 0; ok && i + 1 < a.dim(); ++i) ok = s->size(i) == a.size(i);
    if (!ok) refuse("s must be fp32 [.., M, ceil(K / 128)], contiguous along the blocks");
  }
  if (!q) q = &(qn = at::empty(a.sizes(), a.options().dtype(at::kFloat8_e4m3fn)));
  if (!s) {
    std::vector<int64_t> shape = a.sizes().vec();
    shape.back() = kb;
    s = &(sn = at::empty(shape, a.options().dtype(at::kFloat)));
  }
}

void act_rows(const at::Tensor& a) {
  if ((a.dim() != 2 && a.dim() != 3) || !inner(a)) refuse("a must be [M, K] or [B, M, K], contiguous along K");
}

// (a, q, s) -> (q, s)
PyObject* quant_act_fp8_block(PyObject* const* p, Py_ssize_t n) {
  count(n, 3);
  const at::Tensor& a = tensor(p[0], "a");
  const at::Tensor *q = maybe(p[1], "q"), *s = maybe(p[2], "s");
  const c10::Device d = gpu_of(a);
  one_device(d, q, s);
  act_rows(a);
  const int code = act_code(a, "a");
  const c10::cuda::CUDAGuard guard(d);
  at::Tensor qn, sn;
  block_outputs(a, q, s, qn, sn);
  const bool b = a.dim() == 3;
  done("cb_quant_act_fp8_block",
       api.quant_act_fp8_block(a.data_ptr(), code, b ? a.size(0) : 1, a.size(-2), a.size(-1), b ? a.stride(0) : 0, a.stride(-2),
                               static_cast<uint8_t*>(q->data_ptr()), b ? q->stride(0) : 0, q->stride(-2), fptr(s),
                               b ? s->stride(0) : 0, s->stride(-2), current_stream(d)));
  PyObject* out = PyTuple_New(2);
  if (!out) throw Raised{};
  PyTuple_SET_ITEM(out, 0, same(p[1], *q));
  PyTuple_SET_ITEM(out, 1, same(p[2], *s));
  return out;
}

// ---- block-scaled GEMM --------------------------------------------------------
struct GemmArgs {
  int64_t B, M, N, K, st[11];
  const at::Tensor* out;
  at::Tensor out_new;
  int out_code, bias_code;
};

// Checks of the GEMM; aq's own type is the caller's to check.
void gemm_args(GemmArgs& g, const at::Tensor& aq, const at::Tensor& w, const at::Tensor& a_scale, const at::Tensor& w_scale,
               const at::Tensor* out, at::ScalarType out_type, const at::Tensor* bias) {
  const bool b = aq.dim() == 3;
  if ((aq.dim() != 2 && !b) || w.dim() != aq.dim()) refuse("a must be [M, K] or [B, M, K] and w_nk [N, K] or [B, N, K]");
  g.M = aq.size(-2), g.K = aq.size(-1), g.N = w.size(-2), g.B = b ? aq.size(0) : 1;
  if (w.size(-1) != g.K || (b && w.size(0) != g.B)) refuse("shape mismatch: a and w_nk must agree on K and the batch");
  if (!is_fp8(w) || !inner(w)) refuse("w_nk must be float8_e4m3fn, contiguous along K (K-major [N, K])");
  if (w_scale.scalar_type() != at::kFloat || w_scale.dim() != aq.dim() || w_scale.size(-1) != groups(g.K) ||
      w_scale.size(-2) != groups(g.N) || (b && w_scale.size(0) != g.B) || !inner(w_scale))
    refuse("w_scale must be fp32 [.., ceil(N / 128), ceil(K / 128)], contiguous along K");
  if (out) {
    if (out->dim() != aq.dim() || out->size(-1) != g.N || out->size(-2) != g.M || (b && out->size(0) != g.B) || !inner(*out))
      refuse("out must be [.., M, N], contiguous along N");
  } else if (b) {
    out = &(g.out_new = at::empty({g.B, g.M, g.N}, aq.options().dtype(out_type)));
  } else {
    out = &(g.out_new = at::empty({g.M, g.N}, aq.options().dtype(out_type)));
  }
  g.out = out;
  g.out_code = float_code(*out, "out");
  g.bias_code = CB_DTYPE_F32;
  int64_t bias_b = 0;
  if (bias) {
    if ((bias->dim() != 1 && bias->dim() != 2) || bias->size(-1) != g.N || !inner(*bias) || (bias->dim() == 2 && bias->size(0) != g.B))
      refuse("bias must be [N] or [B, N], contiguous along N");
    g.bias_code = float_code(*bias, "bias");
    if (bias->dim() == 2) bias_b = bias->stride(0);
  }
  const int64_t st[11] = {b ? aq.stride(0) : 0,      aq.stride(-2),      b ? w.stride(0) : 0,       w.stride(-2),
                          b ? out->stride(0) : 0,    out->stride(-2),    b ? a_scale.stride(0) : 0, a_scale.stride(-2),
                          b ? w_scale.stride(0) : 0, w_scale.stride(-2), bias_b};
  for (int i = 0; i < 11; ++i) g.st[i] = st[i];
}

// (aq, w_nk, a_scale, w_scale, out, out_dtype or None, bias) -> out
PyObject* fp8_block_gemm(PyObject* const* p, Py_ssize_t n) {
  count(n, 7);
  const at::Tensor &aq = tensor(p[0], "aq"), &w = tensor(p[1], "w_nk"), &as = tensor(p[2], "a_scale"), &ws = tensor(p[3], "w_scale");
  const at::Tensor *out = maybe(p[4], "out"), *bias = maybe(p[6], "bias");
  if (!out && !THPDtype_Check(p[5])) refuse("out_dtype must be a torch.dtype");
  const at::ScalarType type = out ? out->scalar_type() : reinterpret_cast<THPDtype*>(p[5])->scalar_type;
  const c10::Device d = gpu_of(aq);
  one_device(d, &w, &as, &ws, out, bias);
  if (!is_fp8(aq) || (aq.dim() != 2 && aq.dim() != 3) || !inner(aq)) refuse("aq must be float8_e4m3fn [M, K] or [B, M, K], contiguous along K");
  bool ok = as.dim() == aq.dim() && as.scalar_type() == at::kFloat && inner(as) && as.size(-1) == groups(aq.size(-1));
  for (int64_t i = 0; ok && i + 1 < aq.dim(); ++i) ok = as.size(i) == aq.size(i);
  if (!ok) refuse("a_scale must be fp32 [.., M, ceil(K / 128)], contiguous along the blocks");
  const c10::cuda::CUDAGuard guard(d);
  GemmArgs g;
  gemm_args(g, aq, w, as, ws, out, type, bias);
  const cb_stream_t stream = current_stream(d);
  const Buffer buf = workspace(d, stream, api.workspace_bytes(CB_OP_FP8_BLOCK, g.B, g.M, g.N, g.K));
  done("cb_fp8_block_gemm",
       api.fp8_block_gemm(static_cast<const uint8_t*>(aq.data_ptr()), fptr(&as), static_cast<const uint8_t*>(w.data_ptr()), fptr(&ws),
                          ptr(bias), g.bias_code, g.out->data_ptr(), g.out_code, g.B, g.M, g.N, g.K, g.st, buf.p, buf.bytes, stream));
  return same(p[4], *g.out);
}

// (a, w_nk, w_scale, q, s, out, out_dtype or None, bias) -> out
PyObject* fp8_block_gemm_dynamic(PyObject* const* p, Py_ssize_t n) {
  count(n, 8);
  const at::Tensor &a = tensor(p[0], "a"), &w = tensor(p[1], "w_nk"), &ws = tensor(p[2], "w_scale");
  const at::Tensor *q = maybe(p[3], "q"), *s = maybe(p[4], "s"), *out = maybe(p[5], "out"), *bias = maybe(p[7], "bias");
  if (p[6] != Py_None && !THPDtype_Check(p[6])) refuse("out_dtype must be a torch.dtype");
  const at::ScalarType type = p[6] != Py_None ? reinterpret_cast<THPDtype*>(p[6])->scalar_type : a.scalar_type();
  const c10::Device d = gpu_of(a);
  one_device(d, &w, &ws, q, s, out, bias);
  act_rows(a);
  const int code = act_code(a, "a");
  const c10::cuda::CUDAGuard guard(d);
  at::Tensor qn, sn;
  block_outputs(a, q, s, qn, sn);
  GemmArgs g;
  gemm_args(g, *q, w, *s, ws, out, type, bias);
  const cb_stream_t stream = current_stream(d);
  const Buffer buf = workspace(d, stream, api.workspace_bytes(CB_OP_FP8_BLOCK, g.B, g.M, g.N, g.K));
  done("cb_fp8_block_gemm_dynamic",
       api.fp8_block_gemm_dynamic(a.data_ptr(), code, a.dim() == 3 ? a.stride(0) : 0, a.stride(-2), static_cast<uint8_t*>(q->data_ptr()),
                                  fptr(s), static_cast<const uint8_t*>(w.data_ptr()), fptr(&ws), ptr(bias), g.bias_code, g.out->data_ptr(),
                                  g.out_code, g.B, g.M, g.N, g.K, g.st, buf.p, buf.bytes, stream));
  return same(p[5], *g.out);
}

// ---- paged cache --------------------------------------------------------------
int cache_code(const at::Tensor& k, const at::Tensor& v, const at::Tensor* ks, const at::Tensor* vs) {
  if (k.dim() != 4 || !same_shape(k, v) || k.scalar_type() != v.scalar_type())
    refuse("k_cache and v_cache must be alike: [pages, page_size, heads, D]");
  if (!inner(k) || !inner(v)) refuse("caches must be contiguous along D");
  int code;
  if (k.scalar_type() == at::kFloat8_e4m3fn) code = CB_DTYPE_E4M3;
  else if (k.scalar_type() == at::kBFloat16) code = CB_DTYPE_BF16;
  else if (k.scalar_type() == at::kHalf) code = CB_DTYPE_F16;
  else refuse("caches must be float16, bfloat16 or float8_e4m3fn");
  if (k.size(1) < 1) refuse("the caches' page size must be at least 1");
  for (const at::Tensor* t : {ks, vs}) {
    if (!t) continue;
    if (code != CB_DTYPE_E4M3) refuse("k_scale and v_scale belong to float8_e4m3fn caches");
    if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != k.size(2) || !inner(*t))
      refuse("k_scale and v_scale must be contiguous fp32 [heads]");
  }
  return code;
}

// (k, v, k_cache, v_cache, slots, k_scale, v_scale) -> None
PyObject* paged_kv_append(PyObject* const* p, Py_ssize_t n) {
  count(n, 7);
  const at::Tensor &k = tensor(p[0], "k"), &v = tensor(p[1], "v"), &kc = tensor(p[2], "k_cache"), &vc = tensor(p[3], "v_cache");
  const at::Tensor& slots = tensor(p[4], "slots");
  const at::Tensor *ks = maybe(p[5], "k_scale"), *vs = maybe(p[6], "v_scale");
  const c10::Device d = gpu_of(k);
  one_device(d, &v, &kc, &vc, &slots, ks, vs);
  const int code = act_code(k, "k"), c_code = cache_code(kc, vc, ks, vs);
  if (k.dim() != 3 || k.size(1) != kc.size(2) || k.size(2) != kc.size(3) || !same_shape(v, k) || v.scalar_type() != k.scalar_type())
    refuse("k and v must be alike: [T, heads, D] with the caches' heads and D");
  if (!inner(k) || !inner(v)) refuse("k and v must be contiguous along D");
  const bool wide = slots.scalar_type() == at::kLong;
  if (slots.dim() != 1 || slots.size(0) != k.size(0) || (!wide && slots.scalar_type() != at::kInt) || !inner(slots))
    refuse("slots must be a contiguous int32 or int64 [T] tensor");
  const c10::cuda::CUDAGuard guard(d);
  const cb_stream_t stream = current_stream(d);
  const Buffer buf = workspace(d, stream, sizeof(int));
  const int64_t st[10] = {k.stride(0), k.stride(1), kc.stride(0), kc.stride(1), kc.stride(2),
                          v.stride(0), v.stride(1), vc.stride(0), vc.stride(1), vc.stride(2)};
  done("cb_paged_kv_append",
       api.paged_kv_append(k.data_ptr(), v.data_ptr(), code, kc.data_ptr(), vc.data_ptr(), c_code, fptr(ks), fptr(vs), slots.data_ptr(),
                           wide, k.size(0), k.size(1), k.size(2), kc.size(0), kc.size(1), st, static_cast<int*>(buf.p), stream));
  Py_RETURN_NONE;
}

// (q, k_cache, v_cache, block_table, seq_lens, scale or None, k_scale, v_scale, out, lse) -> out
PyObject* paged_decode_attention(PyObject* const* p, Py_ssize_t n) {
  count(n, 10);
  const at::Tensor &q = tensor(p[0], "q"), &kc = tensor(p[1], "k_cache"), &vc = tensor(p[2], "v_cache");
  const at::Tensor &table = tensor(p[3], "block_table"), &lens = tensor(p[4], "seq_lens");
  const at::Tensor *ks = maybe(p[6], "k_scale"), *vs = maybe(p[7], "v_scale"), *out = maybe(p[8], "out"), *lse = maybe(p[9], "lse");
  const c10::Device d = gpu_of(q);
  one_device(d, &kc, &vc, &table, &lens, ks, vs, out, lse);
  const int code = act_code(q, "q"), c_code = cache_code(kc, vc, ks, vs);
  const int64_t Hkv = kc.size(2), D = kc.size(3);
  if (q.dim() != 3 || q.size(2) != D || !inner(q)) refuse("q must be [B, Hq, D], contiguous along D, with the caches' D");
  const int64_t B = q.size(0), Hq = q.size(1);
  double scale = 1.0 / std::sqrt(static_cast<double>(D > 0 ? D : 1));
  if (p[5] != Py_None) {
    scale = PyFloat_AsDouble(p[5]);
    if (scale == -1.0 && PyErr_Occurred()) throw Raised{};
  }
  if (c_code != code && c_code != CB_DTYPE_E4M3) refuse("the caches must have q's type or be float8_e4m3fn");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != B || !inner(table))
    refuse("block_table must be int32 [B, max_pages], contiguous along the pages");
  if (lens.scalar_type() != at::kInt || lens.dim() != 1 || lens.size(0) != B || !inner(lens))
    refuse("seq_lens must be a contiguous int32 [B] tensor");
  if (out && (!same_shape(*out, q) || out->scalar_type() != q.scalar_type() || !inner(*out))) refuse("out must be like q");
  if (lse && (lse->scalar_type() != at::kFloat || lse->dim() != 2 || lse->size(0) != B || lse->size(1) != Hq || !inner(*lse)))
    refuse("lse must be fp32 [B, Hq], contiguous along Hq");
  const c10::cuda::CUDAGuard guard(d);
  at::Tensor out_new;
  if (!out) out = &(out_new = at::empty(q.sizes(), q.options()));
  const cb_stream_t stream = current_stream(d);
  const Buffer buf = workspace(d, stream, api.workspace_bytes(CB_OP_PAGED_ATTENTION, B, Hq, Hkv, D));
  const int64_t st[12] = {q.stride(0),  q.stride(1),  out->stride(0), out->stride(1), lse ? lse->stride(0) : 0, table.stride(0),
                          kc.stride(0), kc.stride(1), kc.stride(2),   vc.stride(0),   vc.stride(1),             vc.stride(2)};
  done("cb_paged_decode_attention",
       api.paged_decode_attention(q.data_ptr(), code, kc.data_ptr(), vc.data_ptr(), c_code, fptr(ks), fptr(vs),
                                  static_cast<const int*>(table.data_ptr()), static_cast<const int*>(lens.data_ptr()),
                                  static_cast<float>(scale), out->data_ptr(), fptr(lse), B, Hq, Hkv, D, kc.size(0), kc.size(1), table.size(1),
                                  st, buf.p, buf.bytes, stream));
  return same(p[8], *out);
}

// ---- module -------------------------------------------------------------------
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    return F(args, n);
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// ({name: address}, check, workspace)
PyObject* init(PyObject* const* a, Py_ssize_t n) {
  count(n, 3);
  auto address = [&](const char* name) {
    PyObject* o = PyDict_GetItemString(a[0], name);
    void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
    if (!p) {
      PyErr_Format(PyExc_RuntimeError, "no address of %s", name);
      throw Raised{};
    }
    return p;
  };
#define CB_ADDR(f) api.f = reinterpret_cast<decltype(api.f)>(address("cb_" #f))
  CB_ADDR(add_rmsnorm_quant);
  CB_ADDR(quant_act_fp8_block);
  CB_ADDR(fp8_block_gemm);
  CB_ADDR(fp8_block_gemm_dynamic);
  CB_ADDR(paged_kv_append);
  CB_ADDR(paged_decode_attention);
  CB_ADDR(workspace_bytes);
  CB_ADDR(stream_capture_id);
#undef CB_ADDR
  Py_INCREF(a[1]);
  Py_XDECREF(py_check);
  py_check = a[1];
  Py_INCREF(a[2]);
  Py_XDECREF(py_workspace);
  py_workspace = a[2];
  Py_RETURN_NONE;
}

Key key_of(PyObject* const* a) {
  const long device = PyLong_AsLong(a[0]);
  const uint64_t stream = PyLong_AsUnsignedLongLong(a[1]), capture = PyLong_AsUnsignedLongLong(a[2]);
  if (PyErr_Occurred()) throw Raised{};
  return Key{static_cast<int>(device), stream, capture};
}

// (device index, stream, capture, address, bytes)
PyObject* set_workspace(PyObject* const* a, Py_ssize_t n) {
  count(n, 5);
  const Key key = key_of(a);
  void* p = PyLong_AsVoidPtr(a[3]);
  const size_t bytes = PyLong_AsSize_t(a[4]);
  if (PyErr_Occurred()) throw Raised{};
  workspaces[key] = Buffer{p, bytes};
  Py_RETURN_NONE;
}

// (device index, stream, capture)
PyObject* drop_workspace(PyObject* const* a, Py_ssize_t n) {
  count(n, 3);
  workspaces.erase(key_of(a));
  Py_RETURN_NONE;
}

#define CB_ENTRY(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CB_ENTRY(init),
                         CB_ENTRY(set_workspace),
                         CB_ENTRY(drop_workspace),
                         CB_ENTRY(add_rmsnorm_quant),
                         CB_ENTRY(quant_act_fp8_block),
                         CB_ENTRY(fp8_block_gemm),
                         CB_ENTRY(fp8_block_gemm_dynamic),
                         CB_ENTRY(paged_kv_append),
                         CB_ENTRY(paged_decode_attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
