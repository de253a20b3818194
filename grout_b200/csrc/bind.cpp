// Python binding of the window attention and 8-bit cache entry points.
//
// A call of a few microseconds on the GPU should not spend ten on the host: the
// wrappers in attn.py hand their arguments over as they are, and this module
// checks the tensors, fills the C structs and calls the C ABI on the tensors'
// device and its current stream.  (Checks in Python and ctypes took 10 to 12 us a
// call, 5 of them in the entry point with its launch.)  The entry points come as
// addresses from the library that attn.lib() has loaded, so there is one copy
// of its state.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <optional>
#include <string>

#include "grout_attn.h"

namespace {

constexpr int64_t kD = 128;

PyObject* g_error = nullptr;  // GroutError(status, message)

struct Api {
  decltype(&grout_attn_last_error) last_error;
  decltype(&grout_qk_norm_rope_kv_decode_paged_fp8) write_decode;
  decltype(&grout_qk_norm_rope_kv_prefill_paged_fp8) write_prefill;
  decltype(&grout_kv_read_paged_fp8) kv_read;
  decltype(&grout_attn_decode_window_workspace_bytes) decode_workspace;
  decltype(&grout_attn_decode_window) decode_window;
  decltype(&grout_attn_decode_paged_window) decode_paged_window;
  decltype(&grout_attn_decode_paged_fp8) decode_paged_fp8;
  decltype(&grout_attn_prefill_window_splits) prefill_splits;
  decltype(&grout_attn_prefill_window_workspace_bytes) prefill_workspace;
  decltype(&grout_attn_prefill_varlen_window) prefill_varlen;
  decltype(&grout_attn_prefill_paged_window) prefill_paged;
} g_api = {};

// What a check throws: becomes GroutError(status, text).
struct Refused {
  int status;
  std::string text;
};
// A Python error is set.
struct PythonError {};

[[noreturn]] void refuse(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
[[noreturn]] void refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{GROUT_ERR_INVALID_ARG, buf};
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const char* type_name(at::ScalarType t) {
  return t == at::kHalf ? "torch.float16" : t == at::kFloat ? "torch.float32"
       : t == at::kInt ? "torch.int32" : t == at::kFloat8_e4m3fn ? "torch.float8_e4m3fn" : c10::toString(t);
}

// A contiguous CUDA tensor of the type, on device *dev (set by the first one, -1).
const at::Tensor& tensor(PyObject* o, const char* name, at::ScalarType type, int* dev) {
  if (!THPVariable_Check(o)) refuse("%s must be a CUDA tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse("%s must be a CUDA tensor", name);
  if (t.scalar_type() != type) refuse("%s must be %s, got %s", name, type_name(type), type_name(t.scalar_type()));
  if (!t.is_contiguous()) refuse("%s must be contiguous", name);
  if (*dev < 0) *dev = t.get_device();
  if (t.get_device() != *dev) refuse("%s is on cuda:%d, not on cuda:%d", name, (int)t.get_device(), *dev);
  return t;
}

bool same_shape(const at::Tensor& a, const at::Tensor& b) { return a.sizes() == b.sizes(); }

// n as a C long long (anything with __index__); one past 64 bits counts as the nearest.
long long as_ll(PyObject* o) {
  PyObject* n = PyNumber_Index(o);
  if (!n) throw PythonError{};
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(n, &over);
  Py_DECREF(n);
  if (over) return over > 0 ? LLONG_MAX : LLONG_MIN;
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  return v;
}
int32_t as_i32(PyObject* o, const char* name) {
  const long long v = as_ll(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s=%lld is out of range", name, v);
  return (int32_t)v;
}
int32_t i32_of(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s=%lld is out of range", name, (long long)v);
  return (int32_t)v;
}
// A window or sink count: past 32 bits it is as large (or as bad) as the largest that fits.
int32_t span(PyObject* o) {
  const long long v = as_ll(o);
  return v > INT32_MAX ? INT32_MAX : (v < 0 ? -1 : (int32_t)v);
}
float as_float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return (float)v;
}
float scale_of(PyObject* o) { return o == Py_None ? 0.f : as_float(o); }

grout_attn_dims dims_of(int64_t hq, int64_t hkv, int64_t max_seq, float eps, float qk_scale, int32_t flags) {
  grout_attn_dims d;
  d.num_q_heads = i32_of(hq, "num_q_heads");
  d.num_kv_heads = i32_of(hkv, "num_kv_heads");
  d.head_dim = (int32_t)kD;
  d.max_seq = i32_of(max_seq, "max_seq");
  d.rms_eps = eps;
  d.qk_scale = qk_scale;
  d.flags = flags;
  return d;
}

// Device int32/uint32 positions, one entry per sequence.
const uint32_t* positions(PyObject* o, int64_t n, int dev) {
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.is_cuda() && t.get_device() == dev && t.numel() >= n && t.is_contiguous() &&
        (t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32))
      return static_cast<const uint32_t*>(t.data_ptr());
  }
  refuse("position must be a contiguous device int32/uint32 tensor with one entry per sequence on cuda:%d", dev);
}

// [batch, table_stride] page table.
const at::Tensor& page_table(PyObject* o, int64_t batch, int* dev) {
  const at::Tensor& t = tensor(o, "page_table", at::kInt, dev);
  if (t.dim() != 2 || t.size(0) < batch)
    refuse("page_table must be [batch, table_stride]: %s", shape_of(t).c_str());
  return t;
}

struct Pools {
  const at::Tensor &k, &v;
  int64_t num_pages, hkv, page_size;
};
Pools kv_pages(PyObject* ko, PyObject* vo, at::ScalarType type, int* dev) {
  const at::Tensor& k = tensor(ko, "k_pages", type, dev);
  const at::Tensor& v = tensor(vo, "v_pages", type, dev);
  if (k.dim() != 4 || k.size(3) != kD)
    refuse("k_pages must be [num_pages, Hkv, page_size, 128]: %s", shape_of(k).c_str());
  if (!same_shape(k, v)) refuse("v_pages shape mismatch");
  return Pools{k, v, k.size(0), k.size(1), k.size(2)};
}

struct Fp8Pool {
  grout_fp8_pages pages;
  int64_t hkv, page_size;
};
Fp8Pool fp8_pages(PyObject* const* a, int* dev) {  // k_pages, v_pages, k_scales, v_scales
  const Pools p = kv_pages(a[0], a[1], at::kFloat8_e4m3fn, dev);
  const at::Tensor& ks = tensor(a[2], "k_scales", at::kFloat, dev);
  const at::Tensor& vs = tensor(a[3], "v_scales", at::kFloat, dev);
  if (ks.sizes() != p.k.sizes().slice(0, 3) || vs.sizes() != ks.sizes())
    refuse("k_scales and v_scales must be [num_pages, Hkv, page_size]: %s, %s", shape_of(ks).c_str(),
           shape_of(vs).c_str());
  Fp8Pool f;
  f.pages.k = p.k.data_ptr();
  f.pages.v = p.v.data_ptr();
  f.pages.k_scales = static_cast<float*>(ks.data_ptr());
  f.pages.v_scales = static_cast<float*>(vs.data_ptr());
  f.pages.num_pages = i32_of(p.num_pages, "num_pages");
  f.pages.page_size = i32_of(p.page_size, "page_size");
  f.hkv = p.hkv;
  f.page_size = p.page_size;
  return f;
}

const float* rope_table(PyObject* o, int64_t max_seq, int* dev) {
  const at::Tensor& t = tensor(o, "rope_table", at::kFloat, dev);
  if (t.dim() != 2 || t.size(1) != kD || t.size(0) < max_seq)
    refuse("rope_table must be [>= max_seq=%lld, 128] f32: %s", (long long)max_seq, shape_of(t).c_str());
  return static_cast<const float*>(t.data_ptr());
}

void norm_weights(PyObject* qo, PyObject* ko, int* dev, const void** qw, const void** kw) {
  const at::Tensor& q = tensor(qo, "q_norm_w", at::kHalf, dev);
  const at::Tensor& k = tensor(ko, "k_norm_w", at::kHalf, dev);
  if (q.numel() != kD || k.numel() != kD) refuse("q_norm_w and k_norm_w must have 128 entries");
  *qw = q.data_ptr();
  *kw = k.data_ptr();
}

// Device int32 [batch + 1].
const at::Tensor& cu_seqlens(PyObject* o, int* dev) {
  const at::Tensor& t = tensor(o, "cu_seqlens", at::kInt, dev);
  if (t.dim() != 1 || t.numel() < 1) refuse("cu_seqlens must be [batch + 1]: %s", shape_of(t).c_str());
  return t;
}
const int32_t* starts(PyObject* o, int64_t batch, int* dev, const char* name) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name, at::kInt, dev);
  if (t.numel() < batch) refuse("%s needs one entry per sequence", name);
  return static_cast<const int32_t*>(t.data_ptr());
}

struct GilReleased {
  PyThreadState* state = PyEval_SaveThread();
  ~GilReleased() { PyEval_RestoreThread(state); }
};

// Calls f(stream) with dev as the current device, other Python threads running
// meanwhile; a status becomes a GroutError.
template <class F>
void enqueue(int dev, F f) {
  const GilReleased gil;
  const c10::cuda::OptionalCUDAGuard guard(c10::cuda::current_device() == dev
                                               ? std::optional<c10::Device>()
                                               : c10::Device(c10::kCUDA, (c10::DeviceIndex)dev));
  const grout_status st = f(reinterpret_cast<grout_stream_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
  if (st != GROUT_OK) throw Refused{(int)st, g_api.last_error()};
}

// ---- the entry points (positional arguments, as the wrappers in attn.py pass them)

void write_decode(PyObject* const* a) {
  int dev = -1;
  const at::Tensor& qkv = tensor(a[0], "qkv", at::kHalf, &dev);
  const at::Tensor& q_out = tensor(a[4], "q_out", at::kHalf, &dev);
  const void *qw, *kw;
  norm_weights(a[1], a[2], &dev, &qw, &kw);
  const Fp8Pool p = fp8_pages(a + 5, &dev);
  const int64_t hq = as_i32(a[11], "num_q_heads"), hkv = as_i32(a[12], "num_kv_heads");
  if (p.hkv != hkv) refuse("k_pages has %lld KV heads, not %lld", (long long)p.hkv, (long long)hkv);
  const int64_t B = qkv.dim() == 2 ? qkv.size(0) : 1;
  if (qkv.numel() != B * (hq + 2 * hkv) * kD) refuse("qkv shape mismatch: %s", shape_of(qkv).c_str());
  if (q_out.numel() != B * hq * kD) refuse("q_out shape mismatch: %s", shape_of(q_out).c_str());
  const uint32_t* pos = positions(a[10], B, dev);
  const at::Tensor& table = page_table(a[9], B, &dev);
  const int64_t max_seq = a[14] == Py_None ? table.size(1) * p.page_size : as_i32(a[14], "max_seq");
  const float* rope = rope_table(a[3], max_seq, &dev);
  const grout_attn_dims d = dims_of(hq, hkv, max_seq, as_float(a[13]), 0.f, 0);
  enqueue(dev, [&](grout_stream_t s) {
    return g_api.write_decode(qkv.data_ptr(), qw, kw, rope, q_out.data_ptr(), &p.pages,
                              static_cast<const int32_t*>(table.data_ptr()), i32_of(table.size(1), "table_stride"),
                              pos, i32_of(B, "batch"), &d, s);
  });
}

void write_prefill(PyObject* const* a) {
  int dev = -1;
  const at::Tensor& q = tensor(a[0], "q", at::kHalf, &dev);
  const at::Tensor& k = tensor(a[1], "k", at::kHalf, &dev);
  const at::Tensor& v = tensor(a[2], "v", at::kHalf, &dev);
  const at::Tensor& q_out = tensor(a[6], "q_out", at::kHalf, &dev);
  const void *qw, *kw;
  norm_weights(a[3], a[4], &dev, &qw, &kw);
  const Fp8Pool p = fp8_pages(a + 7, &dev);
  if (q.dim() != 3 || q.size(2) != kD) refuse("q shape mismatch: %s", shape_of(q).c_str());
  const int64_t S = q.size(0), hq = q.size(1);
  if (k.dim() != 3 || k.size(0) != S || k.size(1) != p.hkv || k.size(2) != kD || !same_shape(k, v))
    refuse("k/v shape mismatch: %s, %s", shape_of(k).c_str(), shape_of(v).c_str());
  if (!same_shape(q_out, q)) refuse("q_out shape mismatch: %s", shape_of(q_out).c_str());
  const at::Tensor& row = tensor(a[11], "page_table_row", at::kInt, &dev);
  const int64_t most = row.numel() * p.page_size;
  const int64_t max_seq = a[14] == Py_None ? most : as_i32(a[14], "max_seq");
  if (most < max_seq) refuse("page_table_row shorter than max_seq");
  const float* rope = rope_table(a[5], max_seq, &dev);
  const grout_attn_dims d = dims_of(hq, p.hkv, max_seq, as_float(a[13]), 0.f, 0);
  const int32_t start = as_i32(a[12], "position_start");
  enqueue(dev, [&](grout_stream_t s) {
    return g_api.write_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), hq * kD, p.hkv * kD, qw, kw, rope,
                               q_out.data_ptr(), &p.pages, static_cast<const int32_t*>(row.data_ptr()), start,
                               i32_of(S, "seq_len"), &d, s);
  });
}

void kv_read(PyObject* const* a) {
  int dev = -1;
  const at::Tensor& k_out = tensor(a[5], "k_out", at::kHalf, &dev);
  const at::Tensor& v_out = tensor(a[6], "v_out", at::kHalf, &dev);
  const Fp8Pool p = fp8_pages(a, &dev);
  if (k_out.dim() != 3 || k_out.size(1) != p.hkv || k_out.size(2) != kD)
    refuse("k_out must be [rows, %lld, 128]: %s", (long long)p.hkv, shape_of(k_out).c_str());
  if (!same_shape(k_out, v_out)) refuse("v_out shape mismatch");
  const at::Tensor& cu = cu_seqlens(a[7], &dev);
  const int64_t B = cu.numel() - 1;
  const int32_t* start = starts(a[8], B, &dev, "position_start");
  const at::Tensor& table = page_table(a[4], B, &dev);
  const int64_t max_seq = a[9] == Py_None ? table.size(1) * p.page_size : as_i32(a[9], "max_seq");
  const grout_attn_dims d = dims_of(p.hkv, p.hkv, max_seq, 0.f, 0.f, 0);
  enqueue(dev, [&](grout_stream_t s) {
    return g_api.kv_read(&p.pages, static_cast<const int32_t*>(table.data_ptr()),
                         i32_of(table.size(1), "table_stride"), static_cast<const int32_t*>(cu.data_ptr()), start,
                         i32_of(B, "batch"), k_out.size(0), k_out.data_ptr(), v_out.data_ptr(), p.hkv * kD, &d, s);
  });
}

// The caller's workspace, or one of this call's own (given back to the
// stream's allocator after the launch).
struct Workspace {
  bool given;
  void* ptr = nullptr;
  size_t bytes = 0;
  at::Tensor own;
  Workspace(PyObject* o, int dev) : given(o != Py_None) {
    if (!given) return;
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda() || !THPVariable_Unpack(o).is_contiguous() ||
        THPVariable_Unpack(o).get_device() != dev)
      refuse("workspace must be a contiguous tensor on cuda:%d", dev);
    ptr = THPVariable_Unpack(o).data_ptr();
    bytes = (size_t)THPVariable_Unpack(o).nbytes();
  }
  void make(size_t need, const at::Tensor& like) {
    if (!need) return;
    own = at::empty({(int64_t)need}, like.options().dtype(at::kByte));
    ptr = own.data_ptr();
    bytes = need;
  }
};

// A split count, None or 0 the automatic one; refused here, before a workspace
// of that size is asked for.
int32_t splits_of(PyObject* o, int32_t most) {
  const int32_t n = o == Py_None ? 0 : as_i32(o, "num_splits");
  if (n < 0 || n > most) refuse("num_splits=%d must be in [0, %d]", n, most);
  return n;
}
constexpr int32_t kMaxDecodeSplits = 1024, kMaxPrefillSplits = 32;  // as the entry points'
constexpr int32_t kMaxSplitBatch = 65535;                           // of a split prefill

const at::Tensor& decode_query(PyObject* o, int* dev) {
  const at::Tensor& q = tensor(o, "q", at::kHalf, dev);
  if (q.dim() != 3 || q.size(2) != kD) refuse("q must be [B, Hq, 128]: %s", shape_of(q).c_str());
  return q;
}

// The tail that the decode calls share; a: position, out, max_kv_len, window,
// sinks, workspace, num_splits, qk_scale, scale_f16.  f(position, out, batch,
// max_kv_len, window, sinks, splits, dims, workspace, bytes, stream).
template <class F>
void decode_tail(PyObject* const* a, const at::Tensor& q, int64_t hkv, int64_t max_seq, bool fp8, int dev, F f) {
  const at::Tensor& out = tensor(a[1], "out", at::kHalf, &dev);
  if (!same_shape(out, q)) refuse("out shape mismatch");
  const int32_t B = i32_of(q.size(0), "batch");
  const uint32_t* pos = positions(a[0], B, dev);
  const int32_t max_kv_len = as_i32(a[2], "max_kv_len"), window = span(a[3]), sinks = span(a[4]);
  const int32_t splits = splits_of(a[6], kMaxDecodeSplits);
  const int scale_f16 = PyObject_IsTrue(a[8]);
  if (scale_f16 < 0) throw PythonError{};
  const grout_attn_dims d =
      dims_of(q.size(1), hkv, max_seq, 0.f, scale_of(a[7]), scale_f16 ? GROUT_FLAG_DECODE_SCALE_F16 : 0);
  Workspace ws(a[5], dev);
  enqueue(dev, [&](grout_stream_t s) {
    if (!ws.given) ws.make(g_api.decode_workspace(B, max_kv_len, window, sinks, splits, fp8 ? 1 : 0, &d), q);
    return f(pos, out.data_ptr(), B, max_kv_len, window, sinks, splits, &d, ws.ptr, ws.bytes, s);
  });
}

void decode_window(PyObject* const* a) {  // q, k_cache, v_cache, then the tail
  int dev = -1;
  const at::Tensor& q = decode_query(a[0], &dev);
  const at::Tensor& k = tensor(a[1], "k_cache", at::kHalf, &dev);
  const at::Tensor& v = tensor(a[2], "v_cache", at::kHalf, &dev);
  if (k.dim() != 4 || k.size(0) < q.size(0) || k.size(3) != kD)
    refuse("k_cache must be [B, Hkv, max_seq, 128]: %s", shape_of(k).c_str());
  if (!same_shape(k, v)) refuse("v_cache shape mismatch");
  const int64_t hkv = k.size(1), max_seq = k.size(2);
  decode_tail(a + 3, q, hkv, max_seq, false, dev,
              [&](const uint32_t* pos, void* out, int32_t B, int32_t len, int32_t window, int32_t sinks, int32_t splits,
                  const grout_attn_dims* d, void* ws, size_t bytes, grout_stream_t s) {
                return g_api.decode_window(q.data_ptr(), k.data_ptr(), v.data_ptr(), hkv * max_seq * kD, max_seq * kD,
                                           pos, out, B, len, window, sinks, splits, d, ws, bytes, s);
              });
}

void decode_paged_window(PyObject* const* a) {  // q, k_pages, v_pages, page_table, max_seq, then the tail
  int dev = -1;
  const at::Tensor& q = decode_query(a[0], &dev);
  const Pools p = kv_pages(a[1], a[2], at::kHalf, &dev);
  const at::Tensor& table = page_table(a[3], q.size(0), &dev);
  const int64_t max_seq = a[4] == Py_None ? table.size(1) * p.page_size : as_i32(a[4], "max_seq");
  decode_tail(a + 5, q, p.hkv, max_seq, false, dev,
              [&](const uint32_t* pos, void* out, int32_t B, int32_t len, int32_t window, int32_t sinks, int32_t splits,
                  const grout_attn_dims* d, void* ws, size_t bytes, grout_stream_t s) {
                return g_api.decode_paged_window(
                    q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), i32_of(p.num_pages, "num_pages"),
                    i32_of(p.page_size, "page_size"), static_cast<const int32_t*>(table.data_ptr()),
                    i32_of(table.size(1), "table_stride"), pos, out, B, len, window, sinks, splits, d, ws, bytes, s);
              });
}

void decode_paged_fp8(PyObject* const* a) {  // q, the four pools, page_table, max_seq, then the tail
  int dev = -1;
  const at::Tensor& q = decode_query(a[0], &dev);
  const Fp8Pool p = fp8_pages(a + 1, &dev);
  const at::Tensor& table = page_table(a[5], q.size(0), &dev);
  const int64_t max_seq = a[6] == Py_None ? table.size(1) * p.page_size : as_i32(a[6], "max_seq");
  decode_tail(a + 7, q, p.hkv, max_seq, true, dev,
              [&](const uint32_t* pos, void* out, int32_t B, int32_t len, int32_t window, int32_t sinks, int32_t splits,
                  const grout_attn_dims* d, void* ws, size_t bytes, grout_stream_t s) {
                return g_api.decode_paged_fp8(q.data_ptr(), &p.pages, static_cast<const int32_t*>(table.data_ptr()),
                                              i32_of(table.size(1), "table_stride"), pos, out, B, len, window, sinks,
                                              splits, d, ws, bytes, s);
              });
}

// q and out of a chunk call.
const at::Tensor& chunk_query(PyObject* qo, PyObject* oo, int* dev, void** out) {
  const at::Tensor& q = tensor(qo, "q", at::kHalf, dev);
  if (q.dim() != 3 || q.size(2) != kD) refuse("q must be [q_rows, Hq, 128]: %s", shape_of(q).c_str());
  const at::Tensor& o = tensor(oo, "out", at::kHalf, dev);
  if (!same_shape(o, q)) refuse("out shape mismatch");
  *out = o.data_ptr();
  return q;
}
// Batch, lengths and longest sequence of a chunk call.
struct Chunk {
  int32_t batch, max_q_len;
  const int32_t* cu;
};
Chunk chunk_batch(PyObject* cu, PyObject* max_q_len, int64_t rows, int* dev) {
  if (cu == Py_None)
    return Chunk{1, max_q_len == Py_None ? i32_of(rows, "q_rows") : as_i32(max_q_len, "max_q_len"), nullptr};
  if (max_q_len == Py_None) refuse("max_q_len is required with cu_seqlens_q");
  const at::Tensor& t = cu_seqlens(cu, dev);
  return Chunk{i32_of(t.numel() - 1, "batch"), as_i32(max_q_len, "max_q_len"),
               static_cast<const int32_t*>(t.data_ptr())};
}

constexpr size_t kOwnWorkspace = 64u << 20;

// The tail of the chunk calls; a: workspace, num_splits.
template <class Args, class F>
void chunk_call(PyObject* const* a, const at::Tensor& q, const Args& g, int64_t max_keys, int32_t window,
                int32_t sinks, const grout_attn_dims& d, int dev, F f) {
  Workspace ws(a[0], dev);
  int32_t splits = splits_of(a[1], kMaxPrefillSplits);
  if (splits > 1 && g.batch > kMaxSplitBatch)
    refuse("num_splits=%d with batch=%d (at most %d with splits)", splits, g.batch, kMaxSplitBatch);
  enqueue(dev, [&](grout_stream_t s) {
    if (!ws.given) {
      if (splits == 0) {
        // without positions a sequence's keys are the chunk itself
        const int64_t keys = g.position_start ? max_keys : std::min<int64_t>(max_keys, g.max_q_len);
        splits = g_api.prefill_splits(g.batch, g.max_q_len, keys, window, sinks, &d);
        // An item of work per SM needs 20 MB at most; rows of q that no sequence
        // has would need theirs too.
        const size_t one = g_api.prefill_workspace(g.q_rows, 2, &d) / 2;
        if (one) splits = (int32_t)std::min<size_t>(splits, std::max<size_t>(1, kOwnWorkspace / one));
      }
      ws.make(g_api.prefill_workspace(g.q_rows, splits, &d), q);
    }
    return f(&g, window, sinks, splits, &d, ws.ptr, ws.bytes, s);
  });
}

// q, k, v, out, cu_seqlens_q, max_q_len, num_kv_heads, kv_row_stride, kv_head_stride, window, sinks,
// kv_batch_stride, kv_rows, position_start, kv_start, qk_scale, workspace, num_splits
void prefill_varlen(PyObject* const* a) {
  int dev = -1;
  void* out;
  const at::Tensor& q = chunk_query(a[0], a[3], &dev, &out);
  const at::Tensor& k = tensor(a[1], "k", at::kHalf, &dev);
  const at::Tensor& v = tensor(a[2], "v", at::kHalf, &dev);
  const Chunk c = chunk_batch(a[4], a[5], q.size(0), &dev);
  const int64_t hkv = as_i32(a[6], "num_kv_heads"), row = as_ll(a[7]), head = as_ll(a[8]), batch = as_ll(a[11]);
  if (row <= 0 || head <= 0 || batch < 0 || hkv <= 0) refuse("bad kv strides");
  // The furthest element that the strides address lies in k and v.  (In 128
  // bits: a stride may be any number.)
  const __int128 held = std::min(k.numel(), v.numel());
  const __int128 fixed = (__int128)std::max(0, c.batch - 1) * batch + (__int128)(hkv - 1) * head + kD;
  const __int128 left = held - fixed;
  const int64_t most = left < 0 ? 0 : (int64_t)(left / row) + 1;
  const int64_t rows = a[12] == Py_None ? most : as_ll(a[12]);
  if (rows <= 0 || rows > most)
    refuse("kv_rows=%lld: k and v hold %lld rows at these strides", (long long)rows, (long long)most);
  grout_prefill_varlen_args g = {};
  g.q = q.data_ptr();
  g.out = out;
  g.q_row_stride = q.size(1) * kD;
  g.q_rows = q.size(0);
  g.k = k.data_ptr();
  g.v = v.data_ptr();
  g.kv_batch_stride = batch;
  g.kv_row_stride = row;
  g.kv_head_stride = head;
  g.kv_rows = rows;
  g.cu_seqlens_q = c.cu;
  g.position_start = starts(a[13], c.batch, &dev, "position_start");
  g.kv_start = starts(a[14], c.batch, &dev, "kv_start");
  g.batch = c.batch;
  g.max_q_len = c.max_q_len;
  const int32_t window = span(a[9]), sinks = span(a[10]);
  const grout_attn_dims d = dims_of(q.size(1), hkv, 1 << 30, 0.f, scale_of(a[15]), 0);
  chunk_call(a + 16, q, g, rows, window, sinks, d, dev, g_api.prefill_varlen);
}

// q, k_pages, v_pages, page_table, out, window, sinks, cu_seqlens_q, position_start, max_q_len, max_seq, qk_scale,
// workspace, num_splits
void prefill_paged(PyObject* const* a) {
  int dev = -1;
  void* out;
  const at::Tensor& q = chunk_query(a[0], a[4], &dev, &out);
  const Pools p = kv_pages(a[1], a[2], at::kHalf, &dev);
  const Chunk c = chunk_batch(a[7], a[9], q.size(0), &dev);
  const at::Tensor& table = page_table(a[3], c.batch, &dev);
  grout_prefill_paged_args g = {};
  g.q = q.data_ptr();
  g.out = out;
  g.q_row_stride = q.size(1) * kD;
  g.q_rows = q.size(0);
  g.k_pages = p.k.data_ptr();
  g.v_pages = p.v.data_ptr();
  g.num_pages = i32_of(p.num_pages, "num_pages");
  g.page_size = i32_of(p.page_size, "page_size");
  g.page_table = static_cast<const int32_t*>(table.data_ptr());
  g.table_stride = i32_of(table.size(1), "table_stride");
  g.cu_seqlens_q = c.cu;
  g.position_start = starts(a[8], c.batch, &dev, "position_start");
  g.batch = c.batch;
  g.max_q_len = c.max_q_len;
  const int32_t window = span(a[5]), sinks = span(a[6]);
  const int64_t max_seq = a[10] == Py_None ? table.size(1) * p.page_size : as_i32(a[10], "max_seq");
  const grout_attn_dims d = dims_of(q.size(1), p.hkv, max_seq, 0.f, scale_of(a[11]), 0);
  chunk_call(a + 12, q, g, max_seq, window, sinks, d, dev, g_api.prefill_paged);
}

// Sets torch.OutOfMemoryError, as every allocation of PyTorch's own does.
void out_of_memory(const char* what) {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
  if (type) PyErr_SetString(type, what);
  Py_XDECREF(type);
  Py_XDECREF(torch);
}

// Runs an entry point; C++ exceptions end here.
template <void (*kFn)(PyObject* const*), int kArgs>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "takes %d arguments (%zd given)", kArgs, n);
    return nullptr;
  }
  if (!g_api.last_error) {
    PyErr_SetString(PyExc_RuntimeError, "the library is not loaded");
    return nullptr;
  }
  try {
    kFn(args);
    Py_RETURN_NONE;
  } catch (const PythonError&) {
  } catch (const Refused& r) {
    PyObject* e = PyObject_CallFunction(g_error, "is#", r.status, r.text.data(), (Py_ssize_t)r.text.size());
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
  } catch (const c10::OutOfMemoryError& e) {
    out_of_memory(e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// use(GroutError, (addresses of the entry points, in Api's order))
PyObject* use(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kCount = sizeof(Api) / sizeof(void*);
  if (n != 2 || !PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != kCount) {
    PyErr_Format(PyExc_TypeError, "use(error, %zd addresses)", kCount);
    return nullptr;
  }
  void* addr[kCount];
  for (Py_ssize_t i = 0; i < kCount; ++i) {
    addr[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args[1], i));
    if (!addr[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  static_assert(sizeof(addr) == sizeof(g_api), "Api holds pointers only");
  memcpy(&g_api, addr, sizeof(addr));
  Py_INCREF(args[0]);
  Py_XSETREF(g_error, args[0]);
  Py_RETURN_NONE;
}

#define GROUT_FN(name, args) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<name, args>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {
    {"use", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&use)), METH_FASTCALL, nullptr},
    GROUT_FN(write_decode, 15),  GROUT_FN(write_prefill, 15),       GROUT_FN(kv_read, 10),
    GROUT_FN(decode_window, 12), GROUT_FN(decode_paged_window, 14), GROUT_FN(decode_paged_fp8, 16),
    GROUT_FN(prefill_varlen, 18), GROUT_FN(prefill_paged, 14),      {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", "Checks and calls of the window and 8-bit cache entry points.",
                        -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&g_module); }
