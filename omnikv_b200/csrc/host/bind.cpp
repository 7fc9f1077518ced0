// Tensor-level front of the 8-bit entry points: a Python extension that takes torch tensors, checks them, allocates the
// results and calls the C ABI on the current stream.
//
// The kernels behind these calls take one to ten microseconds for a single token, and checking a dozen tensors from Python
// takes longer than that (attention 13.5, append 8.4, rows to codes 9.2 us of host time per call against 4.4, 3.2, 4.0 here).
// Nothing is kept between calls but workspaces (per device, stream and captured graph) and, per device, the SM count and
// the status word's address.
//
// The library is not linked: `init` gets the addresses of its entry points, so that the one the process has loaded is used.
#include <Python.h>

#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "omnikv_b200.h"

namespace {

struct Abi {
  decltype(&omnikv_kv8_store) kv8_store;
  decltype(&omnikv_kv8_append) kv8_append;
  decltype(&omnikv_kv8_load) kv8_load;
  decltype(&omnikv_kv8_attn_workspace_bytes) kv8_attn_workspace_bytes;
  decltype(&omnikv_kv8_decode_attn) kv8_decode_attn;
  decltype(&omnikv_quant_rows) quant_rows;
  decltype(&omnikv_linear_w8a8_workspace_bytes) linear_w8a8_workspace_bytes;
  decltype(&omnikv_linear_w8a8) linear_w8a8;
  decltype(&omnikv_capture_id) capture_id;
  decltype(&omnikv_capture_retain) capture_retain;
} abi;
PyObject *g_error, *g_check, *g_device_info;  // the exception class; check(status, what); device_info(ordinal) -> (SMs, status address)
long long g_launches = 0;

// A refused argument: the message of the exception that the call raises.
struct Refused {
  std::string what;
};
[[noreturn]] void refuse(std::string what) { throw Refused{std::move(what)}; }
struct PythonError {};

// ---- arguments ----------------------------------------------------------------------------------------------------------
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw PythonError();
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
at::ScalarType scalar_type(PyObject* o, const char* name) {
  if (!THPDtype_Check(o)) refuse(std::string(name) + " must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
// The ordinal of the device that all given tensors (null entries allowed) are on.
int one_device(const at::Tensor& first, std::initializer_list<const at::Tensor*> others) {
  const int dev = first.is_cuda() ? (int)first.get_device() : -1;
  for (const at::Tensor* t : others)
    if (t && (t->is_cuda() ? (int)t->get_device() : -1) != dev) refuse("all tensors of a call must be on one CUDA device");
  if (dev < 0) refuse("omnikv_b200 kernels need CUDA tensors; there is no CPU path");
  return dev;
}
int code_of_16bit(at::ScalarType t, const char* what) {
  if (t == at::kBFloat16) return OMNIKV_BF16;
  if (t == at::kHalf) return OMNIKV_F16;
  refuse(std::string(what) + " must be bfloat16 or float16, got " + c10::toString(t));
}
const int32_t* ints(const at::Tensor* t, int64_t n, const char* name) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != n || !t->is_contiguous())
    refuse(std::string(name) + " must be contiguous int32 [" + std::to_string(n) + "]");
  return static_cast<const int32_t*>(t->data_ptr());
}

// The step of a dimension (of one entry: any step will do).
int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : t.size(t.dim() - 1); }
bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  for (int d = 0; d < (int)a.dim(); ++d)
    if (step(a, d) != step(b, d)) return false;
  return true;
}
bool dense_rows(const at::Tensor& t) { return t.size(t.dim() - 1) < 2 || t.stride(t.dim() - 1) == 1; }

// The C description of a cache: codes [B, KVH, rows, 128] (int8 or e4m3), fp32 scales [B, KVH, >= ceil(rows / block)].
omnikv_kv8_cache cache_of(const at::Tensor& k8, const at::Tensor& v8, const at::Tensor& ks, const at::Tensor& vs, int64_t block) {
  const at::ScalarType t = k8.scalar_type();
  if ((t != at::kChar && t != at::kFloat8_e4m3fn) || v8.scalar_type() != t || k8.dim() != 4 || k8.size(3) != 128 ||
      !dense_rows(k8) || !same_layout(k8, v8))
    refuse("kv8: k8 and v8 must be int8 or float8_e4m3fn [B, KVH, rows, 128] of one layout, rows contiguous");
  if (block < 1 || block > 256 || (block & (block - 1)))
    refuse("kv8: block must be a power of two between 1 and 256, got " + std::to_string(block));
  const int64_t B = k8.size(0), KVH = k8.size(1), rows = k8.size(2);
  if (B > INT32_MAX || KVH > INT32_MAX || rows > INT32_MAX) refuse("kv8: a cache has at most 2^31 - 1 rows");
  if (ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat || ks.dim() != 3 || ks.size(0) != B || ks.size(1) != KVH ||
      ks.size(2) * block < rows || !dense_rows(ks) || !same_layout(ks, vs))
    refuse("kv8: scales must be fp32 [" + std::to_string(B) + ", " + std::to_string(KVH) + ", >= " +
           std::to_string((rows + block - 1) / block) + "] of one layout, last dimension contiguous");
  return omnikv_kv8_cache{t == at::kChar ? OMNIKV_KV8_INT8 : OMNIKV_KV8_E4M3, (int32_t)block, (int32_t)B, (int32_t)KVH, 128,
                          (int32_t)rows, k8.data_ptr(), v8.data_ptr(), step(k8, 0), step(k8, 1), step(k8, 2),
                          static_cast<float*>(ks.data_ptr()), static_cast<float*>(vs.data_ptr()), step(ks, 0), step(ks, 1)};
}

// ---- devices, streams, workspaces -----------------------------------------------------------------------------------------
struct Device {
  int64_t sms;
  int32_t* status;
};
const Device& device(int dev) {
  static auto& known = *new std::map<int, Device>;  // never destroyed: the CUDA context may be gone by then
  auto it = known.find(dev);
  if (it == known.end()) {
    PyObject* r = PyObject_CallFunction(g_device_info, "i", dev);
    if (!r) throw PythonError();
    long long sms = 0, addr = 0;
    const int ok = PyArg_ParseTuple(r, "LL", &sms, &addr);
    Py_DECREF(r);
    if (!ok) throw PythonError();
    it = known.emplace(dev, Device{sms, reinterpret_cast<int32_t*>(addr)}).first;
  }
  return it->second;
}
// A zero-filled workspace for calls that follow one another: one per stream, and one per captured graph (two graphs, or a
// graph and eager calls, may run at the same time).  One that was outgrown is kept: a captured graph may still use it.  Those
// of a captured graph go when the graph has been destroyed, of which a driver thread tells (graph_ended).  Their fill is a node
// of the graph and runs at every replay: in a memory pool that graphs share, another one's temporaries may have lain there.
struct Ended {
  std::mutex lock;
  std::vector<unsigned long long> ids;
};
Ended& ended() {
  static auto& e = *new Ended;
  return e;
}
void graph_ended(void* id) {
  Ended& e = ended();
  const std::lock_guard<std::mutex> hold(e.lock);
  e.ids.push_back(reinterpret_cast<uintptr_t>(id));
}
const at::Tensor& workspace(int dev, cudaStream_t stream, int tag, size_t bytes) {
  static auto& kept = *new std::map<std::tuple<unsigned long long, int, int, cudaStream_t>, std::vector<at::Tensor>>;
  const unsigned long long id = abi.capture_id(stream);
  auto it = kept.find({id, dev, tag, stream});
  if (it != kept.end() && (size_t)it->second.back().numel() >= bytes) return it->second.back();
  std::vector<unsigned long long> gone;
  {
    const std::lock_guard<std::mutex> hold(ended().lock);
    gone.swap(ended().ids);
  }
  for (const unsigned long long g : gone)
    kept.erase(kept.lower_bound({g, INT_MIN, INT_MIN, nullptr}), kept.lower_bound({g + 1, INT_MIN, INT_MIN, nullptr}));
  at::Tensor fresh_one = at::zeros({(int64_t)std::max(bytes, (size_t)1 << 20)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev));
  if (id && it == kept.end()) abi.capture_retain(stream, graph_ended, reinterpret_cast<void*>((uintptr_t)id));
  auto& own = kept[{id, dev, tag, stream}];
  own.push_back(std::move(fresh_one));
  return own.back();
}
struct OnDevice {  // the device of the call is current, its current stream at hand
  c10::cuda::OptionalCUDAGuard guard;
  cudaStream_t stream;
  explicit OnDevice(int dev) {
    if (c10::cuda::current_device() != dev) guard.set_index(dev);
    stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  }
};
void done(int status, const char* what) {
  if (status) {
    PyObject* r = PyObject_CallFunction(g_check, "is", status, what);
    Py_XDECREF(r);
    throw PythonError();
  }
  ++g_launches;
}
// A new contiguous tensor on the current device, made past the dispatcher (attention 4.9 -> 4.5 us of host time a call).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType t) {
  c10::Storage memory(c10::Storage::use_byte_size_t(), (size_t)c10::multiply_integers(sizes) * c10::elementSize(t),
                      c10::cuda::CUDACachingAllocator::get(), true);
  at::Tensor r = at::detail::make_tensor<c10::TensorImpl>(std::move(memory), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                          c10::scalarTypeToTypeMeta(t));
  r.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return r;
}

// ---- the calls --------------------------------------------------------------------------------------------------------------
PyObject* kv8_store(PyObject* const* a) {
  const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &k8 = tensor(a[2], "k8"), &v8 = tensor(a[3], "v8"),
                   &ks = tensor(a[4], "k_scale"), &vs = tensor(a[5], "v_scale");
  const int64_t block = integer(a[6]), start = integer(a[8]);
  const at::Tensor* lens = maybe(a[7], "lens");
  const int dev = one_device(k8, {&k, &v, &v8, &ks, &vs, lens});
  const omnikv_kv8_cache c = cache_of(k8, v8, ks, vs, block);
  const int dt = code_of_16bit(k.scalar_type(), "kv8_store: k and v");
  if (v.scalar_type() != k.scalar_type() || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != c.B || k.size(1) != c.KVH ||
      k.size(3) != 128 || !dense_rows(k) || !dense_rows(v))
    refuse("kv8_store: k and v must be [B, KVH, n, 128] of one dtype, rows contiguous");
  const int64_t n = k.size(2);
  if (start < 0 || start % block || start > c.rows || n > c.rows - start)
    refuse("kv8_store: " + std::to_string(n) + " rows from " + std::to_string(start) + " must start at a multiple of " + std::to_string(block) +
           " and lie inside the cache's " + std::to_string(c.rows));
  const int32_t* lens_ptr = ints(lens, c.B, "lens");
  if (n) {
    OnDevice on(dev);
    done(abi.kv8_store(&c, dt, k.data_ptr(), step(k, 0), step(k, 1), step(k, 2), v.data_ptr(), step(v, 0), step(v, 1),
                       step(v, 2), (int)start, (int)n, lens_ptr, on.stream),
         "omnikv_kv8_store");
  }
  Py_RETURN_NONE;
}

PyObject* kv8_append(PyObject* const* a) {
  const at::Tensor &k = tensor(a[0], "k_new"), &v = tensor(a[1], "v_new"), &k8 = tensor(a[2], "k8"), &v8 = tensor(a[3], "v8"),
                   &ks = tensor(a[4], "k_scale"), &vs = tensor(a[5], "v_scale"), &pos = tensor(a[6], "pos");
  const int dev = one_device(k8, {&k, &v, &v8, &ks, &vs, &pos});
  const omnikv_kv8_cache c = cache_of(k8, v8, ks, vs, integer(a[7]));
  const int dt = code_of_16bit(k.scalar_type(), "kv8_append: k_new and v_new");
  if (k.dim() != 3 || k.size(0) != c.B || k.size(1) != c.KVH || k.size(2) != 128 || !dense_rows(k) ||
      v.scalar_type() != k.scalar_type() || !same_layout(k, v))
    refuse("kv8_append: k_new and v_new must be [B, KVH, 128] of one dtype and layout");
  const int32_t* at_row = ints(&pos, c.B, "pos");
  OnDevice on(dev);
  done(abi.kv8_append(&c, dt, k.data_ptr(), v.data_ptr(), step(k, 0), step(k, 1), at_row, on.stream), "omnikv_kv8_append");
  Py_RETURN_NONE;
}

PyObject* kv8_load(PyObject* const* a) {
  const at::Tensor &k8 = tensor(a[0], "k8"), &v8 = tensor(a[1], "v8"), &ks = tensor(a[2], "k_scale"), &vs = tensor(a[3], "v_scale");
  const at::Tensor* idx = maybe(a[8], "idx");
  const int dev = one_device(k8, {&v8, &ks, &vs, idx});
  const omnikv_kv8_cache c = cache_of(k8, v8, ks, vs, integer(a[4]));
  const at::ScalarType t = scalar_type(a[5], "kv8_load: dtype");
  const int dt = code_of_16bit(t, "kv8_load: dtype");
  const int64_t start = integer(a[6]);
  int64_t n, idx_stride = 0;
  if (idx) {
    if (idx->scalar_type() != at::kInt || idx->dim() != 2 || idx->size(0) != c.B || !dense_rows(*idx) || start || a[7] != Py_None)
      refuse("kv8_load: idx must be int32 [B, n] with contiguous rows, without start and rows");
    n = idx->size(1);
    idx_stride = step(*idx, 0);
  } else {
    n = a[7] == Py_None ? -1 : integer(a[7]);
    if (start < 0 || start > c.rows || n > c.rows - start || (n < 0 && a[7] != Py_None))
      refuse("kv8_load: " + std::to_string(n) + " rows from " + std::to_string(start) + " are not inside the cache's " + std::to_string(c.rows));
    if (n < 0) n = c.rows - start;
  }
  if (n > INT32_MAX) refuse("kv8_load: at most 2^31 - 1 rows");
  OnDevice on(dev);
  const at::Tensor k = fresh({c.B, c.KVH, n, 128}, t), v = fresh({c.B, c.KVH, n, 128}, t);
  if (n) {
    done(abi.kv8_load(&c, dt, (int)start, (int)n, idx ? static_cast<const int32_t*>(idx->data_ptr()) : nullptr, idx_stride, k.data_ptr(),
                      v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), on.stream),
         "omnikv_kv8_load");
  }
  PyObject* r = PyTuple_New(2);
  if (!r) throw PythonError();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(v));
  return r;
}

PyObject* kv8_decode_attn(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &k8 = tensor(a[1], "k8"), &v8 = tensor(a[2], "v8"), &ks = tensor(a[3], "k_scale"),
                   &vs = tensor(a[4], "v_scale"), &len = tensor(a[5], "len_a");
  const at::Tensor *idx = maybe(a[7], "idx"), *tail_start = maybe(a[8], "tail_start"), *tail_len = maybe(a[9], "tail_len"),
                   *out_arg = maybe(a[10], "out"), *score = maybe(a[11], "score_out"), *score_len = maybe(a[12], "score_len"),
                   *ws_arg = maybe(a[16], "ws");
  const int dev = one_device(q, {&k8, &v8, &ks, &vs, &len, idx, tail_start, tail_len, out_arg, score, score_len, ws_arg});
  omnikv_kv8_attn_params p = {};
  p.cache = cache_of(k8, v8, ks, vs, integer(a[6]));
  p.dtype = code_of_16bit(q.scalar_type(), "kv8_decode_attn: q");
  const int64_t B = p.cache.B, KVH = p.cache.KVH, rows = p.cache.rows;
  if (q.dim() != 3 || q.size(0) != B || q.size(2) != 128 || !dense_rows(q) || KVH == 0 || q.size(1) % KVH || q.size(1) > INT32_MAX)
    refuse("kv8_decode_attn: q must be [B, H, 128] with contiguous head vectors, H a multiple of KVH");
  p.H = (int32_t)q.size(1);
  p.scale = 0.08838834764831845f;  // 1 / sqrt(128)
  if (a[15] != Py_None) {
    p.scale = (float)PyFloat_AsDouble(a[15]);
    if (PyErr_Occurred()) throw PythonError();
  }
  if (out_arg && (out_arg->sizes() != q.sizes() || !dense_rows(*out_arg) || out_arg->scalar_type() != q.scalar_type()))
    refuse("kv8_decode_attn: out must have the shape and dtype of q, head vectors contiguous");
  p.len = ints(&len, B, "len_a");
  int64_t cap = rows;
  if (idx) {
    if (idx->scalar_type() != at::kInt || idx->dim() != 2 || idx->size(0) != B || idx->size(1) == 0 || idx->size(1) > INT32_MAX ||
        !dense_rows(*idx))
      refuse("kv8_decode_attn: idx must be int32 [B, cap] with contiguous rows");
    p.idx = static_cast<const int32_t*>(idx->data_ptr());
    p.idx_stride = step(*idx, 0);
    p.idx_cap = (int32_t)idx->size(1);
    cap = idx->size(1);
  }
  if (ws_arg && !ws_arg->is_contiguous()) refuse("kv8_decode_attn: ws must be contiguous");
  if (!tail_len != !tail_start) refuse("kv8_decode_attn: tail_start and tail_len go together");
  if (tail_len) {
    p.tail_start = ints(tail_start, B, "tail_start");
    p.tail_len = ints(tail_len, B, "tail_len");
    cap += rows;
  }
  if (score) {
    if (idx || tail_len || !score_len) refuse("kv8_decode_attn: scores need score_len, and neither idx nor a tail");
    if (score->scalar_type() != at::kFloat || score->dim() != 3 || score->size(0) != KVH || score->size(1) != B || score->size(2) == 0 ||
        !score->is_contiguous())
      refuse("kv8_decode_attn: score_out must be contiguous fp32 [KVH, B, stride]");
    p.score_out = static_cast<float*>(score->data_ptr());
    p.score_stride = score->size(2);
    p.score_len = ints(score_len, B, "score_len");
  }
  // one CTA per SM; fewer when there are fewer (sequence, KV head) pairs and not three tiles of 32 rows for each
  const Device& d = device(dev);
  if (a[14] != Py_None) cap = integer(a[14]);
  const int64_t per = a[13] != Py_None ? integer(a[13]) : std::clamp<int64_t>(cap / 96, 0, d.sms) + 1;
  const int64_t segments = B * KVH;
  if (segments > 4096) refuse("kv8_decode_attn: at most 4096 pairs of a sequence and a KV head, got " + std::to_string(segments));
  if (per < 1 || per > 32768 || segments < 1 || (a[13] != Py_None && per * segments > 32768))
    refuse("kv8_decode_attn: n_splits x B x KVH must lie in 1..32768");
  const int64_t n = a[13] != Py_None ? per * segments : std::min(d.sms, per * segments);
  p.n_ctas = (int32_t)n;
  OnDevice on(dev);
  const at::Tensor out = out_arg ? *out_arg : fresh(q.sizes(), q.scalar_type());
  p.q = q.data_ptr();
  p.q_stride_b = step(q, 0);
  p.q_stride_h = step(q, 1);
  p.out = out.data_ptr();
  p.out_stride_b = step(out, 0);
  p.out_stride_h = step(out, 1);
  p.status = d.status;
  const at::Tensor& ws = ws_arg ? *ws_arg : workspace(dev, on.stream, 0, abi.kv8_attn_workspace_bytes((int)B, p.H, (int)KVH, p.n_ctas));
  p.workspace = ws.data_ptr();
  p.workspace_bytes = (size_t)ws.numel() * ws.element_size();
  done(abi.kv8_decode_attn(&p, on.stream), "omnikv_kv8_decode_attn");
  return THPVariable_Wrap(out);
}

PyObject* quant_rows(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x");
  const int dev = one_device(x, {});
  const int dt = code_of_16bit(x.scalar_type(), "quant_rows: x");
  if (x.dim() != 2 || !dense_rows(x) || x.size(1) == 0 || x.size(1) % 16 || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX)
    refuse("quant_rows: x must be [n, K] with contiguous rows and K a multiple of 16");
  const int64_t n = x.size(0), K = x.size(1);
  OnDevice on(dev);
  const at::Tensor codes = fresh({n, K}, at::kChar), scale = fresh({n}, at::kFloat);
  if (n) {
    done(abi.quant_rows(dt, x.data_ptr(), step(x, 0), (int)n, (int)K, static_cast<int8_t*>(codes.data_ptr()), K,
                        static_cast<float*>(scale.data_ptr()), on.stream),
         "omnikv_quant_rows");
  }
  PyObject* r = PyTuple_New(2);
  if (!r) throw PythonError();
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(codes));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(scale));
  return r;
}

PyObject* linear_w8a8(PyObject* const* a) {
  const at::Tensor &x8 = tensor(a[0], "x8"), &xs = tensor(a[1], "x_scale"), &w8 = tensor(a[2], "w8"), &ws = tensor(a[3], "w_scale");
  const at::Tensor *res = maybe(a[4], "residual"), *out_arg = maybe(a[5], "out");
  const int dev = one_device(x8, {&xs, &w8, &ws, res, out_arg});
  if (x8.scalar_type() != at::kChar || w8.scalar_type() != at::kChar || x8.dim() != 2 || w8.dim() != 2 || !dense_rows(x8) || !dense_rows(w8))
    refuse("linear_w8a8: x8 [n, K] and w8 [channels, K] must be int8 with contiguous rows");
  const int64_t n = x8.size(0), K = x8.size(1), N = w8.size(0);
  if (w8.size(1) != K || K == 0 || K % 16 || n > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
    refuse("linear_w8a8: x8 and w8 must share K, a multiple of 16");
  if (xs.scalar_type() != at::kFloat || ws.scalar_type() != at::kFloat || xs.dim() != 1 || ws.dim() != 1 || xs.size(0) != n ||
      ws.size(0) != N || !xs.is_contiguous() || !ws.is_contiguous())
    refuse("linear_w8a8: scales must be contiguous fp32, one per row of x8 and of w8");
  const at::ScalarType t = a[6] != Py_None ? scalar_type(a[6], "out_dtype")
                           : out_arg       ? out_arg->scalar_type()
                           : res           ? res->scalar_type()
                                           : at::kBFloat16;
  for (const at::Tensor* o : {out_arg, res})
    if (o && (o->dim() != 2 || o->size(0) != n || o->size(1) != N || o->scalar_type() != t || !dense_rows(*o)))
      refuse("linear_w8a8: out and residual must be [n, channels] of one floating dtype, rows contiguous");
  if (t != at::kFloat && t != at::kBFloat16 && t != at::kHalf)
    refuse(std::string("linear_w8a8: the result is float32, bfloat16 or float16, not ") + c10::toString(t));
  OnDevice on(dev);
  const at::Tensor out = out_arg ? *out_arg : fresh({n, N}, t);
  if (n && N) {
    omnikv_linear_w8a8_params p = {};
    p.n_tokens = (int32_t)n;
    p.channels = (int32_t)N;
    p.K = (int32_t)K;
    p.x = static_cast<const int8_t*>(x8.data_ptr());
    p.x_stride_row = step(x8, 0);
    p.x_scale = static_cast<const float*>(xs.data_ptr());
    p.w = static_cast<const int8_t*>(w8.data_ptr());
    p.w_stride_row = step(w8, 0);
    p.w_scale = static_cast<const float*>(ws.data_ptr());
    p.out_dtype = t == at::kFloat ? OMNIKV_F32 : t == at::kBFloat16 ? OMNIKV_BF16 : OMNIKV_F16;
    p.out = out.data_ptr();
    p.out_stride_row = step(out, 0);
    if (res) {
      p.residual = res->data_ptr();
      p.residual_stride_row = step(*res, 0);
    }
    if (const size_t need = abi.linear_w8a8_workspace_bytes(p.n_tokens, p.channels, p.K)) {
      const at::Tensor& work = workspace(dev, on.stream, 1, need);
      p.workspace = work.data_ptr();
      p.workspace_bytes = (size_t)work.numel();
    }
    p.status = device(dev).status;
    done(abi.linear_w8a8(&p, on.stream), "omnikv_linear_w8a8");
  }
  return THPVariable_Wrap(out);
}

// ---- the module -------------------------------------------------------------------------------------------------------------
template <PyObject* (*Call)(PyObject* const*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!g_error) {
    PyErr_SetString(PyExc_RuntimeError, "init has not been called");
    return nullptr;
  }
  if (n != ARGS) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", ARGS, n);
    return nullptr;
  }
  try {
    return Call(args);
  } catch (const Refused& r) {
    PyErr_SetString(g_error, r.what.c_str());
  } catch (const PythonError&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

// init(addresses of the entry points in the order of Abi, exception class, check, device_info)
PyObject* init(PyObject*, PyObject* args) {
  PyObject *addresses, *error, *check, *info;
  if (!PyArg_ParseTuple(args, "O!OOO", &PyTuple_Type, &addresses, &error, &check, &info)) return nullptr;
  static_assert(sizeof(Abi) % sizeof(void*) == 0, "a table of function pointers");
  constexpr Py_ssize_t N = sizeof(Abi) / sizeof(void*);
  if (PyTuple_GET_SIZE(addresses) != N) {
    PyErr_Format(PyExc_ValueError, "%zd addresses expected", N);
    return nullptr;
  }
  void* table[N];
  for (Py_ssize_t i = 0; i < N; ++i) {
    table[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(addresses, i));
    if (!table[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  memcpy(&abi, table, sizeof(abi));
  Py_INCREF(error);
  Py_INCREF(check);
  Py_INCREF(info);
  g_error = error;
  g_check = check;
  g_device_info = info;
  Py_RETURN_NONE;
}
PyObject* launches(PyObject*, PyObject*) { return PyLong_FromLongLong(g_launches); }

PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, nullptr},
    {"launches", launches, METH_NOARGS, nullptr},
    {"kv8_store", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<kv8_store, 9>)), METH_FASTCALL, nullptr},
    {"kv8_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<kv8_append, 8>)), METH_FASTCALL, nullptr},
    {"kv8_load", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<kv8_load, 9>)), METH_FASTCALL, nullptr},
    {"kv8_decode_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<kv8_decode_attn, 17>)), METH_FASTCALL, nullptr},
    {"quant_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<quant_rows, 1>)), METH_FASTCALL, nullptr},
    {"linear_w8a8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<linear_w8a8, 7>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_omnikv_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__omnikv_bind() { return PyModule_Create(&module); }
