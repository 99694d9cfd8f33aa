// The host side of one call of a compiled graph, as a CPython extension: check the tensors, allocate
// the results, hand the pointers to kb200_plan_run.  Takes the place of GPUExecutable.__call__ of the
// reference (kiln/gpu/runtime.py:206-217), which copies the inputs into fixed buffers, replays a graph
// and clones the results out.
//
// A small kernel takes 2 to 5 us, so what such a call costs is the host's work and the launches around
// the kernel.  The same steps from Python (current stream, torch.empty, ctypes, a copy in and a clone
// out around a graph replay) took 17.5 us a call whatever the kernel was; these take about 1 us and one
// launch per kernel.
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/clamp.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/copy.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "kb200.h"

namespace {

constexpr int kMaxBuffers = 16;       // what kb200_plan_run takes

struct Caller {
  kb200_plan* plan;
  c10::Device device{c10::kCUDA, 0};
  std::vector<std::vector<int64_t>> in_shapes, out_shapes;
  std::vector<at::Tensor> fixed_inputs;      // where an input goes that the kernels cannot read as it is
  std::mutex copies;                         // held from such a copy to the launches that read it
};

// The interpreter is left to other threads; taken again on the way out, by an exception too.
struct WithoutInterpreter {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutInterpreter() { PyEval_RestoreThread(state); }
};

constexpr const char* kCapsule = "kb200.caller";

void destroy(PyObject* capsule) { delete static_cast<Caller*>(PyCapsule_GetPointer(capsule, kCapsule)); }

bool read_shapes(PyObject* list, std::vector<std::vector<int64_t>>* out) {
  const Py_ssize_t n = PySequence_Size(list);
  if (n < 0) return false;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* shape = PySequence_GetItem(list, i);
    const Py_ssize_t rank = shape ? PySequence_Size(shape) : -1;
    std::vector<int64_t> dims;
    for (Py_ssize_t d = 0; d < rank; ++d) {
      PyObject* v = PySequence_GetItem(shape, d);
      dims.push_back(v ? PyLong_AsLongLong(v) : -1);
      Py_XDECREF(v);
    }
    Py_XDECREF(shape);
    if (rank < 0 || PyErr_Occurred()) return false;
    out->push_back(std::move(dims));
  }
  return true;
}

// caller(plan address, device index, input shapes, output shapes, fixed input tensors)
PyObject* make_caller(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  unsigned long long plan;
  int device;
  PyObject *in_shapes, *out_shapes, *fixed;
  if (!PyArg_ParseTuple(args, "KiOOO", &plan, &device, &in_shapes, &out_shapes, &fixed)) return nullptr;
  auto c = std::make_unique<Caller>();
  c->plan = reinterpret_cast<kb200_plan*>(plan);
  c->device = c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device));
  if (!read_shapes(in_shapes, &c->in_shapes) || !read_shapes(out_shapes, &c->out_shapes)) return nullptr;
  const Py_ssize_t n = PySequence_Size(fixed);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = PySequence_GetItem(fixed, i);
    if (!t || !THPVariable_Check(t)) {
      Py_XDECREF(t);
      PyErr_SetString(PyExc_TypeError, "fixed inputs must be tensors");
      return nullptr;
    }
    c->fixed_inputs.push_back(THPVariable_Unpack(t));
    Py_DECREF(t);
  }
  if (c->in_shapes.size() > kMaxBuffers || c->out_shapes.size() > kMaxBuffers || c->fixed_inputs.size() != c->in_shapes.size()) {
    PyErr_SetString(PyExc_ValueError, "caller: bad number of inputs or outputs");
    return nullptr;
  }
  return PyCapsule_New(c.release(), kCapsule, destroy);
  END_HANDLE_TH_ERRORS
}

std::string text(c10::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + (shape.size() == 1 ? ",)" : ")");
}

PyObject* raise(int status) {
  PyObject* type = status == KB200_ERR_ARGUMENT || status == KB200_ERR_BOUNDS ? PyExc_ValueError
                   : status == KB200_ERR_UNSUPPORTED                          ? PyExc_NotImplementedError
                                                                              : PyExc_RuntimeError;
  PyErr_Format(type, "kb200: %s (status %d)", kb200_last_error(), status);
  return nullptr;
}

// run(caller, *inputs) -> [outputs]
PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Caller* c = n_args > 0 ? static_cast<Caller*>(PyCapsule_GetPointer(args[0], kCapsule)) : nullptr;
  if (!c) return PyErr_Occurred() ? nullptr : (PyErr_SetString(PyExc_TypeError, "run(caller, *inputs)"), nullptr);
  const size_t n_in = c->in_shapes.size(), n_out = c->out_shapes.size();
  if ((size_t)(n_args - 1) != n_in)
    return PyErr_Format(PyExc_TypeError, "expected %zu inputs, got %zd", n_in, n_args - 1);
  for (size_t i = 0; i < n_in; ++i) {
    if (!THPVariable_Check(args[1 + i])) return PyErr_Format(PyExc_TypeError, "input %zu is not a tensor", i);
    const at::Tensor& t = THPVariable_Unpack(args[1 + i]);
    if (t.sizes() != c10::IntArrayRef(c->in_shapes[i]))
      return PyErr_Format(PyExc_ValueError, "Kiln was compiled for input shape %s, got %s", text(c->in_shapes[i]).c_str(),
                          text(t.sizes()).c_str());
  }
  const c10::cuda::CUDAGuard guard(c->device);
  void* in[kMaxBuffers];
  bool copied = false;
  for (size_t i = 0; i < n_in; ++i) {
    const at::Tensor& t = THPVariable_Unpack(args[1 + i]);
    // read where it is: float32, dense, on this device, 16-byte aligned (128-bit loads, tensor maps); a tensor without memory
    // (zeros that autograd made, a wrapper) has its values copied
    const bool direct = t.layout() == c10::kStrided && t.scalar_type() == c10::kFloat && t.device() == c->device && t.is_contiguous() && !t.is_neg() &&
                        !t._is_zerotensor();
    const void* at = direct ? t.const_data_ptr() : nullptr;
    in[i] = (reinterpret_cast<uintptr_t>(at) & 15) == 0 ? const_cast<void*>(at) : nullptr;
    copied = copied || in[i] == nullptr;
  }
  void* out[kMaxBuffers];
  std::vector<at::Tensor> results;
  results.reserve(n_out);
  for (size_t i = 0; i < n_out; ++i) {
    results.push_back(at::detail::empty_cuda(c->out_shapes[i], c10::kFloat, c->device, std::nullopt));
    out[i] = results[i].data_ptr();
  }
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c->device.index()).stream();
  int status;
  {
    const WithoutInterpreter others_run;
    std::unique_lock<std::mutex> one_copy(c->copies, std::defer_lock);
    if (copied) {
      one_copy.lock();
      const c10::NoGradGuard no_grad;
      for (size_t i = 0; i < n_in; ++i)
        if (in[i] == nullptr) c->fixed_inputs[i].copy_(THPVariable_Unpack(args[1 + i]).detach(), /*non_blocking=*/true);
    }
    status = kb200_plan_run(c->plan, in, (int)n_in, out, (int)n_out, stream);
  }
  if (status != KB200_OK) return raise(status);
  PyObject* list = PyList_New((Py_ssize_t)n_out);
  for (size_t i = 0; list && i < n_out; ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, THPVariable_Wrap(std::move(results[i])));
  return list;
  END_HANDLE_TH_ERRORS
}

// ---- the paged cache (kiln_b200/cache.py) ---------------------------------------------------------
// A step of a server that drafts tokens makes two calls per layer and three more, each of a few microseconds of GPU time: from Python
// (checks, ctypes, streams) a call took 12 to 15 us.

struct CacheCaller {
  kb200_cache* cache;
  c10::Device device{c10::kCUDA, 0};
  int64_t sequences, kv_heads, head_dim, width;      // width: tokens that a sequence may have
  c10::ScalarType type;
};
constexpr const char* kCacheCapsule = "kb200.cache";
void destroy_cache_caller(PyObject* capsule) { delete static_cast<CacheCaller*>(PyCapsule_GetPointer(capsule, kCacheCapsule)); }

// cache_caller(cache address, device index, sequences, kv heads, head dim, dtype code, tokens of a sequence)
PyObject* make_cache_caller(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  unsigned long long cache;
  int device, type;
  long long sequences, kv_heads, head_dim, width;
  if (!PyArg_ParseTuple(args, "KiLLLiL", &cache, &device, &sequences, &kv_heads, &head_dim, &type, &width)) return nullptr;
  auto c = std::make_unique<CacheCaller>();
  c->cache = reinterpret_cast<kb200_cache*>(cache);
  c->device = c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device));
  c->sequences = sequences, c->kv_heads = kv_heads, c->head_dim = head_dim, c->width = width;
  c->type = type == KB200_DTYPE_FP32 ? c10::kFloat : type == KB200_DTYPE_BF16 ? c10::kBFloat16 : c10::kHalf;
  return PyCapsule_New(c.release(), kCacheCapsule, destroy_cache_caller);
  END_HANDLE_TH_ERRORS
}

// What a call raises before it reaches the library.
struct Refused {};
#define REFUSE(type, ...) (PyErr_Format(type, __VA_ARGS__), throw Refused())

CacheCaller& cache_of(PyObject* capsule) {
  if (capsule == Py_None) REFUSE(PyExc_ValueError, "the cache is closed");
  auto* c = static_cast<CacheCaller*>(PyCapsule_GetPointer(capsule, kCacheCapsule));
  if (c == nullptr) throw Refused();
  return *c;
}
const at::Tensor& tensor_of(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) REFUSE(PyExc_TypeError, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}
void on_device(const CacheCaller& c, const at::Tensor& t, const char* name) {
  if (t.device() != c.device) REFUSE(PyExc_ValueError, "%s is on %s, the cache on %s", name, t.device().str().c_str(), c.device.str().c_str());
  if (t.layout() != c10::kStrided) REFUSE(PyExc_TypeError, "%s must be a dense tensor", name);
}
bool has_memory(const at::Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }
// A call's integers as the library takes them.
at::Tensor integers(const CacheCaller& c, PyObject* o, const char* name, c10::IntArrayRef shape) {
  const at::Tensor& t = tensor_of(o, name);
  const bool wide = t.scalar_type() == c10::kLong;
  if (!wide && t.scalar_type() != c10::kInt) REFUSE(PyExc_TypeError, "%s must hold int32 or int64", name);
  if (t.sizes() != shape) REFUSE(PyExc_ValueError, "%s must have shape %s, got %s", name, text(shape).c_str(), text(t.sizes()).c_str());
  on_device(c, t, name);
  if (wide) return at::clamp(t, -2147483648ll, 2147483647ll).to(c10::kInt).contiguous();
  return t.is_contiguous() && has_memory(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
at::Tensor integers_or_none(const CacheCaller& c, PyObject* o, const char* name, int64_t n) { return o == Py_None ? at::Tensor() : integers(c, o, name, {n}); }
const int32_t* at_of(const at::Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.const_data_ptr()) : nullptr; }

// Rows of new tokens, [rows, tokens, heads, head_dim]: copied where the kernels cannot read (or write) them as they are.
struct TokenRows {
  at::Tensor t;
  kb200_rows rows;
  TokenRows(const CacheCaller& c, PyObject* o, const char* name, int64_t heads) : t(tensor_of(o, name)) {
    if (t.dim() != 4 || t.size(3) != c.head_dim || (heads >= 0 && t.size(2) != heads))
      REFUSE(PyExc_ValueError, "%s must be [rows, tokens, %s, %lld], got %s", name, heads >= 0 ? std::to_string(heads).c_str() : "heads", (long long)c.head_dim,
             text(t.sizes()).c_str());
    if (t.scalar_type() != c.type && t.scalar_type() != c10::kFloat) REFUSE(PyExc_TypeError, "%s must be of the cache's type or float32", name);
    on_device(c, t, name);
    take();
  }
  explicit TokenRows(at::Tensor of) : t(std::move(of)) { take(); }
  void take() {
    const int64_t unit = 16 / t.element_size();
    if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(has_memory(t) ? t.const_data_ptr() : nullptr) % 16 != 0 || t.stride(0) % unit || t.stride(1) % unit ||
        t.stride(2) % unit || !has_memory(t)) {
      const c10::NoGradGuard no_grad;
      t = t.clone(at::MemoryFormat::Contiguous);
    }
    rows = kb200_rows{const_cast<void*>(t.const_data_ptr()), t.scalar_type() == c10::kFloat ? KB200_DTYPE_FP32 : t.scalar_type() == c10::kBFloat16 ? KB200_DTYPE_BF16 : KB200_DTYPE_FP16,
                      (int32_t)t.size(2), {t.stride(0), t.stride(1), t.stride(2)}};
  }
};

void batch_ok(const CacheCaller& c, int64_t rows, PyObject* slots) {
  if (slots == Py_None && rows > c.sequences) REFUSE(PyExc_ValueError, "%lld rows, but the cache has %lld sequences", (long long)rows, (long long)c.sequences);
  if (rows >= 2147483647) REFUSE(PyExc_ValueError, "too many rows");
}
int layer_of(PyObject* o) {
  const long layer = PyLong_AsLong(o);
  if (layer == -1 && PyErr_Occurred()) throw Refused();
  return layer < 0 || layer > 2147483647 ? -1 : (int)layer;
}
template <typename F>
PyObject* enqueue(const CacheCaller& c, F&& f) {
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.device.index()).stream();
  int status;
  {
    const WithoutInterpreter others_run;
    status = f(stream);
  }
  if (status != KB200_OK) return raise(status);
  Py_RETURN_NONE;
}
bool n_args(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
  return got == want;
}

// cache_fork / cache_reserve / cache_truncate(cache, integers by sequence)
template <int (*Call)(kb200_cache*, const int32_t*, void*)>
PyObject* by_sequence(PyObject* const* args, Py_ssize_t n, const char* name) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 2)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const at::Tensor values = integers(c, args[1], name, {c.sequences});
    return enqueue(c, [&](cudaStream_t s) { return Call(c.cache, at_of(values), s); });
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
PyObject* cache_fork(PyObject*, PyObject* const* args, Py_ssize_t n) { return by_sequence<kb200_cache_fork>(args, n, "sources"); }
PyObject* cache_reserve(PyObject*, PyObject* const* args, Py_ssize_t n) { return by_sequence<kb200_cache_reserve>(args, n, "counts"); }
PyObject* cache_truncate(PyObject*, PyObject* const* args, Py_ssize_t n) { return by_sequence<kb200_cache_truncate>(args, n, "lengths"); }

// cache_compact(cache)
PyObject* cache_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 1)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    return enqueue(c, [&](cudaStream_t s) { return kb200_cache_compact(c.cache, s); });
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// cache_append(cache, layer, k, v, counts, slots)
PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 6)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const int layer = layer_of(args[1]);
    const TokenRows k(c, args[2], "k", c.kv_heads), v(c, args[3], "v", c.kv_heads);
    if (k.t.sizes() != v.t.sizes() || k.t.scalar_type() != v.t.scalar_type())
      REFUSE(PyExc_ValueError, "k and v must be alike, got %s and %s", text(k.t.sizes()).c_str(), text(v.t.sizes()).c_str());
    const int64_t rows = k.t.size(0), tokens = k.t.size(1);
    batch_ok(c, rows, args[5]);
    const at::Tensor counts = integers_or_none(c, args[4], "counts", rows), slots = integers_or_none(c, args[5], "slots", rows);
    return enqueue(c, [&](cudaStream_t s) { return kb200_cache_append(c.cache, layer, &k.rows, &v.rows, (int)rows, (int)tokens, at_of(counts), at_of(slots), s); });
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// cache_accept(cache, counts, kept)
PyObject* cache_accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 3)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const at::Tensor counts = integers(c, args[1], "counts", {c.sequences});
    at::Tensor kept;
    if (args[2] != Py_None) {
      const at::Tensor& t = tensor_of(args[2], "kept");
      if (t.dim() != 2 || t.size(1) >= 2147483647) REFUSE(PyExc_ValueError, "kept must be [sequences, width]");
      kept = integers(c, args[2], "kept", {c.sequences, t.size(1)});
    }
    static const int32_t nothing = 0;                  // (what a tensor of no width points to is not read)
    const int32_t* const at = kept.defined() && kept.numel() == 0 ? &nothing : at_of(kept);
    return enqueue(c, [&](cudaStream_t s) { return kb200_cache_accept(c.cache, at_of(counts), at, kept.defined() ? (int)kept.size(1) : 0, s); });
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// A call's mask, and its strides by batch row, token and drafted token.
at::Tensor mask_of(const CacheCaller& c, PyObject* o, int64_t rows, int64_t tokens, int64_t (&stride)[3]) {
  at::Tensor mask;
  if (o == Py_None) return mask;
  if (!THPVariable_Check(o) || THPVariable_Unpack(o).scalar_type() != c10::kBool) REFUSE(PyExc_TypeError, "mask must be a bool tensor");
  mask = THPVariable_Unpack(o);
  on_device(c, mask, "mask");
  const bool each = mask.dim() == 3;
  if (mask.dim() < 2 || mask.dim() > 3 || mask.size(-1) != tokens || mask.size(-2) != tokens || (each && mask.size(0) != rows))
    REFUSE(PyExc_ValueError, "mask must be [%lld, %lld] or [%lld, %lld, %lld], got %s", (long long)tokens, (long long)tokens, (long long)rows, (long long)tokens,
           (long long)tokens, text(mask.sizes()).c_str());
  if (!has_memory(mask)) mask = mask.clone();
  for (int i = 0; i < (int)mask.dim(); ++i) stride[i + (each ? 0 : 1)] = mask.stride(i);
  return mask;
}
double scale_of(const CacheCaller& c, PyObject* o) {
  if (o == Py_None) return 1.0 / std::sqrt((double)c.head_dim);
  const double scale = PyFloat_AsDouble(o);
  if (scale == -1.0 && PyErr_Occurred()) throw Refused();
  return scale;
}
// A number of tokens.
int tokens_of(PyObject* o, const char* name, long least) {
  const long long value = PyLong_Check(o) && !PyBool_Check(o) ? PyLong_AsLongLong(o) : -1;
  PyErr_Clear();
  if (value < least || value > 2147483647) REFUSE(PyExc_ValueError, "%s must be an integer from %ld on", name, least);
  return (int)value;
}
// float32 numbers that a call reads.
const at::Tensor& floats_of(const CacheCaller& c, PyObject* o, const char* name, c10::IntArrayRef shape) {
  const at::Tensor& t = tensor_of(o, name);
  if (t.scalar_type() != c10::kFloat) REFUSE(PyExc_TypeError, "%s must hold float32", name);
  if (t.sizes() != shape) REFUSE(PyExc_ValueError, "%s must have shape %s, got %s", name, text(shape).c_str(), text(t.sizes()).c_str());
  on_device(c, t, name);
  return t;
}
// ... and that it writes.
const at::Tensor& floats_to(const CacheCaller& c, PyObject* o, const char* name, c10::IntArrayRef shape) {
  const at::Tensor& t = floats_of(c, o, name, shape);
  if (!has_memory(t)) REFUSE(PyExc_ValueError, "%s has no memory of its own", name);
  if (t.requires_grad()) REFUSE(PyExc_ValueError, "%s requires a gradient", name);
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes) REFUSE(PyExc_ValueError, "elements of %s share memory", name);
  return t;
}
// Whether two tensors' memory, from the first to the last element of each, has bytes in common.
bool near_each_other(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0 || !has_memory(a) || !has_memory(b)) return false;
  auto extent = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);      // (strides are not negative)
    return (last + 1) * (int64_t)t.element_size();
  };
  const char *const at_a = static_cast<const char*>(a.const_data_ptr()), *const at_b = static_cast<const char*>(b.const_data_ptr());
  return at_a < at_b + extent(b) && at_b < at_a + extent(a);
}
void apart(const at::Tensor& a, const at::Tensor& b, const char* name_a, const char* name_b) {
  if (near_each_other(a, b)) REFUSE(PyExc_ValueError, "%s shares memory with %s", name_a, name_b);
}

// cache_attend(cache, layer, q, mask, counts, slots, scale, out, window, sinks, places, lse) -> out
PyObject* cache_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 12)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const int layer = layer_of(args[1]);
    const TokenRows q(c, args[2], "q", -1);
    const int64_t rows = q.t.size(0), tokens = q.t.size(1), heads = q.t.size(2);
    if (heads == 0 || heads % c.kv_heads != 0) REFUSE(PyExc_ValueError, "%lld heads are no multiple of the cache's %lld", (long long)heads, (long long)c.kv_heads);
    batch_ok(c, rows, args[5]);
    if (tokens >= 2147483647 || heads >= 2147483647) REFUSE(PyExc_ValueError, "too many tokens or heads");
    int64_t mask_stride[3] = {0, 0, 0};
    const at::Tensor mask = mask_of(c, args[3], rows, tokens, mask_stride);
    const at::Tensor counts = integers_or_none(c, args[4], "counts", rows), slots = integers_or_none(c, args[5], "slots", rows);
    const double scale = scale_of(c, args[6]);
    const int window = args[8] == Py_None ? 0 : tokens_of(args[8], "window", 1), sinks = tokens_of(args[9], "sinks", 0);
    if (window == 0 && (sinks != 0 || args[10] != Py_None)) REFUSE(PyExc_ValueError, "sinks and places go with a window");
    at::Tensor places, lse;
    int64_t lse_stride[3] = {0, 0, 0};
    if (args[10] != Py_None) places = integers(c, args[10], "places", {rows, tokens});
    if (args[11] != Py_None) {
      lse = floats_to(c, args[11], "lse", {rows, tokens, heads});
      apart(lse, q.t, "lse", "q");
      for (int i = 0; i < 3; ++i) lse_stride[i] = lse.stride(i);
    }
    const bool beside = window > 0 || lse.defined();
    at::Tensor out;
    if (args[7] == Py_None) {
      out = at::detail::empty_cuda({rows, tokens, heads, c.head_dim}, c.type, c.device, std::nullopt);
    } else {
      if (!THPVariable_Check(args[7])) REFUSE(PyExc_TypeError, "out must be a tensor");
      out = THPVariable_Unpack(args[7]);
      if (out.sizes() != q.t.sizes() || out.scalar_type() != c.type || out.device() != c.device || out.layout() != c10::kStrided || !has_memory(out))
        REFUSE(PyExc_ValueError, "out must be %s of the cache's type on its device", text(q.t.sizes()).c_str());
      if (out.requires_grad()) REFUSE(PyExc_ValueError, "out requires a gradient");
      // rows are written while others of q are still read: the same tensor is fine, part of it is not
      if (at::has_internal_overlap(out) == at::MemOverlap::Yes) REFUSE(PyExc_ValueError, "elements of out share memory");
      if (at::get_overlap_status(out, q.t) == at::MemOverlapStatus::Partial) REFUSE(PyExc_ValueError, "out shares part of q's memory");
    }
    if (lse.defined()) apart(lse, out, "lse", "out");
    const TokenRows to(out);
    if (rows > 0 && tokens > 0) {
      const uint64_t bytes = beside ? kb200_cache_attend_window_workspace(c.cache, (int)rows, (int)tokens, (int)heads, window, sinks)
                                    : kb200_cache_attend_workspace(c.cache, (int)rows, (int)tokens, (int)heads);
      // the kernels write into it (said first: it raises for a tensor that may not change)
      if (args[7] != Py_None && to.t.is_same(out)) out.unsafeGetTensorImpl()->bump_version();
      if (lse.defined()) lse.unsafeGetTensorImpl()->bump_version();
      at::Tensor workspace;                            // (of this call alone; its memory is used again behind the kernels, on their stream)
      if (bytes > 0) workspace = at::detail::empty_cuda({(int64_t)bytes}, c10::kByte, c.device, std::nullopt);
      PyObject* const done = enqueue(c, [&](cudaStream_t s) {
        if (beside)
          return kb200_cache_attend_window(c.cache, layer, &q.rows, &to.rows, (int)rows, (int)tokens, mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr,
                                           mask_stride, at_of(counts), at_of(slots), (float)scale, window, sinks, at_of(places),
                                           lse.defined() ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr, lse_stride, bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, s);
        return kb200_cache_attend(c.cache, layer, &q.rows, &to.rows, (int)rows, (int)tokens, mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr,
                                  mask_stride, at_of(counts), at_of(slots), (float)scale, bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, s);
      });
      if (done == nullptr) return nullptr;
      Py_DECREF(done);
      if (args[7] != Py_None && !to.t.is_same(out)) {
        const c10::NoGradGuard no_grad;
        out.copy_(to.t);
      }
    }
    if (args[7] != Py_None) {
      Py_INCREF(args[7]);
      return args[7];
    }
    return THPVariable_Wrap(std::move(out));
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// cache_release(cache, window, sinks)
PyObject* cache_release(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 3)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const int window = tokens_of(args[1], "window", 1), sinks = tokens_of(args[2], "sinks", 0);
    return enqueue(c, [&](cudaStream_t s) { return kb200_cache_release(c.cache, window, sinks, s); });
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// A number for each token of each sequence, [sequences, width] of float32: where a call reads and writes them.  What is not laid out row by row is copied.
struct TokenWeights {
  at::Tensor from, to, result;         // result: what the caller gets
  TokenWeights(const CacheCaller& c, PyObject* weights, PyObject* out) {
    const std::vector<int64_t> shape = {c.sequences, c.width};
    if (weights != Py_None) {
      from = floats_of(c, weights, "weights", shape);
      if (!has_memory(from) || !by_rows(from)) {
        const c10::NoGradGuard no_grad;
        from = from.clone(at::MemoryFormat::Contiguous);
      }
    }
    if (out == Py_None) {
      to = result = at::detail::empty_cuda(shape, c10::kFloat, c.device, std::nullopt);
      return;
    }
    to = result = floats_to(c, out, "out", shape);
    if (from.defined() && near_each_other(to, from) && !same_or_beside(to, from)) REFUSE(PyExc_ValueError, "out shares part of the weights' memory");
    if (!by_rows(to)) to = at::detail::empty_cuda(shape, c10::kFloat, c.device, std::nullopt);
  }
  // The same numbers, or rows that lie side by side in a third tensor's.
  static bool same_or_beside(const at::Tensor& a, const at::Tensor& b) {
    if (!by_rows(a) || !by_rows(b) || (a.size(0) > 1 && a.stride(0) != b.stride(0))) return false;
    const int64_t bytes = static_cast<const char*>(a.const_data_ptr()) - static_cast<const char*>(b.const_data_ptr());
    if (bytes == 0) return true;
    const int64_t row = a.stride(0) * 4, width = a.size(1) * 4, off = a.size(0) > 1 ? (bytes % row + row) % row : 0;
    return off >= width && row - off >= width;
  }
  static bool by_rows(const at::Tensor& t) { return t.stride(1) == 1 && (t.size(0) == 1 || t.stride(0) >= t.size(1)); }
  const float* read() const { return from.defined() ? static_cast<const float*>(from.const_data_ptr()) : nullptr; }
  int64_t read_stride() const { return from.defined() ? from.stride(0) : 0; }
  // (said first: it raises for a tensor that may not change)
  float* write() const {
    if (to.is_same(result)) to.unsafeGetTensorImpl()->bump_version();
    return static_cast<float*>(to.mutable_data_ptr());
  }
  PyObject* done(PyObject* out) {
    if (!to.is_same(result)) {
      const c10::NoGradGuard no_grad;
      result.copy_(to);
    }
    if (out == Py_None) return THPVariable_Wrap(std::move(result));
    Py_INCREF(out);
    return out;
  }
};

// cache_weigh(cache, layer, q, lse, weights, mask, counts, slots, scale, committed, out) -> out
PyObject* cache_weigh(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 11)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const int layer = layer_of(args[1]);
    const TokenRows q(c, args[2], "q", -1);
    const int64_t rows = q.t.size(0), tokens = q.t.size(1), heads = q.t.size(2);
    if (heads == 0 || heads % c.kv_heads != 0) REFUSE(PyExc_ValueError, "%lld heads are no multiple of the cache's %lld", (long long)heads, (long long)c.kv_heads);
    batch_ok(c, rows, args[7]);
    if (tokens >= 2147483647 || heads >= 2147483647) REFUSE(PyExc_ValueError, "too many tokens or heads");
    at::Tensor lse = floats_of(c, args[3], "lse", {rows, tokens, heads});
    if (!has_memory(lse)) lse = lse.clone();
    int64_t mask_stride[3] = {0, 0, 0};
    const at::Tensor mask = mask_of(c, args[5], rows, tokens, mask_stride);
    const at::Tensor counts = integers_or_none(c, args[6], "counts", rows), slots = integers_or_none(c, args[7], "slots", rows);
    const double scale = scale_of(c, args[8]);
    const int committed = PyObject_IsTrue(args[9]);
    if (committed < 0) return nullptr;
    TokenWeights w(c, args[4], args[10]);
    apart(w.to, q.t, "out", "q");
    apart(w.to, lse, "out", "lse");
    const int64_t lse_stride[3] = {lse.stride(0), lse.stride(1), lse.stride(2)};
    float* const to = w.write();
    PyObject* const done = enqueue(c, [&](cudaStream_t s) {
      return kb200_cache_weigh(c.cache, layer, &q.rows, static_cast<const float*>(lse.const_data_ptr()), lse_stride, (int)rows, (int)tokens,
                               mask.defined() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr, mask_stride, at_of(counts), at_of(slots), (float)scale, committed, w.read(),
                               w.read_stride(), to, w.to.stride(0), s);
    });
    if (done == nullptr) return nullptr;
    Py_DECREF(done);
    return w.done(args[10]);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// cache_evict(cache, weights, keep, recent, sinks, out) -> out
PyObject* cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 6)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    if (args[1] == Py_None) REFUSE(PyExc_TypeError, "weights must be a tensor");
    const at::Tensor keep = integers(c, args[2], "keep", {c.sequences});
    const int recent = tokens_of(args[3], "recent", 0), sinks = tokens_of(args[4], "sinks", 0);
    TokenWeights w(c, args[1], args[5]);
    const uint64_t bytes = kb200_cache_evict_workspace(c.cache);
    const at::Tensor workspace = at::detail::empty_cuda({(int64_t)bytes}, c10::kByte, c.device, std::nullopt);
    float* const to = w.write();
    PyObject* const done = enqueue(c, [&](cudaStream_t s) {
      return kb200_cache_evict(c.cache, w.read(), w.read_stride(), at_of(keep), recent, sinks, to, w.to.stride(0), workspace.mutable_data_ptr(), bytes, s);
    });
    if (done == nullptr) return nullptr;
    Py_DECREF(done);
    return w.done(args[5]);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// Rows over a vocabulary, [rows, tokens, vocabulary]: copied where the kernels cannot read them as they are.
struct VocabularyRows {
  at::Tensor t;
  kb200_scores scores;
  VocabularyRows(const CacheCaller& c, PyObject* o, const char* name, c10::IntArrayRef shape) : t(tensor_of(o, name)) {
    if (t.dim() != 3 || (!shape.empty() && t.sizes() != shape))
      REFUSE(PyExc_ValueError, "%s must be %s, got %s", name, shape.empty() ? "[rows, tokens, vocabulary]" : text(shape).c_str(), text(t.sizes()).c_str());
    const c10::ScalarType type = t.scalar_type();
    if (type != c10::kFloat && type != c10::kBFloat16 && type != c10::kHalf) REFUSE(PyExc_TypeError, "%s must hold float32, bfloat16 or float16", name);
    on_device(c, t, name);
    if (!has_memory(t) || (t.stride(2) != 1 && t.size(2) != 1)) {
      const c10::NoGradGuard no_grad;
      t = t.clone(at::MemoryFormat::Contiguous);
    }
    scores = kb200_scores{t.const_data_ptr(), type == c10::kFloat ? KB200_DTYPE_FP32 : type == c10::kBFloat16 ? KB200_DTYPE_BF16 : KB200_DTYPE_FP16, 0, {t.stride(0), t.stride(1)}};
  }
};

// cache_verify(cache, logits, tokens, uniform, draft, parents, counts, slots, temperature) -> (n_accepted, accepted, following)
PyObject* cache_verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!n_args(n, 9)) return nullptr;
  try {
    CacheCaller& c = cache_of(args[0]);
    const c10::cuda::CUDAGuard guard(c.device);
    const VocabularyRows logits(c, args[1], "logits", {});
    const int64_t rows = logits.t.size(0), tokens = logits.t.size(1), vocab = logits.t.size(2);
    batch_ok(c, rows, args[7]);
    if (rows > 1 << 20 || tokens > 512 || vocab < 1 || vocab >= 1 << 30)
      REFUSE(PyExc_ValueError, "logits must be of at most 2^20 rows, 512 tokens and fewer than 2^30 numbers each, got %s", text(logits.t.sizes()).c_str());
    const at::Tensor drafted = integers(c, args[2], "tokens", {rows, tokens});
    auto contiguous = [&](PyObject* o, const char* name, c10::IntArrayRef shape) {
      const at::Tensor& t = floats_of(c, o, name, shape);
      return t.is_contiguous() && has_memory(t) ? t : t.clone(at::MemoryFormat::Contiguous);
    };
    const at::Tensor uniform = contiguous(args[3], "uniform", {rows, tokens});
    std::unique_ptr<VocabularyRows> draft;
    if (args[4] != Py_None) draft = std::make_unique<VocabularyRows>(c, args[4], "draft", logits.t.sizes());
    at::Tensor parents, temperature;
    int64_t parents_stride = tokens;
    if (args[5] != Py_None) {
      const bool each = tensor_of(args[5], "parents").dim() != 1;
      parents = each ? integers(c, args[5], "parents", {rows, tokens}) : integers(c, args[5], "parents", {tokens});
      parents_stride = each ? tokens : 0;
    }
    const at::Tensor counts = integers_or_none(c, args[6], "counts", rows), slots = integers_or_none(c, args[7], "slots", rows);
    if (args[8] != Py_None) temperature = contiguous(args[8], "temperature", {rows});
    auto whole = [&](c10::IntArrayRef shape) { return at::detail::empty_cuda(shape, c10::kInt, c.device, std::nullopt); };
    at::Tensor n_accepted = whole({c.sequences}), accepted = whole({c.sequences, tokens}), following = whole({c.sequences});
    const uint64_t bytes = kb200_cache_verify_workspace(c.cache, (int)rows, (int)tokens, (int)vocab);
    at::Tensor workspace;
    if (bytes > 0) workspace = at::detail::empty_cuda({(int64_t)bytes}, c10::kByte, c.device, std::nullopt);
    PyObject* const done = enqueue(c, [&](cudaStream_t s) {
      return kb200_cache_verify(c.cache, &logits.scores, draft ? &draft->scores : nullptr, (int)rows, (int)tokens, (int)vocab, at_of(drafted), at_of(parents), parents_stride,
                                static_cast<const float*>(uniform.const_data_ptr()), temperature.defined() ? static_cast<const float*>(temperature.const_data_ptr()) : nullptr,
                                at_of(counts), at_of(slots), static_cast<int32_t*>(n_accepted.mutable_data_ptr()), static_cast<int32_t*>(accepted.mutable_data_ptr()),
                                static_cast<int32_t*>(following.mutable_data_ptr()), bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, s);
    });
    if (done == nullptr) return nullptr;
    Py_DECREF(done);
    PyObject* const a = THPVariable_Wrap(std::move(n_accepted));
    PyObject* const b = THPVariable_Wrap(std::move(accepted));
    PyObject* const f = THPVariable_Wrap(std::move(following));
    PyObject* const all = a && b && f ? PyTuple_Pack(3, a, b, f) : nullptr;
    Py_XDECREF(a), Py_XDECREF(b), Py_XDECREF(f);
    return all;
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

PyMethodDef methods[] = {
    {"cache_caller", make_cache_caller, METH_VARARGS, "cache_caller(cache, device, sequences, kv_heads, head_dim, dtype, tokens)"},
    {"cache_fork", fast(cache_fork), METH_FASTCALL, "cache_fork(cache, sources)"},
    {"cache_reserve", fast(cache_reserve), METH_FASTCALL, "cache_reserve(cache, counts)"},
    {"cache_truncate", fast(cache_truncate), METH_FASTCALL, "cache_truncate(cache, lengths)"},
    {"cache_compact", fast(cache_compact), METH_FASTCALL, "cache_compact(cache)"},
    {"cache_append", fast(cache_append), METH_FASTCALL, "cache_append(cache, layer, k, v, counts, slots)"},
    {"cache_accept", fast(cache_accept), METH_FASTCALL, "cache_accept(cache, counts, kept)"},
    {"cache_attend", fast(cache_attend), METH_FASTCALL, "cache_attend(cache, layer, q, mask, counts, slots, scale, out, window, sinks, places, lse) -> out"},
    {"cache_release", fast(cache_release), METH_FASTCALL, "cache_release(cache, window, sinks)"},
    {"cache_weigh", fast(cache_weigh), METH_FASTCALL, "cache_weigh(cache, layer, q, lse, weights, mask, counts, slots, scale, committed, out) -> out"},
    {"cache_evict", fast(cache_evict), METH_FASTCALL, "cache_evict(cache, weights, keep, recent, sinks, out) -> out"},
    {"cache_verify", fast(cache_verify), METH_FASTCALL,
     "cache_verify(cache, logits, tokens, uniform, draft, parents, counts, slots, temperature) -> (n_accepted, accepted, following)"},
    {"caller", make_caller, METH_VARARGS, "caller(plan, device, input_shapes, output_shapes, fixed_inputs)"},
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(run)), METH_FASTCALL, "run(caller, *inputs) -> list of output tensors"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kb200_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kb200_call() { return PyModule_Create(&module); }
