// The checks and launches behind the decoding-step operators of
// neso_b200.ops, as a Python extension module. One of their calls passes 5 to
// 12 tensors and as many strides; reading them through Python attributes and
// ctypes took 16 to 30 us, several times what the small kernels run for
// (here 3 to 6 us). The kernels themselves are reached through the addresses of
// the C entry points that neso_b200._lib has loaded (set_entry_points), so
// this module links against torch only and both see one library.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/neso_b200.h"

namespace {

struct Entries {
  decltype(&neso_set_device) set_device;
  decltype(&neso_rope_paged_append) rope_paged_append;
  decltype(&neso_paged_attention) paged_attention;
  decltype(&neso_paged_attention_workspace) paged_attention_workspace;
  decltype(&neso_kv_evict) kv_evict;
  decltype(&neso_process_logits) process_logits;
} entry;
PyObject* raise_status = nullptr;  // raise_status(code, function) raises NesoError

// A refused argument: thrown by the checks, turned into the Python exception
// at the module's boundary.
struct Refusal {
  PyObject* type;
  std::string what;
};
[[noreturn]] void type_error(std::string what) { throw Refusal{PyExc_TypeError, std::move(what)}; }
[[noreturn]] void value_error(std::string what) { throw Refusal{PyExc_ValueError, std::move(what)}; }
struct PythonError {};  // an exception is set already

std::string str(int64_t x) { return std::to_string(x); }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}

using Types = std::initializer_list<at::ScalarType>;

// A CUDA tensor of one of `types` with `dim` dimensions on `device`.
const at::Tensor& cuda_tensor(PyObject* o, const char* name, Types types, int64_t dim, c10::Device device) {
  const at::Tensor& t = tensor(o, name);
  if (!t.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor (got " + t.device().str() + ")");
  if (t.device() != device) {
    value_error(std::string(name) + " is on " + t.device().str() + ", the other tensors on " + device.str());
  }
  bool known = false;
  for (at::ScalarType s : types) known = known || t.scalar_type() == s;
  if (!known) {
    std::string list;
    for (at::ScalarType s : types) list += (list.empty() ? "" : " or ") + std::string(c10::toString(s));
    type_error(std::string(name) + " must be " + list + " (got " + c10::toString(t.scalar_type()) + ")");
  }
  if (t.dim() != dim) value_error(std::string(name) + " must have " + str(dim) + " dimensions (got " + str(t.dim()) + ")");
  return t;
}

c10::Device device_of(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (!t.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor (got " + t.device().str() + ")");
  return t.device();
}

// The last dimension has to be contiguous (a length of one always is).
void rows(const at::Tensor& t, const char* name) {
  if (t.size(-1) > 1 && t.stride(-1) != 1) {
    value_error(std::string("the last dimension of ") + name + " must be contiguous");
  }
}

// Stride of a dimension; 0 where its length leaves the stride without a meaning.
int64_t step_of(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// The dimensions of `t` that are longer than one, the widest stride first.
struct Dims {
  int n = 0;
  int64_t size[4], stride[4];
};
Dims dims_of(const at::Tensor& t) {
  Dims d;
  const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
  for (size_t i = 0; i < sizes.size(); ++i) {
    if (sizes[i] <= 1) continue;
    int at = d.n++;
    for (; at > 0 && d.stride[at - 1] < strides[i]; --at) {
      d.size[at] = d.size[at - 1];
      d.stride[at] = d.stride[at - 1];
    }
    d.size[at] = sizes[i];
    d.stride[at] = strides[i];
  }
  return d;
}

// A tensor that is written to: each step of a dimension passes all that the
// narrower dimensions hold, so that no two elements are one.
void written(const at::Tensor& t, const char* name) {
  if (t.numel() == 0) return;
  const Dims d = dims_of(t);
  int64_t span = 1;
  for (int i = d.n - 1; i >= 0; --i) {
    if (d.stride[i] < span) {
      value_error(std::string(name) + " is written to and must not be an expanded view or overlap itself");
    }
    span += (d.size[i] - 1) * d.stride[i];
  }
}

struct Extent {
  uintptr_t first, end;
};
Extent extent(const at::Tensor& t) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {first, first};
  int64_t span = 1;
  for (int64_t i = 0; i < t.dim(); ++i) span += (t.size(i) - 1) * t.stride(i);
  return {first, first + static_cast<uintptr_t>(span) * t.element_size()};
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const Extent x = extent(a), y = extent(b);
  return x.first < y.end && y.first < x.end;
}
// Whether elements [lo, hi) hold one of the view of dimensions i and on of d
// that starts at 0.
bool holds(const Dims& d, int i, int64_t lo, int64_t hi) {
  if (hi <= 0) return false;
  if (i == d.n) return lo <= 0;
  int64_t span = 1;  // of one step
  for (int j = i + 1; j < d.n; ++j) span += (d.size[j] - 1) * d.stride[j];
  const int64_t step = d.stride[i];
  if (step == 0) return holds(d, i + 1, lo, hi);
  const int64_t first = lo < span ? 0 : (lo - span) / step + 1;  // the first step that ends behind lo
  for (int64_t x = first; x < d.size[i] && x * step < hi; ++x) {
    if (lo <= x * step && x * step < hi) return true;  // its first element
    if (holds(d, i + 1, lo - x * step, hi - x * step)) return true;
  }
  return false;
}

// An output must not touch an input, None or a tensor, or a cache (which may
// surround it: a buffer that holds pages and other things).
void apart(const at::Tensor& out, const char* name, PyObject* other, const char* what) {
  if (other == Py_None || !overlap(out, THPVariable_Unpack(other))) return;
  value_error(std::string(name) + " overlaps " + what);
}
void apart(const at::Tensor& out, const char* name, const at::Tensor& cache, const char* what) {
  if (!overlap(out, cache)) return;
  const Extent x = extent(out);
  const int64_t size = cache.element_size();
  const int64_t lo = static_cast<int64_t>(x.first - reinterpret_cast<uintptr_t>(cache.data_ptr()));
  const int64_t hi = static_cast<int64_t>(x.end - reinterpret_cast<uintptr_t>(cache.data_ptr()));
  // Whole elements of the cache: floor and ceiling of bytes that may be negative.
  if (holds(dims_of(cache), 0, lo >= 0 ? lo / size : -((-lo + size - 1) / size), hi >= 0 ? (hi + size - 1) / size : 0)) {
    value_error(std::string(name) + " overlaps " + what);
  }
}

// An output may be the input itself or must not touch it.
void same_or_apart(const at::Tensor& a, const at::Tensor& b, const char* what) {
  if (!overlap(a, b)) return;
  bool same = a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes();
  for (int64_t i = 0; same && i < a.dim(); ++i) same = step_of(a, i) == step_of(b, i);
  if (same) return;
  value_error(std::string(what) + " overlap without being the same tensor");
}

int32_t size32(int64_t n, const char* name) {
  if (n > INT32_MAX) value_error(std::string(name) + " is too large (" + str(n) + ")");
  return static_cast<int32_t>(n);
}

int32_t int_arg(PyObject* o, const char* name) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw PythonError{};
  if (x > INT32_MAX || x < INT32_MIN) value_error(std::string(name) + " is out of range (" + str(x) + ")");
  return static_cast<int32_t>(x);
}
float float_arg(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw PythonError{};
  return static_cast<float>(x);
}

int32_t code_of(at::ScalarType s) {
  return s == at::kHalf ? NESO_F16 : s == at::kBFloat16 ? NESO_BF16 : NESO_F32;
}

// A pair of caches [num_pages, Hkv, page_size, D] of one 16-bit type.
struct Caches {
  const at::Tensor &k, &v;
  int32_t pages, heads, page_size, dim;
};
Caches caches(PyObject* ko, PyObject* vo, c10::Device device) {
  const at::Tensor& k = cuda_tensor(ko, "k_cache", {at::kHalf, at::kBFloat16}, 4, device);
  const at::Tensor& v = cuda_tensor(vo, "v_cache", {k.scalar_type()}, 4, device);
  if (k.sizes() != v.sizes()) value_error("k_cache and v_cache must share one [num_pages, Hkv, page_size, D] shape");
  rows(k, "k_cache");
  rows(v, "v_cache");
  return {k, v, size32(k.size(0), "num_pages"), size32(k.size(1), "Hkv"), size32(k.size(2), "page_size"),
          size32(k.size(3), "D")};
}

const at::Tensor& table(PyObject* o, const char* name, int64_t batch, c10::Device device) {
  const at::Tensor& t = cuda_tensor(o, name, {at::kInt}, 2, device);
  rows(t, name);
  if (t.size(0) != batch) value_error(std::string(name) + " must have one row per sequence (" + str(batch) + ")");
  size32(t.size(1), name);
  return t;
}

const at::Tensor& vector(PyObject* o, const char* name, at::ScalarType type, int64_t n, c10::Device device) {
  const at::Tensor& t = cuda_tensor(o, name, {type}, 1, device);
  rows(t, name);
  if (t.size(0) != n) value_error(std::string(name) + " must have " + str(n) + " elements (got " + str(t.size(0)) + ")");
  return t;
}

const at::Tensor& weights_of(PyObject* o, const char* name, int64_t batch, int64_t heads, int64_t tokens,
                             c10::Device device) {
  const at::Tensor& t = cuda_tensor(o, name, {at::kFloat}, 3, device);
  rows(t, name);
  if (t.size(0) != batch || t.size(1) != heads || t.size(2) < tokens) {
    value_error(std::string(name) + " must be [" + str(batch) + ", " + str(heads) + ", at least " + str(tokens) +
                " tokens]");
  }
  return t;
}

template <class T>
T* data(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <class T>
T* data_or_null(PyObject* o) {
  return o == Py_None ? nullptr : static_cast<T*>(THPVariable_Unpack(o).data_ptr());
}

// A new tensor, straight from the CUDA allocator on the current stream (through
// the dispatcher it takes half a microsecond more).
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, c10::nullopt));
}

neso_stream_t stream_on(c10::Device device) {
  const int rc = entry.set_device(device.index());
  if (rc != NESO_OK) throw rc;
  return c10::cuda::getCurrentCUDAStream(device.index()).stream();
}

PyObject* rope_paged_append(PyObject* const* a) {
  const c10::Device device = device_of(a[0], "q");
  const c10::cuda::CUDAGuard guard(device);  // the caller's device is back on return
  const at::Tensor& q = cuda_tensor(a[0], "q", {at::kHalf, at::kBFloat16}, 3, device);
  const Caches c = caches(a[7], a[8], device);
  const int64_t N = q.size(0), hq = q.size(1);
  const at::Tensor& k = cuda_tensor(a[1], "k", {q.scalar_type()}, 3, device);
  const at::Tensor& v = cuda_tensor(a[2], "v", {q.scalar_type()}, 3, device);
  if (k.size(0) != N || k.size(1) != c.heads || k.size(2) != c.dim || v.sizes() != k.sizes()) {
    value_error("k and v must be [" + str(N) + ", " + str(c.heads) + ", " + str(c.dim) + "]");
  }
  if (q.size(2) != c.dim || c.k.scalar_type() != q.scalar_type()) {
    value_error("q and the cache must share one head_dim and dtype");
  }
  rows(q, "q");
  rows(k, "k");
  rows(v, "v");
  const at::Tensor& cos = cuda_tensor(a[3], "cos", {at::kFloat}, 2, device);
  const at::Tensor& sin = cuda_tensor(a[4], "sin", {at::kFloat}, 2, device);
  if (!cos.is_contiguous() || !sin.is_contiguous()) value_error("cos and sin must be contiguous");
  if (cos.sizes() != sin.sizes()) value_error("cos and sin must share one shape");
  const int64_t pos_dim = tensor(a[5], "positions").dim();
  const at::Tensor& pos = cuda_tensor(a[5], "positions", {at::kInt}, pos_dim == 1 ? 1 : 2, device);
  const int64_t axes = pos_dim == 1 ? 1 : pos.size(0);
  if (pos.size(-1) != N || !pos.is_contiguous()) {
    value_error("positions must be contiguous [" + str(N) + "] or [axes, " + str(N) + "]");
  }
  int32_t widths[16];
  const bool given = a[9] != Py_None;
  if (!given && axes != 1) value_error("several position axes need sections");
  if (given) {
    PyObject* seq = PySequence_Fast(a[9], "sections must be a sequence of widths");
    if (seq == nullptr) throw PythonError{};
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    bool ok = n == axes && n <= 16;
    bool bad = false;
    for (Py_ssize_t i = 0; ok && !bad && i < n; ++i) {
      const long long w = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
      bad = w == -1 && PyErr_Occurred();
      widths[i] = w < INT32_MIN || w > INT32_MAX ? -1 : static_cast<int32_t>(w);
    }
    Py_DECREF(seq);
    if (bad) throw PythonError{};
    if (!ok) value_error("sections must have one width per axis (" + str(axes) + ")");
  }
  const at::Tensor& slots = vector(a[6], "slots", at::kLong, N, device);
  written(c.k, "k_cache");
  written(c.v, "v_cache");
  at::Tensor out;
  if (a[10] == Py_None) {
    out = empty({N, hq, c.dim}, q.scalar_type(), device);
  } else {
    out = cuda_tensor(a[10], "out", {q.scalar_type()}, 3, device);
    if (out.sizes() != q.sizes() || !out.is_contiguous()) value_error("out must be contiguous and of q's shape");
    same_or_apart(out, q, "out and q");
    static const char* const names[9] = {"q", "k", "v", "cos", "sin", "positions", "slots", "k_cache", "v_cache"};
    for (int i = 1; i < 7; ++i) apart(out, "out", a[i], names[i]);
    apart(out, "out", c.k, names[7]);
    apart(out, "out", c.v, names[8]);
  }
  const neso_stream_t stream = stream_on(device);
  const int rc = entry.rope_paged_append(
      q.data_ptr(), k.data_ptr(), v.data_ptr(), data<float>(cos), data<float>(sin), data<int32_t>(pos),
      data<int64_t>(slots), out.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), code_of(q.scalar_type()), size32(N, "N"),
      size32(hq, "Hq"), c.heads, c.dim, size32(cos.size(1), "half"), size32(cos.size(0), "cos"), size32(axes, "axes"),
      given ? widths : nullptr, step_of(q, 0), step_of(q, 1), step_of(k, 0), step_of(k, 1), step_of(v, 0), step_of(v, 1), c.pages,
      c.page_size, step_of(c.k, 0), step_of(c.k, 1), step_of(c.k, 2), step_of(c.v, 0), step_of(c.v, 1), step_of(c.v, 2), stream);
  if (rc != NESO_OK) throw rc;
  return a[10] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[10]);
}

PyObject* paged_attention(PyObject* const* a) {
  const c10::Device device = device_of(a[0], "q");
  const c10::cuda::CUDAGuard guard(device);  // the caller's device is back on return
  const at::Tensor& q = cuda_tensor(a[0], "q", {at::kHalf, at::kBFloat16}, 3, device);
  rows(q, "q");
  const Caches c = caches(a[1], a[2], device);
  const int64_t B = q.size(0), hq = q.size(1);
  if (q.size(2) != c.dim || c.k.scalar_type() != q.scalar_type()) {
    value_error("q and the cache must share one head_dim and dtype");
  }
  const at::Tensor& tables = table(a[3], "block_tables", B, device);
  const at::Tensor& lens = vector(a[4], "seq_lens", at::kInt, B, device);
  const float scale = a[5] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(c.dim))) : float_arg(a[5]);
  const float softcap = float_arg(a[6]);
  const int32_t window = int_arg(a[7], "window");
  if (a[8] != Py_None) vector(a[8], "slopes", at::kFloat, hq, device);
  const bool weighted = a[9] != Py_None;
  PyObject* wout = a[10] != Py_None ? a[10] : a[9];
  int64_t win_s[2] = {0, 0}, wout_s[2] = {0, 0};
  if (weighted) {
    const int64_t tokens = tables.size(1) * c.page_size;
    const at::Tensor& wi = weights_of(a[9], "weights", B, c.heads, tokens, device);
    const at::Tensor& wo = weights_of(wout, "weights_out", B, c.heads, tokens, device);
    same_or_apart(wo, wi, "weights and weights_out");
    written(wo, "weights_out");
    apart(wo, "weights_out", a[0], "q");
    apart(wo, "weights_out", c.k, "k_cache");
    apart(wo, "weights_out", c.v, "v_cache");
    apart(wo, "weights_out", a[3], "block_tables");
    apart(wo, "weights_out", a[4], "seq_lens");
    apart(wo, "weights_out", a[8], "slopes");
    for (int i = 0; i < 2; ++i) {
      win_s[i] = step_of(wi, i);
      wout_s[i] = step_of(wo, i);
    }
  } else if (a[10] != Py_None) {
    value_error("weights_out needs weights");
  }
  at::Tensor out;
  if (a[11] == Py_None) {
    out = empty({B, hq, c.dim}, q.scalar_type(), device);
  } else {
    out = cuda_tensor(a[11], "out", {q.scalar_type()}, 3, device);
    if (out.sizes() != q.sizes() || !out.is_contiguous()) value_error("out must be contiguous and of q's shape");
    if (overlap(out, q)) value_error("out must not overlap q");
    apart(out, "out", c.k, "k_cache");
    apart(out, "out", c.v, "v_cache");
    apart(out, "out", a[3], "block_tables");
    apart(out, "out", a[4], "seq_lens");
    apart(out, "out", a[8], "slopes");
    if (weighted) {
      apart(out, "out", a[9], "weights");
      apart(out, "out", wout, "weights_out");
    }
  }
  const neso_stream_t stream = stream_on(device);
  const int32_t b32 = size32(B, "B"), hq32 = size32(hq, "Hq"), width = static_cast<int32_t>(tables.size(1));
  const int64_t need = entry.paged_attention_workspace(b32, hq32, c.heads, c.dim, width, c.page_size, weighted);
  if (need < 0) throw static_cast<int>(need);
  // A workspace of the call's own, from torch's allocator: calls on other
  // streams and captured graphs have theirs.
  at::Tensor workspace;
  if (need > 0) workspace = empty({need}, at::kByte, device);
  const int rc = entry.paged_attention(
      q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), data<int32_t>(tables), data<int32_t>(lens), data_or_null<float>(a[8]),
      weighted ? data_or_null<float>(a[9]) : nullptr, weighted ? data_or_null<float>(wout) : nullptr, out.data_ptr(),
      need > 0 ? workspace.data_ptr() : nullptr, need, code_of(q.scalar_type()), b32, hq32, c.heads, c.dim, scale, softcap, window, step_of(q, 0),
      step_of(q, 1), c.pages, c.page_size, step_of(c.k, 0), step_of(c.k, 1), step_of(c.k, 2), step_of(c.v, 0), step_of(c.v, 1),
      step_of(c.v, 2), width, step_of(tables, 0), win_s[0], win_s[1], wout_s[0], wout_s[1], stream);
  if (rc != NESO_OK) throw rc;
  return a[11] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[11]);
}

PyObject* kv_evict(PyObject* const* a) {
  const c10::Device device = device_of(a[0], "k_cache");
  const c10::cuda::CUDAGuard guard(device);
  const Caches c = caches(a[0], a[1], device);
  const int64_t B = tensor(a[2], "block_tables").dim() == 2 ? tensor(a[2], "block_tables").size(0) : 0;
  const at::Tensor& tables = table(a[2], "block_tables", B, device);
  const at::Tensor& lens = vector(a[3], "seq_lens", at::kInt, B, device);
  const int64_t tokens = tables.size(1) * c.page_size;
  const at::Tensor& wi = weights_of(a[4], "weights", B, c.heads, tokens, device);
  const int32_t budget = int_arg(a[5], "budget"), recent = int_arg(a[6], "recent"), sink = int_arg(a[7], "sink");
  if (budget > (1 << 30)) value_error("budget is limited to 2^30 tokens (got " + str(budget) + ")");  // before `kept` is allocated
  const at::Tensor& to = a[8] == Py_None ? tables : table(a[8], "out_tables", B, device);
  const at::Tensor& wo = a[9] == Py_None ? wi : weights_of(a[9], "weights_out", B, c.heads, tokens, device);
  same_or_apart(wo, wi, "weights and weights_out");
  if (to.size(1) * c.page_size < std::min<int64_t>(budget, tokens)) {
    value_error("out_tables hold " + str(to.size(1) * c.page_size) + " tokens per sequence, " +
                str(std::min<int64_t>(budget, tokens)) + " may be kept");
  }
  written(c.k, "k_cache");
  written(c.v, "v_cache");
  written(wo, "weights_out");
  apart(wo, "weights_out", c.k, "k_cache");
  apart(wo, "weights_out", c.v, "v_cache");
  apart(wo, "weights_out", a[2], "block_tables");
  apart(wo, "weights_out", a[3], "seq_lens");
  apart(wo, "weights_out", a[8], "out_tables");
  at::Tensor kept = empty({B, c.heads, budget > 0 ? budget : 0}, at::kInt, device);
  at::Tensor new_lens = empty({B}, at::kInt, device);
  const neso_stream_t stream = stream_on(device);
  const int rc = entry.kv_evict(
      c.k.data_ptr(), c.v.data_ptr(), data<int32_t>(tables), data<int32_t>(to), data<int32_t>(lens), data<float>(wi),
      data<float>(wo), data<int32_t>(kept), data<int32_t>(new_lens), size32(B, "B"), c.heads, c.dim, budget, recent, sink,
      c.pages, c.page_size, step_of(c.k, 0), step_of(c.k, 1), step_of(c.k, 2), step_of(c.v, 0), step_of(c.v, 1), step_of(c.v, 2),
      static_cast<int32_t>(tables.size(1)), step_of(tables, 0), static_cast<int32_t>(to.size(1)), step_of(to, 0), step_of(wi, 0),
      step_of(wi, 1), step_of(wo, 0), step_of(wo, 1), stream);
  if (rc != NESO_OK) throw rc;
  PyObject* x = THPVariable_Wrap(std::move(kept));
  PyObject* y = THPVariable_Wrap(std::move(new_lens));
  PyObject* both = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

PyObject* process_logits(PyObject* const* a) {
  const c10::Device device = device_of(a[0], "logits");
  const c10::cuda::CUDAGuard guard(device);
  const at::Tensor& x = cuda_tensor(a[0], "logits", {at::kFloat, at::kHalf, at::kBFloat16}, 2, device);
  rows(x, "logits");
  const int64_t B = x.size(0), V = x.size(1);
  int64_t T = 0, history_stride = 0, mask_stride = 0, biases = 0;
  if (a[1] != Py_None) {
    const at::Tensor& h = cuda_tensor(a[1], "history", {at::kInt}, 2, device);
    rows(h, "history");
    if (h.size(0) != B || a[2] == Py_None) {
      value_error("history must have one row per sequence (" + str(B) + ") and come with history_lens");
    }
    T = h.size(1);
    history_stride = step_of(h, 0);
    vector(a[2], "history_lens", at::kInt, B, device);
    if (a[3] != Py_None) vector(a[3], "prompt_lens", at::kInt, B, device);
  } else if (a[2] != Py_None || a[3] != Py_None) {
    value_error("history_lens and prompt_lens need a history");
  }
  static const char* const names[3] = {"repetition", "frequency", "presence"};
  for (int i = 0; i < 3; ++i) {
    if (a[4 + i] == Py_None) continue;
    vector(a[4 + i], names[i], at::kFloat, B, device);
    if (a[1] == Py_None) value_error(std::string(names[i]) + " needs a history");
  }
  if ((a[7] == Py_None) != (a[8] == Py_None)) value_error("bias_ids and bias come together");
  if (a[7] != Py_None) {
    const at::Tensor& ids = cuda_tensor(a[7], "bias_ids", {at::kInt}, 2, device);
    const at::Tensor& bias = cuda_tensor(a[8], "bias", {at::kFloat}, 2, device);
    biases = bias.size(1);
    if (bias.sizes() != ids.sizes() || bias.size(0) != B || !bias.is_contiguous() || !ids.is_contiguous()) {
      value_error("bias_ids and bias must be contiguous and share one [" + str(B) + ", n] shape");
    }
  }
  if (a[9] != Py_None) {
    const at::Tensor& mask = cuda_tensor(a[9], "mask", {at::kInt}, 2, device);
    rows(mask, "mask");
    if (mask.size(0) != B || mask.size(1) < (V + 31) / 32) {
      value_error("mask must be [" + str(B) + ", at least " + str((V + 31) / 32) + " words]");
    }
    mask_stride = step_of(mask, 0);
  }
  at::Tensor out;
  if (a[10] == Py_None) {
    out = empty({B, V}, x.scalar_type(), device);
  } else {
    out = cuda_tensor(a[10], "out", {x.scalar_type()}, 2, device);
    rows(out, "out");
    if (out.sizes() != x.sizes()) value_error("out must have the shape of logits");
    same_or_apart(out, x, "out and logits");
    written(out, "out");
    static const char* const inputs[9] = {"history",  "history_lens", "prompt_lens", "repetition", "frequency",
                                          "presence", "bias_ids",     "bias",        "mask"};
    for (int i = 0; i < 9; ++i) apart(out, "out", a[1 + i], inputs[i]);
  }
  const neso_stream_t stream = stream_on(device);
  const int rc = entry.process_logits(
      x.data_ptr(), out.data_ptr(), code_of(x.scalar_type()), size32(B, "B"), size32(V, "V"), step_of(x, 0), step_of(out, 0),
      data_or_null<int32_t>(a[1]), data_or_null<int32_t>(a[2]), data_or_null<int32_t>(a[3]), size32(T, "history"),
      history_stride, data_or_null<float>(a[4]), data_or_null<float>(a[5]), data_or_null<float>(a[6]),
      data_or_null<int32_t>(a[7]), data_or_null<float>(a[8]), size32(biases, "bias"), data_or_null<int32_t>(a[9]),
      mask_stride, stream);
  if (rc != NESO_OK) throw rc;
  return a[10] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[10]);
}

// Positional arguments only, None for what was not given; every C++ exception
// ends here.
template <PyObject* (*kCall)(PyObject* const*), int kArgs>
PyObject* guarded(const char* name, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "%s takes %d arguments (got %zd)", name, kArgs, n);
    return nullptr;
  }
  if (raise_status == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "set_entry_points has not been called");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    return kCall(args);
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.what.c_str());
  } catch (const PythonError&) {
  } catch (int status) {
    PyObject* r = PyObject_CallFunction(raise_status, "is", status, name);
    if (r != nullptr) {
      Py_DECREF(r);
      PyErr_Format(PyExc_RuntimeError, "%s failed with status %d", name, status);
    }
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

PyObject* py_rope_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded<rope_paged_append, 11>("neso_rope_paged_append", args, n);
}
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded<paged_attention, 12>("neso_paged_attention", args, n);
}
PyObject* py_kv_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded<kv_evict, 10>("neso_kv_evict", args, n);
}
PyObject* py_process_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded<process_logits, 11>("neso_process_logits", args, n);
}

// set_entry_points(raise_status, address of each entry in the order of Entries)
PyObject* py_set_entry_points(PyObject*, PyObject* args) {
  PyObject* raise = nullptr;
  unsigned long long at[6];
  if (!PyArg_ParseTuple(args, "OKKKKKK", &raise, &at[0], &at[1], &at[2], &at[3], &at[4], &at[5])) return nullptr;
  entry.set_device = reinterpret_cast<decltype(entry.set_device)>(at[0]);
  entry.rope_paged_append = reinterpret_cast<decltype(entry.rope_paged_append)>(at[1]);
  entry.paged_attention = reinterpret_cast<decltype(entry.paged_attention)>(at[2]);
  entry.paged_attention_workspace = reinterpret_cast<decltype(entry.paged_attention_workspace)>(at[3]);
  entry.kv_evict = reinterpret_cast<decltype(entry.kv_evict)>(at[4]);
  entry.process_logits = reinterpret_cast<decltype(entry.process_logits)>(at[5]);
  Py_INCREF(raise);
  Py_XDECREF(raise_status);
  raise_status = raise;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"set_entry_points", py_set_entry_points, METH_VARARGS, nullptr},
    {"rope_paged_append", reinterpret_cast<PyCFunction>(py_rope_paged_append), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(py_paged_attention), METH_FASTCALL, nullptr},
    {"kv_evict", reinterpret_cast<PyCFunction>(py_kv_evict), METH_FASTCALL, nullptr},
    {"process_logits", reinterpret_cast<PyCFunction>(py_process_logits), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bindings", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__bindings(void) { return PyModule_Create(&module); }
