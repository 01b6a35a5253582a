// CPython binding of the sequence-memory operators (paged attention, cache writes,
// gated delta rule). A decode step calls them once per layer on little data, so the
// call itself counts: reading the tensors' properties, checking them and
// allocating the outputs here takes about a quarter of the time that the same
// checks take in Python. The kernels are reached through the C ABI of d3moe.h, whose
// addresses bind() takes from the library the package has loaded.
//
// Every function runs under guarded(): a refused argument becomes ValueError, a
// negative status the package's D3Error (ValueError for D3_EINVAL, as elsewhere in
// the package), any other C++ exception RuntimeError. None leaves this file.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <limits>
#include <optional>
#include <string>

#include "d3moe.h"

namespace {

using at::Tensor;
using c10::IntArrayRef;

struct Refusal : std::exception {
  std::string text;
  explicit Refusal(std::string t) : text(std::move(t)) {}
  const char* what() const noexcept override { return text.c_str(); }
};
struct PythonError {};  // the Python error is set already

decltype(&d3_kv_append) kv_append_fn;
decltype(&d3_copy_pages) copy_pages_fn;
decltype(&d3_paged_attention) paged_attention_fn;
decltype(&d3_paged_attention_workspace_size) paged_attention_ws_fn;
decltype(&d3_gated_delta_step) step_fn;
decltype(&d3_gated_delta_chunk) chunk_fn;
decltype(&d3_gated_delta_chunk_workspace_size) chunk_ws_fn;
decltype(&d3_last_error_string) last_error_fn;
PyObject* d3_error = nullptr;  // d3moe._lib.D3Error

void require(bool ok, const char* text) {
  if (!ok) throw Refusal(text);
}

void check(int rc, const char* name) {
  if (rc >= 0) return;
  const char* text = last_error_fn();
  if (rc == D3_EINVAL) throw Refusal(std::string(name) + ": " + (text ? text : ""));
  PyObject* e = PyObject_CallFunction(d3_error, "sis", name, rc, text ? text : "");
  if (e) {
    PyErr_SetObject(d3_error, e);
    Py_DECREF(e);
  }
  throw PythonError{};
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Refusal(std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}

const Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  return v;
}

int64_t integer(PyObject* o, const char* what) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  if (v < std::numeric_limits<int>::min() || v > std::numeric_limits<int>::max())
    throw Refusal(std::string(what) + " is out of range");
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError{};
  return v != 0;
}

int to_int(int64_t v) {
  require(v <= std::numeric_limits<int>::max(), "a size is out of range");
  return static_cast<int>(v);
}

// The device of the operator's main tensor.
int cuda_device(const Tensor& t) {
  require(t.is_cuda(), "d3moe operators take CUDA tensors; there is no CPU path");
  return t.get_device();
}

bool on(const Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

const int32_t* index_ptr(const Tensor& t, int64_t n, int dev, const char* what) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !on(t, dev) || !t.is_contiguous())
    throw Refusal(std::string(what) + " must be contiguous int32 [" + std::to_string(n) + "] on the operands' device");
  return static_cast<const int32_t*>(t.data_ptr());
}

int32_t* status_ptr(PyObject* o, int dev) {
  const Tensor* t = maybe(o, "status");
  if (!t) return nullptr;
  require(t->scalar_type() == at::kInt && t->numel() >= 1 && on(*t, dev), "status must be an int32 tensor on the operands' device");
  return static_cast<int32_t*>(t->data_ptr());
}

const float* scale_ptr(PyObject* o, int64_t heads, int dev) {
  const Tensor* t = maybe(o, "a cache scale");
  if (!t) return nullptr;
  require(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == heads && t->is_contiguous() && on(*t, dev),
          "cache scales must be contiguous float32 [heads] on the cache's device");
  return static_cast<const float*>(t->data_ptr());
}

// Stride of an axis; 0 where the axis has one entry and its stride no meaning.
int64_t step(const Tensor& t, int axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

d3_stream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

Tensor empty(IntArrayRef sizes, at::ScalarType type, int dev) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, dev), std::nullopt);
}

// Scratch of `need` bytes: the caller's or a new one (kept alive by `hold`).
void* scratch(PyObject* o, size_t need, int dev, Tensor& hold, size_t& bytes) {
  if (const Tensor* t = maybe(o, "workspace")) {
    require(on(*t, dev) && t->is_contiguous(), "workspace must be contiguous on the operands' device");
    bytes = t->nbytes();
    return t->data_ptr();
  }
  hold = empty({static_cast<int64_t>(need)}, at::kByte, dev);
  bytes = need;
  return hold.data_ptr();
}

int dtype_tag(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return D3_DTYPE_BF16;
    case at::kHalf: return D3_DTYPE_F16;
    case at::kFloat8_e4m3fn: return D3_DTYPE_E4M3;
    default: return -1;
  }
}

d3_kv_cache_t kv_cache(const Tensor& k, const Tensor& v, const Tensor& table, PyObject* k_scale, PyObject* v_scale, int dev) {
  const int dtype = dtype_tag(k.scalar_type());
  require(dtype >= 0 && v.scalar_type() == k.scalar_type(), "k_cache and v_cache must both be bfloat16, float16 or float8_e4m3fn");
  require(k.dim() == 4 && k.sizes() == v.sizes(), "k_cache and v_cache must be [pages, page_size, heads, dim] of one shape");
  const IntArrayRef n = k.sizes();
  require(k.stride(3) == 1 && v.stride(3) == 1, "the last axis of a cache must be contiguous");
  require(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
          "page_table must be int32 [sequences, pages per sequence], rows contiguous");
  require(on(v, dev) && on(table, dev), "caches and page_table must be on one device");
  require(dtype == D3_DTYPE_E4M3 || (k_scale == Py_None && v_scale == Py_None), "only an e4m3 cache has scales");
  d3_kv_cache_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_page_stride = step(k, 0);
  c.k_token_stride = step(k, 1);
  c.k_head_stride = step(k, 2);
  c.v_page_stride = step(v, 0);
  c.v_token_stride = step(v, 1);
  c.v_head_stride = step(v, 2);
  c.k_scale = scale_ptr(k_scale, n[2], dev);
  c.v_scale = scale_ptr(v_scale, n[2], dev);
  c.table = static_cast<const int32_t*>(table.data_ptr());
  c.table_stride = table.stride(0);
  c.sequences = to_int(table.size(0));
  c.table_pages = to_int(table.size(1));
  c.num_pages = to_int(n[0]);
  c.page_size = to_int(n[1]);
  c.heads = to_int(n[2]);
  c.dim = to_int(n[3]);
  c.dtype = dtype;
  return c;
}

// Type of the rows that go with a cache: its own, bf16 for an e4m3 cache.
at::ScalarType row_type(const Tensor& cache) {
  return cache.scalar_type() == at::kFloat8_e4m3fn ? at::kBFloat16 : cache.scalar_type();
}

template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F f) {
  try {
    require(n == want, "wrong number of arguments");
    require(d3_error != nullptr, "the binding is not connected to the library");
    return f(args);
  } catch (const PythonError&) {
  } catch (const Refusal& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// kv_append(k, v, k_cache, v_cache, page_table, positions, seq_ids, k_scale, v_scale, status)
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 10, [](PyObject* const* p) -> PyObject* {
    const Tensor &k = tensor(p[0], "k"), &v = tensor(p[1], "v"), &kc = tensor(p[2], "k_cache"), &vc = tensor(p[3], "v_cache");
    const int dev = cuda_device(kc);
    const d3_kv_cache_t c = kv_cache(kc, vc, tensor(p[4], "page_table"), p[7], p[8], dev);
    const at::ScalarType want = row_type(kc);
    require(k.scalar_type() == want && v.scalar_type() == want, "k and v must be of the cache's dtype (bfloat16 for an e4m3 cache)");
    require(k.dim() == 3 && k.size(1) == c.heads && k.size(2) == c.dim && v.sizes() == k.sizes(),
            "k and v must be [T, heads, dim] with the cache's heads and dim");
    const int64_t T = k.size(0);
    require(T == 0 || (k.stride(2) == 1 && v.stride(2) == 1), "the last axis of k and v must be contiguous");
    require(on(k, dev) && on(v, dev), "k, v and the cache must be on one device");
    const int32_t* pos = index_ptr(tensor(p[5], "positions"), T, dev, "positions");
    const Tensor* seq = maybe(p[6], "seq_ids");
    const int32_t* sp = seq ? index_ptr(*seq, T, dev, "seq_ids") : nullptr;
    int32_t* status = status_ptr(p[9], dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    check(kv_append_fn(k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1), dtype_tag(want), to_int(T),
                       sp, pos, &c, status, stream_of(dev)),
          "d3_kv_append");
    Py_RETURN_NONE;
  });
}

// copy_pages(pool, src, dst, page_dim, status)
PyObject* copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 5, [](PyObject* const* p) -> PyObject* {
    const Tensor& pool = tensor(p[0], "pool");
    const int dev = cuda_device(pool);
    const int64_t axis = integer(p[3], "page_dim");
    require(axis >= 0 && axis < pool.dim(), "page_dim must be an axis of pool");
    const IntArrayRef size = pool.sizes(), stride = pool.strides();
    const bool none = pool.numel() == 0;  // nothing to copy: no stride of it means anything
    int64_t elements = 1, planes = 1, plane_stride = 0;
    for (int64_t i = pool.dim() - 1; i > axis; --i) {
      require(none || size[i] == 1 || stride[i] == elements, "the axes behind page_dim must be contiguous");
      elements *= size[i];
    }
    for (int64_t i = axis - 1; i >= 0; --i) {
      if (size[i] == 1) continue;
      if (planes == 1) plane_stride = stride[i];
      else require(none || stride[i] == planes * plane_stride, "the axes before page_dim must step evenly");
      planes *= size[i];
    }
    const Tensor& src = tensor(p[1], "src");
    const int64_t count = src.numel(), b = static_cast<int64_t>(pool.element_size());
    const int32_t* sp = index_ptr(src, count, dev, "src");
    const int32_t* dp = index_ptr(tensor(p[2], "dst"), count, dev, "dst");
    int32_t* status = status_ptr(p[4], dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    if (none) Py_RETURN_NONE;
    check(copy_pages_fn(pool.data_ptr(), to_int(planes), plane_stride * b, to_int(size[axis]), stride[axis] * b, elements * b, sp, dp,
                        to_int(count), status, stream_of(dev)),
          "d3_copy_pages");
    Py_RETURN_NONE;
  });
}

// paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale, k_scale, v_scale, window, max_seq_len, out,
//                 return_lse, workspace, status)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 14, [](PyObject* const* p) -> PyObject* {
    const Tensor &q = tensor(p[0], "q"), &kc = tensor(p[1], "k_cache"), &vc = tensor(p[2], "v_cache");
    const int dev = cuda_device(kc);
    const d3_kv_cache_t c = kv_cache(kc, vc, tensor(p[3], "page_table"), p[6], p[7], dev);
    require(q.dim() == 3 && q.size(2) == c.dim && on(q, dev), "q must be [B, heads, dim] with the cache's dim, on its device");
    const at::ScalarType want = row_type(kc);
    require(q.scalar_type() == want, "q must be of the cache's dtype (bfloat16 for an e4m3 cache)");
    const int64_t B = q.size(0), Hq = q.size(1);
    require(c.sequences == B, "page_table must have one row per query");
    const int32_t* lens = index_ptr(tensor(p[4], "seq_lens"), B, dev, "seq_lens");
    int32_t* status = status_ptr(p[13], dev);
    const double scale = p[5] == Py_None ? 1.0 / std::sqrt(static_cast<double>(c.dim)) : number(p[5]);
    const int window = static_cast<int>(integer(p[8], "window"));
    const int64_t held = static_cast<int64_t>(c.table_pages) * c.page_size;
    int64_t limit = p[9] == Py_None ? held : integer(p[9], "max_seq_len");
    limit = limit < held ? limit : held;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    Tensor out, lse, hold;
    if (const Tensor* o = maybe(p[10], "out")) {
      require(o->sizes() == q.sizes() && o->scalar_type() == want && on(*o, dev), "out must have the shape, dtype and device of q");
      out = *o;
    } else {
      out = empty(q.sizes(), want, dev);
    }
    require(q.stride(2) == 1 && out.stride(2) == 1, "the last axis of q and out must be contiguous");
    const bool with_lse = truth(p[11]);
    if (with_lse) lse = empty({B, Hq}, at::kFloat, dev);
    size_t need = 0, bytes = 0;
    check(paged_attention_ws_fn(to_int(B), to_int(Hq), c.heads, c.dim, &need), "d3_paged_attention_workspace_size");
    void* ws = scratch(p[12], need, dev, hold, bytes);
    check(paged_attention_fn(q.data_ptr(), step(q, 0), step(q, 1), dtype_tag(want), to_int(B), to_int(Hq), &c, lens, to_int(limit),
                             window, static_cast<float>(scale), out.data_ptr(), step(out, 0), step(out, 1),
                             with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, ws, bytes, status, stream_of(dev)),
          "d3_paged_attention");
    if (!with_lse) return THPVariable_Wrap(out);
    PyObject *a = THPVariable_Wrap(out), *b = THPVariable_Wrap(lse);
    PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    return both;
  });
}

struct Delta {
  d3_gated_delta_t a{};
  Tensor out;
  int64_t T = 0;
  int dev = 0;
};

// Operands 0-5 (q, k, v, g, beta, state) and the others where they are given.
Delta delta(PyObject* const* p, PyObject* slots, int64_t n, PyObject* scale, PyObject* l2norm, PyObject* eps, PyObject* out) {
  const Tensor &q = tensor(p[0], "q"), &k = tensor(p[1], "k"), &v = tensor(p[2], "v"), &g = tensor(p[3], "g"), &beta = tensor(p[4], "beta"),
               &state = tensor(p[5], "state");
  Delta d;
  const int dev = d.dev = cuda_device(state);
  require(q.dim() == 3 && v.dim() == 3 && state.dim() == 4, "q, k, v must be [T, heads, dim] and state [slots, heads, key_dim, value_dim]");
  const int64_t T = d.T = q.size(0), Hk = q.size(1), dk = q.size(2), Hv = v.size(1), dv = v.size(2);
  auto gates = [&](const Tensor& t) { return t.dim() == 2 && t.size(0) == T && t.size(1) == Hv; };
  require(k.sizes() == q.sizes() && v.size(0) == T && gates(g) && gates(beta),
          "k must have the shape of q, v its tokens, g and beta [T, value_heads]");
  require(state.size(1) == Hv && state.size(2) == dk && state.size(3) == dv, "state must be [slots, value_heads, key_dim, value_dim]");
  require(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16, "q, k and v must be bfloat16");
  require(g.scalar_type() == at::kFloat && beta.scalar_type() == at::kFloat && state.scalar_type() == at::kFloat,
          "g, beta and state must be float32");
  require(on(q, dev) && on(k, dev) && on(v, dev) && on(g, dev) && on(beta, dev), "all operands must be on one device");
  auto packed = [&](const Tensor& t, int64_t heads, int64_t dim) { return T == 0 || (t.stride(2) == 1 && (heads == 1 || t.stride(1) == dim)); };
  if (out == Py_None) {
    d.out = empty({T, Hv, dv}, at::kBFloat16, dev);
  } else {
    d.out = tensor(out, "out");
    require(d.out.sizes() == v.sizes() && d.out.scalar_type() == at::kBFloat16 && on(d.out, dev),
            "out must be bfloat16 with the shape and device of v");
  }
  require(packed(q, Hk, dk) && packed(k, Hk, dk) && packed(v, Hv, dv) && packed(d.out, Hv, dv),
          "heads and dims of q, k, v and out must be contiguous (tokens may be strided)");
  require(state.stride(3) == 1 && state.stride(2) == dv && (Hv == 1 || state.stride(1) == dk * dv), "each slot of state must be contiguous");
  require(T == 0 || Hv == 1 || (g.stride(1) == 1 && beta.stride(1) == 1), "heads of g and beta must be contiguous");
  const Tensor* s = maybe(slots, "slots");
  require(s || n <= state.size(0), "state has fewer slots than there are sequences");
  d3_gated_delta_t& a = d.a;
  a.slot = s ? index_ptr(*s, n, dev, "slots") : nullptr;
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.g = static_cast<const float*>(g.data_ptr());
  a.beta = static_cast<const float*>(beta.data_ptr());
  a.out = d.out.data_ptr();
  a.state = static_cast<float*>(state.data_ptr());
  a.q_stride = step(q, 0);
  a.k_stride = step(k, 0);
  a.v_stride = step(v, 0);
  a.g_stride = step(g, 0);
  a.beta_stride = step(beta, 0);
  a.out_stride = step(d.out, 0);
  a.slot_stride = step(state, 0);
  a.slots = to_int(state.size(0));
  a.key_heads = to_int(Hk);
  a.value_heads = to_int(Hv);
  a.key_dim = to_int(dk);
  a.value_dim = to_int(dv);
  a.l2norm = truth(l2norm);
  a.scale = static_cast<float>(scale == Py_None ? 1.0 / std::sqrt(static_cast<double>(dk)) : number(scale));
  a.eps = static_cast<float>(number(eps));
  return d;
}

// gated_delta_step(q, k, v, g, beta, state, slots, scale, l2norm, eps, out, status)
PyObject* gated_delta_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 12, [](PyObject* const* p) -> PyObject* {
    const Tensor& q = tensor(p[0], "q");
    const Delta d = delta(p, p[6], q.dim() ? q.size(0) : 0, p[7], p[8], p[9], p[10]);
    int32_t* status = status_ptr(p[11], d.dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(d.dev));
    check(step_fn(&d.a, to_int(d.T), status, stream_of(d.dev)), "d3_gated_delta_step");
    return THPVariable_Wrap(d.out);
  });
}

// gated_delta_chunk(q, k, v, g, beta, state, cu_seqlens, slots, fresh, scale, l2norm, eps, out, workspace, status)
PyObject* gated_delta_chunk(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 15, [](PyObject* const* p) -> PyObject* {
    const Tensor& cu = tensor(p[6], "cu_seqlens");
    const int64_t seqs = cu.numel() - 1;
    require(seqs >= 0, "cu_seqlens must hold n + 1 row starts");
    const Delta d = delta(p, p[7], seqs, p[9], p[10], p[11], p[12]);
    const int32_t* cp = index_ptr(cu, seqs + 1, d.dev, "cu_seqlens");
    const Tensor* fresh = maybe(p[8], "fresh");
    if (fresh && !((fresh->scalar_type() == at::kBool || fresh->scalar_type() == at::kByte) && fresh->dim() == 1 && fresh->size(0) == seqs &&
                   fresh->is_contiguous() && on(*fresh, d.dev)))
      throw Refusal("fresh must be contiguous bool [" + std::to_string(seqs) + "] on the operands' device");
    int32_t* status = status_ptr(p[14], d.dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(d.dev));
    size_t need = 0, bytes = 0;
    check(chunk_ws_fn(to_int(d.T), to_int(seqs), d.a.value_heads, d.a.key_dim, d.a.value_dim, &need), "d3_gated_delta_chunk_workspace_size");
    Tensor hold;
    void* ws = scratch(p[13], need, d.dev, hold, bytes);
    check(chunk_fn(&d.a, cp, to_int(d.T), to_int(seqs), fresh ? static_cast<const uint8_t*>(fresh->data_ptr()) : nullptr, ws, bytes, status,
                   stream_of(d.dev)),
          "d3_gated_delta_chunk");
    return THPVariable_Wrap(d.out);
  });
}

// bind(D3Error, [addresses in the order below])
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* error = nullptr;
  unsigned long long x[8];
  if (!PyArg_ParseTuple(args, "OKKKKKKKK", &error, &x[0], &x[1], &x[2], &x[3], &x[4], &x[5], &x[6], &x[7])) return nullptr;
  kv_append_fn = reinterpret_cast<decltype(kv_append_fn)>(x[0]);
  copy_pages_fn = reinterpret_cast<decltype(copy_pages_fn)>(x[1]);
  paged_attention_fn = reinterpret_cast<decltype(paged_attention_fn)>(x[2]);
  paged_attention_ws_fn = reinterpret_cast<decltype(paged_attention_ws_fn)>(x[3]);
  step_fn = reinterpret_cast<decltype(step_fn)>(x[4]);
  chunk_fn = reinterpret_cast<decltype(chunk_fn)>(x[5]);
  chunk_ws_fn = reinterpret_cast<decltype(chunk_ws_fn)>(x[6]);
  last_error_fn = reinterpret_cast<decltype(last_error_fn)>(x[7]);
  Py_INCREF(error);
  Py_XSETREF(d3_error, error);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(kv_append),        FAST(copy_pages),        FAST(paged_attention),
                         FAST(gated_delta_step), FAST(gated_delta_chunk), {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_d3native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__d3native() {
  PyObject* m = PyModule_Create(&module);
  // the text is also what build.py looks for in the file
  if (m && PyModule_AddStringConstant(m, "built_for", D3_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
