// serving.cpp — the host side of the serving calls (kv_cache.py): argument checks,
// outputs, current stream and the C call (include/dwa_decode.h) as one Python
// extension function each.
//
// A decoding step makes three or four of these calls per layer on small tensors, whose
// kernels take 3 to 6 us; checked in Python and called through ctypes each call took
// 11 to 18 us of the host's time, here 3 to 4.5, 2.3 of them the launch.  Nothing is kept
// between calls but the C entry points' addresses, which kv_cache.py binds from the loaded
// library.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <exception>
#include <sstream>
#include <string>
#include <tuple>

#include "dwa_decode.h"

namespace {

decltype(&dwa_kv_write) g_write = nullptr;
decltype(&dwa_kv_read) g_read = nullptr;
decltype(&dwa_paged_attention) g_attend = nullptr;
decltype(&dwa_verify_drafts) g_verify = nullptr;
decltype(&dwa_kv_append) g_append = nullptr;
decltype(&dwa_kv_keep) g_keep = nullptr;
decltype(&dwa_paged_tree_attention) g_attend_tree = nullptr;
decltype(&dwa_paged_tree_attention_workspace) g_tree_workspace = nullptr;
decltype(&dwa_tree_masks) g_masks = nullptr;
decltype(&dwa_verify_tree) g_verify_tree = nullptr;
PyObject* g_raise = nullptr;  // raises the package's error for a status and a function's name

struct Refusal {
  PyObject* type;
  std::string what;
};

[[noreturn]] void refuse(std::string what) { throw Refusal{PyExc_ValueError, std::move(what)}; }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Refusal{PyExc_TypeError, std::string(name) + " must be a torch.Tensor"};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(std::string(name) + " requires grad: the serving calls have no gradients (use torch.no_grad())");
  return t;
}

std::string describe(const at::Tensor& t) {
  std::ostringstream s;
  s << t.scalar_type() << " " << t.sizes() << ", strides " << t.strides() << ", on " << t.device();
  return s.str();
}

int device_of(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(std::string(name) + " must live on a CUDA device (got " + describe(t) + ")");
  return t.get_device();
}

bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }

struct Cache {
  int dev = 0;
  int64_t n_pages = 0, heads = 0, page = 0, d = 0, ld_page = 0, ld_scale = 0;
  void *k = nullptr, *v = nullptr;
  float *k_scale = nullptr, *v_scale = nullptr;
};

// The distance between pages; a dimension of size 1 may have any stride.
int64_t page_stride(const at::Tensor& t, const char* what) {
  int64_t dense = 1;
  for (int64_t i = t.dim() - 1; i > 0; --i) {
    if (t.size(i) > 1 && t.stride(i) != dense) refuse(what);
    dense *= t.size(i);
  }
  return t.size(0) > 1 ? t.stride(0) : dense;
}

Cache cache_of(PyObject* k_o, PyObject* v_o, PyObject* ks_o, PyObject* vs_o) {
  const at::Tensor &k = tensor(k_o, "k_cache"), &v = tensor(v_o, "v_cache");
  Cache c;
  c.dev = device_of(k, "k_cache");
  if (k.dim() != 4) refuse("k_cache must be [n_pages, H_kv, page_size, d]");
  if (v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes() || v.strides() != k.strides() ||
      !on(v, c.dev))
    refuse("v_cache must be like k_cache (type, shape, strides, device)");
  c.n_pages = k.size(0);
  c.heads = k.size(1);
  c.page = k.size(2);
  c.d = k.size(3);
  c.ld_page = page_stride(k, "a cache's pages must be contiguous inside");
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  const bool scales = ks_o != Py_None && vs_o != Py_None;
  if (k.scalar_type() == at::kFloat8_e4m3fn) {
    if (!scales) refuse("a float8_e4m3fn cache needs k_scale and v_scale");
    const at::Tensor &ks = tensor(ks_o, "k_scale"), &vs = tensor(vs_o, "v_scale");
    if (ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat ||
        ks.sizes() != k.sizes().slice(0, 3) || vs.sizes() != ks.sizes() || vs.strides() != ks.strides() ||
        !on(ks, c.dev) || !on(vs, c.dev))
      refuse("k_scale and v_scale must be f32 [n_pages, H_kv, page_size] with the same strides on the "
             "cache's device");
    c.ld_scale = page_stride(ks, "the scales of a page must be contiguous");
    c.k_scale = static_cast<float*>(ks.data_ptr());
    c.v_scale = static_cast<float*>(vs.data_ptr());
  } else if (k.scalar_type() != at::kBFloat16) {
    refuse("k_cache must be bfloat16 or float8_e4m3fn");
  } else if (ks_o != Py_None || vs_o != Py_None) {
    refuse("a bfloat16 cache has no scales");
  }
  if (c.heads > INT32_MAX || c.page > INT32_MAX || c.d > INT32_MAX) refuse("k_cache is too large");
  return c;
}

// A contiguous tensor's pointer.
template <typename T>
T* array(PyObject* o, at::ScalarType type, at::IntArrayRef shape, int dev, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.sizes() != shape || !on(t, dev) || !t.is_contiguous()) {
    std::ostringstream s;
    s << name << " must be a contiguous " << type << " " << shape << " on the same device as the others (got "
      << describe(t) << ")";
    refuse(s.str());
  }
  return static_cast<T*>(t.data_ptr());
}

int32_t* status_of(PyObject* o, int dev) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "status");
  if (t.scalar_type() != at::kInt || t.numel() != 1 || !on(t, dev))
    refuse("status must be one int32 on the cache's device");
  return static_cast<int32_t*>(t.data_ptr());
}

// Rows [T, heads, d], contiguous along d: their token and head strides (a dimension of
// size 1 may have any).  heads < 0: any number.
void rows_of(const at::Tensor& t, int64_t heads, int64_t d, int dev, const char* name, int64_t* tok,
             int64_t* head) {
  if (t.dim() != 3 || (heads >= 0 && t.size(1) != heads) || t.size(2) != d || !on(t, dev) ||
      (d > 1 && t.stride(2) != 1)) {
    std::ostringstream s;
    s << name << " must be [T, ";
    if (heads >= 0) s << heads;
    else s << "H";
    s << ", " << d << "], contiguous along d, on the cache's device (got " << describe(t) << ")";
    refuse(s.str());
  }
  *tok = t.size(0) > 1 ? t.stride(0) : 0;
  *head = t.size(1) > 1 ? t.stride(1) : d;
}

// An output.  (Through the dispatcher, at::empty, it takes 1.2 us.)
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::Tensor(at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)),
                                           std::nullopt));
}

// A tensor of its own over a part of an allocation, `at` elements in: calls with two outputs
// allocate once (1 us).
at::Tensor part_of(const at::Tensor& whole, int64_t at, at::IntArrayRef shape) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                          whole.dtype());
  t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  return t;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

// None, or an exception set where the call was refused or failed.
PyObject* finish(int32_t status, const char* name) {
  if (status == DWA_OK) Py_RETURN_NONE;
  PyObject* r = PyObject_CallFunction(g_raise, "is", static_cast<int>(status), name);
  if (r != nullptr) {  // it has to raise
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, name);
  }
  return nullptr;
}

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
  if (got != want || g_raise == nullptr) {
    PyErr_SetString(PyExc_TypeError, "unbound, or called with a wrong number of arguments");
    return nullptr;
  }
  try {
    return body();
  } catch (const Refusal& e) {
    PyErr_SetString(e.type, e.what.c_str());
  } catch (...) {  // as torch's own functions raise it: out of memory has a type of its own
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// bind(write, read, attend, verify, append, keep, attend_tree, its workspace, masks, verify_tree,
// raise): the entry points' addresses.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[10];
  PyObject* raise;
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9],
                        &raise))
    return nullptr;
  g_write = reinterpret_cast<decltype(g_write)>(a[0]);
  g_read = reinterpret_cast<decltype(g_read)>(a[1]);
  g_attend = reinterpret_cast<decltype(g_attend)>(a[2]);
  g_verify = reinterpret_cast<decltype(g_verify)>(a[3]);
  g_append = reinterpret_cast<decltype(g_append)>(a[4]);
  g_keep = reinterpret_cast<decltype(g_keep)>(a[5]);
  g_attend_tree = reinterpret_cast<decltype(g_attend_tree)>(a[6]);
  g_tree_workspace = reinterpret_cast<decltype(g_tree_workspace)>(a[7]);
  g_masks = reinterpret_cast<decltype(g_masks)>(a[8]);
  g_verify_tree = reinterpret_cast<decltype(g_verify_tree)>(a[9]);
  Py_INCREF(raise);
  Py_XDECREF(g_raise);
  g_raise = raise;
  Py_RETURN_NONE;
}

// (k, v, k_cache, v_cache, slots, k_scale, v_scale, status)
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Cache c = cache_of(a[2], a[3], a[5], a[6]);
    const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v");
    const at::ScalarType type = k.scalar_type();
    if ((type != at::kBFloat16 && type != at::kFloat) || v.scalar_type() != type)
      refuse("k and v must both be bfloat16 or float32");
    int64_t kt, kh, vt, vh;
    rows_of(k, c.heads, c.d, c.dev, "k", &kt, &kh);
    rows_of(v, c.heads, c.d, c.dev, "v", &vt, &vh);
    const int64_t T = k.size(0);
    if (v.size(0) != T) refuse("k and v must have the same number of tokens");
    const int64_t* slots = array<int64_t>(a[4], at::kLong, {T}, c.dev, "slots");
    int32_t* status = status_of(a[7], c.dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    return finish(g_write(k.data_ptr(), v.data_ptr(), type == at::kBFloat16, T,
                          static_cast<int32_t>(c.heads), static_cast<int32_t>(c.d), kt, kh, vt, vh, slots,
                          c.k, c.v, c.k_scale, c.v_scale, c.n_pages, static_cast<int32_t>(c.page),
                          c.ld_page, c.ld_scale, status, c10::cuda::getCurrentCUDAStream(c.dev).stream()),
                  "dwa_kv_write");
  });
}

// (k_cache, v_cache, slots, k_scale, v_scale, out pair or None, status) -> (k, v)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Cache c = cache_of(a[0], a[1], a[3], a[4]);
    const at::Tensor& slots_t = tensor(a[2], "slots");
    const int64_t T = slots_t.dim() == 1 ? slots_t.size(0) : 0;
    const int64_t* slots = array<int64_t>(a[2], at::kLong, {T}, c.dev, "slots");
    int32_t* status = status_of(a[6], c.dev);
    at::Tensor k, v;
    void *k_out, *v_out;
    const bool own = a[5] == Py_None;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    if (own) {
      const int64_t size = T * c.heads * c.d;  // a multiple of 16: both start on 32 bytes
      const at::Tensor both = fresh({2 * size}, at::kBFloat16, c.dev);
      k = part_of(both, 0, {T, c.heads, c.d});
      v = part_of(both, size, {T, c.heads, c.d});
      k_out = k.data_ptr();
      v_out = v.data_ptr();
    } else {
      if (!PyTuple_Check(a[5]) || PyTuple_GET_SIZE(a[5]) != 2)
        throw Refusal{PyExc_TypeError, "out must be a pair of tensors"};
      k_out = array<void>(PyTuple_GET_ITEM(a[5], 0), at::kBFloat16, {T, c.heads, c.d}, c.dev, "out");
      v_out = array<void>(PyTuple_GET_ITEM(a[5], 1), at::kBFloat16, {T, c.heads, c.d}, c.dev, "out");
    }
    PyObject* ok = finish(
        g_read(c.k, c.v, c.k_scale, c.v_scale, slots, T, static_cast<int32_t>(c.heads),
               static_cast<int32_t>(c.d), c.n_pages, static_cast<int32_t>(c.page), c.ld_page, c.ld_scale,
               k_out, v_out, own, status, c10::cuda::getCurrentCUDAStream(c.dev).stream()),
        "dwa_kv_read");
    if (ok == nullptr) return nullptr;
    Py_DECREF(ok);
    if (!own) {
      Py_INCREF(a[5]);
      return a[5];
    }
    return Py_BuildValue("(NN)", wrap(k), wrap(v));
  });
}

const at::Tensor& block_table_of(PyObject* o, int dev) {
  const at::Tensor& table = tensor(o, "block_table");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || !on(table, dev) ||
      (table.size(1) > 1 && table.stride(1) != 1))
    refuse("block_table must be int32 [B, max_pages], contiguous along its rows, on the cache's device "
           "(got " + describe(table) + ")");
  return table;
}

// (q, k_cache, v_cache, block_table, lengths, q_start, max_q, k_scale, v_scale, scale, out,
// status), and with a tree also (..., tree_mask) -> out
template <bool kTree>
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, kTree ? 13 : 12, [&]() -> PyObject* {
    const Cache c = cache_of(a[1], a[2], a[7], a[8]);
    const at::Tensor& q = tensor(a[0], "q");
    int64_t q_ld, q_head;
    rows_of(q, -1, c.d, c.dev, "q", &q_ld, &q_head);
    if (q.scalar_type() != at::kBFloat16) refuse("q must be bfloat16 (got " + describe(q) + ")");
    if (q_head != c.d) refuse("q must be contiguous over heads and d");
    const int64_t T = q.size(0), heads = q.size(1), width = heads * c.d;
    const at::Tensor& table = block_table_of(a[3], c.dev);
    const int64_t B = table.size(0), max_pages = table.size(1);
    const int32_t* lengths = array<int32_t>(a[4], at::kInt, {B}, c.dev, "lengths");
    const int32_t* q_start = nullptr;
    int64_t max_q = B ? T / B : 0;
    if (a[5] != Py_None) {
      q_start = array<int32_t>(a[5], at::kInt, {B + 1}, c.dev, "q_start");
      max_q = T;
    }
    if (a[6] != Py_None) {
      max_q = PyLong_AsLongLong(a[6]);
      if (PyErr_Occurred()) return nullptr;
    }
    double scale = 1.0 / std::sqrt(static_cast<double>(c.d));
    if (a[9] != Py_None) {
      scale = PyFloat_AsDouble(a[9]);
      if (PyErr_Occurred()) return nullptr;
    }
    if (heads > INT32_MAX || B > INT32_MAX || max_pages > INT32_MAX || max_q > INT32_MAX || max_q < INT32_MIN)
      refuse("paged_attention: too many heads, sequences, pages or rows");
    int32_t* status = status_of(a[11], c.dev);
    const int64_t* mask = nullptr;
    int64_t words = 0;
    if constexpr (kTree) {
      const at::Tensor& m = tensor(a[12], "tree_mask");
      words = m.dim() == 2 ? m.size(1) : 0;
      mask = array<int64_t>(a[12], at::kLong, {T, words}, c.dev, "tree_mask");
      if (words < 1 || words > INT32_MAX) refuse("tree_mask must have a word at least for every row");
      if (a[6] == Py_None && max_q > 64 * words) max_q = 64 * words;  // T bounds a tree, and so do the words
    }
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    at::Tensor made;
    int64_t out_ld = width;
    void* out;
    if (a[10] == Py_None) {
      made = fresh({T, heads, c.d}, at::kBFloat16, c.dev);
      out = made.data_ptr();
    } else {
      const at::Tensor& o = tensor(a[10], "out");
      int64_t o_head;
      rows_of(o, heads, c.d, c.dev, "out", &out_ld, &o_head);
      if (o.scalar_type() != at::kBFloat16 || o.size(0) != T || o_head != c.d)
        refuse("out must be like q, contiguous over heads and d");
      out = o.data_ptr();
      if (T <= 1) out_ld = width;
    }
    const void* stream = c10::cuda::getCurrentCUDAStream(c.dev).stream();
    auto call = [&](auto entry, auto tree, auto space) {
      const auto before = std::make_tuple(
          q.data_ptr(), T, static_cast<int32_t>(heads), static_cast<int32_t>(c.d), T > 1 ? q_ld : width, c.k, c.v,
          c.k_scale, c.v_scale, static_cast<int32_t>(c.heads), c.n_pages, static_cast<int32_t>(c.page), c.ld_page,
          c.ld_scale, static_cast<int32_t*>(table.data_ptr()), B > 1 ? table.stride(0) : max_pages,
          static_cast<int32_t>(max_pages), lengths, q_start, static_cast<int32_t>(B), static_cast<int32_t>(max_q));
      return std::apply(entry, std::tuple_cat(before, tree, std::make_tuple(static_cast<float>(scale), out, out_ld),
                                              space, std::make_tuple(status, const_cast<void*>(stream))));
    };
    PyObject* ok;
    if constexpr (kTree) {
      const size_t bytes =
          T > 0 && max_q > 0 ? g_tree_workspace(static_cast<int32_t>(heads), static_cast<int32_t>(c.d),
                                                static_cast<int32_t>(c.heads), static_cast<int32_t>(c.page),
                                                static_cast<int32_t>(max_pages), static_cast<int32_t>(B),
                                                static_cast<int32_t>(max_q))
                             : 0;
      at::Tensor held;  // freed in the stream's order
      if (bytes > 0) held = fresh({static_cast<int64_t>(bytes)}, at::kByte, c.dev);
      ok = finish(call(g_attend_tree, std::make_tuple(mask, static_cast<int32_t>(words)),
                       std::make_tuple(bytes > 0 ? held.data_ptr() : nullptr, bytes)),
                  "dwa_paged_tree_attention");
    } else {
      ok = finish(call(g_attend, std::tuple<>(), std::tuple<>()), "dwa_paged_attention");
    }
    if (ok == nullptr) return nullptr;
    Py_DECREF(ok);
    if (a[10] == Py_None) return wrap(made);
    Py_INCREF(a[10]);
    return a[10];
  });
}

// (target_probs, draft_tokens, draft_probs, accept_u, sample_u, draft_lengths) -> (accepted, tokens)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const at::Tensor& target = tensor(a[0], "target_probs");
    const int dev = device_of(target, "target_probs");
    const at::ScalarType type = target.scalar_type();
    if ((type != at::kFloat && type != at::kBFloat16) || target.dim() != 3 || target.size(1) < 1 ||
        !target.is_contiguous())
      refuse("target_probs must be a contiguous float32 or bfloat16 [B, K + 1, V] (got " + describe(target) +
             ")");
    const int64_t B = target.size(0), K = target.size(1) - 1, V = target.size(2);
    if (K > INT32_MAX || V > INT32_MAX) refuse("verify_drafts: too many drafts or tokens");
    const void* draft = a[2] == Py_None ? nullptr : array<void>(a[2], type, {B, K, V}, dev, "draft_probs");
    const int32_t* drafted = array<int32_t>(a[1], at::kInt, {B, K}, dev, "draft_tokens");
    const float* u = array<float>(a[3], at::kFloat, {B, K}, dev, "accept_u");
    const float* r = array<float>(a[4], at::kFloat, {B}, dev, "sample_u");
    const int32_t* lengths =
        a[5] == Py_None ? nullptr : array<int32_t>(a[5], at::kInt, {B}, dev, "draft_lengths");
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    const at::Tensor both = fresh({B * (K + 2)}, at::kInt, dev);
    at::Tensor tokens = part_of(both, 0, {B, K + 1}), accepted = part_of(both, B * (K + 1), {B});
    PyObject* ok = finish(
        g_verify(target.data_ptr(), draft, type == at::kBFloat16, drafted, u, r, lengths, B,
                 static_cast<int32_t>(K), static_cast<int32_t>(V), static_cast<int32_t*>(accepted.data_ptr()),
                 static_cast<int32_t*>(tokens.data_ptr()), c10::cuda::getCurrentCUDAStream(dev).stream()),
        "dwa_verify_drafts");
    if (ok == nullptr) return nullptr;
    Py_DECREF(ok);
    return Py_BuildValue("(NN)", wrap(accepted), wrap(tokens));
  });
}

// (q or None, k, v, cos, sin, k_cache, v_cache, slots, positions or None, k_scale, v_scale,
// q_out or None, status) -> the rotated q, or None
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const Cache c = cache_of(a[5], a[6], a[9], a[10]);
    const at::Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    const at::ScalarType type = k.scalar_type();
    if ((type != at::kBFloat16 && type != at::kFloat) || v.scalar_type() != type)
      refuse("q, k and v must all be bfloat16 or float32");
    int64_t qt = 0, qh = 0, kt, kh, vt, vh;
    rows_of(k, c.heads, c.d, c.dev, "k", &kt, &kh);
    rows_of(v, c.heads, c.d, c.dev, "v", &vt, &vh);
    const int64_t T = k.size(0);
    if (v.size(0) != T) refuse("k and v must have the same number of tokens");
    const at::Tensor &cos = tensor(a[3], "cos"), &sin = tensor(a[4], "sin");
    const at::ScalarType table = cos.scalar_type();
    if ((table != at::kBFloat16 && table != at::kFloat) || sin.scalar_type() != table || cos.dim() != 2 ||
        cos.size(1) != c.d / 2 || sin.sizes() != cos.sizes() || !on(cos, c.dev) || !on(sin, c.dev) ||
        (c.d > 2 && (cos.stride(1) != 1 || sin.stride(1) != 1)) ||
        (cos.size(0) > 1 && cos.stride(0) != sin.stride(0)))
      refuse("cos and sin must both be bfloat16 or float32 [n_positions, d / 2] with the same row stride, on the "
             "cache's device (got " + describe(cos) + " and " + describe(sin) + ")");
    const int64_t n_positions = cos.size(0), ld_table = n_positions > 1 ? cos.stride(0) : c.d / 2;
    const int64_t* slots = array<int64_t>(a[7], at::kLong, {T}, c.dev, "slots");
    const int64_t* positions = a[8] == Py_None ? nullptr : array<int64_t>(a[8], at::kLong, {T}, c.dev, "positions");
    if (positions == nullptr && T > n_positions)
      refuse("without positions cos and sin need a row for every token");
    int32_t* status = status_of(a[12], c.dev);
    const void* q_ptr = nullptr;
    void* q_out = nullptr;
    int64_t heads = 0;
    at::Tensor made;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    if (a[0] != Py_None) {
      const at::Tensor& q = tensor(a[0], "q");
      rows_of(q, -1, c.d, c.dev, "q", &qt, &qh);
      heads = q.size(1);
      if (q.scalar_type() != type || q.size(0) != T || heads < 1 || heads > INT32_MAX)
        refuse("q must have k's type and number of tokens, and a head at least (got " + describe(q) + ")");
      q_ptr = q.data_ptr();
      if (a[11] == Py_None) {
        made = fresh({T, heads, c.d}, at::kBFloat16, c.dev);
        q_out = made.data_ptr();
      } else {
        q_out = array<void>(a[11], at::kBFloat16, {T, heads, c.d}, c.dev, "q_out");
      }
    } else if (a[11] != Py_None) {
      refuse("q_out goes with q");
    }
    PyObject* ok = finish(
        g_append(q_ptr, k.data_ptr(), v.data_ptr(), type == at::kBFloat16, T, static_cast<int32_t>(heads),
                 static_cast<int32_t>(c.heads), static_cast<int32_t>(c.d), qt, qh, kt, kh, vt, vh, cos.data_ptr(),
                 sin.data_ptr(), table == at::kBFloat16, ld_table, n_positions, positions, slots, c.k, c.v,
                 c.k_scale, c.v_scale, c.n_pages, static_cast<int32_t>(c.page), c.ld_page, c.ld_scale, q_out,
                 status, c10::cuda::getCurrentCUDAStream(c.dev).stream()),
        "dwa_kv_append");
    if (ok == nullptr || a[0] == Py_None) return ok;
    Py_DECREF(ok);
    if (a[11] == Py_None) return wrap(made);
    Py_INCREF(a[11]);
    return a[11];
  });
}

// (parents, q_start or None, B or None, max_q or None, status) -> (mask, depth)
PyObject* masks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor& parents_t = tensor(a[0], "parents");
    const int dev = device_of(parents_t, "parents");
    if (parents_t.dim() != 1) refuse("parents must be int32 [T] (got " + describe(parents_t) + ")");
    const int64_t T = parents_t.size(0);
    const int32_t* parents = array<int32_t>(a[0], at::kInt, {T}, dev, "parents");
    const int32_t* q_start = nullptr;
    int64_t B = 1, max_q = T;
    if (a[1] != Py_None) {
      const at::Tensor& s = tensor(a[1], "q_start");
      B = s.dim() == 1 ? s.size(0) - 1 : -1;
      if (B < 0) refuse("q_start must be int32 [B + 1]");
      q_start = array<int32_t>(a[1], at::kInt, {B + 1}, dev, "q_start");
      if (a[2] != Py_None) refuse("n_trees goes without q_start");
    } else if (a[2] != Py_None) {
      B = PyLong_AsLongLong(a[2]);
      if (PyErr_Occurred()) return nullptr;
      if (B < 1 || T % B) refuse("n_trees must be positive and divide the number of nodes");
      max_q = T / B;
    }
    if (a[3] != Py_None) {
      max_q = PyLong_AsLongLong(a[3]);
      if (PyErr_Occurred()) return nullptr;
    }
    if (B > INT32_MAX || max_q < 0 || max_q > INT32_MAX) refuse("tree_masks: too many trees, or a bad max_q");
    int32_t* status = status_of(a[4], dev);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    const int64_t words = max_q > 64 ? (max_q + 63) / 64 : 1;
    const at::Tensor mask = fresh({T, words}, at::kLong, dev), depth = fresh({T}, at::kInt, dev);
    PyObject* ok = finish(g_masks(parents, q_start, T, static_cast<int32_t>(B), static_cast<int32_t>(max_q),
                                  static_cast<int64_t*>(mask.data_ptr()), static_cast<int32_t>(words),
                                  static_cast<int32_t*>(depth.data_ptr()), status,
                                  c10::cuda::getCurrentCUDAStream(dev).stream()),
                          "dwa_tree_masks");
    if (ok == nullptr) return nullptr;
    Py_DECREF(ok);
    return Py_BuildValue("(NN)", wrap(mask), wrap(depth));
  });
}

// (target_probs, tree_tokens, parents, sample_u, q_start or None) -> (accepted, tokens, path)
PyObject* verify_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor& target = tensor(a[0], "target_probs");
    const int dev = device_of(target, "target_probs");
    const at::ScalarType type = target.scalar_type();
    if ((type != at::kFloat && type != at::kBFloat16) || target.dim() != 2 || !target.is_contiguous())
      refuse("target_probs must be a contiguous float32 or bfloat16 [T, V] (got " + describe(target) + ")");
    const int64_t T = target.size(0), V = target.size(1);
    const int32_t* tokens = array<int32_t>(a[1], at::kInt, {T}, dev, "tree_tokens");
    const int32_t* parents = array<int32_t>(a[2], at::kInt, {T}, dev, "parents");
    const at::Tensor& u = tensor(a[3], "sample_u");
    if (u.dim() != 2) refuse("sample_u must be float32 [B, steps] (got " + describe(u) + ")");
    const int64_t B = u.size(0), steps = u.size(1);
    const float* uniform = array<float>(a[3], at::kFloat, {B, steps}, dev, "sample_u");
    const int32_t* q_start =
        a[4] == Py_None ? nullptr : array<int32_t>(a[4], at::kInt, {B + 1}, dev, "q_start");
    if (B > INT32_MAX || steps > INT32_MAX || V > INT32_MAX) refuse("verify_tree: too many sequences, steps or tokens");
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    const at::Tensor all = fresh({B * (2 * steps + 1)}, at::kInt, dev);
    at::Tensor drawn = part_of(all, 0, {B, steps}), path = part_of(all, B * steps, {B, steps}),
               accepted = part_of(all, 2 * B * steps, {B});
    PyObject* ok = finish(g_verify_tree(target.data_ptr(), type == at::kBFloat16, tokens, parents, q_start, uniform, T,
                                        static_cast<int32_t>(B), static_cast<int32_t>(steps),
                                        static_cast<int32_t>(V), static_cast<int32_t*>(accepted.data_ptr()),
                                        static_cast<int32_t*>(drawn.data_ptr()),
                                        static_cast<int32_t*>(path.data_ptr()),
                                        c10::cuda::getCurrentCUDAStream(dev).stream()),
                          "dwa_verify_tree");
    if (ok == nullptr) return nullptr;
    Py_DECREF(ok);
    return Py_BuildValue("(NNN)", wrap(accepted), wrap(drawn), wrap(path));
  });
}

// (k_cache, v_cache, block_table, start, path, n_accepted, k_scale, v_scale, status); the caches are
// one layer's, or [layers, n_pages, H_kv, page_size, d]
PyObject* kv_keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const at::Tensor& k = tensor(a[0], "k_cache");
    Cache c;
    int64_t layers = 1, ld_layer = 0, ld_scale_layer = 0;
    if (k.dim() == 5) {
      const at::Tensor& v = tensor(a[1], "v_cache");
      layers = k.size(0);
      if (layers < 1) refuse("k_cache must have a layer at least");
      if (v.sizes() != k.sizes() || v.strides() != k.strides())
        refuse("v_cache must be like k_cache (type, shape, strides, device)");
      ld_layer = k.stride(0);
      at::Tensor parts[4] = {k.select(0, 0), v.select(0, 0)};
      PyObject* of[4] = {nullptr, nullptr, a[6], a[7]};
      for (int i = 2; i < 4; ++i)
        if (of[i] != Py_None) {
          const at::Tensor& scale = tensor(of[i], "scale");
          if (scale.dim() != 4 || scale.size(0) != layers) refuse("scales must be f32 [layers, n_pages, H_kv, page_size]");
          if (i == 3 && scale.stride(0) != ld_scale_layer) refuse("k_scale and v_scale must have the same strides");
          ld_scale_layer = scale.stride(0);
          parts[i] = scale.select(0, 0);
        }
      // of the first layer, as every call's
      PyObject* held[4];
      for (int i = 0; i < 4; ++i) {
        if (parts[i].defined()) {
          held[i] = wrap(parts[i]);
        } else {
          Py_INCREF(Py_None);
          held[i] = Py_None;
        }
      }
      struct Release {
        PyObject** p;
        ~Release() {
          for (int i = 0; i < 4; ++i) Py_DECREF(p[i]);
        }
      } release{held};
      c = cache_of(held[0], held[1], held[2], held[3]);
    } else {
      c = cache_of(a[0], a[1], a[6], a[7]);
    }
    const at::Tensor& table = block_table_of(a[2], c.dev);
    const int64_t B = table.size(0), max_pages = table.size(1);
    const int32_t* start = array<int32_t>(a[3], at::kInt, {B}, c.dev, "start");
    const at::Tensor& path_t = tensor(a[4], "path");
    if (path_t.dim() != 2) refuse("path must be int32 [B, steps] (got " + describe(path_t) + ")");
    const int64_t steps = path_t.size(1);
    const int32_t* path = array<int32_t>(a[4], at::kInt, {B, steps}, c.dev, "path");
    const int32_t* kept = array<int32_t>(a[5], at::kInt, {B}, c.dev, "n_accepted");
    int32_t* status = status_of(a[8], c.dev);
    if (layers > INT32_MAX || B > INT32_MAX || steps > INT32_MAX || max_pages > INT32_MAX)
      refuse("kv_cache_keep: too many layers, sequences, steps or pages");
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    return finish(g_keep(c.k, c.v, c.k_scale, c.v_scale, static_cast<int32_t>(layers), ld_layer, ld_scale_layer,
                         static_cast<int32_t>(c.heads), static_cast<int32_t>(c.d), c.n_pages,
                         static_cast<int32_t>(c.page), c.ld_page, c.ld_scale, static_cast<int32_t*>(table.data_ptr()),
                         B > 1 ? table.stride(0) : max_pages, static_cast<int32_t>(max_pages), start, path, kept,
                         static_cast<int32_t>(B), static_cast<int32_t>(steps), status,
                         c10::cuda::getCurrentCUDAStream(c.dev).stream()),
                  "dwa_kv_keep");
  });
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"kv_write", reinterpret_cast<PyCFunction>(kv_write), METH_FASTCALL, nullptr},
    {"kv_read", reinterpret_cast<PyCFunction>(kv_read), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(attend<false>), METH_FASTCALL, nullptr},
    {"verify", reinterpret_cast<PyCFunction>(verify), METH_FASTCALL, nullptr},
    {"kv_append", reinterpret_cast<PyCFunction>(kv_append), METH_FASTCALL, nullptr},
    {"kv_keep", reinterpret_cast<PyCFunction>(kv_keep), METH_FASTCALL, nullptr},
    {"attend_tree", reinterpret_cast<PyCFunction>(attend<true>), METH_FASTCALL, nullptr},
    {"masks", reinterpret_cast<PyCFunction>(masks), METH_FASTCALL, nullptr},
    {"verify_tree", reinterpret_cast<PyCFunction>(verify_tree), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&g_module); }
