// The calls of a decoding step from Python.
//
// A step's kernels take a few microseconds each, and Python's checks of their
// arguments, the allocations and a ctypes call of 20 to 36 arguments (0.1 us
// each) took 12 to 19.  Two layers take their place:
//
//   hier_*     an entry point of hier_b200.h as it is, called with ints
//              (pointers too; None is NULL), bools and floats; an int that its
//              C type cannot hold is refused
//   layout, append, attention, page_step, head_norm
//              the checks, allocations and call of a cache over tensors and of
//              the operators' Python functions, for well-formed tensors.  They
//              return None, having done nothing, for anything else (another device than the
//              current one, rows that need a copy, arguments to refuse), which
//              the Python functions then do or refuse; an int is a status.
//
// and words_beside_capture, what a capture must not make by itself.
//
// The module holds no code of the library: bind() gives it the addresses of
// the one that is loaded.

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstring>

#include "hier_b200.h"
#include "pycall.h"

namespace {

using pycall::attempt;
using pycall::unlocked;

// ---- entry points as they are ----------------------------------------------

constexpr int kMaxArgs = 40;

struct Words {
  int64_t w[kMaxArgs];
  float f;  // no entry has more than one
};

// `sig` names the parameters: p pointer, q int64, i int32, f float
bool read_words(const char* name, const char* sig, PyObject* const* a, Py_ssize_t n, Words* out) {
  if (n != (Py_ssize_t)strlen(sig)) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, (Py_ssize_t)strlen(sig), n);
    return false;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (sig[i] == 'f') {
      out->f = (float)PyFloat_AsDouble(a[i]);
      if (out->f == -1.f && PyErr_Occurred()) return false;
      continue;
    }
    if (sig[i] == 'p' && a[i] == Py_None) {
      out->w[i] = 0;
      continue;
    }
    const long long v = PyLong_AsLongLong(a[i]);
    if (v == -1 && PyErr_Occurred()) return false;
    if (sig[i] == 'i' && (v < INT32_MIN || v > INT32_MAX)) {
      PyErr_Format(PyExc_ValueError, "%s: argument %zd (%lld) passes 32 bits", name, i, v);
      return false;
    }
    out->w[i] = v;
  }
  return true;
}

struct Pointer {  // any data pointer
  void* p;
  template <class T>
  operator T*() const { return static_cast<T*>(p); }
};

#define P(i) (Pointer{reinterpret_cast<void*>(static_cast<uintptr_t>(x.w[i]))})
#define Q(i) (x.w[i])
#define I(i) (static_cast<int32_t>(x.w[i]))

// One entry: its bound address, and a method that reads `SIG` (its doc string
// too) and calls it.
#define ENTRY(NAME, SIG, ...)                                                   \
  const char SIG_##NAME[] = SIG;                                                \
  decltype(&NAME) at_##NAME;                                                    \
  PyObject* py_##NAME(PyObject*, PyObject* const* a, Py_ssize_t n) {            \
    Words x;                                                                    \
    if (!read_words(#NAME, SIG_##NAME, a, n, &x)) return nullptr;               \
    if (!at_##NAME) {                                                           \
      PyErr_SetString(PyExc_RuntimeError, #NAME " is not bound");               \
      return nullptr;                                                           \
    }                                                                           \
    return PyLong_FromLong(unlocked([&] { return at_##NAME(__VA_ARGS__); }));   \
  }

ENTRY(hier_head_norm_rope, "pqpqqiiippipqpfpqpqpqpqipp", P(0), Q(1), P(2), Q(3), Q(4), I(5), I(6),
      I(7), P(8), P(9), I(10), P(11), Q(12), P(13), x.f, P(15), Q(16), P(17), Q(18), P(19), Q(20),
      P(21), Q(22), I(23), P(24), P(25))
ENTRY(hier_head_norm_rope_bwd, "pqpqqiiippipqpfpqpqpqpqpipppp", P(0), Q(1), P(2), Q(3), Q(4), I(5),
      I(6), I(7), P(8), P(9), I(10), P(11), Q(12), P(13), x.f, P(15), Q(16), P(17), Q(18), P(19),
      Q(20), P(21), Q(22), P(23), I(24), P(25), P(26), P(27), P(28))
ENTRY(hier_page_step, "ppipqipipiippppppp", P(0), P(1), I(2), P(3), Q(4), I(5), P(6), I(7), P(8),
      I(9), I(10), P(11), P(12), P(13), P(14), P(15), P(16), P(17))
ENTRY(hier_paged8_append, "pqpqiiippppipqippipp", P(0), Q(1), P(2), Q(3), I(4), I(5), I(6), P(7),
      P(8), P(9), P(10), I(11), P(12), Q(13), I(14), P(15), P(16), I(17), P(18), P(19))
ENTRY(hier_paged8_attn, "pqiiiiippppipqippiiiifipqpipppp", P(0), Q(1), I(2), I(3), I(4), I(5),
      I(6), P(7), P(8), P(9), P(10), I(11), P(12), Q(13), I(14), P(15), P(16), I(17), I(18), I(19),
      I(20), x.f, I(22), P(23), Q(24), P(25), I(26), P(27), P(28), P(29), P(30))

decltype(&hier_paged8_attn_workspace) at_hier_paged8_attn_workspace;
decltype(&hier_head_norm_rope_bwd_partials) at_hier_head_norm_rope_bwd_partials;
decltype(&hier_last_error) at_hier_last_error;

// ---- whole calls -------------------------------------------------------------

constexpr int kDim = 128, kPage = 64;

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool int_of(PyObject* o, int64_t lo, int64_t hi, int64_t* out) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *out = v;
  return v >= lo && v <= hi;
}

template <class T>
T* data(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// bf16 [T, width] that a kernel can read as it is
bool is_rows(const at::Tensor* t, int64_t width, at::Device dev) {
  return t && t->scalar_type() == at::kBFloat16 && t->device() == dev && t->dim() == 2 &&
         t->size(1) == width && t->size(0) > 0 && t->size(0) <= INT32_MAX && t->stride(1) == 1 &&
         t->stride(0) >= width && t->stride(0) % 8 == 0 && aligned(*t);
}

bool is_vector(const at::Tensor* t, int64_t n, at::Device dev) {
  return t && t->scalar_type() == at::kInt && t->device() == dev && t->dim() == 1 &&
         t->size(0) == n && t->is_contiguous();
}

// a block table of at least one request and page
bool is_table(const at::Tensor* t, at::Device dev) {
  return t && t->scalar_type() == at::kInt && t->device() == dev && t->dim() == 2 && t->size(0) > 0 &&
         t->size(1) > 0 && t->size(0) < INT32_MAX && t->size(1) <= INT32_MAX / kPage &&
         t->stride(1) == 1 && t->stride(0) >= t->size(1);
}

// the current device, and its current stream
bool on_current(at::Device dev) { return dev.is_cuda() && dev.index() == c10::cuda::current_device(); }
void* stream_of(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

struct Cache {
  const at::Tensor *k, *v, *k_scale, *v_scale, *status;
  int64_t format, pages, heads;
};

// k, v, k_scale, v_scale, status, format of a cache that its class has checked
bool cache_of(PyObject* const* a, Cache* c) {
  c->k = tensor_of(a[0]), c->v = tensor_of(a[1]), c->k_scale = tensor_of(a[2]), c->v_scale = tensor_of(a[3]);
  c->status = tensor_of(a[4]);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->status || !int_of(a[5], 0, 1, &c->format))
    return false;
  c->pages = c->k->size(0), c->heads = c->k->size(1);
  return c->pages <= INT32_MAX && aligned(*c->k) && aligned(*c->v) && on_current(c->k->device());
}

// one table row of pages, a length and row starts for each request
struct Requests {
  const at::Tensor *table, *lengths, *q_start;
};
bool requests_of(PyObject* const* a, at::Device dev, Requests* r) {
  r->table = tensor_of(a[0]), r->lengths = tensor_of(a[1]), r->q_start = tensor_of(a[2]);
  return is_table(r->table, dev) && is_vector(r->lengths, r->table->size(0), dev) &&
         is_vector(r->q_start, r->table->size(0) + 1, dev);
}

// words_beside_capture(device, count) -> int32 [count], zeros: allocated and zeroed on a stream of
// its own, so that neither is a part of the graph that this thread captures.
PyObject* words_beside_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
  int64_t dev, count;
  if (n != 2 || !int_of(a[0], 0, 127, &dev) || !int_of(a[1], 1, INT32_MAX, &count)) {
    PyErr_SetString(PyExc_TypeError, "words_beside_capture(device, count)");
    return nullptr;
  }
  try {
    const c10::InferenceMode mode(false);
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};
    const c10::cuda::CUDAStreamGuard stream(c10::cuda::getStreamFromPool(false, (c10::DeviceIndex)dev));
    at::Tensor words = at::zeros({count}, at::device(stream.current_stream().device()).dtype(at::kInt));
    stream.current_stream().synchronize();
    return THPVariable_Wrap(std::move(words));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// layout(k, v, k_scale, v_scale) -> format of a cache over them
PyObject* layout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    if (n != 4) return nullptr;
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i) {
      t[i] = tensor_of(a[i]);
      if (!t[i] || t[i]->device() != t[0]->device() || !t[i]->is_contiguous()) return nullptr;
    }
    const auto type = t[0]->scalar_type();
    if ((type != at::kChar && type != at::kFloat8_e4m3fn) || t[1]->scalar_type() != type ||
        t[2]->scalar_type() != at::kFloat || t[3]->scalar_type() != at::kFloat || t[0]->dim() != 5)
      return nullptr;
    const int64_t pages = t[0]->size(0), heads = t[0]->size(1);
    if (pages < 1 || heads < 1 || t[0]->sizes() != at::IntArrayRef({pages, heads, 2, kPage, 64}) ||
        t[1]->sizes() != at::IntArrayRef({pages, heads, kDim, kPage}) ||
        t[2]->sizes() != at::IntArrayRef({pages, heads}) || t[3]->sizes() != t[2]->sizes())
      return nullptr;
    return PyLong_FromLong(type == at::kFloat8_e4m3fn);
  });
}

// append(*cache, k, v, table, lengths, q_start) -> status
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    Cache c;
    Requests r;
    if (n != 11 || !at_hier_paged8_append || !cache_of(a, &c)) return nullptr;
    const at::Device dev = c.k->device();
    const at::Tensor *k = tensor_of(a[6]), *v = tensor_of(a[7]);
    if (!is_rows(k, c.heads * kDim, dev) || !is_rows(v, c.heads * kDim, dev) || k->size(0) != v->size(0) ||
        !requests_of(a + 8, dev, &r))
      return nullptr;
    void* stream = stream_of(dev);
    return PyLong_FromLong(unlocked([&] {
      return at_hier_paged8_append(
          k->data_ptr(), k->stride(0), v->data_ptr(), v->stride(0), (int32_t)k->size(0), (int32_t)c.heads,
          (int32_t)c.format, c.k->data_ptr(), c.v->data_ptr(), data<float>(*c.k_scale),
          data<float>(*c.v_scale), (int32_t)c.pages, data<int32_t>(*r.table), r.table->stride(0),
          (int32_t)r.table->size(1), data<int32_t>(*r.lengths), data<int32_t>(*r.q_start),
          (int32_t)r.table->size(0), data<int32_t>(*c.status), stream);
    }));
  });
}

// attention(*cache, q, table, lengths, q_start, heads, frame, block, window, scale, max_rows, out,
// return_lse, dev_err) -> out or (out, lse), or a status
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    Cache c;
    Requests r;
    int64_t heads, frame, block, window, most = 0;
    constexpr int64_t kMost = 1 << 30;
    if (n != 19 || !at_hier_paged8_attn || !at_hier_paged8_attn_workspace || !cache_of(a, &c) ||
        !int_of(a[10], 1, INT32_MAX / kDim, &heads) || !int_of(a[11], 1, kMost, &frame) ||
        !int_of(a[12], 0, kMost, &block) || !int_of(a[13], -1, kMost, &window) || window == 0 ||
        heads % c.heads)
      return nullptr;
    float scale = (float)(1.0 / std::sqrt((double)kDim));
    if (a[14] != Py_None) {
      scale = (float)PyFloat_AsDouble(a[14]);
      if (PyErr_Occurred()) {
        PyErr_Clear();
        return nullptr;
      }
    }
    if (!(scale > 0.f && scale < INFINITY)) return nullptr;
    if (a[15] != Py_None && !int_of(a[15], 0, INT32_MAX, &most)) return nullptr;
    const at::Device dev = c.k->device();
    const at::Tensor *q = tensor_of(a[6]), *err = tensor_of(a[18]);
    if (!is_rows(q, heads * kDim, dev) || !requests_of(a + 7, dev, &r) || !err) return nullptr;
    const int64_t rows = q->size(0);
    const bool given = a[16] != Py_None;
    const at::Tensor* to = given ? tensor_of(a[16]) : nullptr;
    if (given && (!is_rows(to, heads * kDim, dev) || to->size(0) != rows)) return nullptr;
    const int with_lse = PyObject_IsTrue(a[17]);
    if (with_lse < 0) return nullptr;
    int64_t floats = 0;
    int rc = at_hier_paged8_attn_workspace((int32_t)rows, (int32_t)heads, (int32_t)c.heads,
                                           (int32_t)r.table->size(0), (int32_t)r.table->size(1),
                                           (int32_t)most, &floats);
    if (rc) return PyLong_FromLong(rc);
    at::Tensor out, lse, workspace;
    const auto f32 = c.k_scale->options();
    if (!given) out = at::empty({rows, heads * kDim}, q->options());
    if (with_lse) lse = at::empty({rows, heads}, f32);
    if (floats) workspace = at::empty({floats}, f32);
    const at::Tensor& o = given ? *to : out;
    void* stream = stream_of(dev);
    rc = unlocked([&] {
      return at_hier_paged8_attn(
          q->data_ptr(), q->stride(0), (int32_t)rows, (int32_t)heads, (int32_t)c.heads, kDim,
          (int32_t)c.format, c.k->data_ptr(), c.v->data_ptr(), data<float>(*c.k_scale),
          data<float>(*c.v_scale), (int32_t)c.pages, data<int32_t>(*r.table), r.table->stride(0),
          (int32_t)r.table->size(1), data<int32_t>(*r.lengths), data<int32_t>(*r.q_start),
          (int32_t)r.table->size(0), (int32_t)frame, (int32_t)block, (int32_t)window, scale,
          (int32_t)most, o.data_ptr(), o.stride(0), with_lse ? data<float>(lse) : nullptr,
          !given ? 1 : with_lse ? 2 : 0,
          floats ? data<float>(workspace) : nullptr, data<int32_t>(*c.status), data<int32_t>(*err),
          stream);
    });
    if (rc) return PyLong_FromLong(rc);
    PyObject* result;
    if (given) {
      Py_INCREF(a[16]);
      result = a[16];
    } else {
      result = THPVariable_Wrap(std::move(out));
    }
    if (!with_lse || !result) return result;
    PyObject* second = THPVariable_Wrap(std::move(lse));
    PyObject* both = second ? PyTuple_Pack(2, result, second) : nullptr;
    Py_DECREF(result);
    Py_XDECREF(second);
    return both;
  });
}

// n elements of a vector from `at` on, as a tensor over the same memory
at::Tensor part_of(const at::Tensor& t, int64_t at, int64_t n) {
  auto r = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  r.unsafeGetTensorImpl()->set_storage_offset(at);
  r.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return r;
}

// page_step(lengths, add, table, free_pages, free_count, rows, most_new, in_place) -> (lengths,
// free_count, q_start, status, slots, positions), or a status
PyObject* page_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    int64_t rows, most = -1;
    if (n != 8 || !at_hier_page_step || !int_of(a[5], 0, INT32_MAX, &rows) ||
        (a[6] != Py_None && !int_of(a[6], 0, INT32_MAX, &most)))
      return nullptr;
    const at::Tensor *lengths = tensor_of(a[0]), *add = tensor_of(a[1]), *table = tensor_of(a[2]);
    const at::Tensor *list = tensor_of(a[3]), *count = tensor_of(a[4]);
    if (!table || !on_current(table->device())) return nullptr;
    const at::Device dev = table->device();
    if (!is_table(table, dev) || !list || list->dim() != 1 || list->size(0) > INT32_MAX) return nullptr;
    const int64_t requests = table->size(0);
    if (!is_vector(lengths, requests, dev) || !is_vector(add, requests, dev) ||
        !is_vector(list, list->size(0), dev) || !is_vector(count, 1, dev))
      return nullptr;
    const int in_place = PyObject_IsTrue(a[7]);
    if (in_place < 0) return nullptr;
    // [lengths, free_count,] q_start, status, slots, positions
    const int64_t sizes[6] = {requests, 1, requests + 1, 1, rows, rows};
    const int first = in_place ? 2 : 0;
    int64_t starts[7] = {};
    for (int i = first; i < 6; ++i) starts[i + 1] = starts[i] + sizes[i];
    const at::Tensor all = at::empty({starts[6]}, lengths->options());
    // (made before the launch: nothing may fail once the step has been taken)
    PyObject* result = PyTuple_New(6);
    if (!result) return nullptr;
    const pycall::Owned owned{result};
    for (int i = 0; i < 6; ++i) {
      PyObject* one;
      if (i < first) {
        one = a[i ? 4 : 0];
        Py_INCREF(one);
      } else {
        one = THPVariable_Wrap(part_of(all, starts[i], sizes[i]));
      }
      if (!one) return nullptr;
      PyTuple_SET_ITEM(result, i, one);
    }
    int32_t* base = data<int32_t>(all);
    int32_t* new_lengths = in_place ? data<int32_t>(*lengths) : base;
    int32_t* new_count = in_place ? data<int32_t>(*count) : base + starts[1];
    void* stream = stream_of(dev);
    const int rc = unlocked([&] {
      return at_hier_page_step(
          data<int32_t>(*lengths), data<int32_t>(*add), (int32_t)requests, data<int32_t>(*table),
          table->stride(0), (int32_t)table->size(1), data<int32_t>(*list), (int32_t)list->size(0),
          data<int32_t>(*count), (int32_t)rows, (int32_t)most, new_lengths, new_count,
          base + starts[2], base + starts[4], base + starts[5], base + starts[3], stream);
    });
    if (rc) return PyLong_FromLong(rc);
    Py_INCREF(result);
    return result;
  });
}

// The arguments of the per-head norm: q, k, freqs, heads, key heads, weights, positions (or None), eps
// and the device's error word.
struct HeadNorm {
  const at::Tensor *q, *k, *freqs, *wq, *wk, *pos, *err;
  int64_t rows, heads, kv_heads, D;
  float eps;
  bool f32;  // the weights
};

bool head_norm_of(PyObject* const* a, Py_ssize_t n, HeadNorm* h) {
  if (n != 10 || !at_hier_head_norm_rope || !int_of(a[3], 1, 4096, &h->heads) ||
      !int_of(a[4], 1, 4096, &h->kv_heads))
    return false;
  h->q = tensor_of(a[0]), h->k = tensor_of(a[1]), h->freqs = tensor_of(a[2]);
  h->wq = tensor_of(a[5]), h->wk = tensor_of(a[6]), h->err = tensor_of(a[9]);
  if (!h->q || !h->k || !h->freqs || !h->wq || !h->wk || !h->err || h->q->dim() != 2 ||
      !on_current(h->q->device()))
    return false;
  const at::Device dev = h->q->device();
  h->D = h->q->size(1) / h->heads, h->rows = h->q->size(0);
  if (h->D * h->heads != h->q->size(1) || (h->D != 64 && h->D != 128 && h->D != 256) ||
      !is_rows(h->q, h->heads * h->D, dev) || !is_rows(h->k, h->kv_heads * h->D, dev) ||
      h->k->size(0) != h->rows)
    return false;
  for (const at::Tensor* w : {h->wq, h->wk})
    if (w->dim() != 1 || w->size(0) != h->D || w->device() != dev || !w->is_contiguous() ||
        w->scalar_type() != h->wq->scalar_type())
      return false;
  h->f32 = h->wq->scalar_type() == at::kFloat;
  if (!h->f32 && h->wq->scalar_type() != at::kBFloat16) return false;
  const at::Tensor& f = *h->freqs;
  if (f.scalar_type() != at::kFloat || f.device() != dev || f.dim() != 3 || f.size(0) < 1 ||
      f.size(1) * 2 != h->D || f.size(2) != 2 || !f.is_contiguous() || !aligned(f))
    return false;
  h->pos = nullptr;
  if (a[7] != Py_None) {
    h->pos = tensor_of(a[7]);
    if (!is_vector(h->pos, h->rows, dev)) return false;
  } else if (h->rows % f.size(0)) {
    return false;
  }
  h->eps = (float)PyFloat_AsDouble(a[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

int head_norm_forward(const HeadNorm& h, at::Tensor* q, at::Tensor* k) {
  *q = at::empty({h.rows, h.heads * h.D}, h.q->options());
  *k = at::empty({h.rows, h.kv_heads * h.D}, h.k->options());
  return at_hier_head_norm_rope(
      h.q->data_ptr(), h.q->stride(0), h.k->data_ptr(), h.k->stride(0), h.rows, (int32_t)h.heads,
      (int32_t)h.kv_heads, (int32_t)h.D, h.wq->data_ptr(), h.wk->data_ptr(), h.f32, data<float>(*h.freqs),
      h.freqs->size(0), h.pos ? data<int32_t>(*h.pos) : nullptr, h.eps, q->data_ptr(), q->stride(0),
      nullptr, h.rows, k->data_ptr(), k->stride(0), nullptr, h.rows, 1, data<int32_t>(*h.err),
      stream_of(h.q->device()));
}

PyObject* pair_of(at::Tensor a, at::Tensor b) {
  PyObject *first = THPVariable_Wrap(std::move(a)), *second = THPVariable_Wrap(std::move(b));
  PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
  Py_XDECREF(first);
  Py_XDECREF(second);
  return both;
}

// head_norm(*arguments) -> (q, k), or a status
PyObject* head_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    HeadNorm h;
    if (!head_norm_of(a, n, &h)) return nullptr;
    at::Tensor q, k;
    const int rc = unlocked([&] { return head_norm_forward(h, &q, &k); });
    return rc ? PyLong_FromLong(rc) : pair_of(std::move(q), std::move(k));
  });
}

// The same with gradients for q, k and the weights.  The engine calls back
// without Python; differentiating twice is an error, as of any kernel.
struct HeadNormFn : torch::autograd::Function<HeadNormFn> {
  using Context = torch::autograd::AutogradContext;
  using Tensors = torch::autograd::variable_list;

  static Tensors forward(Context* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq,
                         const at::Tensor& wk, const HeadNorm* h, int* rc) {
    at::Tensor qo, ko;
    *rc = head_norm_forward(*h, &qo, &ko);
    ctx->save_for_backward({q, k, wq, wk, *h->freqs, h->pos ? *h->pos : at::Tensor()});
    ctx->saved_data["err"] = *h->err;  // (no input: cleared when a caller likes)
    ctx->saved_data["sizes"] = std::vector<int64_t>{h->heads, h->kv_heads, h->D};
    ctx->saved_data["eps"] = (double)h->eps;
    return {qo, ko};
  }

  static Tensors backward(Context* ctx, Tensors g) {
    const Tensors s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3], &freqs = s[4], &pos = s[5];
    const at::Tensor err = ctx->saved_data["err"].toTensor();
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const float eps = (float)ctx->saved_data["eps"].toDouble();
    const int64_t rows = q.size(0), D = sizes[2];
    const int32_t heads = (int32_t)sizes[0], kv_heads = (int32_t)sizes[1];
    const at::Device dev = q.device();
    for (int i = 0; i < 2; ++i)  // (already of the outputs' type and shape)
      if (!is_rows(&g[i], sizes[i] * D, dev)) g[i] = g[i].clone(at::MemoryFormat::Contiguous);
    Tensors d;
    {
      const at::NoGradGuard none;
      d = {at::empty({rows, heads * D}, q.options()), at::empty({rows, kv_heads * D}, k.options()),
           at::empty_like(wq), at::empty_like(wk)};
    }
    int32_t blocks = 0;
    int rc = at_hier_head_norm_rope_bwd_partials(rows, heads, kv_heads, (int32_t)D, &blocks);
    const at::Tensor part = at::empty({blocks, D}, freqs.options());
    if (!rc)
      rc = at_hier_head_norm_rope_bwd(
          q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), rows, heads, kv_heads, (int32_t)D,
          wq.data_ptr(), wk.data_ptr(), wq.scalar_type() == at::kFloat, data<float>(freqs), freqs.size(0),
          pos.defined() ? data<int32_t>(pos) : nullptr, eps, g[0].data_ptr(), g[0].stride(0),
          g[1].data_ptr(), g[1].stride(0), d[0].data_ptr(), heads * D, d[1].data_ptr(), kv_heads * D,
          data<float>(part), blocks, d[2].data_ptr(), d[3].data_ptr(), data<int32_t>(err), stream_of(dev));
    TORCH_CHECK(!rc, at_hier_last_error());
    if (at::GradMode::is_enabled()) {
      for (at::Tensor& t : d) t.set_requires_grad(true);
      const auto twice = std::make_shared<torch::autograd::DelayedError>(
          "the per-head norm's gradients cannot be differentiated again", (int64_t)d.size());
      d = (*twice)(std::move(d));
    }
    return {d[0], d[1], d[2], d[3], at::Tensor(), at::Tensor()};
  }
};

// head_norm_grad(*arguments) -> (q, k) with their graph, or a status
PyObject* head_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    HeadNorm h;
    if (!at_hier_head_norm_rope_bwd || !at_hier_head_norm_rope_bwd_partials || !at_hier_last_error ||
        !head_norm_of(a, n, &h))
      return nullptr;
    int rc = 0;
    const auto out = HeadNormFn::apply(*h.q, *h.k, *h.wq, *h.wk, &h, &rc);
    return rc ? PyLong_FromLong(rc) : pair_of(out[0], out[1]);
  });
}

// ---- the module ----------------------------------------------------------------

#define BOUND(NAME) {#NAME, reinterpret_cast<void**>(&at_##NAME)}

const struct {
  const char* name;
  void** at;
} entries[] = {BOUND(hier_head_norm_rope), BOUND(hier_head_norm_rope_bwd), BOUND(hier_page_step),
               BOUND(hier_paged8_append),  BOUND(hier_paged8_attn),
               BOUND(hier_paged8_attn_workspace),
               BOUND(hier_head_norm_rope_bwd_partials),
               BOUND(hier_last_error)};

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "bind(name, address)");
    return nullptr;
  }
  const char* name = PyUnicode_AsUTF8(a[0]);
  if (!name) return nullptr;
  void* address = PyLong_AsVoidPtr(a[1]);
  if (!address && PyErr_Occurred()) return nullptr;
  for (const auto& e : entries)
    if (!strcmp(e.name, name)) {
      memcpy(e.at, &address, sizeof(address));
      Py_RETURN_NONE;
    }
  return PyErr_Format(PyExc_ValueError, "no entry %s", name);
}

#define METHOD(NAME, FN, DOC) \
  {NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(FN)), METH_FASTCALL, DOC}
#define RAW(NAME) METHOD(#NAME, py_##NAME, SIG_##NAME)

PyMethodDef methods[] = {
    METHOD("bind", bind, "bind(name, address): where an entry point is"),
    METHOD("words_beside_capture", words_beside_capture, "zeros that no graph owns"),
    METHOD("layout", layout, "format of a cache over tensors of its layout"),
    METHOD("append", append, "paged8_append of well-formed tensors"),
    METHOD("attention", attention, "paged8_attention of well-formed tensors"),
    METHOD("page_step", page_step, "page_step of well-formed tensors"),
    METHOD("head_norm", head_norm, "hier_head_norm_rope of well-formed tensors"),
    METHOD("head_norm_grad", head_norm_grad, "head_norm_rope_grad of well-formed tensors"),
    RAW(hier_head_norm_rope),
    RAW(hier_head_norm_rope_bwd),
    RAW(hier_page_step),
    RAW(hier_paged8_append),
    RAW(hier_paged8_attn),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Calls of libhier_b200.so's entry points.", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&module); }
