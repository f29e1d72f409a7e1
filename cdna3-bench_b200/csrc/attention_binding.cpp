// Python binding of the attention operators (mxfp4_b200/attention.py): argument checks, output and
// workspace allocation and the C call in one step, for calls whose work on the GPU is a few
// microseconds (measured per call, checks in Python and ctypes against this: 17 -> 4.5 us for
// qk_norm_rope).  The C entries' addresses come from the library that _lib.py loaded, so that
// both bindings call the same one.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/mxfp4_b200.h"

namespace {

struct Entries {
  decltype(&mxfp4_error_string) error_string;
  decltype(&mxfp4_qk_norm_rope) qk_norm_rope;
  decltype(&mxfp4_qk_norm_rope_cache) qk_norm_rope_cache;
  decltype(&mxfp4_kv_cache_write) write;
  decltype(&mxfp4_kv_cache_read) read;
  decltype(&mxfp4_paged_attention_workspace_bytes) attention_bytes;
  decltype(&mxfp4_paged_attention) attention;
};
Entries g_entries = {};

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error(what); }

void check(int code, const char* what) {
  if (code) refuse(std::string(what) + ": " + g_entries.error_string(code) + " (code " + std::to_string(code) + ")");
}

// The tensor behind an argument; null if it is none.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int integer(PyObject* o, const char* what) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(what) + " out of range");
  return static_cast<int>(v);
}
int64_t as_int(int64_t n, const char* what) {
  if (n > INT32_MAX) refuse(std::string(what) + " out of range");
  return n;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

// An int32 vector of n on `dev`.
const int* index_vector(PyObject* o, int64_t n, c10::Device dev, const char* what) {
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != at::kInt || t->device() != dev || t->dim() != 1 || t->size(0) != n ||
      (n > 1 && t->stride(0) != 1))
    refuse(std::string(what) + " must be a contiguous int32 vector of " + std::to_string(n) + " on " + dev.str());
  return static_cast<const int*>(t->data_ptr());
}

struct Cache {
  mxfp4_kv_cache c;
  c10::Device dev;
};
// From an MXKVCache: its four tensors, the address of the C structure that describes them and the device's index.
// The memory is the tensors' own as they are now: they may have been given another storage since, or lost it.
Cache cache_of(PyObject* native) {
  if (!PyTuple_Check(native) || PyTuple_GET_SIZE(native) != 6) refuse("cache must be an MXKVCache");
  const void* p = PyLong_AsVoidPtr(PyTuple_GET_ITEM(native, 4));
  if (!p && PyErr_Occurred()) throw python_error();
  Cache r = {*static_cast<const mxfp4_kv_cache*>(p),
             c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(integer(PyTuple_GET_ITEM(native, 5), "device")))};
  uint8_t* at[4];
  for (int i = 0; i < 4; ++i) {
    const at::Tensor* t = tensor(PyTuple_GET_ITEM(native, i));
    const int64_t width = i >= 2 ? r.c.head_dim / 32 : (r.c.format == MXFP4_KV_MXFP8 ? r.c.head_dim : r.c.head_dim / 2);
    const int64_t rows = int64_t(r.c.num_pages) * r.c.num_kv_heads * r.c.page_size;
    if (!t || t->scalar_type() != at::kByte || t->device() != r.dev || !t->is_contiguous() || t->dim() != 4 ||
        t->size(0) != r.c.num_pages || t->size(1) != r.c.num_kv_heads || t->size(2) != r.c.page_size || t->size(3) != width ||
        static_cast<int64_t>(t->storage().nbytes()) < t->storage_offset() + rows * width)
      refuse("the cache's tensors are no longer those it was made of: type, shape, device or storage has changed");
    at[i] = static_cast<uint8_t*>(t->data_ptr());
  }
  r.c.k_codes = at[0], r.c.v_codes = at[1], r.c.k_scales = at[2], r.c.v_scales = at[3];
  return r;
}

// Uninitialised contiguous memory: at::empty without the dispatcher's walk (0.3 us less each).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// What the two norm-and-rotation calls share.
struct Rope {
  const at::Tensor* qkv;
  int tokens = 0, rows = 0, rot = 0, weight_dtype = MXFP4_DTYPE_BF16;
  int64_t stride = 0;
  const float *cos = nullptr, *sin = nullptr;
  const int* positions = nullptr;
  const void *q_weight = nullptr, *k_weight = nullptr;
};
// dim 0: taken from qkv's width.  args: cos, sin, positions, q_weight, k_weight.
Rope rope_of(PyObject* qkv, int heads, int kv_heads, int& dim, PyObject* const* args) {
  Rope r;
  r.qkv = tensor(qkv);
  if (!r.qkv || r.qkv->scalar_type() != at::kBFloat16 || !r.qkv->is_cuda() || r.qkv->dim() != 2 || r.qkv->stride(1) != 1)
    refuse("qkv must be bfloat16 [tokens, width] on the GPU with contiguous rows");
  const int64_t width = r.qkv->size(1), all = int64_t(heads) + 2 * int64_t(kv_heads);
  if (heads <= 0 || kv_heads <= 0) refuse("num_heads and num_kv_heads must be positive");
  if (dim == 0) dim = static_cast<int>(as_int(width / all, "qkv's width"));
  if (width != all * dim || dim == 0) refuse("qkv's width must be (num_heads + 2 * num_kv_heads) * head_dim");
  const c10::Device dev = r.qkv->device();
  r.tokens = static_cast<int>(as_int(r.qkv->size(0), "tokens"));
  r.stride = r.tokens > 1 ? r.qkv->stride(0) : width;
  if (args[0] != Py_None || args[1] != Py_None) {
    const at::Tensor *c = tensor(args[0]), *s = tensor(args[1]);
    if (!c || !s || c->scalar_type() != at::kFloat || s->scalar_type() != at::kFloat || c->device() != dev || s->device() != dev ||
        c->dim() != 2 || c->sizes() != s->sizes() || !c->is_contiguous() || !s->is_contiguous())
      refuse("cos and sin must be contiguous float32 [rows, rot / 2] of one shape on " + dev.str());
    if (c->numel() == 0) refuse("cos and sin must not be empty");
    r.rows = static_cast<int>(as_int(c->size(0), "rows of cos and sin"));
    r.rot = static_cast<int>(as_int(2 * c->size(1), "rot"));
    r.cos = static_cast<const float*>(c->data_ptr()), r.sin = static_cast<const float*>(s->data_ptr());
  }
  if (args[2] != Py_None) {
    if (!r.rot) refuse("positions without cos and sin");
    r.positions = index_vector(args[2], r.tokens, dev, "positions");
  } else if (r.rot && r.rows < r.tokens) {
    refuse("cos and sin need a row per token when no positions are given");
  }
  if (args[3] != Py_None || args[4] != Py_None) {
    const at::Tensor *q = tensor(args[3]), *k = tensor(args[4]);
    for (const at::Tensor* w : {q, k})
      if (!w || (w->scalar_type() != at::kBFloat16 && w->scalar_type() != at::kFloat) || w->scalar_type() != q->scalar_type() ||
          w->device() != dev || w->dim() != 1 || w->size(0) != dim || !w->is_contiguous())
        refuse("q_weight and k_weight come together, contiguous [head_dim], both bfloat16 or both float32, on " + dev.str());
    r.q_weight = q->data_ptr(), r.k_weight = k->data_ptr();
    if (q->scalar_type() == at::kFloat) r.weight_dtype = MXFP4_DTYPE_F32;
  }
  return r;
}

#define ENTRY(name, count)                                                                     \
  PyObject* name(PyObject*, PyObject* const* args, Py_ssize_t n) {                             \
    HANDLE_TH_ERRORS                                                                           \
    if (n != (count)) refuse(#name ": wrong number of arguments");                             \
    if (!g_entries.error_string) refuse("the library is not bound");

// qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps, interleaved
ENTRY(qk_norm_rope, 10)
  const int heads = integer(args[1], "num_heads"), kv_heads = integer(args[2], "num_kv_heads");
  int dim = 0;
  const Rope r = rope_of(args[0], heads, kv_heads, dim, args + 3);
  const double eps = real(args[8]);
  const bool inter = truth(args[9]);
  const c10::Device dev = r.qkv->device();
  const c10::DeviceGuard guard(dev);
  at::Tensor q = fresh({r.tokens, heads, dim}, at::kBFloat16, dev), k = fresh({r.tokens, kv_heads, dim}, at::kBFloat16, dev);
  check(g_entries.qk_norm_rope(r.qkv->data_ptr(), r.stride, r.tokens, heads, kv_heads, dim, r.cos, r.sin, r.rows, r.rot, inter,
                               r.positions, r.q_weight, r.k_weight, r.weight_dtype, eps, q.data_ptr(), k.data_ptr(),
                               stream_of(dev)),
        "mxfp4_qk_norm_rope");
  PyObject *pq = THPVariable_Wrap(std::move(q)), *pk = THPVariable_Wrap(std::move(k));
  PyObject* both = pq && pk ? PyTuple_Pack(2, pq, pk) : nullptr;
  Py_XDECREF(pq);
  Py_XDECREF(pk);
  return both;
  END_HANDLE_TH_ERRORS
}

// qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps, interleaved, cache, slots
ENTRY(qk_norm_rope_cache, 12)
  const int heads = integer(args[1], "num_heads"), kv_heads = integer(args[2], "num_kv_heads");
  const Cache c = cache_of(args[10]);
  if (kv_heads != c.c.num_kv_heads) refuse("num_kv_heads differs from the cache's");
  int dim = c.c.head_dim;
  const Rope r = rope_of(args[0], heads, kv_heads, dim, args + 3);
  const double eps = real(args[8]);
  const bool inter = truth(args[9]);
  if (r.qkv->device() != c.dev) refuse("qkv must be on the cache's GPU");
  const int* slots = index_vector(args[11], r.tokens, c.dev, "slots");
  const c10::DeviceGuard guard(c.dev);
  at::Tensor q = fresh({r.tokens, heads, dim}, at::kBFloat16, c.dev);
  check(g_entries.qk_norm_rope_cache(r.qkv->data_ptr(), r.stride, r.tokens, heads, r.cos, r.sin, r.rows, r.rot, inter,
                                     r.positions, r.q_weight, r.k_weight, r.weight_dtype, eps, q.data_ptr(), &c.c, slots,
                                     stream_of(c.dev)),
        "mxfp4_qk_norm_rope_cache");
  return THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

// cache, k, v, slots
ENTRY(kv_cache_write, 4)
  const Cache c = cache_of(args[0]);
  const int64_t heads = c.c.num_kv_heads, dim = c.c.head_dim;
  const at::Tensor* t[2] = {tensor(args[1]), tensor(args[2])};
  int64_t stride[2];
  for (int i = 0; i < 2; ++i) {
    if (!t[i] || t[i]->scalar_type() != at::kBFloat16 || t[i]->device() != c.dev || t[i]->dim() != 3 || t[i]->size(0) != t[0]->size(0) ||
        t[i]->size(1) != heads || t[i]->size(2) != dim || t[i]->stride(2) != 1 || (heads > 1 && t[i]->stride(1) != dim))
      refuse("k and v must be bfloat16 [tokens, num_kv_heads, head_dim] on the cache's GPU, a token's heads contiguous");
    stride[i] = t[0]->size(0) > 1 ? t[i]->stride(0) : heads * dim;
  }
  const int tokens = static_cast<int>(as_int(t[0]->size(0), "tokens"));
  const int* slots = index_vector(args[3], tokens, c.dev, "slots");
  const c10::DeviceGuard guard(c.dev);
  check(g_entries.write(&c.c, t[0]->data_ptr(), stride[0], t[1]->data_ptr(), stride[1], slots, tokens, stream_of(c.dev)),
        "mxfp4_kv_cache_write");
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// cache, slots
ENTRY(kv_cache_read, 2)
  const Cache c = cache_of(args[0]);
  const at::Tensor* s = tensor(args[1]);
  if (!s || s->dim() != 1) refuse("slots must be a vector");
  const int tokens = static_cast<int>(as_int(s->size(0), "tokens"));
  const int* slots = index_vector(args[1], tokens, c.dev, "slots");
  const c10::DeviceGuard guard(c.dev);
  at::Tensor k = fresh({tokens, c.c.num_kv_heads, c.c.head_dim}, at::kBFloat16, c.dev);
  at::Tensor v = fresh({tokens, c.c.num_kv_heads, c.c.head_dim}, at::kBFloat16, c.dev);
  check(g_entries.read(&c.c, slots, tokens, k.data_ptr(), v.data_ptr(), stream_of(c.dev)), "mxfp4_kv_cache_read");
  PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
  PyObject* both = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return both;
  END_HANDLE_TH_ERRORS
}

// q, cache, page_table, lengths, scale, return_lse, out
ENTRY(paged_attention, 7)
  const Cache c = cache_of(args[1]);
  const int64_t dim = c.c.head_dim;
  const at::Tensor *q = tensor(args[0]), *table = tensor(args[2]);
  if (!q || q->scalar_type() != at::kBFloat16 || q->device() != c.dev || q->dim() != 3 || q->size(2) != dim || q->stride(2) != 1)
    refuse("q must be bfloat16 [seqs, num_heads, head_dim] on the cache's GPU");
  const int seqs = static_cast<int>(as_int(q->size(0), "seqs")), heads = static_cast<int>(as_int(q->size(1), "num_heads"));
  if (heads == 0 || heads % c.c.num_kv_heads || (heads > 1 && q->stride(1) != dim))
    refuse("q: num_heads must be a multiple of num_kv_heads, a sequence's heads contiguous");
  if (!table || table->scalar_type() != at::kInt || table->device() != c.dev || table->dim() != 2 || table->size(0) != seqs ||
      table->size(1) == 0 || (table->size(1) > 1 && table->stride(1) != 1))
    refuse("page_table must be int32 [seqs, max_pages] on the cache's GPU with contiguous rows");
  const int pages = static_cast<int>(as_int(table->size(1), "max_pages"));
  const int* lengths = index_vector(args[3], seqs, c.dev, "lengths");
  const double scale = args[4] == Py_None ? 1.0 / std::sqrt(static_cast<double>(dim)) : real(args[4]);
  if (!std::isfinite(static_cast<float>(scale))) refuse("scale must be finite in fp32");
  const c10::DeviceGuard guard(c.dev);
  at::Tensor out, lse;
  if (args[6] == Py_None) {
    out = fresh({seqs, heads, dim}, at::kBFloat16, c.dev);
  } else {
    const at::Tensor* o = tensor(args[6]);
    if (!o || o->scalar_type() != at::kBFloat16 || o->device() != c.dev || o->sizes() != q->sizes() || !o->is_contiguous())
      refuse("out must be contiguous bfloat16 [seqs, num_heads, head_dim] on the cache's GPU");
    const int64_t row = heads * dim, stride = seqs > 1 ? q->stride(0) : row, size = seqs * row;
    const int64_t off = (static_cast<const char*>(o->data_ptr()) - static_cast<const char*>(q->data_ptr())) / 2;  // of out in q
    if (size > 0 && off < (seqs - 1) * stride + row && -off < size && !(off == 0 && stride == row)) {
      const int64_t in_row = off >= 0 && stride > row ? off % stride : 0;  // q's rows may leave room for all of out
      if (in_row < row || in_row + size > stride) refuse("out overlaps q without being q itself");
    }
    out = *o;
  }
  const bool want_lse = truth(args[5]);
  if (want_lse) lse = fresh({seqs, heads}, at::kFloat, c.dev);
  const size_t bytes = g_entries.attention_bytes(&c.c, seqs, heads, pages);
  at::Tensor workspace;
  if (bytes) workspace = fresh({static_cast<int64_t>(bytes)}, at::kByte, c.dev);
  check(g_entries.attention(q->data_ptr(), seqs > 1 ? q->stride(0) : heads * dim, &c.c, static_cast<const int*>(table->data_ptr()),
                            seqs > 1 ? table->stride(0) : pages, pages, lengths, seqs, heads, static_cast<float>(scale), out.data_ptr(),
                            want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, bytes ? workspace.data_ptr() : nullptr, bytes,
                            stream_of(c.dev)),
        "mxfp4_paged_attention");
  PyObject* po = THPVariable_Wrap(std::move(out));
  if (!want_lse) return po;
  PyObject* pl = THPVariable_Wrap(std::move(lse));
  PyObject* both = po && pl ? PyTuple_Pack(2, po, pl) : nullptr;
  Py_XDECREF(po);
  Py_XDECREF(pl);
  return both;
  END_HANDLE_TH_ERRORS
}

// Addresses of the C entries, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) refuse("bind: wrong number of arguments");
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) throw python_error();
  }
  g_entries = {reinterpret_cast<decltype(Entries::error_string)>(p[0]), reinterpret_cast<decltype(Entries::qk_norm_rope)>(p[1]),
               reinterpret_cast<decltype(Entries::qk_norm_rope_cache)>(p[2]), reinterpret_cast<decltype(Entries::write)>(p[3]),
               reinterpret_cast<decltype(Entries::read)>(p[4]), reinterpret_cast<decltype(Entries::attention_bytes)>(p[5]),
               reinterpret_cast<decltype(Entries::attention)>(p[6])};
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD(bind),           METHOD(qk_norm_rope),    METHOD(qk_norm_rope_cache), METHOD(kv_cache_write),
                           METHOD(kv_cache_read),  METHOD(paged_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_attention", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// MXFP4_BUILT_FOR: the torch and the Python compiled against; build.py looks for it in the file.
PyMODINIT_FUNC PyInit__attention() {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "built_for", MXFP4_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
