// Python's way into the paged-cache serving operators (ops.rotary, paged_kv_append,
// paged_tree_attention, sample): checks torch tensors and calls the C ABI.
//
// These calls are short on the GPU (3 us for a decode step's rotation), so what stands
// before a launch counts: checking and passing twenty arguments through ctypes took
// 13 us a call, this module 5. It holds no arithmetic; libbm_layer_ops.so beside it does.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <exception>

#include "bm_layer_ops.h"

namespace {

PyObject* g_error = nullptr;  // BMError

// Raises BMError(status, message).
PyObject* raise(int status, const char* message) {
  PyObject* e = PyObject_CallFunction(g_error, "is", status, message);
  if (e != nullptr) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  return nullptr;
}
struct Refused : std::exception {};

[[noreturn]] void invalid(const char* format, ...) {
  char message[256];
  va_list ap;
  va_start(ap, format);
  vsnprintf(message, sizeof(message), format, ap);
  va_end(ap);
  raise(BM_ERR_INVALID_ARGUMENT, message);
  throw Refused();
}

void check(int status) {
  if (status == BM_OK) return;
  raise(status, bm_last_error_message());
  throw Refused();
}

// A tensor argument, or NULL for None.
const at::Tensor* tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) invalid("%s must be a tensor", name);
  return &THPVariable_Unpack(o);
}
const at::Tensor& required(PyObject* o, const char* name) {
  const at::Tensor* t = tensor(o, name);
  if (t == nullptr) invalid("%s must be a tensor", name);
  return *t;
}

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    invalid("%s must be an integer", name);
  }
  return v;
}
int32_t integer32(PyObject* o, const char* name) {
  const int64_t v = integer(o, name);
  if (v < INT32_MIN || v > INT32_MAX) invalid("%s outside 32 bits", name);
  return static_cast<int32_t>(v);
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v != 0;
}

c10::Device cuda_device(const at::Tensor& t) {
  if (!t.is_cuda()) invalid("tensor is not on a CUDA device");
  return t.device();
}

bm_dtype_t dtype_of(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return BM_F32;
  if (t.scalar_type() == at::kBFloat16) return BM_BF16;
  invalid("unsupported dtype (float32 or bfloat16)");
}

void* data(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// [rows, heads, hd] with dense heads; rows may be slices of wider ones.
struct HeadRows {
  int64_t rows = 0, heads = 0, stride = 0;
};
HeadRows head_rows(const at::Tensor& t, const char* name, const at::Tensor& like, int64_t hd) {
  if (t.dim() != 3 || t.size(2) != hd || t.scalar_type() != like.scalar_type() || t.device() != like.device()) {
    invalid("%s must be [rows, heads, head_dim] of the other tensors' device, dtype and head_dim", name);
  }
  HeadRows r{t.size(0), t.size(1), 0};
  if (t.is_contiguous()) {
    r.stride = r.heads * hd;
    return r;
  }
  if ((hd > 1 && t.stride(2) != 1) || (r.heads > 1 && t.stride(1) != hd)) invalid("%s must have dense heads", name);
  r.stride = r.rows > 1 ? t.stride(0) : r.heads * hd;
  return r;
}

void i32(const at::Tensor* t, const char* name, c10::Device device, int64_t numel) {
  if (t == nullptr) return;
  if (t->scalar_type() != at::kInt || !t->is_contiguous() || t->device() != device) {
    invalid("%s must be a contiguous int32 tensor on %s", name, device.str().c_str());
  }
  if (t->numel() != numel) invalid("%s must have %lld entries", name, static_cast<long long>(numel));
}

// A rope table's entries: max_pos rows of rotary_dim / 2 fp32 pairs.
void rope_table(const at::Tensor& t, c10::Device device, int64_t max_pos, int64_t rotary_dim) {
  if (t.device() != device) invalid("the rope table is on another device");
  if (t.scalar_type() != at::kFloat || !t.is_contiguous() || max_pos < 0 || rotary_dim < 0 || t.numel() < max_pos * (rotary_dim / 2) * 2) {
    invalid("the rope table must be contiguous float32 [max_pos, rotary_dim / 2, 2]");
  }
}

int32_t* status_word(PyObject* o, c10::Device device) {
  const at::Tensor* t = tensor(o, "status");
  if (t == nullptr) return nullptr;
  if (t->device() != device) invalid("the status word is on another device");
  return t->data_ptr<int32_t>();
}

// The stream's handle: an integer, or None for the device's current stream.
void* stream_of(PyObject* o, c10::Device device) {
  if (o == Py_None) return c10::cuda::getCurrentCUDAStream(device.index()).stream();
  return reinterpret_cast<void*>(static_cast<uintptr_t>(integer(o, "stream")));
}

// An output argument: the tensor given, or a new one like `shape_of`.
PyObject* output(PyObject* given, const at::Tensor& shape_of) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(at::empty(shape_of.sizes(), shape_of.options()));
}

struct Owned {
  PyObject* p = nullptr;
  ~Owned() { Py_XDECREF(p); }
  PyObject* release() {
    PyObject* r = p;
    p = nullptr;
    return r;
  }
};

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd expected", n, want);
  return false;
}

// q, k, positions, pos0, table, max_pos, rotary_dim, interleaved, q_out, k_out, status, stream
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 12)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q = tensor(a[0], "q"), *k = tensor(a[1], "k"), *pos = tensor(a[2], "positions");
    const at::Tensor* ref = q != nullptr ? q : k;
    if (ref == nullptr) invalid("neither q nor k given");
    if (ref->dim() != 3) invalid("q and k must be [rows, heads, head_dim]");
    if (q == nullptr && a[8] != Py_None) invalid("q_out without q");
    if (k == nullptr && a[9] != Py_None) invalid("k_out without k");
    const c10::Device device = cuda_device(*ref);
    const bm_dtype_t dtype = dtype_of(*ref);
    const at::Tensor& table = required(a[4], "table");
    const int64_t hd = ref->size(2);
    HeadRows qr, kr, qor, kor;
    Owned q_out, k_out;
    if (q != nullptr) {
      qr = head_rows(*q, "q", *ref, hd);
      q_out.p = output(a[8], *q);
      qor = head_rows(required(q_out.p, "q_out"), "q_out", *ref, hd);
      if (qor.rows != qr.rows || qor.heads != qr.heads) invalid("q_out must have q's shape");
    }
    if (k != nullptr) {
      kr = head_rows(*k, "k", *ref, hd);
      k_out.p = output(a[9], *k);
      kor = head_rows(required(k_out.p, "k_out"), "k_out", *ref, hd);
      if (kor.rows != kr.rows || kor.heads != kr.heads) invalid("k_out must have k's shape");
      if (q != nullptr && kr.rows != qr.rows) invalid("q and k must have the same rows");
    }
    const int64_t rows = q != nullptr ? qr.rows : kr.rows;
    i32(pos, "positions", device, rows);
    const int32_t max_pos = integer32(a[5], "max_pos"), rotary_dim = integer32(a[6], "rotary_dim");
    rope_table(table, device, max_pos, rotary_dim);
    const c10::cuda::CUDAGuard guard(device);
    check(bm_rotary(q ? THPVariable_Unpack(q_out.p).data_ptr() : nullptr, k ? THPVariable_Unpack(k_out.p).data_ptr() : nullptr,
                    data(q), data(k), static_cast<const int32_t*>(data(pos)), integer32(a[3], "positions"),
                    table.data_ptr(), max_pos, rotary_dim, truth(a[7]), rows,
                    static_cast<int32_t>(qr.heads), static_cast<int32_t>(kr.heads), static_cast<int32_t>(hd), qr.stride,
                    kr.stride, qor.stride, kor.stride, dtype, status_word(a[10], device), stream_of(a[11], device)));
    if (q_out.p == nullptr) {
      Py_INCREF(Py_None);
      q_out.p = Py_None;
    }
    if (k_out.p == nullptr) {
      Py_INCREF(Py_None);
      k_out.p = Py_None;
    }
    return PyTuple_Pack(2, q_out.p, k_out.p);
  });
}

// The cache as its tensors are now: k_pages, v_pages, page_table.
struct Cache {
  const at::Tensor& k;
  bm_paged_kv_t c;
};
int32_t size32(const at::Tensor& t, int64_t dim, const char* name) {
  if (t.size(dim) > INT32_MAX) invalid("%s has more than 2^31 - 1 entries in a dimension", name);
  return static_cast<int32_t>(t.size(dim));
}
Cache cache_of(PyObject* k_pages, PyObject* v_pages, PyObject* page_table) {
  const at::Tensor &k = required(k_pages, "k_pages"), &v = required(v_pages, "v_pages"), &t = required(page_table, "page_table");
  if (k.dim() != 4 || v.sizes() != k.sizes() || !k.is_contiguous() || !v.is_contiguous() || v.scalar_type() != k.scalar_type() ||
      v.device() != k.device()) {
    invalid("k_pages and v_pages must be contiguous [num_pages, kv_heads, page_size, head_dim] of one dtype and device");
  }
  if (t.dim() != 2 || t.scalar_type() != at::kInt || !t.is_contiguous() || t.device() != k.device()) {
    invalid("page_table must be a contiguous int32 tensor [num_seqs, max_pages] on the pages' device");
  }
  return Cache{k, {k.data_ptr(), v.data_ptr(), static_cast<const int32_t*>(t.data_ptr()), size32(k, 0, "k_pages"),
                   size32(k, 2, "k_pages"), size32(t, 1, "page_table"), size32(t, 0, "page_table"), size32(k, 1, "k_pages"),
                   size32(k, 3, "k_pages")}};
}

// q, k, v, positions, slots, seq_ids, k_pages, v_pages, page_table, table, max_pos, rotary_dim,
// interleaved, q_out, status, stream
PyObject* paged_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 16)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* q = tensor(a[0], "q");
    const at::Tensor &k = required(a[1], "k"), &v = required(a[2], "v");
    const at::Tensor *pos = tensor(a[3], "positions"), *slots = tensor(a[4], "slots"), *seqs = tensor(a[5], "seq_ids");
    const at::Tensor* table = tensor(a[9], "table");
    const Cache cache = cache_of(a[6], a[7], a[8]);
    if (k.dim() != 3) invalid("k and v must be [rows, kv_heads, head_dim]");
    if (q == nullptr && a[13] != Py_None) invalid("q_out without q");
    const c10::Device device = cuda_device(k);
    const bm_dtype_t dtype = dtype_of(k);
    if (cache.k.scalar_type() != k.scalar_type() || cache.k.device() != device) invalid("the cache has another dtype or device");
    const int64_t hd = cache.c.head_dim;
    const HeadRows kr = head_rows(k, "k", k, hd), vr = head_rows(v, "v", k, hd);
    if (kr.heads != cache.c.num_kv_heads || vr.heads != kr.heads || vr.rows != kr.rows) {
      invalid("k and v do not match the cache or each other");
    }
    HeadRows qr, qor;
    Owned q_out;
    if (q != nullptr) {
      qr = head_rows(*q, "q", k, hd);
      q_out.p = output(a[13], *q);
      qor = head_rows(required(q_out.p, "q_out"), "q_out", k, hd);
      if (qr.rows != kr.rows || qor.rows != qr.rows || qor.heads != qr.heads) invalid("q must have k's rows, and q_out q's shape");
    }
    i32(pos, "positions", device, kr.rows);
    i32(slots, "slots", device, kr.rows);
    i32(seqs, "seq_ids", device, kr.rows);
    const int32_t max_pos = integer32(a[10], "max_pos"), rotary_dim = integer32(a[11], "rotary_dim");
    if (table != nullptr) rope_table(*table, device, max_pos, rotary_dim);
    const c10::cuda::CUDAGuard guard(device);
    check(bm_paged_kv_append(q ? THPVariable_Unpack(q_out.p).data_ptr() : nullptr, data(q), k.data_ptr(), v.data_ptr(),
                             static_cast<const int32_t*>(data(pos)), static_cast<const int32_t*>(data(slots)),
                             static_cast<const int32_t*>(data(seqs)), &cache.c, data(table), max_pos,
                             rotary_dim, truth(a[12]), kr.rows, static_cast<int32_t>(qr.heads),
                             qr.stride, kr.stride, vr.stride, qor.stride, dtype, status_word(a[14], device),
                             stream_of(a[15], device)));
    if (q_out.p == nullptr) Py_RETURN_NONE;
    return q_out.release();
  });
}

// q, k_pages, v_pages, page_table, ctx_lens, q_starts, max_ctx, max_tree, tree_mask, seq_ids, scale,
// out, workspace, status, stream
PyObject* paged_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 15)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& q = required(a[0], "q");
    const at::Tensor &ctx = required(a[4], "ctx_lens"), &starts = required(a[5], "q_starts"), &ws = required(a[12], "workspace");
    const at::Tensor *mask = tensor(a[8], "tree_mask"), *seqs = tensor(a[9], "seq_ids");
    const Cache cache = cache_of(a[1], a[2], a[3]);
    const c10::Device device = cuda_device(q);
    if (q.dim() != 3 || !q.is_contiguous() || q.size(2) != cache.c.head_dim) {
      invalid("q must be contiguous [rows, heads, head_dim] with the cache's head_dim");
    }
    const bm_dtype_t dtype = dtype_of(q);
    if (cache.k.scalar_type() != q.scalar_type() || cache.k.device() != device) invalid("the cache has another dtype or device");
    const int64_t batch = ctx.numel();
    i32(&ctx, "ctx_lens", device, batch);
    i32(&starts, "q_starts", device, batch + 1);
    i32(seqs, "seq_ids", device, batch);
    int64_t words = 0;
    if (mask != nullptr) {
      if (mask->scalar_type() != at::kLong || mask->dim() != 2 || mask->size(0) != q.size(0) || !mask->is_contiguous() ||
          mask->device() != device) {
        invalid("tree_mask must be contiguous int64 [rows, words] on q's device");
      }
      words = mask->size(1);
    }
    Owned out;
    out.p = output(a[11], q);
    const at::Tensor& o = required(out.p, "out");
    if (o.sizes() != q.sizes() || o.scalar_type() != q.scalar_type() || o.device() != device || !o.is_contiguous()) {
      invalid("out must be contiguous and like q");
    }
    if (ws.device() != device || !ws.is_contiguous()) invalid("workspace must be contiguous on q's device");
    const double scale = PyFloat_AsDouble(a[10]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused();
    const c10::cuda::CUDAGuard guard(device);
    check(bm_paged_tree_attention(o.data_ptr(), q.data_ptr(), &cache.c, static_cast<const int32_t*>(data(seqs)),
                                  ctx.data_ptr<int32_t>(), starts.data_ptr<int32_t>(), static_cast<const uint64_t*>(data(mask)),
                                  static_cast<int32_t>(words), q.size(0), batch, static_cast<int32_t>(q.size(1)),
                                  integer32(a[6], "max_ctx"), integer32(a[7], "max_tree"), static_cast<float>(scale),
                                  ws.data_ptr(), static_cast<size_t>(ws.numel()) * ws.element_size(), dtype,
                                  status_word(a[13], device), stream_of(a[14], device)));
    return out.release();
  });
}

// logits, uniforms, temperature, top_k, top_p, min_p, out, status, stream
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& x = required(a[0], "logits");
    const c10::Device device = cuda_device(x);
    if (x.dim() != 2 || x.size(1) == 0 || (x.size(1) > 1 && x.stride(1) != 1)) {
      invalid("logits must be [rows, vocab] with unit inner stride");
    }
    const bm_dtype_t dtype = dtype_of(x);
    const int64_t rows = x.size(0), vocab = x.size(1);
    static const char* names[] = {"uniforms", "temperature", "top_k", "top_p", "min_p"};
    const at::Tensor* s[5];
    for (int i = 0; i < 5; ++i) {
      s[i] = i == 0 ? &required(a[1], names[0]) : tensor(a[1 + i], names[i]);
      const at::ScalarType want = i == 2 ? at::kInt : at::kFloat;
      if (s[i] != nullptr && (s[i]->scalar_type() != want || s[i]->numel() != rows || !s[i]->is_contiguous() || s[i]->device() != device)) {
        invalid("%s must be a contiguous %s tensor of one entry per row on the logits' device", names[i], i == 2 ? "int32" : "float32");
      }
    }
    Owned out;
    if (a[6] != Py_None) {
      const at::Tensor& given = required(a[6], "out");
      i32(&given, "out", device, rows);
      out.p = a[6];
      Py_INCREF(out.p);
    } else {
      out.p = THPVariable_Wrap(at::empty({rows}, x.options().dtype(at::kInt)));
    }
    const c10::cuda::CUDAGuard guard(device);
    check(bm_sample(static_cast<int32_t*>(THPVariable_Unpack(out.p).data_ptr()), x.data_ptr(), static_cast<const float*>(data(s[0])),
                    static_cast<const float*>(data(s[1])), static_cast<const int32_t*>(data(s[2])),
                    static_cast<const float*>(data(s[3])), static_cast<const float*>(data(s[4])), rows, vocab,
                    rows > 1 ? x.stride(0) : vocab, dtype, status_word(a[7], device), stream_of(a[8], device)));
    return out.release();
  });
}

PyMethodDef g_methods[] = {
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"paged_kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_kv_append)), METH_FASTCALL, nullptr},
    {"paged_tree_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_tree_attention)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving_ops() {
  PyObject* lib = PyImport_ImportModule("baremetalinferenceengine_b200._lib");
  if (lib == nullptr) return nullptr;
  g_error = PyObject_GetAttrString(lib, "BMError");
  Py_DECREF(lib);
  if (g_error == nullptr) return nullptr;
  return PyModule_Create(&g_module);
}
