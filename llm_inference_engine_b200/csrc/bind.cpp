// The short way from Python to the C ABI for ordinary calls of the 8-bit operators: the checks, the allocations and the launch
// of fp8.linear, cache8.rope_append and cache8.attention on torch tensors, in one step of 3 us where the same in
// Python takes 10 to 15 (a small call on the GPU is shorter than that). A call that is not plain (a tensor that has to be
// copied first, another device than the current one, an argument that will be refused, a first call that has to make
// something) gets None back before anything has happened, and the Python code takes it from the start. The entry points
// are those of libmuse_proj.so, handed in as addresses by the ctypes binding that loaded it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <math.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/muse_proj.h"

namespace {

struct Entries {
  decltype(&muse_fp8_walk) walk;
  decltype(&muse_fp8_quantize) quantize;
  decltype(&muse_fp8_gemm) gemm;
  decltype(&muse_fp8_gemm_ws_bytes) gemm_ws;
  decltype(&muse_rope_append) rope;
  decltype(&muse_cache_attention) attention;
  decltype(&muse_cache_attention_ws_bytes) attention_ws;
} entry;
bool loaded = false;
constexpr int MAX_DEVICES = 64;
int* status_of[MAX_DEVICES];

// Argument i as a tensor of this type and number of dimensions on device `index` (-1: any CUDA device); null if it is not.
const at::Tensor* tensor(PyObject* o, at::ScalarType type, int dims, int index) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.scalar_type() != type || t.dim() != dims || (index >= 0 && t.get_device() != index)) return nullptr;
  return &t;
}
uintptr_t addr(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }
bool whole(PyObject* o, long long* v) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0 && *v >= INT32_MIN && *v <= INT32_MAX;
}
// The device is current.
bool here(int index) { return loaded && index >= 0 && index < MAX_DEVICES && c10::cuda::current_device() == index; }
// And its status word exists.
bool ready(int index) { return here(index) && status_of[index]; }
void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }
PyObject* wrap(at::Tensor&& t) { return THPVariable_Wrap(std::move(t)); }

// Rows of [m, cols] values at 16-byte vectors' alignment.
bool vector_rows(const at::Tensor& t, int64_t m, int64_t cols) {
  return t.stride(1) == 1 && addr(t) % 16 == 0 && (m <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= cols));
}

PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n_args) {   // x, w8, w_exp
  if (n_args != 3) Py_RETURN_NONE;
  const at::Tensor* w = tensor(args[1], at::kFloat8_e4m3fn, 2, -1);
  if (!w || !here(w->get_device())) Py_RETURN_NONE;
  const int index = w->get_device();
  const at::Tensor *x = tensor(args[0], at::kBFloat16, 2, index), *e = tensor(args[2], at::kByte, 2, index);
  if (!x || !e) Py_RETURN_NONE;
  const int64_t m = x->size(0), k = x->size(1), n = w->size(0), kb = (k + 127) / 128;
  if (m < 1 || n < 1 || k < 16 || k % 16 || w->size(1) != k || e->size(0) != (n + 127) / 128 || e->size(1) != kb || !w->is_contiguous() ||
      !e->is_contiguous() || addr(*w) % 16 || !vector_rows(*x, m, k) || m > INT32_MAX || n > INT32_MAX || k > INT32_MAX)
    Py_RETURN_NONE;
  const int64_t ld = m > 1 ? x->stride(0) : k;
  if (ld > INT32_MAX) Py_RETURN_NONE;
  const bool walk = m <= MUSE_FP8_WALK_TOKENS && k <= MUSE_FP8_WALK_K && n * k <= MUSE_FP8_WALK_BYTES;
  if (!walk && !status_of[index]) Py_RETURN_NONE;
  void* stream = stream_of(index);
  at::Tensor out = at::empty({m, n}, x->options());
  int rc;
  if (walk) {
    rc = entry.walk(w->data_ptr(), e->data_ptr(), x->data_ptr(), out.data_ptr(), m, n, k, ld, n, stream);
  } else {
    at::Tensor xq = at::empty({m, k}, w->options()), xe = at::empty({m, kb}, e->options()), ws;
    const long long bytes = entry.gemm_ws(m, n, k);
    if (bytes < 0) Py_RETURN_NONE;
    if (bytes > 0) ws = at::empty({bytes}, e->options());
    rc = entry.quantize(x->data_ptr(), xq.data_ptr(), xe.data_ptr(), m, k, ld, stream);
    if (rc == 0)
      rc = entry.gemm(w->data_ptr(), e->data_ptr(), xq.data_ptr(), xe.data_ptr(), out.data_ptr(), bytes > 0 ? ws.data_ptr() : nullptr, status_of[index], m, n,
                      k, n, stream);
  }
  if (rc != 0) Py_RETURN_NONE;   // the Python code meets it again and says what it is
  return wrap(std::move(out));
}

struct Batch {
  const at::Tensor *k, *v, *ke, *ve, *table, *lens, *cu;
  int index, pages, heads, dim, batch, width;
};
// cache (a tuple of four), page_table, seq_lens, cu_q or None: the checks that rope_append and attention share.
bool batch_of(PyObject* cache, PyObject* table, PyObject* lens, PyObject* cu, long long m, long long max_q, long long q_heads, Batch* b) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 4) return false;
  b->k = tensor(PyTuple_GET_ITEM(cache, 0), at::kFloat8_e4m3fn, 4, -1);
  if (!b->k) return false;
  b->index = b->k->get_device();
  if (!ready(b->index)) return false;
  b->v = tensor(PyTuple_GET_ITEM(cache, 1), at::kFloat8_e4m3fn, 4, b->index);
  b->ke = tensor(PyTuple_GET_ITEM(cache, 2), at::kByte, 2, b->index);
  b->ve = tensor(PyTuple_GET_ITEM(cache, 3), at::kByte, 2, b->index);
  b->table = tensor(table, at::kInt, 2, b->index);
  b->lens = tensor(lens, at::kInt, 1, b->index);
  b->cu = cu == Py_None ? nullptr : tensor(cu, at::kInt, 1, b->index);
  if (!b->v || !b->ke || !b->ve || !b->table || !b->lens || (cu != Py_None && !b->cu)) return false;
  const int64_t pages = b->k->size(0), heads = b->k->size(1), dim = b->k->size(3), batch = b->table->size(0), width = b->table->size(1);
  if (b->k->size(2) != MUSE_PAGE_TOKENS || (dim != 64 && dim != 128) || pages < 1 || heads < 1 || pages > INT32_MAX || batch < 1 || width < 1 ||
      batch > INT32_MAX || width > INT32_MAX)
    return false;
  if (b->v->size(0) != pages || b->v->size(1) != heads || b->v->size(2) != dim || b->v->size(3) != MUSE_PAGE_TOKENS || b->ke->size(0) != pages ||
      b->ke->size(1) != heads || b->ve->size(0) != pages || b->ve->size(1) != heads || b->lens->size(0) != batch)
    return false;
  for (const at::Tensor* t : {b->k, b->v, b->ke, b->ve, b->table, b->lens})
    if (!t->is_contiguous()) return false;
  if ((addr(*b->k) | addr(*b->v)) % 16) return false;
  if (b->cu ? !b->cu->is_contiguous() || b->cu->size(0) != batch + 1 : m != batch || max_q != 1) return false;
  if (max_q < 1 || q_heads < heads || q_heads % heads) return false;
  b->pages = static_cast<int>(pages);
  b->heads = static_cast<int>(heads);
  b->dim = static_cast<int>(dim);
  b->batch = static_cast<int>(batch);
  b->width = static_cast<int>(width);
  return true;
}
const void* cu_ptr(const Batch& b) { return b.cu ? b.cu->data_ptr() : nullptr; }

// qkv, cache, cos_sin, page_table, seq_lens, cu_q, q_heads, max_q, interleaved, values
PyObject* rope_append(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  long long q_heads, max_q;
  if (n_args != 10 || !whole(args[6], &q_heads) || !whole(args[7], &max_q)) Py_RETURN_NONE;
  const at::Tensor* x = tensor(args[0], at::kBFloat16, 2, -1);
  Batch b;
  if (!x || x->size(0) < 1 || x->size(0) > INT32_MAX) Py_RETURN_NONE;
  const int64_t m = x->size(0);
  if (!batch_of(args[1], args[3], args[4], args[5], m, max_q, q_heads, &b) || x->get_device() != b.index) Py_RETURN_NONE;
  const at::Tensor* cs = tensor(args[2], at::kFloat, 3, b.index);
  const int64_t cols = (q_heads + 2 * b.heads) * b.dim;
  if (!cs || !cs->is_contiguous() || addr(*cs) % 16 || cs->size(2) != 2 || cs->size(1) % 8 || cs->size(1) < 8 || 2 * cs->size(1) > b.dim ||
      cs->size(0) < static_cast<int64_t>(b.width) * MUSE_PAGE_TOKENS || cs->size(0) > INT32_MAX || x->size(1) < cols || !vector_rows(*x, m, x->size(1)))
    Py_RETURN_NONE;
  const int turns = PyObject_IsTrue(args[8]), values = PyObject_IsTrue(args[9]);
  if (turns < 0 || values < 0) return nullptr;
  at::Tensor q = at::empty({m, q_heads, b.dim}, x->options()), kv, vv;
  if (values) {
    kv = at::empty({m, b.heads, b.dim}, x->options());
    vv = at::empty({m, b.heads, b.dim}, x->options());
  }
  const int rc = entry.rope(x->data_ptr(), cs->data_ptr(), b.table->data_ptr(), b.lens->data_ptr(), cu_ptr(b), b.k->data_ptr(), b.v->data_ptr(),
                            b.ke->data_ptr(), b.ve->data_ptr(), q.data_ptr(), values ? kv.data_ptr() : nullptr, values ? vv.data_ptr() : nullptr,
                            status_of[b.index], m > 1 ? x->stride(0) : cols, m, b.batch, b.width, b.pages, max_q, q_heads, b.heads, b.dim,
                            2 * cs->size(1), turns, cs->size(0), stream_of(b.index));
  if (rc != 0) Py_RETURN_NONE;
  if (!values) return wrap(std::move(q));
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  at::Tensor* t[3] = {&q, &kv, &vv};
  for (int i = 0; i < 3; ++i) {
    PyObject* o = wrap(std::move(*t[i]));
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
}

// q, cache, page_table, seq_lens, cu_q, max_q, scale or None, window, gate or None
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  long long max_q, window;
  if (n_args != 9 || !whole(args[5], &max_q) || !whole(args[7], &window) || window < 0) Py_RETURN_NONE;
  const at::Tensor* q = tensor(args[0], at::kBFloat16, 3, -1);
  if (!q || q->size(0) < 1 || q->size(0) > INT32_MAX || q->size(1) > INT32_MAX) Py_RETURN_NONE;
  const int64_t m = q->size(0), q_heads = q->size(1);
  Batch b;
  if (!batch_of(args[1], args[2], args[3], args[4], m, max_q, q_heads, &b) || q->get_device() != b.index || q->size(2) != b.dim) Py_RETURN_NONE;
  if (max_q > m) max_q = m;   // no sequence has more new tokens than the batch has rows
  const int64_t cols = q_heads * b.dim;
  if (q->stride(2) != 1 || q->stride(1) != b.dim || addr(*q) % 16 || (m > 1 && (q->stride(0) % 8 || q->stride(0) < cols))) Py_RETURN_NONE;
  double scale = b.dim == 128 ? 0.08838834764831845 : 0.125;
  if (args[6] != Py_None) {
    scale = PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    if (!(scale > 0.0) || std::isinf(scale)) Py_RETURN_NONE;
  }
  const at::Tensor* gate = nullptr;
  if (args[8] != Py_None) {
    gate = tensor(args[8], at::kBFloat16, 2, b.index);
    if (!gate || gate->size(0) != m || gate->size(1) != cols || gate->stride(1) != 1 || (m > 1 && gate->stride(0) < cols)) Py_RETURN_NONE;
  }
  const long long bytes = entry.attention_ws(b.batch, max_q, q_heads, b.heads, b.dim);
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor out = at::empty({m, cols}, q->options()), ws = at::empty({bytes}, b.ke->options());
  const int rc = entry.attention(q->data_ptr(), b.k->data_ptr(), b.v->data_ptr(), b.ke->data_ptr(), b.ve->data_ptr(), b.table->data_ptr(),
                                 b.lens->data_ptr(), cu_ptr(b), gate ? gate->data_ptr() : nullptr, out.data_ptr(), ws.data_ptr(), status_of[b.index],
                                 m > 1 ? q->stride(0) : cols, gate && m > 1 ? gate->stride(0) : cols, cols, static_cast<float>(scale), m, b.batch,
                                 b.width, b.pages, max_q, q_heads, b.heads, b.dim, window, stream_of(b.index));
  if (rc != 0) Py_RETURN_NONE;
  return wrap(std::move(out));
}

// Addresses of the entry points, in the order of Entries.
PyObject* set_entries(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  void* p[7];
  if (n_args != 7) {
    PyErr_SetString(PyExc_TypeError, "seven addresses are wanted");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is null");
      return nullptr;
    }
  }
  entry = {reinterpret_cast<decltype(entry.walk)>(p[0]), reinterpret_cast<decltype(entry.quantize)>(p[1]), reinterpret_cast<decltype(entry.gemm)>(p[2]),
           reinterpret_cast<decltype(entry.gemm_ws)>(p[3]), reinterpret_cast<decltype(entry.rope)>(p[4]), reinterpret_cast<decltype(entry.attention)>(p[5]),
           reinterpret_cast<decltype(entry.attention_ws)>(p[6])};
  loaded = true;
  Py_RETURN_NONE;
}

// Device index, address of its status word (0: there is none).
PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  long long index;
  if (n_args != 2 || !whole(args[0], &index) || index < 0 || index >= MAX_DEVICES) {
    PyErr_SetString(PyExc_ValueError, "a device index and an address are wanted");
    return nullptr;
  }
  status_of[index] = static_cast<int*>(PyLong_AsVoidPtr(args[1]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// at::empty can throw (out of memory): a C++ exception must not leave through the interpreter.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const std::exception&) {
    Py_RETURN_NONE;   // the Python code meets the same condition and raises torch's own error
  }
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F>)), METH_FASTCALL, nullptr};
}

}  // namespace

PyMODINIT_FUNC PyInit__bind() {
  static PyMethodDef methods[] = {method<linear>("linear"),           method<rope_append>("rope_append"), method<attention>("attention"),
                                  method<set_entries>("set_entries"), method<set_status>("set_status"),   {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef def = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods};
  return PyModule_Create(&def);
}
