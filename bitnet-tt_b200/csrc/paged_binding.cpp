// Python entry points of the paged KV cache's calls (bitnet_tt/_paged.so).
//
// The other entry points are bound through ctypes, where such a call costs the
// host 9 to 12 us: 3 us to convert twenty arguments, the rest to look at the
// tensors from Python.  A decode step makes two of these calls per layer, whose
// kernels take 3 to 6 us, so here one function looks at the tensors, allocates
// what is missing and calls the library: one after the other, appends of 32
// tokens take 3.2 us (ctypes 9.0), decode rows over 300 keys 6.2 us (11.4).
//
// Each returns its result, None when an argument is not as it should be (the
// caller finds out which and raises), or the library's status as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/version.h>

#include <climits>

#include "../../include/bitnet_b200.h"

namespace {

struct Cache {
  bitnet_paged_kv_t kv;
  int device;
};
const char* const kName = "bitnet_tt.paged_cache";

void free_cache(PyObject* o) { delete static_cast<Cache*>(PyCapsule_GetPointer(o, kName)); }
const Cache* cache_of(PyObject* o) { return static_cast<const Cache*>(PyCapsule_GetPointer(o, kName)); }

// cache(k, v, k_scale, v_scale, num_pages, page_size, n_kv_heads, head_dim, kv_type, device): pointers as ints
PyObject* py_cache(PyObject*, PyObject* args) {
  unsigned long long p[4];
  Cache c;
  if (!PyArg_ParseTuple(args, "KKKKiiiiii", &p[0], &p[1], &p[2], &p[3], &c.kv.num_pages, &c.kv.page_size,
                        &c.kv.n_kv_heads, &c.kv.head_dim, &c.kv.kv_type, &c.device))
    return nullptr;
  c.kv.k_pages = reinterpret_cast<void*>(p[0]);
  c.kv.v_pages = reinterpret_cast<void*>(p[1]);
  c.kv.k_scale = reinterpret_cast<float*>(p[2]);
  c.kv.v_scale = reinterpret_cast<float*>(p[3]);
  return PyCapsule_New(new Cache(c), kName, free_cache);
}

bool on(const at::Tensor& t, at::ScalarType type, int device) {
  return t.scalar_type() == type && t.is_cuda() && t.get_device() == device;
}
// A contiguous int32 tensor; a vector of n entries if n >= 0.
const at::Tensor* index_arg(PyObject* o, int device, int64_t n) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return on(t, at::kInt, device) && t.is_contiguous() && (n < 0 || t.numel() == n) ? &t : nullptr;
}
// bf16 rows [tokens, features], the features contiguous.
const at::Tensor* rows_arg(PyObject* o, int device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return on(t, at::kBFloat16, device) && t.dim() == 2 && t.stride(1) == 1 && t.size(0) <= INT_MAX &&
                 (t.size(0) <= 1 || t.stride(0) <= INT_MAX)
             ? &t
             : nullptr;
}
// The stride of rows: of one row or none it may be anything.  (heads_of() has bounded the features.)
int ld_of(const at::Tensor& t) { return (int)(t.size(0) <= 1 ? t.size(1) : t.stride(0)); }
// Lets other Python threads run while this one allocates or launches: either may wait for the GPU,
// and what the GPU waits for may be a callback in Python.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, int device) {
  const Unlocked u;
  return at::empty(shape, at::TensorOptions(type).device(at::kCUDA, device));
}

// An output of this shape: the caller's (a new reference to it), or a new one.  Null with `bad` set
// when the caller's does not fit.
PyObject* out_arg(PyObject* o, at::IntArrayRef shape, int device, void** data, bool* bad) {
  if (o == Py_None) {
    at::Tensor t = fresh(shape, at::kBFloat16, device);
    *data = t.data_ptr();
    return THPVariable_Wrap(std::move(t));
  }
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (on(t, at::kBFloat16, device) && t.sizes() == shape && t.is_contiguous()) {
      *data = t.data_ptr();
      return Py_NewRef(o);
    }
  }
  *bad = true;
  return nullptr;
}

// The arguments that every call shares: a table of some sequences.
struct Table {
  const int32_t* data;
  int b, pages;
};
bool table_arg(PyObject* o, int device, Table* t) {
  const at::Tensor* x = index_arg(o, device, -1);
  if (!x || x->dim() != 2 || x->size(0) < 1 || x->size(1) < 1 || x->size(0) >= INT_MAX || x->size(1) > INT_MAX) return false;
  *t = {x->const_data_ptr<int32_t>(), (int)x->size(0), (int)x->size(1)};
  return true;
}
// Heads of `features` beside `shared` others; 0 when they do not come out.
int heads_of(int64_t features, int shared, const Cache& c) {
  if (features % c.kv.head_dim || features > INT_MAX) return 0;
  const int64_t n = features / c.kv.head_dim - shared;
  return n >= 1 && n % c.kv.n_kv_heads == 0 ? (int)n : 0;
}

// C++ exceptions as torch's own calls raise them (an allocation that fails: torch.OutOfMemoryError).
template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}
template <typename F>
PyObject* launched(PyObject* result, F call) {
  int st;
  {
    const Unlocked u;
    st = call();
  }
  if (st == BITNET_OK) return result;
  Py_DECREF(result);
  return PyLong_FromLong(st);
}

// append(cache, qkv, cu_seqlens, kv_lens, block_table, cos, sin, q_out | None, interleaved, stepwise) -> q
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "append takes 10 arguments"), nullptr;
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    if (!c) return nullptr;
    const int dev = c->device;
    Table t;
    const at::Tensor *qkv = rows_arg(a[1], dev), *cu = nullptr, *lens = nullptr;
    if (!qkv || !table_arg(a[4], dev, &t) || !(cu = index_arg(a[2], dev, t.b + 1)) || !(lens = index_arg(a[3], dev, t.b)) ||
        !THPVariable_Check(a[5]) || !THPVariable_Check(a[6]))
      Py_RETURN_NONE;
    const at::Tensor &cos = THPVariable_Unpack(a[5]), &sin = THPVariable_Unpack(a[6]);
    const at::ScalarType tab = cos.scalar_type();
    const int heads = heads_of(qkv->size(1), 2 * c->kv.n_kv_heads, *c);
    if ((tab != at::kFloat && tab != at::kBFloat16) || !on(cos, tab, dev) || !on(sin, tab, dev) || cos.dim() != 2 ||
        cos.sizes() != sin.sizes() || !cos.is_contiguous() || !sin.is_contiguous() || cos.size(0) > INT_MAX ||
        cos.size(1) > c->kv.head_dim || !heads)
      Py_RETURN_NONE;
    const int inter = PyObject_IsTrue(a[8]), step = PyObject_IsTrue(a[9]);
    if (inter < 0 || step < 0) return nullptr;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    void* q = nullptr;
    bool bad = false;
    PyObject* out = out_arg(a[7], {qkv->size(0), (int64_t)heads * c->kv.head_dim}, dev, &q, &bad);
    if (bad) Py_RETURN_NONE;
    if (!out) return nullptr;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    return launched(out, [&] {
      return bitnet_paged_append(&c->kv, t.data, t.b, t.pages, cu->const_data_ptr<int32_t>(),
                                 lens->const_data_ptr<int32_t>(), qkv->data_ptr(), ld_of(*qkv),
                                 (int)qkv->size(0), heads, cos.data_ptr(), sin.data_ptr(), (int)cos.size(0),
                                 2 * (int)cos.size(1), tab == at::kFloat, inter, step, q, stream);
    });
  });
}

// attend(cache, q, cu_seqlens, kv_lens, block_table, max_seqlen, max_kv_len, scale, out | None, workspace | None) -> out
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "attend takes 10 arguments"), nullptr;
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    if (!c) return nullptr;
    const int dev = c->device;
    Table t;
    const at::Tensor *q = rows_arg(a[1], dev), *cu = nullptr, *lens = nullptr;
    if (!q || !table_arg(a[4], dev, &t) || !(cu = index_arg(a[2], dev, t.b + 1)) || !(lens = index_arg(a[3], dev, t.b)))
      Py_RETURN_NONE;
    const long long max_q = PyLong_AsLongLong(a[5]), max_kv = PyLong_AsLongLong(a[6]);
    const double scale = PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) return nullptr;
    const int heads = heads_of(q->size(1), 0, *c);
    if (max_q < INT_MIN || max_q > INT_MAX || max_kv < INT_MIN || max_kv > INT_MAX || !heads) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const int tokens = (int)q->size(0);
    at::Tensor own;
    void* ws = nullptr;
    size_t bytes = 0;
    if (a[9] == Py_None) {
      bytes = bitnet_paged_attention_workspace_bytes(t.b, tokens, (int)max_q, (int)max_kv, heads, c->kv.n_kv_heads,
                                                     c->kv.head_dim);
      if (bytes) {
        own = fresh({(int64_t)bytes}, at::kByte, dev);
        ws = own.data_ptr();
      }
    } else {
      if (!THPVariable_Check(a[9])) Py_RETURN_NONE;
      const at::Tensor& w = THPVariable_Unpack(a[9]);
      if (!w.is_cuda() || w.get_device() != dev || !w.is_contiguous()) Py_RETURN_NONE;
      ws = w.data_ptr();
      bytes = w.nbytes();
    }
    void* o = nullptr;
    bool bad = false;
    PyObject* out = out_arg(a[8], q->sizes(), dev, &o, &bad);
    if (bad) Py_RETURN_NONE;
    if (!out) return nullptr;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    return launched(out, [&] {
      return bitnet_paged_attention(&c->kv, t.data, t.b, t.pages, cu->const_data_ptr<int32_t>(),
                                    lens->const_data_ptr<int32_t>(), q->data_ptr(), ld_of(*q), tokens,
                                    (int)max_q, (int)max_kv, heads, (float)scale, ws, bytes, o, stream);
    });
  });
}

// read(cache, block_table, starts | None, cu_rows, total_rows, k_out | None, v_out | None) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "read takes 7 arguments"), nullptr;
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    if (!c) return nullptr;
    const int dev = c->device;
    Table t;
    const at::Tensor *starts = nullptr, *cu = nullptr;
    if (!table_arg(a[1], dev, &t) || !(cu = index_arg(a[3], dev, t.b + 1)) ||
        (a[2] != Py_None && !(starts = index_arg(a[2], dev, t.b))))
      Py_RETURN_NONE;
    const long long rows = PyLong_AsLongLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    if (rows < 0 || rows > INT_MAX) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    void *k = nullptr, *v = nullptr;
    bool bad = false;
    const int64_t shape[3] = {rows, c->kv.n_kv_heads, c->kv.head_dim};
    const THPObjectPtr ko(out_arg(a[5], shape, dev, &k, &bad));  // let go where the next allocation throws
    if (bad) Py_RETURN_NONE;
    if (!ko) return nullptr;
    const THPObjectPtr vo(out_arg(a[6], shape, dev, &v, &bad));
    if (bad) Py_RETURN_NONE;
    if (!vo) return nullptr;
    PyObject* pair = PyTuple_Pack(2, ko.get(), vo.get());
    if (!pair) return nullptr;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    return launched(pair, [&] {
      return bitnet_paged_read(&c->kv, t.data, t.b, t.pages, starts ? starts->const_data_ptr<int32_t>() : nullptr,
                               cu->const_data_ptr<int32_t>(), (int)rows, k, v, stream);
    });
  });
}

PyMethodDef methods[] = {
    {"cache", py_cache, METH_VARARGS, "cache(k, v, k_scale, v_scale, num_pages, page_size, n_kv_heads, head_dim, kv_type, device)"},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_append)), METH_FASTCALL, "bitnet_paged_append"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_attend)), METH_FASTCALL, "bitnet_paged_attention"},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(py_read)), METH_FASTCALL, "bitnet_paged_read"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
