// Native calls of the 8-bit decoder-step operators on torch tensors (Python module _b2torch): the
// tensors' addresses, types and shapes are read in C++ and handed to the C ABI of
// include/onnxl_b200.h.  A single-token step is a chain of kernels of a few microseconds, so the
// host's time per call sets its pace: building the descriptors in Python takes 25 to 40 us a call.
//
// Each function allocates the outputs it is not given, on the current stream of the inputs' device.
// The C ABI's functions come as addresses from the library the package has loaded (connect), with the
// Python function that raises their errors.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <utility>

#include "../../include/onnxl_b200.h"

namespace {

PyObject *g_check = nullptr; // callable: raises for a status
decltype(&b2_rms_normalization_quantize) f_norm = nullptr;
decltype(&b2_scaled_matmul) f_product = nullptr;
decltype(&b2_kv_cache_append) f_append = nullptr;
decltype(&b2_cache_attention) f_attention = nullptr;
PyObject *s_data, *s_dtype, *s_shape, *s_k, *s_v, *s_k_scale, *s_v_scale, *s_table, *s_lengths;

constexpr int32_t kInt8 = 3, kF8E4M3FN = 17; // ONNX TensorProto.DataType codes

int32_t onnx_type(at::ScalarType t) {
  switch (t) {
  case at::kFloat: return 1;
  case at::kByte: return 2;
  case at::kChar: return 3;
  case at::kShort: return 5;
  case at::kInt: return 6;
  case at::kLong: return 7;
  case at::kBool: return 9;
  case at::kHalf: return 10;
  case at::kDouble: return 11;
  case at::kBFloat16: return 16;
  case at::kFloat8_e4m3fn: return kF8E4M3FN;
  default: return 0;
  }
}

// Bits of an element of an ONNX type as the framework's tensors store it; 0: none of them.
int bits_of(long dtype) {
  switch (dtype) {
  case 21: case 22: case 23: return 4;                            // UINT4, INT4, FLOAT4E2M1
  case 2: case 3: case 9: case 17: case 18: case 19: case 20: return 8; // UINT8, INT8, BOOL, FLOAT8*
  case 4: case 5: case 10: case 16: return 16;                    // UINT16, INT16, FLOAT16, BFLOAT16
  case 1: case 6: case 12: return 32;                             // FLOAT, INT32, UINT32
  case 7: case 11: case 13: return 64;                            // INT64, DOUBLE, UINT64
  default: return 0;
  }
}

bool fail(PyObject *type, const char *message) {
  PyErr_SetString(type, message);
  return false;
}

// A tensor argument as the C ABI takes it.  Keeps its tensor alive.
struct Arg {
  at::Tensor t;
  b2_tensor d{};
  int64_t dims[8];

  bool set(const at::Tensor &x, int device) {
    if (!x.is_cuda()) return fail(PyExc_ValueError, "onnxl_b200 tensors must live on a CUDA device (no CPU fallback)");
    if (!x.is_contiguous()) return fail(PyExc_ValueError, "onnxl_b200 tensors must be contiguous");
    if (device >= 0 && x.get_device() != device)
      return fail(PyExc_ValueError, "onnxl_b200 tensors of one call must live on one device");
    t = x;
    d.data = t.data_ptr();
    d.dtype = onnx_type(t.scalar_type());
    d.ndim = (int32_t)t.dim();
    d.shape = t.sizes().data();
    return true;
  }
  // Whether `dims` elements of the declared type lie in the storage, on the type's boundary: the kernels
  // read and write what the shape says.
  bool fits(long dtype, Py_ssize_t n) {
    const int bits = bits_of(dtype);
    if (!bits) return fail(PyExc_ValueError, "a QTensor's dtype is not a numeric ONNX type");
    int64_t count = bits;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (dims[i] == 0) return true;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (__builtin_mul_overflow(count, dims[i], &count))
        return fail(PyExc_ValueError, "a QTensor's storage is smaller than its shape");
    if (t.nbytes() < (size_t)(count / 8 + (count % 8 != 0)))
      return fail(PyExc_ValueError, "a QTensor's storage is smaller than its shape");
    if (bits > 8 && reinterpret_cast<uintptr_t>(d.data) % (bits / 8) != 0)
      return fail(PyExc_ValueError, "a QTensor's storage must start on a boundary of its type");
    return true;
  }
  // A torch.Tensor, or a QTensor (data, dtype, shape).  `dtype` replaces the type of 8-bit storage.
  bool parse(PyObject *o, int device, int32_t dtype = 0) {
    if (THPVariable_Check(o)) {
      if (!set(THPVariable_Unpack(o), device)) return false;
      if (dtype) d.dtype = dtype;
      return true;
    }
    PyObject *data = PyObject_GetAttr(o, s_data), *code = data ? PyObject_GetAttr(o, s_dtype) : nullptr,
             *shape = code ? PyObject_GetAttr(o, s_shape) : nullptr;
    bool ok = false;
    if (!shape || !THPVariable_Check(data) || !PyLong_Check(code) || !PySequence_Check(shape)) {
      PyErr_Clear();
      fail(PyExc_TypeError, "expected a torch.Tensor or QTensor");
    } else if (set(THPVariable_Unpack(data), device)) {
      const Py_ssize_t n = PySequence_Size(shape);
      ok = n <= 8 || fail(PyExc_ValueError, "a QTensor has at most 8 dimensions");
      for (Py_ssize_t i = 0; ok && i < n; ++i) {
        PyObject *v = PySequence_GetItem(shape, i);
        dims[i] = v ? PyLong_AsLongLong(v) : -1;
        Py_XDECREF(v);
        ok = !PyErr_Occurred() && (dims[i] >= 0 || fail(PyExc_ValueError, "a QTensor's shape is not negative"));
      }
      const long type = ok ? PyLong_AsLong(code) : 0;
      ok = ok && !PyErr_Occurred() && fits(type, n);
      if (ok) {
        d.dtype = (int32_t)type;
        d.ndim = (int32_t)n;
        d.shape = dims;
      }
    }
    Py_XDECREF(data);
    Py_XDECREF(code);
    Py_XDECREF(shape);
    return ok;
  }
};

bool given(PyObject *o) { return o != Py_None; }

// Raises for a status other than B2_OK.
bool checked(int rc) {
  if (rc == B2_OK) return true;
  PyObject *r = PyObject_CallFunction(g_check, "i", rc);
  if (r) {
    Py_DECREF(r);
    PyErr_SetString(PyExc_RuntimeError, "onnxl_b200 call failed");
  }
  return false;
}

at::Tensor empty_like_shape(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// One zeroed buffer per (device, stream), grown on demand: calls on one stream are ordered, and
// every call leaves its counters at zero.  A call that is being captured into a graph gets its own
// buffer, which the graph clears (the whole of it, counters and partial results), since a replay may run
// beside calls on any stream.
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_workspaces;

void *workspace(int device, cudaStream_t st, size_t need, at::Tensor *keep) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &capture) == cudaSuccess && capture != cudaStreamCaptureStatusNone) {
    *keep = at::zeros({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
    return keep->data_ptr();
  }
  at::Tensor &t = g_workspaces[{device, st}];
  if (!t.defined() || t.nbytes() < need)
    t = at::zeros({(int64_t)std::max<size_t>(need, (size_t)1 << 20)},
                  at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
  return t.data_ptr();
}

bool connected() {
  return g_check != nullptr || fail(PyExc_RuntimeError, "_b2torch: connect() has not been called");
}

bool arity(const char *name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  return false;
}

// (x, scale, residual, epsilon, dtype, group_size, out, out_scale, out_sum) -> (codes, scales, sum)
PyObject *rms_norm_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!connected() || !arity("rms_norm_quantize", n, 9)) return nullptr;
  Arg x, w, r, y, s, h;
  if (!x.parse(args[0], -1)) return nullptr;
  const int device = x.t.get_device();
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  if (!w.parse(args[1], device) || (given(args[2]) && !r.parse(args[2], device))) return nullptr;
  const double eps = PyFloat_AsDouble(args[3]);
  const long dtype = PyLong_AsLong(args[4]);
  const long long group = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (given(args[6])) {
    if (!y.parse(args[6], device)) return nullptr;
  } else {
    if (dtype != kInt8 && dtype != kF8E4M3FN) {
      fail(PyExc_ValueError, "8-bit codes are INT8 or FLOAT8E4M3FN");
      return nullptr;
    }
    y.set(empty_like_shape(x.t.sizes(), dtype == kInt8 ? at::kChar : at::kByte, device), device);
    y.d.dtype = (int32_t)dtype;
  }
  if (given(args[7])) {
    if (!s.parse(args[7], device)) return nullptr;
  } else {
    const int64_t width = x.t.dim() ? x.t.size(-1) : 1;
    if (group < 0 || (group && width % group)) {
      fail(PyExc_ValueError, "b200::RMSNormalizationQuantize: group_size must divide the number of columns (0: one group per row).");
      return nullptr;
    }
    auto shape = x.t.sizes().vec();
    if (!shape.empty()) shape.back() = group ? width / group : 1;
    s.set(empty_like_shape(shape, at::kFloat, device), device);
  }
  const bool sum = given(args[8]) || given(args[2]);
  if (given(args[8])) {
    if (!h.parse(args[8], device)) return nullptr;
  } else if (sum) {
    h.set(empty_like_shape(x.t.sizes(), x.t.scalar_type(), device), device);
  }
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  if (!checked(f_norm(&x.d, given(args[2]) ? &r.d : nullptr, &w.d, (float)eps, group, &y.d,
                                             &s.d, sum ? &h.d : nullptr, st)))
    return nullptr;
  PyObject *out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, given(args[6]) ? Py_NewRef(args[6]) : THPVariable_Wrap(y.t));
  PyTuple_SET_ITEM(out, 1, given(args[7]) ? Py_NewRef(args[7]) : THPVariable_Wrap(s.t));
  PyTuple_SET_ITEM(out, 2, given(args[8]) ? Py_NewRef(args[8]) : sum ? THPVariable_Wrap(h.t) : Py_NewRef(Py_None));
  return out;
  END_HANDLE_TH_ERRORS
}

// (a, a_scale, w, w_scale, dtype, out) -> y; dtype: a torch.dtype
PyObject *scaled_matmul(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!connected() || !arity("scaled_matmul", n, 6)) return nullptr;
  Arg a, as, w, ws, y;
  if (!a.parse(args[0], -1)) return nullptr;
  const int device = a.t.get_device();
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  if (!as.parse(args[1], device) || !w.parse(args[2], device) || !ws.parse(args[3], device)) return nullptr;
  if (given(args[5])) {
    if (!y.parse(args[5], device)) return nullptr;
  } else {
    if (!THPDtype_Check(args[4])) {
      fail(PyExc_TypeError, "dtype must be a torch.dtype");
      return nullptr;
    }
    if (a.d.ndim < 1 || w.d.ndim != 2) {
      fail(PyExc_ValueError, "b200::ScaledMatMul: W must be [N, K] with K the last dimension of A.");
      return nullptr;
    }
    std::vector<int64_t> shape(a.d.shape, a.d.shape + a.d.ndim);
    shape.back() = w.d.shape[0];
    y.set(empty_like_shape(shape, reinterpret_cast<THPDtype *>(args[4])->scalar_type, device), device);
  }
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  if (!checked(f_product(&a.d, &as.d, &w.d, &ws.d, &y.d, nullptr, nullptr, st))) return nullptr;
  return given(args[5]) ? Py_NewRef(args[5]) : THPVariable_Wrap(y.t);
  END_HANDLE_TH_ERRORS
}

// The tensors of a QuantizedKVCache.
struct Cache {
  Arg k, v, ks, vs, table, lengths;
  b2_quantized_cache c{};
  bool parse(PyObject *o, int device) {
    PyObject *code = PyObject_GetAttr(o, s_dtype);
    const long dtype = code ? PyLong_AsLong(code) : 0;
    Py_XDECREF(code);
    if (PyErr_Occurred()) return false;
    const std::pair<PyObject *, Arg *> parts[] = {{s_k, &k}, {s_v, &v}, {s_k_scale, &ks},
                                                  {s_v_scale, &vs}, {s_table, &table}, {s_lengths, &lengths}};
    for (const auto &p : parts) {
      PyObject *t = PyObject_GetAttr(o, p.first);
      const bool pool = p.second == &k || p.second == &v;
      const bool ok = t && p.second->parse(t, device, pool ? (int32_t)dtype : 0);
      Py_XDECREF(t);
      if (!ok) return false;
      if (pool && p.second->t.element_size() != 1)
        return fail(PyExc_ValueError, "QuantizedKVCache: k and v must hold 8-bit codes");
    }
    c = b2_quantized_cache{&k.d, &v.d, &ks.d, &vs.d, &table.d, &lengths.d};
    return true;
  }
};

// (K, V, cache, new_lengths) -> None
PyObject *kv_cache_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!connected() || !arity("kv_cache_append", n, 4)) return nullptr;
  Arg k, v, counts;
  Cache c;
  if (!k.parse(args[0], -1)) return nullptr;
  const int device = k.t.get_device();
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  if (!v.parse(args[1], device) || !c.parse(args[2], device) || (given(args[3]) && !counts.parse(args[3], device)))
    return nullptr;
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  if (!checked(f_append(&k.d, &v.d, &c.c, given(args[3]) ? &counts.d : nullptr, st))) return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (Q, cache, new_lengths, out, has_scale, scale, is_causal, softcap, left_window_size, sink_tokens) -> y
PyObject *cache_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!connected() || !arity("cache_attention", n, 10)) return nullptr;
  Arg q, counts, y;
  Cache c;
  if (!q.parse(args[0], -1)) return nullptr;
  const int device = q.t.get_device();
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  if (!c.parse(args[1], device) || (given(args[2]) && !counts.parse(args[2], device))) return nullptr;
  b2_cache_attention_attrs at{};
  at.has_scale = PyObject_IsTrue(args[4]);
  at.scale = (float)PyFloat_AsDouble(args[5]);
  at.is_causal = PyObject_IsTrue(args[6]);
  at.softcap = (float)PyFloat_AsDouble(args[7]);
  at.left_window_size = PyLong_AsLongLong(args[8]);
  at.sink_tokens = PyLong_AsLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  if (given(args[3])) {
    if (!y.parse(args[3], device)) return nullptr;
  } else {
    y.set(empty_like_shape(q.t.sizes(), q.t.scalar_type(), device), device);
  }
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  const b2_tensor *nd = given(args[2]) ? &counts.d : nullptr;
  size_t need = 0;
  if (!checked(f_attention(&q.d, &c.c, nd, &at, &y.d, nullptr, &need, st))) return nullptr;
  at::Tensor keep;
  void *ws = need ? workspace(device, st, need, &keep) : nullptr;
  if (!checked(f_attention(&q.d, &c.c, nd, &at, &y.d, ws, need ? &need : nullptr, st))) return nullptr;
  return given(args[3]) ? Py_NewRef(args[3]) : THPVariable_Wrap(y.t);
  END_HANDLE_TH_ERRORS
}

// (check, addresses of b2_rms_normalization_quantize, b2_scaled_matmul, b2_kv_cache_append and
// b2_cache_attention)
PyObject *connect(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!arity("connect", n, 5)) return nullptr;
  void *p[4];
  for (int i = 0; i < 4; ++i)
    if (!(p[i] = PyLong_AsVoidPtr(args[i + 1]))) {
      if (!PyErr_Occurred()) fail(PyExc_ValueError, "connect: a function has no address");
      return nullptr;
    }
  f_norm = reinterpret_cast<decltype(f_norm)>(p[0]);
  f_product = reinterpret_cast<decltype(f_product)>(p[1]);
  f_append = reinterpret_cast<decltype(f_append)>(p[2]);
  f_attention = reinterpret_cast<decltype(f_attention)>(p[3]);
  Py_INCREF(args[0]);
  Py_XDECREF(g_check);
  g_check = args[0];
  Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *, PyObject *const *, Py_ssize_t)> PyMethodDef fast(const char *name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {fast<rms_norm_quantize>("rms_norm_quantize"), fast<scaled_matmul>("scaled_matmul"),
                         fast<kv_cache_append>("kv_cache_append"), fast<cache_attention>("cache_attention"),
                         fast<connect>("connect"), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b2torch", "Native calls of onnxl_b200 on torch tensors.", -1, methods};

} // namespace

PyMODINIT_FUNC PyInit__b2torch() {
  const std::pair<PyObject **, const char *> names[] = {
      {&s_data, "data"}, {&s_dtype, "dtype"}, {&s_shape, "shape"}, {&s_k, "k"}, {&s_v, "v"}, {&s_k_scale, "k_scale"},
      {&s_v_scale, "v_scale"}, {&s_table, "block_table"}, {&s_lengths, "lengths"}};
  for (const auto &n : names)
    if (!(*n.first = PyUnicode_InternFromString(n.second))) return nullptr;
  return PyModule_Create(&module);
}
