// The row-group calls with torch tensors, without the interpreter's part: a Python extension module that reads the
// tensors' addresses, shapes and strides itself and enters the library at once.  `grouped.py` offers a call here first; a
// call that is not plain (an array that is no tensor, another device than the current one, a wrong type or length, the
// first call of a thread) is "not taken" and goes the way through ctypes, which checks, explains and launches the same
// entry point.  Small calls are bound by the host: gemm_lora takes 10.2 us of it through ctypes, 4.2 of them the launch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/moye_b200.h"

// Read from the file before anything of it runs: another torch or interpreter may lay its objects out differently.
#define MOYE_TEXT2(x) #x
#define MOYE_TEXT(x) MOYE_TEXT2(x)
extern "C" __attribute__((used, visibility("default"))) const char moye_calls_built_for[] =
    "moye_calls for " MOYE_BUILT_FOR ", library " MOYE_TEXT(MOYE_B200_VERSION) ";";

namespace {

struct Entries {
  decltype(&moye_b200_group_rows) group_rows;
  decltype(&moye_b200_gather_rows) gather_rows;
  decltype(&moye_b200_combine_rows) combine_rows;
  decltype(&moye_b200_combine_rows_grad) combine_rows_grad;
  decltype(&moye_b200_gemm_grouped) gemm_grouped;
  decltype(&moye_b200_gemm_grouped_grad) gemm_grouped_grad;
  decltype(&moye_b200_gemm_lora) gemm_lora;
} entry = {};
PyObject* handles = nullptr;  // (thread, device) -> object whose `value` is the handle, kept by _lib.py
PyObject* value_name = nullptr;

constexpr long kNotTaken = 1;  // 0: launched, below: the library's error code

int moye_type(c10::ScalarType t) {
  switch (t) {
    case c10::ScalarType::Float: return MOYE_F32;
    case c10::ScalarType::Half: return MOYE_F16;
    case c10::ScalarType::BFloat16: return MOYE_BF16;
    case c10::ScalarType::Int: return MOYE_S32;
    case c10::ScalarType::Long: return MOYE_U64;
    case c10::ScalarType::Char: return MOYE_S8;
    case c10::ScalarType::Byte: return MOYE_U8;
    case c10::ScalarType::Short: return MOYE_U16;
    case c10::ScalarType::Float8_e4m3fn: return MOYE_E4M3;
    default: return -1;
  }
}

// The arguments of one call; `ok` falls as soon as one of them is not plain.
struct Arguments {
  moye_tensor_t arrays[5];
  int used = 0, dev = -1;
  bool ok = true;

  const at::Tensor* tensor(PyObject* o) {
    if (!ok || !THPVariable_Check(o)) return ok = false, nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided) return ok = false, nullptr;
    const int at = t.get_device();
    if (dev < 0) dev = at;
    if (at != dev) return ok = false, nullptr;
    return &t;
  }
  const moye_tensor_t* array(PyObject* o, int rank) {
    const at::Tensor* t = tensor(o);
    if (!ok || t->dim() != rank) return ok = false, nullptr;
    moye_tensor_t& d = arrays[used++];
    d = {};
    d.ptr = t->data_ptr();
    d.dtype = moye_type(t->scalar_type());
    d.rank = rank;
    if (d.dtype < 0) return ok = false, nullptr;
    const auto sizes = t->sizes(), strides = t->strides();
    for (int i = 0; i < rank; ++i) {
      d.shape[i] = sizes[i];
      d.stride[i] = strides[i];
    }
    return &d;
  }
  // A contiguous vector of `numel` values (any number: -1).
  template <typename T>
  const T* vector(PyObject* o, long long numel, long long* count = nullptr) {
    const at::Tensor* t = tensor(o);
    if (!ok || t->scalar_type() != (std::is_same<T, float>::value ? c10::ScalarType::Float : c10::ScalarType::Int) || !t->is_contiguous() ||
        (numel >= 0 && t->numel() != numel))
      return ok = false, nullptr;
    if (count) *count = t->numel();
    return static_cast<const T*>(t->data_ptr());
  }
  long long number(PyObject* o) {
    const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
    if (v < 0) ok = false;
    return v;
  }
  float real(PyObject* o) {
    if (PyFloat_Check(o)) return (float)PyFloat_AS_DOUBLE(o);
    if (!PyLong_Check(o)) return ok = false, 0.f;
    return (float)PyLong_AsDouble(o);
  }
};

// f(handle, stream) without the interpreter lock; `stream` None is the current one of the operands' device.
template <typename F>
long launch(Arguments& a, PyObject* stream, F f) {
  if (PyErr_Occurred()) a.ok = false;
  if (!a.ok || a.dev < 0 || c10::cuda::current_device() != a.dev) return kNotTaken;
  void* on = nullptr;
  if (stream == Py_None) on = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)a.dev).stream();
  else if (PyLong_Check(stream)) on = PyLong_AsVoidPtr(stream);
  else return kNotTaken;
  PyObject* key = Py_BuildValue("(ki)", PyThread_get_thread_ident(), a.dev);
  PyObject* kept = key ? PyDict_GetItem(handles, key) : nullptr;  // borrowed
  Py_XDECREF(key);
  PyObject* value = kept ? PyObject_GetAttr(kept, value_name) : nullptr;
  moye_handle_t h = value && PyLong_Check(value) ? static_cast<moye_handle_t>(PyLong_AsVoidPtr(value)) : nullptr;
  Py_XDECREF(value);
  if (!h || PyErr_Occurred()) return kNotTaken;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(h, on);
  Py_END_ALLOW_THREADS
  return rc;
}

// Runs `body`; whatever it cannot digest is a call not taken, which the other way explains.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F body) {
  long rc = kNotTaken;
  if (got == want && handles) {
    try {
      rc = body();
    } catch (...) {
      rc = kNotTaken;
    }
  }
  PyErr_Clear();
  return PyLong_FromLong(rc);
}

// A plan comes as its buffer (order, inverse, offsets), tokens and choices.
const int* inverse_of(Arguments& a, PyObject* buf, long long tokens, long long choices) {
  const int* p = a.vector<int>(buf, -1);
  return a.ok ? p + tokens * choices : nullptr;
}

// group_rows(ids, buf, tokens, choices, groups, stream)
PyObject* group_rows(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> long {
    Arguments a;
    const at::Tensor* t = a.tensor(v[0]);
    if (!a.ok) return kNotTaken;
    const int rank = (int)t->dim();
    const long long tokens = a.number(v[2]), choices = a.number(v[3]), groups = a.number(v[4]);
    if (!a.ok || rank < 1 || rank > 2 || t->size(0) != tokens || (rank == 2 ? t->size(1) : 1) != choices) return kNotTaken;
    const moye_tensor_t* ids = a.array(v[0], rank);
    int* buf = const_cast<int*>(a.vector<int>(v[1], 2 * tokens * choices + groups + 1));
    return launch(a, v[5], [&](moye_handle_t h, void* s) {
      return entry.group_rows(h, ids, (int)groups, buf, buf + 2 * tokens * choices, buf + tokens * choices, s);
    });
  });
}

// new_plan(ids, groups): the buffer of a new plan, filled on the current stream, or a number like the other calls
PyObject* new_plan(PyObject*, PyObject* const* v, Py_ssize_t n) {
  at::Tensor made;
  PyObject* rc = guarded(n, 2, [&]() -> long {
    Arguments a;
    const at::Tensor* t = a.tensor(v[0]);
    const long long groups = a.number(v[1]);
    if (!a.ok || t->dim() < 1 || t->dim() > 2 || groups < 1 || groups > 1024 || c10::cuda::current_device() != a.dev) return kNotTaken;
    const moye_tensor_t* ids = a.array(v[0], (int)t->dim());
    if (!a.ok) return kNotTaken;
    const long long all = t->numel();
    made = at::empty({2 * all + groups + 1}, t->options().dtype(at::kInt));
    int* buf = made.data_ptr<int>();
    return launch(a, Py_None, [&](moye_handle_t h, void* s) {
      return entry.group_rows(h, ids, (int)groups, buf, buf + 2 * all, buf + all, s);
    });
  });
  if (!rc || PyLong_AsLong(rc) != 0) return rc;
  Py_DECREF(rc);
  return THPVariable_Wrap(std::move(made));
}

// gather_rows(dst, src, buf, tokens, choices, stream)
PyObject* gather_rows(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> long {
    Arguments a;
    const moye_tensor_t *dst = a.array(v[0], 2), *src = a.array(v[1], 2);
    const long long tokens = a.number(v[3]), choices = a.number(v[4]);
    const int* inverse = inverse_of(a, v[2], tokens, choices);
    if (!a.ok || src->shape[0] != tokens) return kNotTaken;
    return launch(a, v[5], [&](moye_handle_t h, void* s) { return entry.gather_rows(h, dst, src, inverse, (int)choices, s); });
  });
}

// combine_rows(dst, src, buf, tokens, choices, weights or None, stream)
PyObject* combine_rows(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> long {
    Arguments a;
    const moye_tensor_t *dst = a.array(v[0], 2), *src = a.array(v[1], 2), *w = v[5] == Py_None ? nullptr : a.array(v[5], 2);
    const long long tokens = a.number(v[3]), choices = a.number(v[4]);
    const int* inverse = inverse_of(a, v[2], tokens, choices);
    if (!a.ok || dst->shape[0] != tokens) return kNotTaken;
    return launch(a, v[6], [&](moye_handle_t h, void* s) { return entry.combine_rows(h, dst, src, w, inverse, (int)choices, s); });
  });
}

// combine_rows_grad(dsrc, dweights, ddst, src, buf, tokens, choices, weights, stream)
PyObject* combine_rows_grad(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> long {
    Arguments a;
    const moye_tensor_t *dsrc = a.array(v[0], 2), *dw = a.array(v[1], 2), *ddst = a.array(v[2], 2), *src = a.array(v[3], 2),
                        *w = a.array(v[7], 2);
    const long long tokens = a.number(v[5]), choices = a.number(v[6]);
    const int* inverse = inverse_of(a, v[4], tokens, choices);
    if (!a.ok || ddst->shape[0] != tokens) return kNotTaken;
    return launch(a, v[8], [&](moye_handle_t h, void* s) {
      return entry.combine_rows_grad(h, dsrc, dw, ddst, src, w, inverse, (int)choices, s);
    });
  });
}

// gemm_grouped(D, A, B, borders, first, alpha, beta, stream): B's groups + 1 borders end `borders` and start at `first`
// gemm_grouped_grad(dB, dD, A, ...): the same
template <bool GRAD>
PyObject* gemm_grouped(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> long {
    Arguments a;
    const moye_tensor_t *x = a.array(v[0], GRAD ? 3 : 2), *y = a.array(v[1], 2), *z = a.array(v[2], GRAD ? 2 : 3);
    if (!a.ok) return kNotTaken;
    const long long first = a.number(v[4]), groups = (GRAD ? x : z)->shape[0];
    const int* borders = a.vector<int>(v[3], first + groups + 1);
    const float alpha = a.real(v[5]), beta = a.real(v[6]);
    return launch(a, v[7], [&](moye_handle_t h, void* s) {
      return (GRAD ? entry.gemm_grouped_grad : entry.gemm_grouped)(h, x, y, z, borders + first, alpha, beta, s);
    });
  });
}

// gemm_lora(D, X, A, B, adapters, offsets, scales, C, stream), None for what is absent
PyObject* gemm_lora(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> long {
    Arguments a;
    const moye_tensor_t *d = a.array(v[0], 2), *x = a.array(v[1], 2), *fa = a.array(v[2], 3), *fb = a.array(v[3], 3),
                        *c = v[7] == Py_None ? nullptr : a.array(v[7], 2);
    long long requests = 0;
    const int* which = a.vector<int>(v[4], -1, &requests);
    if (!a.ok || requests > INT32_MAX) return kNotTaken;
    const int* offsets = v[5] == Py_None ? nullptr : a.vector<int>(v[5], requests + 1);
    const float* scales = v[6] == Py_None ? nullptr : a.vector<float>(v[6], fa->shape[0]);
    return launch(a, v[8], [&](moye_handle_t h, void* s) {
      return entry.gemm_lora(h, d, x, fa, fb, c, which, offsets, (int)requests, scales, s);
    });
  });
}

// bind(addresses of the entry points in the order of `Entries`, handles)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[7];
  PyObject* kept;
  if (!PyArg_ParseTuple(args, "(KKKKKKK)O!", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, &PyDict_Type, &kept)) return nullptr;
  static_assert(sizeof(Entries) == sizeof(p), "one address per entry point");
  memcpy(&entry, p, sizeof(p));
  Py_INCREF(kept);
  Py_XDECREF(handles);
  handles = kept;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"group_rows", FAST(group_rows)},
                         {"new_plan", FAST(new_plan)},
                         {"gather_rows", FAST(gather_rows)},
                         {"combine_rows", FAST(combine_rows)},
                         {"combine_rows_grad", FAST(combine_rows_grad)},
                         {"gemm_grouped", FAST(gemm_grouped<false>)},
                         {"gemm_grouped_grad", FAST(gemm_grouped<true>)},
                         {"gemm_lora", FAST(gemm_lora)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "moye_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_moye_calls() {
  value_name = PyUnicode_InternFromString("value");
  return value_name ? PyModule_Create(&module) : nullptr;
}
