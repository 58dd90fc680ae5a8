// The Python calls of a decoder's serving step (fluidml_b200/cabi.py) straight onto the C ABI: a description of each tensor on the
// stack and the call.  Through ctypes the descriptions of a call's nine tensors and its conversions took 10 us, three times the
// kernel of a small call.
//
// A tensor is None, an object of the type that set_tensor_type() named (torch.Tensor: its data_ptr(), dtype, shape, stride() and
// is_cuda are read here), or anything else that the function given to set_describe() turns into the bytes of an fml_tensor; that
// function also raises for what no operator takes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cstring>
#include "fluidml_cuda.h"

namespace {

PyObject *g_data_ptr, *g_dtype, *g_shape, *g_stride, *g_is_cuda;  // attribute names
PyObject *g_describe = nullptr;
PyTypeObject *g_tensor_type = nullptr;
struct { PyObject *dtype; int code; } g_codes[8];
int g_n_codes = 0;

// 64-bit integers of a tuple.
bool integers(PyObject *tuple, int rank, int64_t *out) {
  if (!tuple || !PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != rank) return false;
  for (int i = 0; i < rank; ++i) {
    out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
    if (out[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}

int code_of(PyObject *dtype) {
  for (int i = 0; i < g_n_codes; ++i)
    if (g_codes[i].dtype == dtype) return g_codes[i].code;
  return 0;
}

// True with *t filled in; false when the describe function has to look at it (no exception set), or has raised (set).
bool read_tensor(PyObject *o, fml_tensor *t) {
  PyObject *dtype = PyObject_GetAttr(o, g_dtype);
  if (!dtype) return false;
  t->dtype = code_of(dtype);
  Py_DECREF(dtype);
  if (t->dtype == 0) return false;
  PyObject *cuda = PyObject_GetAttr(o, g_is_cuda);
  if (!cuda) return false;
  const bool on_device = cuda == Py_True;
  Py_DECREF(cuda);
  if (!on_device) return false;
  PyObject *shape = PyObject_GetAttr(o, g_shape);
  if (!shape) return false;
  bool ok = PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) <= FML_MAX_RANK;
  if (ok) {
    t->rank = (int32_t)PyTuple_GET_SIZE(shape);
    ok = integers(shape, t->rank, t->shape);
  }
  Py_DECREF(shape);
  if (!ok) return false;
  PyObject *stride = PyObject_CallMethodNoArgs(o, g_stride);
  ok = integers(stride, t->rank, t->stride);
  Py_XDECREF(stride);
  if (!ok) return false;
  PyObject *ptr = PyObject_CallMethodNoArgs(o, g_data_ptr);
  if (!ptr) return false;
  t->data = PyLong_AsVoidPtr(ptr);
  Py_DECREF(ptr);
  return !PyErr_Occurred();
}

// The description of one argument: `at` points at `t`, or is null for None.  False with an exception set.
struct Arg {
  fml_tensor t;
  const fml_tensor *at = nullptr;
  bool set(PyObject *o) {
    if (o == Py_None) return true;
    at = &t;
    if (Py_TYPE(o) == g_tensor_type) {
      if (read_tensor(o, &t)) return true;
      if (PyErr_Occurred()) return false;
    }
    if (!g_describe) {
      PyErr_SetString(PyExc_RuntimeError, "set_describe() has not been called");
      return false;
    }
    PyObject *bytes = PyObject_CallOneArg(g_describe, o);
    if (!bytes) return false;
    const bool ok = PyBytes_Check(bytes) && PyBytes_GET_SIZE(bytes) == (Py_ssize_t)sizeof(fml_tensor);
    if (ok) memcpy(&t, PyBytes_AS_STRING(bytes), sizeof(t));
    else PyErr_SetString(PyExc_TypeError, "a description must be the bytes of an fml_tensor");
    Py_DECREF(bytes);
    return ok;
  }
};
template <int N> bool set_all(PyObject *const *args, Arg (&a)[N]) {
  for (int i = 0; i < N; ++i)
    if (!a[i].set(args[i])) return false;
  return true;
}
bool number(PyObject *o, float *out) {
  *out = (float)PyFloat_AsDouble(o);
  return !PyErr_Occurred();
}
bool address(PyObject *o, void **out) {  // None or an integer
  *out = o == Py_None ? nullptr : PyLong_AsVoidPtr(o);
  return !PyErr_Occurred();
}
bool count_is(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments are needed, %zd were given", want, n);
  return false;
}

// q, k, v, positions, slots, frequencies, q_out, k_out, v_out, magnitude, layout, stream
PyObject *rotary_positions(PyObject *, PyObject *const *args, Py_ssize_t n) {
  Arg a[9];
  float magnitude;
  void *stream;
  if (!count_is(n, 12) || !set_all(args, a) || !number(args[9], &magnitude) || !address(args[11], &stream)) return nullptr;
  const long layout = PyLong_AsLong(args[10]);
  if (PyErr_Occurred()) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fml_rotary_positions(a[0].at, a[1].at, a[2].at, a[3].at, a[4].at, a[5].at, magnitude, (int)layout, a[6].at, a[7].at, a[8].at, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

bool rules_of(PyObject *divisor, PyObject *cap, PyObject *causal, fml_score_rules *r) {
  if (!number(divisor, &r->divisor) || !number(cap, &r->cap)) return false;
  r->causal = causal ? PyObject_IsTrue(causal) : 1;
  return !PyErr_Occurred();
}

// q, k, v, slopes, prefix, q_documents, k_documents, out, divisor, cap, causal, stream
PyObject *attention_rules(PyObject *, PyObject *const *args, Py_ssize_t n) {
  Arg a[8];
  fml_score_rules r;
  void *stream;
  if (!count_is(n, 12) || !set_all(args, a) || !rules_of(args[8], args[9], args[10], &r) || !address(args[11], &stream)) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fml_attention_rules(a[0].at, a[1].at, a[2].at, a[3].at, a[4].at, a[5].at, a[6].at, &r, a[7].at, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

// q, k_cache, v_cache, block_table, context, query_start, tree, slopes, out, divisor, cap, workspace, its bytes, stream
PyObject *attention_tree(PyObject *, PyObject *const *args, Py_ssize_t n) {
  Arg a[9];
  fml_score_rules r;
  void *workspace, *stream;
  if (!count_is(n, 14) || !set_all(args, a) || !rules_of(args[9], args[10], nullptr, &r) || !address(args[11], &workspace) ||
      !address(args[13], &stream))
    return nullptr;
  const size_t bytes = PyLong_AsSize_t(args[12]);
  if (PyErr_Occurred()) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fml_attention_tree(a[0].at, a[1].at, a[2].at, a[3].at, a[4].at, a[5].at, a[6].at, a[7].at, &r, a[8].at, workspace, bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

// logits, uniform, temperature, top_k, top_p, min_p, tokens, probabilities, stream
PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
  Arg a[8];
  void *stream;
  if (!count_is(n, 9) || !set_all(args, a) || !address(args[8], &stream)) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fml_sample(a[0].at, a[1].at, a[2].at, a[3].at, a[4].at, a[5].at, a[6].at, a[7].at, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

PyObject *set_describe(PyObject *, PyObject *f) {
  Py_INCREF(f);
  Py_XSETREF(g_describe, f);
  Py_RETURN_NONE;
}
PyObject *set_tensor_type(PyObject *, PyObject *type) {
  if (!PyType_Check(type)) {
    PyErr_SetString(PyExc_TypeError, "a type is needed");
    return nullptr;
  }
  Py_INCREF(type);
  Py_XDECREF(reinterpret_cast<PyObject *>(g_tensor_type));
  g_tensor_type = reinterpret_cast<PyTypeObject *>(type);
  Py_RETURN_NONE;
}
// dtype object, code: how read_tensor knows a tensor's type (the objects are singletons and live on).
PyObject *add_dtype(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 2)) return nullptr;
  const long code = PyLong_AsLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (code_of(args[0]) == 0 && g_n_codes < 8) {
    Py_INCREF(args[0]);
    g_codes[g_n_codes].dtype = args[0];
    g_codes[g_n_codes++].code = (int)code;
  }
  Py_RETURN_NONE;
}

template <typename F> PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }
PyMethodDef g_methods[] = {{"rotary_positions", fast(rotary_positions), METH_FASTCALL, nullptr},
                           {"attention_rules", fast(attention_rules), METH_FASTCALL, nullptr},
                           {"attention_tree", fast(attention_tree), METH_FASTCALL, nullptr},
                           {"sample", fast(sample), METH_FASTCALL, nullptr},
                           {"set_describe", set_describe, METH_O, nullptr},
                           {"set_tensor_type", set_tensor_type, METH_O, nullptr},
                           {"add_dtype", fast(add_dtype), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject *PyInit__serving(void) {
  g_data_ptr = PyUnicode_InternFromString("data_ptr");
  g_dtype = PyUnicode_InternFromString("dtype");
  g_shape = PyUnicode_InternFromString("shape");
  g_stride = PyUnicode_InternFromString("stride");
  g_is_cuda = PyUnicode_InternFromString("is_cuda");
  if (!g_data_ptr || !g_dtype || !g_shape || !g_stride || !g_is_cuda) return nullptr;
  return PyModule_Create(&g_module);
}
