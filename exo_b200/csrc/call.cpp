// The calls of the checked entry points (exo_b200/api.py, CheckedProc) for the ordinary case: no context, and torch
// tensors of the right types and sizes, the first of them on a GPU.  The interpreter and ctypes take 5.5 us for
// such a call, longer than the launch behind it; this takes 2 us (linear_i8_bf16_exo on 11 arguments, launch included:
// 6.1 us, 9.7 through the interpreter).  Whatever is not the ordinary case is left to the Python
// path, which also finds the words for what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

namespace {

constexpr int kMaxArgs = 18, kKinds = 3, kMaxTypes = 3;

struct Plan {
  void* fn;
  int sizes, tensors;
  struct {
    int kind, d0, d1;  // argument positions of the dimensions; d1 = 0: one dimension
  } tensor[kMaxArgs];
};

PyObject *tensor_type, *parameter_type, *raw_stream, *stream_cell, *dtypes[kKinds][kMaxTypes];
PyObject *s_dtype, *s_shape, *s_is_contiguous, *s_data_ptr, *s_get_device, *s_value;
void (*set_default_stream)(void*);
int (*last_error)();

// setup(Tensor, Parameter, ((dtype, ...), ...) by kind, current raw stream of a device, the cell of the thread's default
//       stream, address of exo_b200_set_default_stream, address of exo_b200_last_error)
PyObject* setup(PyObject*, PyObject* args) {
  PyObject *tensor, *parameter, *kinds, *stream, *cell;
  unsigned long long set, last;
  if (!PyArg_ParseTuple(args, "OOO!OOKK", &tensor, &parameter, &PyTuple_Type, &kinds, &stream, &cell, &set, &last))
    return nullptr;
  if (PyTuple_GET_SIZE(kinds) != kKinds) return PyErr_Format(PyExc_ValueError, "expected %d kinds", kKinds);
  for (int k = 0; k < kKinds; k++) {
    PyObject* of = PyTuple_GET_ITEM(kinds, k);
    if (!PyTuple_Check(of) || PyTuple_GET_SIZE(of) > kMaxTypes) return PyErr_Format(PyExc_ValueError, "types of a kind");
    for (int t = 0; t < kMaxTypes; t++)
      Py_XSETREF(dtypes[k][t], t < PyTuple_GET_SIZE(of) ? Py_NewRef(PyTuple_GET_ITEM(of, t)) : nullptr);
  }
  Py_XSETREF(tensor_type, Py_NewRef(tensor));
  Py_XSETREF(parameter_type, Py_NewRef(parameter));
  Py_XSETREF(raw_stream, Py_NewRef(stream));
  Py_XSETREF(stream_cell, Py_NewRef(cell));
  set_default_stream = reinterpret_cast<void (*)(void*)>((uintptr_t)set);
  last_error = reinterpret_cast<int (*)()>((uintptr_t)last);
  Py_RETURN_NONE;
}

void free_plan(PyObject* capsule) { PyMem_Free(PyCapsule_GetPointer(capsule, "exo_b200.plan")); }

// plan(address, number of sizes, ((kind, d0, d1), ...)) -> what call() takes
PyObject* plan(PyObject*, PyObject* args) {
  unsigned long long fn;
  int sizes;
  PyObject* tensors;
  if (!PyArg_ParseTuple(args, "KiO!", &fn, &sizes, &PyTuple_Type, &tensors)) return nullptr;
  const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
  if (sizes < 0 || 1 + sizes + n > kMaxArgs) return PyErr_Format(PyExc_ValueError, "too many arguments");
  Plan* p = static_cast<Plan*>(PyMem_Calloc(1, sizeof(Plan)));
  if (!p) return PyErr_NoMemory();
  p->fn = reinterpret_cast<void*>((uintptr_t)fn);
  p->sizes = sizes;
  p->tensors = (int)n;
  for (Py_ssize_t i = 0; i < n; i++) {
    auto& t = p->tensor[i];
    if (!PyArg_ParseTuple(PyTuple_GET_ITEM(tensors, i), "iii", &t.kind, &t.d0, &t.d1) || t.kind < 0 ||
        t.kind >= kKinds || t.d0 < 1 || t.d0 > sizes || t.d1 < 0 || t.d1 > sizes) {
      PyMem_Free(p);
      return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a tensor of the plan");
    }
  }
  return PyCapsule_New(p, "exo_b200.plan", free_plan);
}

// The integer that a method without arguments returns; false (and no exception) where it is none.
bool method_int(PyObject* o, PyObject* name, long long* v) {
  PyObject* r = PyObject_CallMethodNoArgs(o, name);
  if (!r) {
    PyErr_Clear();
    return false;
  }
  *v = PyLong_AsLongLong(r);  // a bool counts as 0 or 1
  Py_DECREF(r);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// Whether a tensor has `rows` elements, or `rows` rows of *width of them (in one dimension, or any whose last is the row).
bool fits(PyObject* o, long long rows, const long long* width) {
  PyObject* shape = PyObject_GetAttr(o, s_shape);
  if (!shape || !PyTuple_Check(shape)) {
    PyErr_Clear();
    Py_XDECREF(shape);
    return false;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(shape);
  __int128 have = 1;  // (a tensor's element count is below 2^63)
  long long last = 1;
  for (Py_ssize_t i = 0; i < n; i++) {
    last = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
    if (last < 0) {
      PyErr_Clear();
      Py_DECREF(shape);
      return false;
    }
    have *= last;
  }
  Py_DECREF(shape);
  // sizes that would not fit a product are the Python path's to refuse
  return have == (__int128)rows * (width ? *width : 1) && (!width || n < 2 || last == *width);
}

// The thread's default stream as the Python path last set it; sets it where it differs.
bool use_stream(long long device) {
  PyObject* index = PyLong_FromLongLong(device);
  PyObject* stream = index ? PyObject_CallOneArg(raw_stream, index) : nullptr;
  Py_XDECREF(index);
  if (!stream) {
    PyErr_Clear();
    return false;
  }
  PyObject* old = PyObject_GetAttr(stream_cell, s_value);
  if (!old) PyErr_Clear();
  const int same = old ? PyObject_RichCompareBool(old, stream, Py_EQ) : 0;
  Py_XDECREF(old);
  bool ok = same == 1;
  if (same == 0) {
    void* handle = PyLong_AsVoidPtr(stream);
    if (!PyErr_Occurred()) {
      set_default_stream(handle);
      ok = PyObject_SetAttr(stream_cell, s_value, stream) == 0;
    }
  }
  Py_DECREF(stream);
  if (!ok) PyErr_Clear();
  return ok;
}

// call(plan, arguments) -> the entry point's error code, or -1 where the Python path has to make the call
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2 || !tensor_type) return PyLong_FromLong(-1);
  const Plan* p = static_cast<const Plan*>(PyCapsule_GetPointer(args[0], "exo_b200.plan"));
  if (!p) return nullptr;
  PyObject* a = args[1];
  const PyObject* none = Py_None;
  if (!PyTuple_Check(a) || PyTuple_GET_SIZE(a) != 1 + p->sizes + p->tensors || PyTuple_GET_ITEM(a, 0) != none)
    return PyLong_FromLong(-1);
  long long v[kMaxArgs] = {};
  for (int i = 1; i <= p->sizes; i++) {
    PyObject* o = PyTuple_GET_ITEM(a, i);
    if (!PyLong_CheckExact(o)) return PyLong_FromLong(-1);
    v[i] = PyLong_AsLongLong(o);
    if (v[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return PyLong_FromLong(-1);
    }
  }
  long long device = -1;
  for (int i = 0; i < p->tensors; i++) {
    const auto& t = p->tensor[i];
    const int at = 1 + p->sizes + i;
    PyObject* o = PyTuple_GET_ITEM(a, at);
    if (o == none) continue;
    PyObject* cls = (PyObject*)Py_TYPE(o);
    if (cls != tensor_type && cls != parameter_type) return PyLong_FromLong(-1);
    PyObject* type = PyObject_GetAttr(o, s_dtype);
    if (!type) {
      PyErr_Clear();
      return PyLong_FromLong(-1);
    }
    Py_DECREF(type);  // torch keeps its types
    if (type != dtypes[t.kind][0] && type != dtypes[t.kind][1] && type != dtypes[t.kind][2]) return PyLong_FromLong(-1);
    long long dense;
    if (!fits(o, v[t.d0], t.d1 ? &v[t.d1] : nullptr) || !method_int(o, s_is_contiguous, &dense) || dense != 1 ||
        !method_int(o, s_data_ptr, &v[at]) || !v[at])  // (no memory: not the same as no operand)
      return PyLong_FromLong(-1);
    if (device < 0 && (!method_int(o, s_get_device, &device) || device < 0)) return PyLong_FromLong(-1);
  }
  if (device < 0 || !use_stream(device)) return PyLong_FromLong(-1);
  int code;
  Py_BEGIN_ALLOW_THREADS
  // every argument is an integer or a pointer, which the System V ABI passes alike; those past the last are ignored
  reinterpret_cast<void (*)(long long, long long, long long, long long, long long, long long, long long, long long,
                            long long, long long, long long, long long, long long, long long, long long, long long,
                            long long, long long)>(p->fn)(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9],
                                                          v[10], v[11], v[12], v[13], v[14], v[15], v[16], v[17]);
  code = last_error();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

PyMethodDef methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                         {"plan", plan, METH_VARARGS, nullptr},
                         {"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call() {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_value = PyUnicode_InternFromString("value");
  if (!s_dtype || !s_shape || !s_is_contiguous || !s_data_ptr || !s_get_device || !s_value) return nullptr;
  return PyModule_Create(&module);
}
