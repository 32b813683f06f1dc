/* Calls of the operators inside a model's block for Python, past ctypes: that takes 0.1 us an argument, as long as a small kernel's
 * launch for the longer lists.  Each function takes the arguments of the C function of its name, whole numbers (None for a null
 * pointer), and returns its status; the interpreter's lock is released meanwhile, as ctypes does.
 *
 * place(tensor, dtype, shape, device) checks what a call's tensor usually is: of that type and shape, contiguous, on that device.  It
 * returns (address, last extent), or None where it is not: the caller finds out what it is. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/tc_b200.h"

static int numbers(PyObject* const* args, Py_ssize_t given, Py_ssize_t wanted, int64_t* out) {
  if (given != wanted) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
    return 0;
  }
  for (Py_ssize_t i = 0; i < wanted; ++i) {
    out[i] = 0;
    if (args[i] == Py_None) continue;
    out[i] = (int64_t)PyLong_AsLongLong(args[i]);
    if (out[i] == -1 && PyErr_Occurred()) return 0;
  }
  return 1;
}

#define P(i) ((void*)(intptr_t)a[i])
#define CALL(name, count, ...)                                                              \
  static PyObject* name(PyObject* self, PyObject* const* args, Py_ssize_t given) {          \
    int64_t a[count];                                                                       \
    int status;                                                                             \
    (void)self;                                                                             \
    if (!numbers(args, given, count, a)) return NULL;                                       \
    Py_BEGIN_ALLOW_THREADS status = tc_##name((tc_op_plan*)P(0), __VA_ARGS__);              \
    Py_END_ALLOW_THREADS return PyLong_FromLong(status);                                    \
  }

CALL(microscale_execute, 9, P(1), a[2], P(3), P(4), a[5], (int)a[6], a[7], P(8))
CALL(microscale_restore, 8, P(1), a[2], P(3), a[4], P(5), a[6], P(7))
CALL(micro_product_execute, 14, P(1), a[2], P(3), a[4], P(5), P(6), a[7], P(8), a[9], (int)a[10], P(11), (size_t)a[12], P(13))
CALL(checkpoint_execute, 9, P(1), a[2], P(3), P(4), P(5), a[6], a[7], P(8))
CALL(checkpoint_restore, 7, P(1), a[2], P(3), P(4), a[5], P(6))
CALL(checkpoint_execute_grad, 9, P(1), a[2], P(3), a[4], P(5), P(6), a[7], P(8))
CALL(checkpoint_execute_product, 14, P(1), a[2], (int)a[3], P(4), a[5], P(6), P(7), a[8], a[9], (int)a[10], P(11), (size_t)a[12], P(13))
CALL(residual_norm_execute, 15, P(1), a[2], P(3), a[4], P(5), a[6], P(7), a[8], P(9), P(10), P(11), a[12], a[13], P(14))
CALL(residual_norm_execute_grad, 25, P(1), a[2], P(3), a[4], P(5), a[6], P(7), P(8), P(9), a[10], P(11), a[12], P(13), a[14], P(15), a[16], P(17), P(18), P(19), a[20], a[21],
     P(22), (size_t)a[23], P(24))

static PyObject *s_dtype, *s_shape, *s_get_device, *s_is_contiguous, *s_data_ptr;

static int same_shape(PyObject* tensor, PyObject* shape) {
  PyObject* have = PyObject_GetAttr(tensor, s_shape);
  int same = have && PyTuple_Check(have) && PyTuple_Check(shape) && PyTuple_GET_SIZE(have) == PyTuple_GET_SIZE(shape);
  for (Py_ssize_t i = 0; same && i < PyTuple_GET_SIZE(shape); ++i)
    same = PyLong_AsLongLong(PyTuple_GET_ITEM(have, i)) == PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
  Py_XDECREF(have);
  return same;
}
static int same_object(PyObject* have, PyObject* want) {
  Py_XDECREF(have);  /* types and truth values live as long as the program */
  return have && have == want;
}
static int same_number(PyObject* have, PyObject* want) {
  const int same = have && PyLong_Check(have) && PyLong_Check(want) && PyLong_AsLongLong(have) == PyLong_AsLongLong(want);
  Py_XDECREF(have);
  return same;
}
static PyObject* place(PyObject* self, PyObject* const* args, Py_ssize_t given) {
  (void)self;
  if (given != 4 || !PyTuple_Check(args[2]) || !PyTuple_GET_SIZE(args[2])) {
    PyErr_SetString(PyExc_TypeError, "place: expected a tensor, a type, a shape and a device");
    return NULL;
  }
  PyObject* t = args[0];
  if (same_object(PyObject_GetAttr(t, s_dtype), args[1]) && same_shape(t, args[2]) && same_object(PyObject_CallMethodNoArgs(t, s_is_contiguous), Py_True) &&
      same_number(PyObject_CallMethodNoArgs(t, s_get_device), args[3])) {
    PyObject* address = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (address) {
      PyObject* both = PyTuple_Pack(2, address, PyTuple_GET_ITEM(args[2], PyTuple_GET_SIZE(args[2]) - 1));
      Py_DECREF(address);
      return both;
    }
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {ENTRY(microscale_execute),      ENTRY(microscale_restore),         ENTRY(micro_product_execute),
                                ENTRY(checkpoint_execute),      ENTRY(checkpoint_restore),         ENTRY(checkpoint_execute_grad),
                                ENTRY(checkpoint_execute_product), ENTRY(residual_norm_execute), ENTRY(residual_norm_execute_grad),
                                ENTRY(place),
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tc_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__tc_calls(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  return s_dtype && s_shape && s_get_device && s_is_contiguous && s_data_ptr ? PyModule_Create(&module) : NULL;
}
