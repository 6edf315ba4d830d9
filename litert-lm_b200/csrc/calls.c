/* The operators over device memory as functions of a Python extension module: those that a serving loop calls once per layer and step.
 * Twenty arguments take ctypes 4 us to convert, as long as the launch itself; here they take 0.4.  Integers and addresses in,
 * None out, or (status code, message). */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdlib.h>

#include "../../include/b200lm_ops.h"

#define MOST 24

static int numbers(PyObject* const* args, Py_ssize_t have, Py_ssize_t want, int float_at, long long* v, double* f) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments are wanted, not %zd", want, have);
    return -1;
  }
  for (Py_ssize_t i = 0; i < want; ++i) {
    if (i == float_at) *f = PyFloat_AsDouble(args[i]);
    else v[i] = PyLong_AsLongLong(args[i]);
  }
  return PyErr_Occurred() ? -1 : 0;
}
static int narrow(const long long* v, const char* wide, Py_ssize_t n) {   /* wide[i] == 'i': an int32 */
  for (Py_ssize_t i = 0; i < n; ++i)
    if (wide[i] == 'i' && (v[i] < INT32_MIN || v[i] > INT32_MAX)) {
      PyErr_Format(PyExc_OverflowError, "argument %zd does not fit 32 bits", i);
      return -1;
    }
  return 0;
}
static PyObject* answer(int code, char* err) {
  PyObject* r;
  if (code == 0) Py_RETURN_NONE;
  r = Py_BuildValue("(is)", code, err ? err : "");
  free(err);
  return r;
}
#define P(i) ((void*)(intptr_t)v[i])
#define I(i) ((int32_t)v[i])
/* kinds: p address, l int64, i int32, f float */
#define BEGIN(kinds, float_at)                                                        \
  static const char kind[] = kinds;                                                   \
  long long v[MOST] = {0};                                                            \
  double f = 0;                                                                       \
  char* err = NULL;                                                                   \
  int code;                                                                           \
  (void)self;                                                                         \
  (void)f;                                                                            \
  if (numbers(args, n, sizeof kind - 1, float_at, v, &f) || narrow(v, kind, n)) return NULL; \
  Py_BEGIN_ALLOW_THREADS
#define END Py_END_ALLOW_THREADS return answer(code, err);

/* device, w, scale_type, has_offset, n, k, group, x, x_type, ldx, ncols, y, y_type, ldy, stream */
static PyObject* gemv_w4_grouped(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN("ipiillipilipilp", -1)
  code = B200LmOps_GemvW4Grouped(I(0), P(1), I(2), I(3), v[4], v[5], I(6), P(7), I(8), v[9], I(10), P(11), I(12), v[13], P(14), &err);
  END
}
/* device, qkv, type, qkv_stride, tokens, hq, hkv, hd, rot, q_gain, k_gain, eps, cos, sin, rope_rows, pos, q_out, q_stride, k_out,
 * k_stride, status, stream */
static PyObject* qk_norm_rope(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN("ipiliiiiippfppipplplpp", 11)
  code = B200LmOps_QkNormRope(I(0), P(1), I(2), v[3], I(4), I(5), I(6), I(7), I(8), P(9), P(10), (float)f, P(12), P(13), I(14), P(15), P(16), v[17], P(18), v[19],
                              P(20), P(21), &err);
  END
}
/* the same up to q_stride, then cache, seq, status, stream */
static PyObject* qk_norm_rope_append_kv4(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN("ipiliiiiippfppipplpppp", 11)
  code = B200LmOps_QkNormRopeAppendKv4(I(0), P(1), I(2), v[3], I(4), I(5), I(6), I(7), I(8), P(9), P(10), (float)f, P(12), P(13), I(14), P(15), P(16), v[17], P(18),
                                       P(19), P(20), P(21), &err);
  END
}
/* device, cache, seq, pos, tokens, out_type, k_out, v_out, status, stream */
static PyObject* kv4_read(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN("ipppiipppp", -1)
  code = B200LmOps_Kv4Read(I(0), P(1), P(2), P(3), I(4), I(5), P(6), P(7), P(8), P(9), &err);
  END
}
/* device, cache, q, q_type, q_stride, kv_len, q_start, tokens, max_q, max_kv, hq, window, scale, out, out_stride, workspace,
 * workspace_bytes, status, stream */
static PyObject* attention_kv4(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN("ippilppiiiiifplplpp", 12)
  code = B200LmOps_AttentionKv4(I(0), P(1), P(2), I(3), v[4], P(5), P(6), I(7), I(8), I(9), I(10), I(11), (float)f, P(13), v[14], P(15), v[16], P(17), P(18), &err);
  END
}

static PyMethodDef methods[] = {
    {"gemv_w4_grouped", (PyCFunction)(void (*)(void))gemv_w4_grouped, METH_FASTCALL, NULL},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, NULL},
    {"qk_norm_rope_append_kv4", (PyCFunction)(void (*)(void))qk_norm_rope_append_kv4, METH_FASTCALL, NULL},
    {"kv4_read", (PyCFunction)(void (*)(void))kv4_read, METH_FASTCALL, NULL},
    {"attention_kv4", (PyCFunction)(void (*)(void))attention_kv4, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
