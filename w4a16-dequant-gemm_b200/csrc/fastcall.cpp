// CPython binding of the entries a serving loop calls every step (page_tables, kv_write_b8, attention_b8_paged): the
// same C ABI (include/w4b_abi.h) without ctypes, whose conversion of twenty arguments costs as much as the launch
// (attention: 6.7 us a call through ctypes, 4.2 us so, launch included). Arguments are positional, in the order of the ABI with
// the cache descriptor's eight fields in place of its address; addresses are integers or None. Every function returns
// the entry's status code; capi.py turns it into the exceptions.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits.h>

#include "../../include/w4b_abi.h"

namespace {

// Converts arguments one after the other; stops at the first that does not fit.
struct Args {
  PyObject* const* v;
  Py_ssize_t i;
  bool bad;
  long long wide() {
    const long long x = bad ? 0 : PyLong_AsLongLong(v[i++]);
    bad = bad || (x == -1 && PyErr_Occurred());
    return x;
  }
  int num() {
    const long long x = wide();
    if (!bad && (x > INT_MAX || x < INT_MIN)) {
      PyErr_SetString(PyExc_OverflowError, "argument does not fit a 32-bit int");
      bad = true;
    }
    return (int)x;
  }
  template <typename T>
  T* ptr() {
    if (!bad && v[i] == Py_None) {
      ++i;
      return nullptr;
    }
    const unsigned long long x = bad ? 0 : PyLong_AsUnsignedLongLong(v[i++]);
    bad = bad || (x == (unsigned long long)-1 && PyErr_Occurred());
    return (T*)x;
  }
  float real() {
    const double x = bad ? 0.0 : PyFloat_AsDouble(v[i++]);
    bad = bad || (x == -1.0 && PyErr_Occurred());
    return (float)x;
  }
  w4b_kv_b8 cache() {  // braces: evaluated in order
    return w4b_kv_b8{num(), num(), num(), num(), ptr<uint8_t>(), ptr<float>(), ptr<uint8_t>(), ptr<float>()};
  }
};

bool count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments given, %zd wanted", n, want);
  return false;
}

PyObject* status(int rc) { return PyLong_FromLong(rc); }

PyObject* page_tables(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (!count(n, 17)) return nullptr;
  Args a{v, 0, false};
  const int *cached = a.ptr<int>(), *fresh = a.ptr<int>();
  const int nseq = a.num(), page = a.num(), npages = a.num();
  const int* free_pages = a.ptr<int>();
  const int nfree = a.num();
  const int* taken_in = a.ptr<int>();
  int *taken_out = a.ptr<int>(), *bt = a.ptr<int>();
  const int bt_stride = a.num();
  int *seq_lens = a.ptr<int>(), *q_offsets = a.ptr<int>(), *slots = a.ptr<int>(), *positions = a.ptr<int>();
  const int max_tokens = a.num();
  void* stream = a.ptr<void>();
  if (a.bad) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = w4b_page_tables(cached, fresh, nseq, page, npages, free_pages, nfree, taken_in, taken_out, bt, bt_stride, seq_lens,
                       q_offsets, slots, positions, max_tokens, stream);
  Py_END_ALLOW_THREADS;
  return status(rc);
}

PyObject* kv_write_b8(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (!count(n, 16)) return nullptr;
  Args a{v, 0, false};
  const w4b_kv_b8 p = a.cache();
  const int* slots = a.ptr<int>();
  const int T = a.num();
  const void *k = a.ptr<void>(), *vals = a.ptr<void>();
  const long long ks = a.wide(), vs = a.wide();
  const int dtype = a.num();
  void* stream = a.ptr<void>();
  if (a.bad) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = w4b_kv_write_b8(&p, slots, T, k, vals, ks, vs, dtype, stream);
  Py_END_ALLOW_THREADS;
  return status(rc);
}

PyObject* attn_b8_paged(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (!count(n, 27)) return nullptr;
  Args a{v, 0, false};
  const w4b_kv_b8 p = a.cache();
  const int* bt = a.ptr<int>();
  const int bt_stride = a.num();
  const int *seq_lens = a.ptr<int>(), *q_offsets = a.ptr<int>();
  const int nseq = a.num(), max_q = a.num(), max_len = a.num();
  const void* q = a.ptr<void>();
  const long long q_stride = a.wide();
  const int Hq = a.num(), dtype = a.num();
  const float scale = a.real();
  const int causal = a.num();
  void* out = a.ptr<void>();
  const long long out_stride = a.wide();
  float* lse = a.ptr<float>();
  void* ws = a.ptr<void>();
  const long long ws_bytes = a.wide();
  void* stream = a.ptr<void>();
  if (a.bad) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = w4b_attn_b8_paged(&p, bt, bt_stride, seq_lens, q_offsets, nseq, max_q, max_len, q, q_stride, Hq, dtype, scale, causal,
                         out, out_stride, lse, ws, ws_bytes, stream);
  Py_END_ALLOW_THREADS;
  return status(rc);
}

PyMethodDef methods[] = {
    {"page_tables", (PyCFunction)(void (*)(void))page_tables, METH_FASTCALL, "w4b_page_tables"},
    {"kv_write_b8", (PyCFunction)(void (*)(void))kv_write_b8, METH_FASTCALL, "w4b_kv_write_b8"},
    {"attn_b8_paged", (PyCFunction)(void (*)(void))attn_b8_paged, METH_FASTCALL, "w4b_attn_b8_paged"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_w4b_fastcall", "Per-step entries of libw4b200.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__w4b_fastcall(void) { return PyModule_Create(&module); }
