// The operators of the 4-bit cache and of the step's index arrays, called from Python without the interpreter's share: one
// call checks the operands, allocates outputs and scratch from torch's allocator and enters the kernels' library on the
// current stream.  A few microseconds of work on the device cost about as much host time as the checks in Python alone
// did (per call 12 to 18 us, of which 3 per launch).
//
// A function here returns None when an operand is not what it handles; nothing has been launched then, and the caller's own path
// in Python handles the call or says what is wrong.  Otherwise the library's status (0: success), or the outputs.
// `entry` arguments are addresses of the library's functions.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {
struct Call {
  bool ok = true;
  int device;
  Call() : device((int)c10::cuda::current_device()) {}
  void* stream() const { return (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

  const at::Tensor* tensor(PyObject* o) {
    if (!THPVariable_Check(o)) { ok = false; return nullptr; }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != device) { ok = false; return nullptr; }
    return &t;
  }
  // A contiguous int32 tensor of n elements (n < 0: any number); None becomes null when that is allowed.
  int* words(PyObject* o, long n, bool optional = false) {
    if (o == Py_None) { ok = ok && optional; return nullptr; }
    const at::Tensor* t = tensor(o);
    if (!t || t->scalar_type() != at::kInt || !t->is_contiguous() || (n >= 0 && t->numel() != n)) { ok = false; return nullptr; }
    return (int*)t->data_ptr();
  }
  long number(PyObject* o) {
    if (!PyLong_Check(o)) { ok = false; return 0; }
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over || v > 0x7fffffffL || v < -0x7fffffffL) ok = false;
    return v;
  }
  // The two caches of 4-bit pages; returns the number of pages.
  long caches(PyObject* k, PyObject* v, long nkv, long hd, long page_size, void** k_at, void** v_at) {
    const at::Tensor *kt = tensor(k), *vt = tensor(v);
    if (!kt || !vt || hd < 32 || hd > 256 || hd % 32 || page_size < 16 || page_size % 16) { ok = false; return 0; }
    for (const at::Tensor* t : {kt, vt})
      if (t->scalar_type() != at::kByte || t->dim() != 4 || !t->is_contiguous() || t->size(1) != nkv || t->size(2) != page_size / 16 ||
          t->size(3) != 10 * hd)
        ok = false;
    if (!ok || kt->size(0) != vt->size(0) || kt->size(0) > 0x7fffffffL) { ok = false; return 0; }
    *k_at = kt->data_ptr();
    *v_at = vt->data_ptr();
    return (long)kt->size(0);
  }
  // Rows of float32 or bfloat16 (dtype code 0, 1) with neighbouring columns.
  const at::Tensor* rows(PyObject* o, long columns, int* code) {
    const at::Tensor* t = tensor(o);
    if (!t || t->dim() != 2 || t->size(1) != columns || (t->size(0) > 0 && t->stride(1) != 1) || t->size(0) > 0x7fffffffL) { ok = false; return nullptr; }
    if (t->scalar_type() == at::kFloat) *code = 0;
    else if (t->scalar_type() == at::kBFloat16) *code = 1;
    else { ok = false; return nullptr; }
    return t;
  }
};

void* address(PyObject* o) { return PyLong_AsVoidPtr(o); }
PyObject* none() { Py_RETURN_NONE; }

// What throws inside torch (an allocation) leaves as a Python exception.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// layout(entry, starts, q_lens, page_cu, pages, page_size, block_table, slots, cu_q, kv_lens, positions, token_req, first, status)
PyObject* layout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 14) return none();
  return guarded([&]() -> PyObject* {
    Call c;
    const at::Tensor* starts = c.tensor(a[1]);
    if (!starts || starts->numel() < 1 || starts->numel() > 0x7fffffffL) return none();
    const long B = (long)starts->numel();
    int* p_starts = c.words(a[1], B);
    int* q_lens = c.words(a[2], B);
    int* page_cu = c.words(a[3], B + 1);
    int* pages = c.words(a[4], -1);
    const long page_size = c.number(a[5]);
    int* table = c.words(a[6], -1);
    PyObject* per_token = a[7] != Py_None ? a[7] : a[10] != Py_None ? a[10] : a[11];
    long T = 0;
    if (per_token != Py_None) {
      const at::Tensor* t = c.tensor(per_token);
      if (!t) return none();
      T = (long)t->numel();
    }
    int *slots = c.words(a[7], T, true), *cu_q = c.words(a[8], B + 1, true), *kv_lens = c.words(a[9], B, true), *positions = c.words(a[10], T, true),
        *token_req = c.words(a[11], T, true), *first = c.words(a[12], B, true), *status = c.words(a[13], 1, true);
    if (!c.ok) return none();
    const at::Tensor &pt = THPVariable_Unpack(a[4]), &tt = THPVariable_Unpack(a[6]);
    if (tt.dim() != 2 || tt.size(0) != B || tt.size(1) > 0x7fffffffL || pt.numel() > 0x7fffffffL || T > 0x7fffffffL) return none();
    typedef int (*Fn)(const int*, const int*, const int*, const int*, int, const int*, int, int, int, int*, int*, int*, int*, int*, int, int*, int*, void*);
    return PyLong_FromLong(((Fn)address(a[0]))(p_starts, q_lens, page_cu, pages, (int)pt.numel(), first, (int)B, (int)T, (int)page_size, cu_q, kv_lens,
                                               positions, token_req, table, (int)tt.size(1), slots, status, c.stream()));
  });
}

// write(entry, qkv, positions, cos_sin, slots, k_cache, v_cache, heads, kv heads, head_dim, rotary_dim, page_size, status) -> the rotated queries
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) return none();
  return guarded([&]() -> PyObject* {
    Call c;
    const long nh = c.number(a[7]), nkv = c.number(a[8]), hd = c.number(a[9]), rot = c.number(a[10]), page_size = c.number(a[11]);
    if (!c.ok || rot <= 0 || nh < 0) return none();
    void *k = nullptr, *v = nullptr;
    const long pages = c.caches(a[5], a[6], nkv, hd, page_size, &k, &v);
    int code = 0;
    const at::Tensor *qkv = c.ok ? c.rows(a[1], (nh + 2 * nkv) * hd, &code) : nullptr, *turn = c.tensor(a[3]);
    if (!c.ok || !qkv || !turn) return none();
    const long T = (long)qkv->size(0);
    int *positions = c.words(a[2], T), *slots = c.words(a[4], T), *status = c.words(a[12], 1);
    if (!c.ok || turn->scalar_type() != at::kFloat || turn->dim() != 3 || !turn->is_contiguous() || turn->size(1) != rot / 2 || turn->size(2) != 2 ||
        turn->size(0) > 0x7fffffffL)
      return none();
    at::Tensor q = at::empty({T, nh * hd}, qkv->options());
    typedef int (*Fn)(const void*, long, int, const int*, const float*, int, const int*, void*, void*, int, void*, int, int, int, int, int, int*, void*);
    const int rc = ((Fn)address(a[0]))(qkv->data_ptr(), (long)qkv->stride(0), code, positions, (const float*)turn->data_ptr(), (int)turn->size(0), slots, k, v,
                                       (int)pages, q.data_ptr(), (int)T, (int)nh, (int)nkv, (int)rot, (int)page_size, status, c.stream());
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(q);
  });
}

// pages(entry, k_cache, v_cache, pages, head_dim, page_size, dtype code, status) -> (keys, values)
PyObject* pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return none();
  return guarded([&]() -> PyObject* {
    Call c;
    const long hd = c.number(a[4]), page_size = c.number(a[5]), code = c.number(a[6]);
    const at::Tensor* kt = c.tensor(a[1]);
    if (!c.ok || kt->dim() != 4 || code < 0 || code > 1) return none();
    const long nkv = (long)kt->size(1);
    void *k = nullptr, *v = nullptr;
    const long num_pages = c.caches(a[1], a[2], nkv, hd, page_size, &k, &v);
    int *list = c.words(a[3], -1), *status = c.words(a[7], 1);
    if (!c.ok) return none();
    const long m = (long)THPVariable_Unpack(a[3]).numel();
    if (m > 0x7fffffffL) return none();
    at::Tensor both = at::empty({2, m, nkv, page_size, hd}, kt->options().dtype(code ? at::kBFloat16 : at::kFloat));
    at::Tensor ko = both.select(0, 0), vo = both.select(0, 1);
    typedef int (*Fn)(const void*, const void*, int, int, int, const int*, int, void*, void*, int, int*, void*);
    const int rc = ((Fn)address(a[0]))(k, v, (int)num_pages, (int)nkv, (int)page_size, list, (int)m, ko.data_ptr(), vo.data_ptr(), (int)code, status,
                                       c.stream());
    if (rc) return PyLong_FromLong(rc);
    PyObject *x = THPVariable_Wrap(ko), *y = THPVariable_Wrap(vo);
    if (!x || !y) { Py_XDECREF(x); Py_XDECREF(y); return nullptr; }
    PyObject* pair = PyTuple_Pack(2, x, y);
    Py_DECREF(x);
    Py_DECREF(y);
    return pair;
  });
}

// attention(scratch entry, entry, simple entry, q, out, k_cache, v_cache, block_tables, token_req, positions, heads, kv heads, head_dim, page_size, window,
//           scale, cu_q, kv_lens, q_lens, max_kv_len, most rows, status, parts entry): bfloat16 requests of at most `most rows` rows each,
// and float32
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 23) return none();
  return guarded([&]() -> PyObject* {
    Call c;
    const long nh = c.number(a[10]), nkv = c.number(a[11]), hd = c.number(a[12]), page_size = c.number(a[13]);
    const long window = a[14] == Py_None ? 0 : c.number(a[14]), most = c.number(a[20]);
    if (!c.ok || nkv < 1 || nh < 1 || nh % nkv || (a[14] != Py_None && window < 1) || !PyFloat_Check(a[15])) return none();
    void *k = nullptr, *v = nullptr;
    const long pages = c.caches(a[5], a[6], nkv, hd, page_size, &k, &v);
    int code = 0, out_code = 0;
    const at::Tensor *q = c.ok ? c.rows(a[3], nh * hd, &code) : nullptr, *out = c.ok ? c.rows(a[4], nh * hd, &out_code) : nullptr;
    int *table = c.words(a[7], -1), *status = c.words(a[21], 1);
    if (!c.ok || code != out_code || q->size(0) != out->size(0) || q->size(0) < 1) return none();
    const long T = (long)q->size(0);
    const at::Tensor& tt = THPVariable_Unpack(a[7]);
    if (tt.dim() != 2 || tt.size(0) > 0x7fffffffL || tt.size(1) > 0x7fffffffL) return none();
    const float scale = (float)PyFloat_AS_DOUBLE(a[15]);
    // The requests' tokens; rows behind the last one's stay as they are.
    const bool runs = PyList_Check(a[18]);
    const long B = runs ? (long)PyList_GET_SIZE(a[18]) : 0;
    long longest = 0, tokens = 0;
    for (long b = 0; b < B; ++b) {
      const long x = c.number(PyList_GET_ITEM(a[18], b));
      if (x < 0) return none();
      longest = x > longest ? x : longest;
      tokens += x;
    }
    if (!c.ok || tokens > T || (runs ? tokens < 1 : a[18] != Py_None)) return none();
    if (code == 0) {
      int *req = c.words(a[8], T), *pos = c.words(a[9], T);
      const long rows = runs ? tokens : T, longest_kv = a[19] == Py_None ? 0 : c.number(a[19]);
      if (!c.ok || longest_kv < 0) return none();
      typedef int (*Parts)(int, int, int, int);
      const int parts = ((Parts)address(a[22]))((int)rows, (int)nkv, (int)longest_kv, (int)window);
      const long floats = parts > 1 ? rows * nh * parts * (hd + 2) : 0;
      at::Tensor scratch;
      if (floats) scratch = at::empty({floats}, q->options().dtype(at::kFloat));
      typedef int (*Fn)(const void*, long, void*, long, int, const void*, const void*, int, const int*, int, int, const int*, const int*, int, int, int, int, int,
                        float, int, float*, long, int*, void*);
      return PyLong_FromLong(((Fn)address(a[2]))(q->data_ptr(), (long)q->stride(0), out->data_ptr(), (long)out->stride(0), code, k, v, (int)pages, table,
                                                 (int)tt.size(1), (int)tt.size(0), req, pos, (int)rows, (int)nh, (int)nkv, (int)page_size, (int)window, scale, parts,
                                                 floats ? (float*)scratch.data_ptr() : nullptr, floats, status, c.stream()));
    }
    if (!runs || a[16] == Py_None || a[17] == Py_None || a[19] == Py_None) return none();
    const long G = nh / nkv, longest_kv = c.number(a[19]);
    int *cu_q = c.words(a[16], B + 1), *kv_lens = c.words(a[17], B);
    if (!c.ok || B < 1 || B > 65535 || tt.size(0) != B || longest * G > most || longest_kv < 0) return none();
    if (q->stride(0) % 8 || (uintptr_t)q->data_ptr() % 16 || out->stride(0) % 4 || (uintptr_t)out->data_ptr() % 8) return none();
    // The positions that a request's rows see, from a multiple of 16 on: by these the kernel's units are counted.
    const long seen = window > 0 ? std::min(longest_kv, window + longest + 14) : longest_kv;
    typedef long (*Scratch)(int, int, int, int);
    const long floats = ((Scratch)address(a[0]))((int)B, (int)nkv, (int)(longest * G), (int)seen);
    at::Tensor scratch = at::empty({floats}, q->options().dtype(at::kFloat));
    typedef int (*Fn)(const void*, long, void*, long, const void*, const void*, int, const int*, int, const int*, const int*, int, int, int, int, int, float,
                      int, int, float*, long, int*, void*);
    return PyLong_FromLong(((Fn)address(a[1]))(q->data_ptr(), (long)q->stride(0), out->data_ptr(), (long)out->stride(0), k, v, (int)pages, table,
                                               (int)tt.size(1), cu_q, kv_lens, (int)B, (int)nh, (int)nkv, (int)page_size, (int)window, scale,
                                               (int)(longest * G), (int)seen, (float*)scratch.data_ptr(), floats, status, c.stream()));
  });
}

PyMethodDef methods[] = {{"layout", (PyCFunction)(void*)layout, METH_FASTCALL, nullptr},
                         {"write", (PyCFunction)(void*)write, METH_FASTCALL, nullptr},
                         {"pages", (PyCFunction)(void*)pages, METH_FASTCALL, nullptr},
                         {"attention", (PyCFunction)(void*)attention, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "coheryn_calls", nullptr, -1, methods};
}  // namespace

PyMODINIT_FUNC PyInit_coheryn_calls() { return PyModule_Create(&module); }
