// The short way from Python to the library for calls whose kernels are shorter than their checks in Python: it takes what a
// step passes (tensors that the Python checks would pass too) and answers -1 to everything else, which those checks then get.
// No entry point of its own: the library's are given by address, so that both ways run the same ones.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../include/fdllm.h"

namespace {

struct Spec {
  fdllm_ctx* ctx;
  decltype(&fdllm_rotate_heads) rotate;
  decltype(&fdllm_paged4_append) append;
  decltype(&fdllm_paged4_read) read;
  decltype(&fdllm_paged_attn_workspace) workspace[2];  // over 8-bit pages, over 4-bit ones
  void* attn[2];                                       // fdllm_paged_attn, fdllm_paged4_attn
  int nq, nkv, index;
  at::ScalarType dtype;
};
constexpr int HD = 128;
constexpr const char* NAME = "fdllm.spec";

// other threads run meanwhile (a launch may wait for room in its queue)
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
// an argument that may be None, or no tensor of the call's device
struct Arg {
  const at::Tensor* t = nullptr;
  bool none = false, ok = false;
  Arg(PyObject* o, int index) {
    if (o == Py_None) {
      none = ok = true;
    } else if (THPVariable_Check(o)) {
      t = &THPVariable_Unpack(o);
      ok = t->is_cuda() && t->get_device() == index;
    }
  }
};
struct Rows { void* p = nullptr; int64_t n = 0, ld = 0; };
// [rows, heads, 128] of the model's dtype, heads contiguous; rows < 0: any number but 0
bool head_rows(const Arg& a, const Spec& s, int heads, int64_t rows, Rows& out) {
  if (!a.ok || a.none || a.t->dim() != 3 || a.t->scalar_type() != s.dtype) return false;
  const auto size = a.t->sizes(), stride = a.t->strides();
  if (size[0] < 1 || (rows >= 0 && size[0] != rows) || size[1] != heads || size[2] != HD || stride[2] != 1 || (heads > 1 && stride[1] != HD))
    return false;
  out = Rows{a.t->data_ptr(), size[0], size[0] > 1 ? stride[0] : (int64_t)heads * HD};  // (a single row has no stride)
  return true;
}
// a contiguous vector; none where it may be
bool vector(const Arg& a, at::ScalarType type, int64_t n, bool may_be_none, void*& out) {
  out = nullptr;
  if (!a.ok) return false;
  if (a.none) return may_be_none;
  if (a.t->dim() != 1 || a.t->scalar_type() != type || a.t->size(0) != n || !a.t->is_contiguous()) return false;
  out = a.t->data_ptr();
  return true;
}
bool whole(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0;
}
bool address(PyObject* o, const void*& p) {
  int64_t v = 0;
  if (o != Py_None && !whole(o, v)) return false;
  p = reinterpret_cast<const void*>((uintptr_t)v);
  return true;
}
// a page table and the rows of its sequences
struct Sequences { int32_t *table = nullptr, *start = nullptr, *row_start = nullptr; int64_t nseq = 0, width = 0, ld = 0, max_rows = 0; };
bool sequences(const Spec& s, int64_t rows, PyObject* table, PyObject* start, PyObject* row_start, PyObject* max_rows, Sequences& q) {
  const Arg t(table, s.index);
  if (!t.ok || t.none || t.t->dim() != 2 || t.t->scalar_type() != at::kInt || t.t->size(0) < 1 || t.t->size(1) < 1 || t.t->stride(1) != 1)
    return false;
  q.table = (int32_t*)t.t->data_ptr();
  q.nseq = t.t->size(0);
  q.width = t.t->size(1);
  q.ld = t.t->stride(0);
  void *a = nullptr, *b = nullptr;
  if (!vector(Arg(start, s.index), at::kInt, q.nseq, false, a) || !vector(Arg(row_start, s.index), at::kInt, q.nseq + 1, true, b)) return false;
  q.start = (int32_t*)a;
  q.row_start = (int32_t*)b;
  int64_t most = -1;
  if (max_rows != Py_None && (!whole(max_rows, most) || most < 0)) return false;
  if (b == nullptr) {
    if (rows % q.nseq || (most >= 0 && (most > rows || most * q.nseq != rows))) return false;
    q.max_rows = rows / q.nseq;
  } else {
    q.max_rows = most < 0 || most > rows ? rows : most;
  }
  return q.nseq <= INT32_MAX && q.width <= INT32_MAX;
}

PyObject* make_spec(PyObject*, PyObject* args) {
  unsigned long long ctx, rotate, append, read, ws8, attn8, ws4, attn4;
  int nq, nkv, half, index;
  if (!PyArg_ParseTuple(args, "K(KKKKKKK)iiii", &ctx, &rotate, &append, &read, &ws8, &attn8, &ws4, &attn4, &nq, &nkv, &half, &index))
    return nullptr;
  using Workspace = decltype(&fdllm_paged_attn_workspace);
  auto* s = new (std::nothrow) Spec{(fdllm_ctx*)ctx, (decltype(&fdllm_rotate_heads))rotate, (decltype(&fdllm_paged4_append))append,
                                    (decltype(&fdllm_paged4_read))read, {(Workspace)ws8, (Workspace)ws4}, {(void*)attn8, (void*)attn4},
                                    nq, nkv, index, half ? at::kHalf : at::kBFloat16};
  if (s == nullptr) return PyErr_NoMemory();
  PyObject* c = PyCapsule_New(s, NAME, [](PyObject* o) { delete (Spec*)PyCapsule_GetPointer(o, NAME); });
  if (c == nullptr) delete s;
  return c;
}

// runs `call(spec, stream, args)` for n arguments behind the spec and the stream; -1 where it throws
template <class F>
PyObject* with_spec(PyObject* const* args, Py_ssize_t nargs, Py_ssize_t n, F call) {
  if (nargs != n + 2) return PyErr_Format(PyExc_TypeError, "%zd arguments, got %zd", n + 2, nargs);
  auto* s = (const Spec*)PyCapsule_GetPointer(args[0], NAME);
  if (s == nullptr) return nullptr;
  int rc = -1;
  try {
    const void* stream = nullptr;
    if (address(args[1], stream)) rc = call(*s, const_cast<void*>(stream), args + 2);
  } catch (...) {
    rc = -1;
  }
  if (PyErr_Occurred()) return nullptr;
  return PyLong_FromLong(rc);
}

// one of queries and keys, its result and its norm: the three of them, or none; rows: as head_rows takes them
bool side(const Spec& s, PyObject* x, PyObject* out, PyObject* norm, int heads, int64_t rows, Rows& in, Rows& to, void*& w) {
  const Arg a(x, s.index), b(out, s.index);
  if (!vector(Arg(norm, s.index), s.dtype, HD, true, w)) return false;
  if (a.none) return b.none && w == nullptr;
  return head_rows(a, s, heads, rows, in) && head_rows(b, s, heads, in.n, to);
}

// q, k, pos, rotary, q_norm, k_norm, q_out, k_out
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return with_spec(args, nargs, 8, [](const Spec& s, void* stream, PyObject* const* a) {
    Rows q, k, qo, ko;
    void *pos = nullptr, *qn, *kn;
    int64_t first = 0;
    const void* rotary;
    if (!side(s, a[0], a[6], a[4], s.nq, -1, q, qo, qn) || !side(s, a[1], a[7], a[5], s.nkv, q.p ? q.n : -1, k, ko, kn)) return -1;
    const int64_t n = q.p ? q.n : k.n;  // (0: neither)
    if (n < 1 || n > INT32_MAX || !address(a[3], rotary)) return -1;
    if (PyLong_CheckExact(a[2]) ? !whole(a[2], first) || first < INT32_MIN || first > INT32_MAX
                                : !vector(Arg(a[2], s.index), at::kInt, n, false, pos))
      return -1;
    const Unlocked unlocked;
    return s.rotate(s.ctx, q.p, q.ld, k.p, k.ld, (int)n, (const int32_t*)pos, first, (const fdllm_rotary*)rotary, qn, kn, qo.p, qo.ld, ko.p,
                    ko.ld, stream);
  });
}

// k, v, cache, layer, page_table, start, pos, q, q_out, rotary, q_norm, k_norm, row_start, max_rows
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return with_spec(args, nargs, 14, [](const Spec& s, void* stream, PyObject* const* a) {
    Rows k, v, q, qo;
    void *pos, *qn, *kn;
    const void *cache, *rotary;
    int64_t layer;
    Sequences seq;
    if (!head_rows(Arg(a[0], s.index), s, s.nkv, -1, k) || !head_rows(Arg(a[1], s.index), s, s.nkv, k.n, v) || k.n > INT32_MAX ||
        !address(a[2], cache) || !whole(a[3], layer) || layer < 0 || layer > INT32_MAX ||
        !sequences(s, k.n, a[4], a[5], a[12], a[13], seq) || !vector(Arg(a[6], s.index), at::kInt, seq.nseq, true, pos) ||
        !side(s, a[7], a[8], a[10], s.nq, k.n, q, qo, qn) || (qo.p && qo.ld != (int64_t)s.nq * HD) || !address(a[9], rotary) ||
        !vector(Arg(a[11], s.index), s.dtype, HD, true, kn))
      return -1;
    const Unlocked unlocked;
    return s.append(s.ctx, q.p, q.ld, k.p, k.ld, v.p, v.ld, (int)k.n, seq.row_start, (int)seq.nseq, (int)seq.max_rows,
                    (const fdllm_paged4_cache*)cache, (int)layer, seq.table, (int)seq.width, seq.ld, seq.start, (const int32_t*)pos,
                    (const fdllm_rotary*)rotary, qn, kn, qo.p, stream);
  });
}

// cache, layer, page_table, start, rows, k_out, v_out, row_start, max_rows
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return with_spec(args, nargs, 9, [](const Spec& s, void* stream, PyObject* const* a) {
    Rows k, v;
    const void* cache;
    int64_t layer, rows;
    Sequences seq;
    if (!address(a[0], cache) || !whole(a[1], layer) || layer < 0 || layer > INT32_MAX || !whole(a[4], rows) || rows < 1 || rows > INT32_MAX ||
        !sequences(s, rows, a[2], a[3], a[7], a[8], seq) || !head_rows(Arg(a[5], s.index), s, s.nkv, rows, k) ||
        !head_rows(Arg(a[6], s.index), s, s.nkv, rows, v))
      return -1;
    const Unlocked unlocked;
    return s.read(s.ctx, (const fdllm_paged4_cache*)cache, (int)layer, seq.table, (int)seq.width, seq.ld, seq.start, (int)rows,
                  seq.row_start, (int)seq.nseq, (int)seq.max_rows, k.p, k.ld, v.p, v.ld, stream);
  });
}

// kind (0: 8-bit pages, 1: 4-bit ones), cache, layer, page_size, q, page_table, kv_len, mask_block, max_len, out, row_start, max_rows
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return with_spec(args, nargs, 12, [](const Spec& s, void* stream, PyObject* const* a) {
    Rows q, o;
    const void* cache;
    int64_t kind, layer, page, mask, most = 0;
    Sequences seq;
    if (!whole(a[0], kind) || kind < 0 || kind > 1 || !address(a[1], cache) || !whole(a[2], layer) || layer < 0 || layer > INT32_MAX ||
        !whole(a[3], page) || page < 1 || page > INT32_MAX || !head_rows(Arg(a[4], s.index), s, s.nq, -1, q) || q.n > INT32_MAX ||
        !sequences(s, q.n, a[5], a[6], a[10], a[11], seq) || !whole(a[7], mask) || mask < 0 || mask > INT32_MAX ||
        (a[8] != Py_None && (!whole(a[8], most) || most < 0)) || !head_rows(Arg(a[9], s.index), s, s.nq, q.n, o) || o.ld != (int64_t)s.nq * HD)
      return -1;
    const Unlocked unlocked;
    const size_t need = s.workspace[kind](s.ctx, (int)q.n, (int)seq.nseq, (int)seq.max_rows, (int)page, (int)seq.width, most);
    at::Tensor ws;  // of this call's own: the allocator gives it to none before what the stream has of it has run
    if (need) ws = at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(at::Device(at::kCUDA, (at::DeviceIndex)s.index)));
    auto run = [&](auto fn) {
      return fn(s.ctx, q.p, q.ld, (int)q.n, seq.row_start, (int)seq.nseq, (int)seq.max_rows, cache, (int)layer, seq.table,
                (int)seq.width, seq.ld, seq.start, most, (int)mask, o.p, need ? ws.data_ptr() : nullptr, need, stream);
    };
    using Attn = int (*)(fdllm_ctx*, const void*, int64_t, int, const int32_t*, int, int, const void*, int, const int32_t*, int, int64_t,
                         const int32_t*, int64_t, int, void*, void*, size_t, void*);
    return run((Attn)s.attn[kind]);
  });
}

PyMethodDef methods[] = {
    {"make_spec", make_spec, METH_VARARGS, "(ctx, the entry points' addresses, nq, nkv, half, device) -> what the other calls take first"},
    {"rotate", (PyCFunction)(void (*)(void))rotate, METH_FASTCALL, "fdllm_rotate_heads; -1: not a call for the short way"},
    {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, "fdllm_paged4_append; -1: not a call for the short way"},
    {"read", (PyCFunction)(void (*)(void))read, METH_FASTCALL, "fdllm_paged4_read; -1: not a call for the short way"},
    {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, "fdllm_paged_attn, fdllm_paged4_attn; -1: not a call for the short way"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fdllm_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `torch` and `python` say what it was compiled against, whose layouts of tensors and objects it holds: it is not to be called
// under another
PyMODINIT_FUNC PyInit_fdllm_calls() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddStringConstant(m, "torch", FDLLM_TORCH) != 0 || PyModule_AddIntConstant(m, "python", PY_VERSION_HEX) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
