// The kernel modules' ordinary calls, from torch tensors to the C entry points, without Python in between.
//
// prompt_b200, accept_b200 and pages_b200 first ask these functions.  Each looks whether everything is as it ordinarily is
// (plain CUDA tensors on the current device, right types, shapes and layouts), allocates what the call returns, calls the C
// entry point on torch's current stream and returns the result; where anything is not, or the entry point refuses, it
// returns None having done nothing, and the module goes on with its own checks, which name what is wrong.  Why this
// exists: the checks, allocations and argument conversions of a call took 10 to 12 us in Python, twice what its kernels
// take when the call is small (acceptance of a chain: 14 us a call, of which 6.6 on the device).
//
// Scratch comes from torch's caching allocator for the call alone: it follows the stream, and a captured graph has its own.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/vmk_b200.h"

namespace {

struct Entries {
  decltype(&vmk_prompt_workspace_bytes) prompt_ws;
  decltype(&vmk_prompt) prompt;
  decltype(&vmk_prompt_paged) prompt_paged;
  decltype(&vmk_accept) accept;
  decltype(&vmk_pages_workspace_bytes) pages_ws;
  decltype(&vmk_pages_reserve) reserve;
  decltype(&vmk_pages_append_granted) append;
  decltype(&vmk_pages_fork) fork;
  decltype(&vmk_pages_compact_granted) compact;
  decltype(&vmk_pages_free) free;
  decltype(&vmk_pages_copy) copy;
} g_entry = {};
constexpr int kEntries = sizeof(Entries) / sizeof(void*);
bool g_ready = false;                          // entry points known, and a status word: a device is there
int32_t* g_status[64] = {nullptr};             // status word of each device, once the Python side has made it

struct Call {
  int dev;
  void* stream;
  int32_t* status;
};

// False: not a call for this file.
bool begin(Call& c) {
  if (!g_ready) return false;
  c.dev = c10::cuda::current_device();
  if (c.dev < 0 || c.dev >= 64 || g_status[c.dev] == nullptr) return false;
  c.status = g_status[c.dev];
  c.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c.dev).stream();
  return true;
}

const at::Tensor* tensor(PyObject* o, const Call& c) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.device().index() == c.dev && t.layout() == at::kStrided ? &t : nullptr;
}

// A contiguous int32 tensor of `dims` axes (and, where they are not negative, these lengths).
const at::Tensor* ints(PyObject* o, const Call& c, int dims, int64_t n0 = -1, int64_t n1 = -1) {
  const at::Tensor* t = tensor(o, c);
  if (t == nullptr || t->scalar_type() != at::kInt || t->dim() != dims || !t->is_contiguous()) return nullptr;
  if ((n0 >= 0 && t->size(0) != n0) || (n1 >= 0 && t->size(1) != n1)) return nullptr;
  return t;
}

int32_t* ip(const at::Tensor* t) { return static_cast<int32_t*>(t->data_ptr()); }
bool fits(int64_t n) { return n <= 0x7fffffff; }

at::Tensor empty(at::IntArrayRef sizes, const at::TensorOptions& o) {
  at::AutoDispatchBelowADInplaceOrView guard;
  return at::empty(sizes, o);
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return empty({(int64_t)(bytes < 256 ? 256 : bytes)}, like.options().dtype(at::kByte));
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* yes() { Py_RETURN_TRUE; }

// Any C++ exception (an allocation that fails, say) becomes the Python one that torch makes of it.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

bool half(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// prompt(q, k, v, cu_q, cu_k or None, causal)
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    if (n != 6 || !begin(c)) return none();
    const at::Tensor *q = tensor(a[0], c), *k = tensor(a[1], c), *v = tensor(a[2], c), *cu_q = ints(a[3], c, 1);
    if (!q || !k || !v || !cu_q || cu_q->size(0) < 1 || !half(*q) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type()) return none();
    if (q->dim() != 3 || k->dim() != 3 || !q->is_contiguous() || !k->is_contiguous() || !v->is_contiguous() || v->sizes() != k->sizes()) return none();
    const at::Tensor* cu_k = a[4] == Py_None ? cu_q : ints(a[4], c, 1, cu_q->size(0));
    const int64_t Tq = q->size(0), Hq = q->size(1), D = q->size(2), Tk = k->size(0), Hkv = k->size(1), S = cu_q->size(0) - 1;
    if (!cu_k || k->size(2) != D || !fits(Tq) || !fits(Tk) || !fits(S) || !fits(Hq) || !fits(Hkv) || !aligned(*q) || !aligned(*k) || !aligned(*v)) return none();
    const int causal = PyObject_IsTrue(a[5]);
    const size_t bytes = g_entry.prompt_ws((int)S, (int)Tq, Tk, (int)Hq, (int)Hkv, (int)D);
    if (causal < 0 || bytes == 0) { PyErr_Clear(); return none(); }
    at::Tensor out = empty(q->sizes(), q->options()), ws = scratch(bytes, *q);
    const int rc = g_entry.prompt(q->data_ptr(), k->data_ptr(), v->data_ptr(), ip(cu_q), ip(cu_k), nullptr, out.data_ptr(), (int)S, (int)Tq, (int)Tk,
                                  (int)Hq, (int)Hkv, (int)D, causal, q->scalar_type() == at::kBFloat16, ws.data_ptr(), (size_t)ws.numel(), c.status, c.stream);
    return rc == VMK_OK ? THPVariable_Wrap(std::move(out)) : none();
  });
}

// prompt_paged(q, k_pages, v_pages, page_table, cu_q, lens, causal)
PyObject* prompt_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    if (n != 7 || !begin(c)) return none();
    const at::Tensor *q = tensor(a[0], c), *k = tensor(a[1], c), *v = tensor(a[2], c), *cu_q = ints(a[4], c, 1);
    if (!q || !k || !v || !cu_q || cu_q->size(0) < 1 || !half(*q) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type()) return none();
    if (q->dim() != 3 || k->dim() != 4 || !q->is_contiguous() || !k->is_contiguous() || !v->is_contiguous() || v->sizes() != k->sizes()) return none();
    const int64_t Tq = q->size(0), Hq = q->size(1), D = q->size(2), pages = k->size(0), Hkv = k->size(1), ps = k->size(2), S = cu_q->size(0) - 1;
    const at::Tensor *table = ints(a[3], c, 2, S), *lens = ints(a[5], c, 1, S);
    if (!table || !lens || k->size(3) != D || ps == 0 || ps % 64 != 0 || !fits(Tq) || !fits(pages) || !fits(ps) || !fits(S) || !fits(Hq) || !fits(Hkv) ||
        !fits(table->size(1)) || !aligned(*q) || !aligned(*k) || !aligned(*v))
      return none();
    const int causal = PyObject_IsTrue(a[6]);
    const size_t bytes = g_entry.prompt_ws((int)S, (int)Tq, table->size(1) * ps, (int)Hq, (int)Hkv, (int)D);
    if (causal < 0 || bytes == 0) { PyErr_Clear(); return none(); }
    at::Tensor out = empty(q->sizes(), q->options()), ws = scratch(bytes, *q);
    const int rc = g_entry.prompt_paged(q->data_ptr(), k->data_ptr(), v->data_ptr(), ip(table), (int)pages, (int)ps, (int)table->size(1), ip(cu_q), ip(lens),
                                        nullptr, out.data_ptr(), (int)S, (int)Tq, (int)Hq, (int)Hkv, (int)D, causal, q->scalar_type() == at::kBFloat16,
                                        ws.data_ptr(), (size_t)ws.numel(), c.status, c.stream);
    return rc == VMK_OK ? THPVariable_Wrap(std::move(out)) : none();
  });
}

// accept(target_probs, tokens, bits, u, draft_probs or None)
PyObject* accept(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    if (n != 5 || !begin(c)) return none();
    const at::Tensor *p = tensor(a[0], c), *q = nullptr, *u = tensor(a[3], c);
    if (!p || p->dim() != 3 || !p->is_contiguous()) return none();
    const int64_t B = p->size(0), kd = p->size(1), V = p->size(2);
    const int dtype = p->scalar_type() == at::kFloat ? 0 : p->scalar_type() == at::kHalf ? 1 : p->scalar_type() == at::kBFloat16 ? 2 : -1;
    if (dtype < 0 || !fits(B) || !fits(kd) || !fits(V)) return none();
    if (a[4] != Py_None) {
      q = tensor(a[4], c);
      if (!q || q->scalar_type() != p->scalar_type() || q->sizes() != p->sizes() || !q->is_contiguous()) return none();
    }
    const at::Tensor *tokens = ints(a[1], c, 2, B, kd), *bits = ints(a[2], c, 2, B, kd);
    int words = 1;
    if (!bits) {
      bits = ints(a[2], c, 3, B, kd);
      if (!bits || !fits(bits->size(2))) return none();
      words = (int)bits->size(2);
    }
    if (!tokens || !u || u->scalar_type() != at::kFloat || u->dim() != 2 || u->size(0) != B || u->size(1) != kd || !u->is_contiguous()) return none();
    at::Tensor path = empty({B, kd}, tokens->options()), count = empty({B}, tokens->options()), next = empty({B}, tokens->options());
    const int rc = g_entry.accept(p->data_ptr(), q ? q->data_ptr() : nullptr, ip(tokens), reinterpret_cast<const uint32_t*>(ip(bits)), words,
                                  static_cast<const float*>(u->data_ptr()), ip(&path), ip(&count), ip(&next), (int)B, (int)kd, (int)V, dtype, c.status, c.stream);
    if (rc != VMK_OK) return none();
    PyObject* r = PyTuple_New(3);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(path)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(count)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(next)));
    return r;
  });
}

struct State {
  const at::Tensor *table, *lens, *refs;
  int R, T;
};

bool state(State& s, const Call& c, PyObject* table, PyObject* lens, PyObject* refs) {
  s.table = ints(table, c, 2);
  if (!s.table || !fits(s.table->size(0)) || !fits(s.table->size(1))) return false;
  s.R = (int)s.table->size(0);
  s.T = (int)s.table->size(1);
  s.lens = ints(lens, c, 1, s.R);
  s.refs = refs != nullptr ? ints(refs, c, 1) : nullptr;
  return s.lens && (refs == nullptr || (s.refs && fits(s.refs->size(0))));
}

bool whole(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0 && v > 0 && fits(v);
}

struct Pools {
  int64_t d[8 * 4];
  int n = 0;
  int64_t pages = 0, page_size = 0;
};

bool pool(Pools& p, const at::Tensor* t) {
  if (!t || p.n == 8 || t->dim() < 3 || t->dim() > 5 || !t->is_contiguous() || t->numel() == 0) return false;
  const int at = t->dim() == 5;
  const int64_t pages = t->size(at), ps = t->size(-2), row = t->size(-1) * (int64_t)t->element_size();
  if (row % 16 != 0 || !fits(pages) || !fits(ps) || (p.n > 0 && (pages != p.pages || ps != p.page_size))) return false;
  p.pages = pages;
  p.page_size = ps;
  int64_t* d = p.d + 4 * p.n++;
  d[0] = reinterpret_cast<int64_t>(t->data_ptr());
  d[1] = at ? t->size(0) : 1;
  d[2] = t->dim() > 3 ? t->size(-3) : 1;
  d[3] = row;
  return true;
}

bool pools(Pools& p, const Call& c, PyObject* o) {
  const bool list = PyList_CheckExact(o), tuple = PyTuple_CheckExact(o);
  if (!list && !tuple) return false;
  const Py_ssize_t n = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
  if (n < 1 || n > 8) return false;
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!pool(p, tensor(list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i), c))) return false;
  return true;
}

// reserve(page_table, lens, refs, extra, page_size)
PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    State s;
    int64_t ps;
    if (n != 5 || !begin(c) || !state(s, c, a[0], a[1], a[2]) || !whole(a[4], ps)) return none();
    const at::Tensor* extra = ints(a[3], c, 1, s.R);
    const int64_t pages = s.refs->size(0);
    if (!extra) return none();
    at::Tensor granted = empty({s.R}, s.lens->options()), ws = scratch(g_entry.pages_ws(s.R, 0, (int)pages), *s.lens);
    const int rc = g_entry.reserve(ip(s.table), s.R, s.T, ip(s.lens), ip(s.refs), (int)pages, (int)ps, ip(extra), ip(&granted), ws.data_ptr(),
                                   (size_t)ws.numel(), c.status, c.stream);
    return rc == VMK_OK ? THPVariable_Wrap(std::move(granted)) : none();
  });
}

// An int32 tensor of n entries or None: false if it is neither.
bool ints_or_none(int32_t*& p, const Call& c, PyObject* o, int64_t n) {
  p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = ints(o, c, 1, n);
  if (t) p = ip(t);
  return t != nullptr;
}

// append(k, v, k_pages, v_pages, page_table, cu, lens, granted=None, refs=None)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    State s;
    Pools p;
    int32_t *granted, *refs;
    if (n < 7 || n > 9 || !begin(c) || !state(s, c, a[4], a[6], nullptr) || !ints_or_none(granted, c, n > 7 ? a[7] : Py_None, s.R)) return none();
    const at::Tensor* cu = ints(a[5], c, 1);
    if (!cu || cu->size(0) < 1 || cu->size(0) - 1 > s.R) return none();
    int64_t src[6], tokens = -1;
    for (int i = 0; i < 2; ++i) {
      const at::Tensor *t = tensor(a[i], c), *into = tensor(a[2 + i], c);
      if (!t || !into || into->dim() > 4 || !pool(p, into) || t->scalar_type() != into->scalar_type() || t->dim() != 3) return none();
      if (i == 0) tokens = t->size(0);
      if (t->size(0) != tokens || t->size(1) != (into->dim() == 4 ? into->size(1) : 1) || t->size(2) != into->size(-1) || tokens == 0 || !fits(tokens)) return none();
      const int64_t e = (int64_t)t->element_size(), by_token = tokens > 1 ? t->stride(0) * e : 0, by_head = t->size(1) > 1 ? t->stride(1) * e : 0;
      if (t->stride(2) != 1 || !aligned(*t) || by_token < 0 || by_head < 0 || by_token % 16 != 0 || by_head % 16 != 0) return none();
      src[3 * i] = reinterpret_cast<int64_t>(t->data_ptr());
      src[3 * i + 1] = by_token;
      src[3 * i + 2] = by_head;
    }
    if (!ints_or_none(refs, c, n > 8 ? a[8] : Py_None, p.pages)) return none();
    const int rc = g_entry.append(p.d, src, (int)p.pages, (int)p.page_size, ip(s.table), s.T, ip(cu), ip(s.lens), refs, granted, (int)cu->size(0) - 1, (int)tokens,
                                  c.status, c.stream);
    return rc == VMK_OK ? yes() : none();
  });
}

// fork(pools, page_table, lens, refs, parents, children)
PyObject* fork_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    State s;
    Pools p;
    if (n != 6 || !begin(c) || !state(s, c, a[1], a[2], a[3]) || !pools(p, c, a[0]) || s.refs->size(0) != p.pages) return none();
    const at::Tensor* par = ints(a[4], c, 1);
    const at::Tensor* ch = par ? ints(a[5], c, 1, par->size(0)) : nullptr;
    if (!ch || !fits(par->size(0))) return none();
    at::Tensor ws = scratch(g_entry.pages_ws(s.R, (int)par->size(0), 0), *s.lens);
    const int rc = g_entry.fork(p.d, p.n, ip(s.table), s.R, s.T, ip(s.lens), ip(s.refs), (int)p.pages, (int)p.page_size, ip(par), ip(ch), (int)par->size(0),
                                ws.data_ptr(), (size_t)ws.numel(), c.status, c.stream);
    return rc == VMK_OK ? yes() : none();
  });
}

// compact(pools, page_table, lens, refs, path, count, granted=None)
PyObject* compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    State s;
    Pools p;
    int32_t* granted;
    if ((n != 6 && n != 7) || !begin(c) || !state(s, c, a[1], a[2], a[3]) || !pools(p, c, a[0]) || s.refs->size(0) != p.pages || !ints_or_none(granted, c, n == 7 ? a[6] : Py_None, s.R))
      return none();
    const at::Tensor *path = ints(a[4], c, 2, s.R), *count = ints(a[5], c, 1, s.R);
    if (!path || !count || !fits(path->size(1))) return none();
    const int rc = g_entry.compact(p.d, p.n, ip(s.table), s.R, s.T, ip(s.lens), ip(s.refs), (int)p.pages, (int)p.page_size, ip(path), ip(count),
                                   granted, (int)path->size(1), c.status, c.stream);
    return rc == VMK_OK ? yes() : none();
  });
}

// free(page_table, lens, refs, keep, page_size)
PyObject* free_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    State s;
    int64_t ps;
    if (n != 5 || !begin(c) || !state(s, c, a[0], a[1], a[2]) || !whole(a[4], ps)) return none();
    const at::Tensor* keep = ints(a[3], c, 1, s.R);
    if (!keep) return none();
    const int rc = g_entry.free(ip(s.table), s.R, s.T, ip(s.lens), ip(s.refs), (int)s.refs->size(0), (int)ps, ip(keep), c.status, c.stream);
    return rc == VMK_OK ? yes() : none();
  });
}

// copy(pools, src, dst)
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c;
    Pools p;
    if (n != 3 || !begin(c) || !pools(p, c, a[0])) return none();
    const at::Tensor* src = ints(a[1], c, 1);
    const at::Tensor* dst = src ? ints(a[2], c, 1, src->size(0)) : nullptr;
    if (!dst || !fits(src->size(0))) return none();
    const int rc = g_entry.copy(p.d, p.n, (int)p.pages, (int)p.page_size, ip(src), ip(dst), (int)src->size(0), c.status, c.stream);
    return rc == VMK_OK ? yes() : none();
  });
}

// init(addresses of the C entry points, in the order of Entries)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != kEntries) {
    PyErr_SetString(PyExc_ValueError, "init: wrong number of entry points");
    return nullptr;
  }
  void* p[kEntries];
  for (Py_ssize_t i = 0; i < n; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "init: null entry point");
      return nullptr;
    }
  }
  memcpy(&g_entry, p, sizeof(p));
  Py_RETURN_NONE;
}

// set_status(device, address of its status word)
PyObject* set_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const long dev = n == 2 ? PyLong_AsLong(a[0]) : -1;
  void* p = n == 2 ? PyLong_AsVoidPtr(a[1]) : nullptr;
  if (PyErr_Occurred()) return nullptr;
  if (dev >= 0 && dev < 64) g_status[dev] = static_cast<int32_t*>(p);
  g_ready = g_entry.copy != nullptr;
  Py_RETURN_NONE;
}

#define VMK_FN(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {VMK_FN("prompt", prompt),   VMK_FN("prompt_paged", prompt_paged), VMK_FN("accept", accept),     VMK_FN("reserve", reserve),
                           VMK_FN("append", append),   VMK_FN("fork", fork_rows),            VMK_FN("compact", compact),   VMK_FN("free", free_pages),
                           VMK_FN("copy", copy),       VMK_FN("init", init),                 VMK_FN("set_status", set_status), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_vmk_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__vmk_torch() { return PyModule_Create(&g_module); }
