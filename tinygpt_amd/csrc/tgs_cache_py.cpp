// tgs_cache_py.cpp -- the Python side's checks of the beam, attention and cache
// calls, in native code: reading shapes, strides, types and addresses of eight
// to twelve tensors from Python took 10 to 16 us a call, more than the small
// calls' kernels (about 5 us).  Each function takes the handle, the device
// index, the raw stream and the tensors in the order of the method of
// tinygpt_amd/cache.py that calls it, raises ValueError or TypeError for
// tensors that do not fit, and returns the C ABI's status.
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <dlfcn.h>
#include <initializer_list>

#include "../../include/tgs_sampler.h"

namespace {

decltype(&tgs_beam_select) p_beam = nullptr;
decltype(&tgs_tree_attention) p_attention = nullptr;
decltype(&tgs_kv_append) p_append = nullptr;
decltype(&tgs_tree_commit) p_commit = nullptr;
decltype(&tgs_kv_fork) p_fork = nullptr;

struct Raised {};  // a Python error is set

[[noreturn]] void bad(const char* fn, const char* msg) {
  PyErr_Format(PyExc_ValueError, "%s: %s", fn, msg);
  throw Raised{};
}
[[noreturn]] void bad_tensor(const char* fn, const char* name, const char* what) {
  PyErr_Format(PyExc_ValueError, "%s: %s must be %s", fn, name, what);
  throw Raised{};
}

typedef std::initializer_list<int64_t> Shape;

struct Call {
  const char* fn;
  tgs_handle h;
  int dev;
  tgs_stream stream;

  Call(const char* f, PyObject* const* args, Py_ssize_t got, Py_ssize_t want) : fn(f) {
    if (got != want) {
      PyErr_Format(PyExc_TypeError, "%s: %zd arguments, %zd expected", f, got, want);
      throw Raised{};
    }
    h = (tgs_handle)PyLong_AsVoidPtr(args[0]);
    dev = (int)number(args[1]);
    stream = (tgs_stream)PyLong_AsVoidPtr(args[2]);
    if (PyErr_Occurred()) throw Raised{};
  }

  long number(PyObject* o) const {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) throw Raised{};
    if (x < INT32_MIN || x > INT32_MAX) bad(fn, "a number beyond 32 bits");
    return x;
  }
  const at::Tensor* maybe(PyObject* o, const char* name) const {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", fn, name);
      throw Raised{};
    }
    return &THPVariable_Unpack(o);
  }
  const at::Tensor& tensor(PyObject* o, const char* name) const {
    const at::Tensor* t = maybe(o, name);
    if (!t) bad_tensor(fn, name, "a tensor");
    return *t;
  }
  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == dev; }
  // Contiguous, of that type and shape, on the handle's device.
  void* exact(const at::Tensor& t, const char* name, at::ScalarType dt, Shape shape) const {
    if (t.scalar_type() != dt || t.sizes() != at::IntArrayRef(shape) || !t.is_contiguous() || !here(t)) {
      char what[160];
      int n = std::snprintf(what, sizeof(what), "a contiguous %s tensor of shape (", dt == at::kInt ? "int32" : dt == at::kFloat ? "float32" : "cache-typed");
      for (int64_t x : shape) n += std::snprintf(what + n, sizeof(what) - n, "%lld, ", (long long)x);
      std::snprintf(what + n - (shape.size() ? 2 : 0), sizeof(what) - n, ") on the handle's device (cuda:%d)", dev);
      bad_tensor(fn, name, what);
    }
    return t.data_ptr();
  }
  int32_t* ints(PyObject* o, const char* name, Shape shape) const {
    return (int32_t*)exact(tensor(o, name), name, at::kInt, shape);
  }
  int32_t* ints_or_null(PyObject* o, const char* name, Shape shape) const {
    const at::Tensor* t = maybe(o, name);
    return t ? (int32_t*)exact(*t, name, at::kInt, shape) : nullptr;
  }
  void apart(const void* out, const char* name, std::initializer_list<const void*> ins) const {
    for (const void* p : ins)
      if (out && p == out) bad_tensor(fn, name, "no input");
  }

  // The cache: keys [layers,] pages, kv_heads, page, D; values [..., page / 8, D, 8].
  at::ScalarType cache(PyObject* ko, PyObject* vo, bool layered, tgs_kv_cache& c) const {
    const at::Tensor &k = tensor(ko, "k"), &v = tensor(vo, "v");
    const int f = layered ? 1 : 0;
    if (k.dim() != 4 + f || v.dim() != 5 + f)
      bad(fn, layered ? "k must be [layers, pages, kv_heads, page, D], v [layers, pages, kv_heads, page / 8, D, 8]"
                      : "k must be [pages, kv_heads, page, D], v [pages, kv_heads, page / 8, D, 8]");
    const auto ks = k.sizes(), vs = v.sizes(), kt = k.strides(), vt = v.strides();
    if (layered && ks[0] != vs[0]) bad(fn, "k and v differ in layers");
    const int64_t N = ks[f], H = ks[f + 1], page = ks[f + 2], D = ks[f + 3];
    if (page % 8 || vs[f] != N || vs[f + 1] != H || vs[f + 2] != page / 8 || vs[f + 3] != D || vs[f + 4] != 8)
      bad(fn, "v must be [..., pages, kv_heads, page / 8, D, 8] for k [..., pages, kv_heads, page, D]");
    if (kt[f + 1] != page * D || kt[f + 2] != D || kt[f + 3] != 1 || vt[f + 1] != page * D || vt[f + 2] != 8 * D ||
        vt[f + 3] != 8 || vt[f + 4] != 1)
      bad(fn, "a page of the cache must be contiguous");
    const at::ScalarType dt = k.scalar_type();
    if ((dt != at::kBFloat16 && dt != at::kHalf) || v.scalar_type() != dt) {
      PyErr_Format(PyExc_TypeError, "%s: the cache must be bfloat16 or float16", fn);
      throw Raised{};
    }
    if (!here(k) || !here(v)) bad(fn, "the cache must be on the handle's device");
    if ((layered && ks[0] > INT32_MAX) || N > INT32_MAX || H > INT32_MAX || page > INT32_MAX || D > INT32_MAX)
      bad(fn, "a cache dimension beyond 32 bits");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.layers = layered ? (int)ks[0] : 1;
    c.k_layer = c.layers > 1 ? kt[0] : 0;
    c.v_layer = c.layers > 1 ? vt[0] : 0;
    c.k_page = kt[f];
    c.v_page = vt[f];
    c.n_pages = (int)N;
    c.kv_heads = (int)H;
    c.page = (int)page;
    c.head_dim = (int)D;
    c.dtype = dt == at::kHalf ? TGS_F16 : TGS_BF16;
    return dt;
  }
  void seqs(PyObject* to, PyObject* lo, tgs_kv_seqs& s) const {
    const at::Tensor& t = tensor(to, "tables");
    if (t.dim() != 2 || t.size(0) > INT32_MAX || t.size(1) > INT32_MAX) bad(fn, "tables must be int32 [sequences, slots]");
    s.B = (int)t.size(0);
    s.width = (int)t.size(1);
    s.tables = (const int32_t*)exact(t, "tables", at::kInt, {s.B, s.width});
    s.lens = ints(lo, "lens", {s.B});
  }
  // Rows [layers,] B, T, heads, D of any strides, D contiguous.
  const at::Tensor& rows(PyObject* o, const char* name, at::ScalarType dt, Shape shape) const {
    const at::Tensor& t = tensor(o, name);
    if (t.scalar_type() != dt || t.sizes() != at::IntArrayRef(shape) || t.strides().back() != 1 || !here(t))
      bad_tensor(fn, name, "of the cache's type and device and of the shape that the other tensors give, its last dimension contiguous");
    return t;
  }
  void new_rows(PyObject* ko, PyObject* vo, at::ScalarType dt, Shape shape, tgs_kv_rows& r) const {
    const at::Tensor &k = rows(ko, "k_new", dt, shape), &v = rows(vo, "v_new", dt, shape);
    const int f = shape.size() == 5 ? 1 : 0;
    const auto a = k.strides(), b = v.strides();
    r.k = k.data_ptr();
    r.v = v.data_ptr();
    r.k_layer = f ? a[0] : 0;
    r.v_layer = f ? b[0] : 0;
    r.k_seq = a[f], r.k_tok = a[f + 1], r.k_head = a[f + 2];
    r.v_seq = b[f], r.v_tok = b[f + 1], r.v_head = b[f + 2];
  }
  int64_t nodes(PyObject* o) const {
    const at::Tensor& t = tensor(o, "k_new");
    if (t.dim() != 5 || t.size(2) > INT32_MAX) bad(fn, "k_new and v_new must be [layers, B, T, kv_heads, D]");
    return t.size(2);
  }
};

template <class F>
PyObject* guarded(F f) {
  try {
    return PyLong_FromLong(f());
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "cache call");
  }
  return nullptr;
}

// handle, device, stream, logits, scores, W, n_out, vocab (-1: all), hist, hist_len, out scores, parents, tokens, hist, hist_len
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("beam_select", a, n, 15);
    const at::Tensor& x = c.tensor(a[3], "logits");
    if (x.dim() != 2 || x.stride(1) != 1 || x.size(0) > INT32_MAX || x.size(1) > INT32_MAX)
      bad(c.fn, "logits must be [G * W, V] with unit stride along V");
    const at::ScalarType dt = x.scalar_type();
    if (dt != at::kFloat && dt != at::kBFloat16) {
      PyErr_SetString(PyExc_TypeError, "beam_select: logits must be float32 or bfloat16");
      throw Raised{};
    }
    const int64_t rows = x.size(0), W = c.number(a[5]), no = c.number(a[6]);
    if (!c.here(x)) bad(c.fn, "logits must be on the handle's device");
    int64_t V = c.number(a[7]);
    if (V < 0) V = x.size(1);
    if (V < 1 || V > x.size(1)) bad(c.fn, "vocab outside the logits' width");
    if (W < 1 || rows % W) bad(c.fn, "logits are not requests of W beams");
    if (no < 0) bad(c.fn, "n_out");
    const int64_t G = rows / W, m = G * no;
    float* scores = (float*)c.exact(c.tensor(a[4], "scores"), "scores", at::kFloat, {rows});
    const at::Tensor* hist = c.maybe(a[8], "hist");
    int64_t H = 0;
    int32_t *hp = nullptr, *lp = nullptr, *ohp = nullptr, *olp = nullptr;
    if ((a[8] == Py_None) != (a[9] == Py_None)) bad(c.fn, "hist and hist_len go together");
    if (hist) {
      if (hist->dim() != 2 || hist->size(1) < 1 || hist->size(1) > INT32_MAX) bad(c.fn, "hist must be int32 [G * W, H]");
      H = hist->size(1);
      hp = c.ints(a[8], "hist", {rows, H});
      lp = c.ints(a[9], "hist_len", {rows});
      ohp = c.ints(a[13], "out hist", {m, H});
      olp = c.ints(a[14], "out hist_len", {m});
      c.apart(ohp, "out hist", {hp, lp});
      c.apart(olp, "out hist_len", {hp, lp});
    }
    float* os = (float*)c.exact(c.tensor(a[10], "out scores"), "out scores", at::kFloat, {m});
    int32_t *op = c.ints(a[11], "out parents", {m}), *ot = c.ints(a[12], "out tokens", {m});
    c.apart(os, "out scores", {scores});
    c.apart(op, "out parents", {hp, lp});
    c.apart(ot, "out tokens", {hp, lp});
    return p_beam(c.h, x.data_ptr(), dt == at::kFloat ? TGS_F32 : TGS_BF16, (int)G, (int)W, (int)V, x.stride(0), scores,
                  (int)no, hp, lp, (int)H, os, op, ot, ohp, olp, c.stream);
  });
}

// handle, device, stream, q, k_new, v_new, k, v, tables, lens, parents, max_len (-1: the tables'), scale (None: 1 / sqrt(D)), out, lse
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("tree_attention", a, n, 15);
    tgs_kv_cache cache;
    tgs_kv_rows rows;
    tgs_kv_seqs seqs;
    tgs_attn t;
    const at::Tensor& q = c.tensor(a[3], "q");
    const at::ScalarType dt = c.cache(a[6], a[7], false, cache);
    c.seqs(a[8], a[9], seqs);
    if (q.dim() != 4 || q.size(1) > INT32_MAX || q.size(2) > INT32_MAX) bad(c.fn, "q must be [B, T, q_heads, D]");
    const int64_t B = seqs.B, T = q.size(1), Hq = q.size(2), H = cache.kv_heads, D = cache.head_dim;
    c.rows(a[3], "q", dt, {B, T, Hq, D});
    if (H == 0 || Hq % H) bad(c.fn, "query heads are no multiple of key heads");
    c.new_rows(a[4], a[5], dt, {B, T, H, D}, rows);
    t.q = q.data_ptr();
    t.q_seq = q.stride(0), t.q_tok = q.stride(1), t.q_head = q.stride(2);
    t.parents = c.ints_or_null(a[10], "parents", {B, T});
    t.T = (int)T;
    t.q_heads = (int)Hq;
    const long most = c.number(a[11]);
    t.max_len = most >= 0 ? (int)most : (int)std::min<int64_t>((int64_t)seqs.width * cache.page, INT32_MAX);
    t.scale = a[12] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)PyFloat_AsDouble(a[12]);
    if (PyErr_Occurred()) throw Raised{};
    t.out = c.exact(c.tensor(a[13], "out"), "out", dt, {B, T, Hq, D});
    const at::Tensor* lse = c.maybe(a[14], "lse");
    t.lse = lse ? (float*)c.exact(*lse, "lse", at::kFloat, {B, T, Hq}) : nullptr;
    c.apart(t.out, "out", {t.q, rows.k, rows.v});
    return p_attention(c.h, &cache, &rows, &seqs, &t, c.stream);
  });
}

// handle, device, stream, k_new, v_new, k, v, tables, lens, counts, lens_out
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("kv_append", a, n, 11);
    tgs_kv_cache cache;
    tgs_kv_rows rows;
    tgs_kv_seqs seqs;
    const at::ScalarType dt = c.cache(a[5], a[6], true, cache);
    c.seqs(a[7], a[8], seqs);
    const int64_t T = c.nodes(a[3]);
    c.new_rows(a[3], a[4], dt, {cache.layers, seqs.B, T, cache.kv_heads, cache.head_dim}, rows);
    int32_t *counts = c.ints_or_null(a[9], "counts", {seqs.B}), *out = c.ints(a[10], "lens_out", {seqs.B});
    c.apart(out, "lens_out", {seqs.lens, seqs.tables, counts});
    return p_append(c.h, &cache, &rows, &seqs, (int)T, counts, out, c.stream);
  });
}

// handle, device, stream, k_new, v_new, k, v, tables, lens, parents, draft, sampled, out n_acc, tokens, path, lens
PyObject* tree_commit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("tree_commit", a, n, 16);
    tgs_kv_cache cache;
    tgs_kv_rows rows;
    tgs_kv_seqs seqs;
    const at::ScalarType dt = c.cache(a[5], a[6], true, cache);
    c.seqs(a[7], a[8], seqs);
    const int64_t B = seqs.B, T = c.nodes(a[3]);
    c.new_rows(a[3], a[4], dt, {cache.layers, B, T, cache.kv_heads, cache.head_dim}, rows);
    int32_t *par = c.ints(a[9], "parents", {B, T}), *draft = c.ints(a[10], "draft", {B, T}),
            *smp = c.ints(a[11], "sampled", {B, T});
    int32_t *acc = c.ints(a[12], "out n_acc", {B}), *tok = c.ints(a[13], "out tokens", {B, T}),
            *path = c.ints(a[14], "out path", {B, T}), *lens = c.ints(a[15], "out lens", {B});
    const char* names[] = {"out n_acc", "out tokens", "out path", "out lens"};
    int32_t* outs[] = {acc, tok, path, lens};
    for (int i = 0; i < 4; i++) c.apart(outs[i], names[i], {seqs.lens, seqs.tables, par, draft, smp});
    return p_commit(c.h, &cache, &rows, &seqs, (int)T, par, draft, smp, acc, tok, path, lens, c.stream);
  });
}

// handle, device, stream, k, v, tables, lens, parents, room, tables_out, lens_out
PyObject* kv_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("kv_fork", a, n, 11);
    tgs_kv_cache cache;
    tgs_kv_seqs seqs;
    c.cache(a[3], a[4], true, cache);
    c.seqs(a[5], a[6], seqs);
    int32_t* par = c.ints(a[7], "parents", {seqs.B});
    int32_t *tab = c.ints(a[9], "tables_out", {seqs.B, seqs.width}), *lens = c.ints(a[10], "lens_out", {seqs.B});
    c.apart(tab, "tables_out", {seqs.lens, seqs.tables, par});
    c.apart(lens, "lens_out", {seqs.lens, seqs.tables, par});
    return p_fork(c.h, &cache, &seqs, par, (int)c.number(a[8]), tab, lens, c.stream);
  });
}

// The library whose entry points the calls go to.
PyObject* bind(PyObject*, PyObject* path) {
  const char* p = PyUnicode_AsUTF8(path);
  if (!p) return nullptr;
  void* lib = dlopen(p, RTLD_NOW | RTLD_LOCAL);
  if (!lib) {
    PyErr_SetString(PyExc_RuntimeError, dlerror());
    return nullptr;
  }
  p_beam = (decltype(p_beam))dlsym(lib, "tgs_beam_select");
  p_attention = (decltype(p_attention))dlsym(lib, "tgs_tree_attention");
  p_append = (decltype(p_append))dlsym(lib, "tgs_kv_append");
  p_commit = (decltype(p_commit))dlsym(lib, "tgs_tree_commit");
  p_fork = (decltype(p_fork))dlsym(lib, "tgs_kv_fork");
  if (!p_beam || !p_attention || !p_append || !p_commit || !p_fork) {
    PyErr_Format(PyExc_RuntimeError, "%s lacks an entry point: build it again", p);
    return nullptr;
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    {"beam_select", (PyCFunction)(void (*)(void))beam_select, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
    {"kv_append", (PyCFunction)(void (*)(void))kv_append, METH_FASTCALL, nullptr},
    {"tree_commit", (PyCFunction)(void (*)(void))tree_commit, METH_FASTCALL, nullptr},
    {"kv_fork", (PyCFunction)(void (*)(void))kv_fork, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cache_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cache_calls(void) { return PyModule_Create(&module); }
