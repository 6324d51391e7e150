// binding.cpp — the attention operators' arguments from torch tensors.  A decode step makes several of these calls per
// layer and the kernels behind them take a few microseconds; with the tensors looked at and packed in Python, calls of
// one token's rotation followed each other after 8.3 us, with this after 2.6 (a decode step's write and read back: 12.1
// and 5.7, nearly the launches' own time).  The entry points come from the library that ctypes has loaded (`entries`), so there is one
// copy of it in the process.  What a call cannot take is a ValueError before anything is launched; the library's own
// checks answer with their status.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <stdexcept>
#include <string>

#include "../../include/moestream_cuda.h"

namespace {

struct Entries {
  decltype(&ms_qk_norm_rope) rope;
  decltype(&ms_prompt_attention) prompt;
  decltype(&ms_kv4_write) write;
  decltype(&ms_kv4_read) read;
  decltype(&ms_kv4_attention) attention;
} entry = {};

using Tensor = at::Tensor;
struct NotTensor : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct PythonError {};                     // is set already

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t d : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(d);
  return s + "]";
}
[[noreturn]] void bad(const std::string& why) { throw std::invalid_argument(why); }

const Tensor& tensor(const char* what, PyObject* o, int64_t device) {
  if (!THPVariable_Check(o)) throw NotTensor(std::string(what) + ": a torch tensor is needed");
  const Tensor& t = THPVariable_Unpack(o);
  if (t.get_device() != device) bad(std::string(what) + " is on " + t.device().str() + ", the context on cuda:" + std::to_string(device));
  return t;
}
int as_int(const char* what, int64_t v) {
  if (v < INT_MIN || v > INT_MAX) bad(std::string(what) + " does not fit 32 bits");
  return (int)v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return (float)v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError();
  return v == 1;
}
void* pointer(PyObject* o) {
  if (o == Py_None) return nullptr;
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw PythonError();
  return p;
}
int type_id(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kFloat ? MS_Q_F32 : s == at::kHalf ? MS_Q_F16 : s == at::kBFloat16 ? MS_Q_BF16 : -1;
}
void rank3(const char* what, const Tensor& t) {
  if (t.dim() != 3) bad(std::string(what) + ": shape " + shape_of(t) + " is not [tokens, heads, head_dim]");
}
// the stride between the tokens of a [n, heads, hd] tensor whose heads are contiguous
int64_t rows(const char* what, const Tensor& t, int64_t n, int64_t heads, int64_t hd) {
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != hd)
    bad(std::string(what) + ": shape " + shape_of(t) + " is not [" + std::to_string(n) + ", " + std::to_string(heads) + ", " + std::to_string(hd) + "]");
  if (n && ((t.stride(1) != hd && heads > 1) || (t.stride(2) != 1 && hd > 1)))
    bad(std::string(what) + ": the heads of a token must be contiguous");
  return n > 1 ? t.stride(0) : heads * hd;
}
const int32_t* index(const char* what, const Tensor& t, int64_t n) {
  if (t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || t.scalar_type() != at::kInt)
    bad(std::string(what) + ": a contiguous int32 tensor of " + std::to_string(n) + " values is needed, got " + toString(t.scalar_type()) + " " + shape_of(t));
  return static_cast<const int32_t*>(t.data_ptr());
}
// n f32 values, or NULL for None
const float* floats(const char* what, PyObject* o, int64_t n, int64_t device) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(what, o, device);
  if (t.numel() != n || !t.is_contiguous() || t.scalar_type() != at::kFloat)
    bad(std::string(what) + ": " + std::to_string(n) + " contiguous f32 values are needed, got " + toString(t.scalar_type()) + " " + shape_of(t));
  return static_cast<const float*>(t.data_ptr());
}

template <class F>
PyObject* launched(F f) {                  // the status of a call of the library, made without the interpreter's lock
  ms_status st;
  Py_BEGIN_ALLOW_THREADS
  st = f();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}
// no C++ exception leaves a function
template <class F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
  if (n != want || !entry.rope) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments, or entries() was not called");
    return nullptr;
  }
  try {
    return f();
  } catch (const PythonError&) {
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const NotTensor& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// entries(rope, prompt, write, read, attention): their addresses
PyObject* entries(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[5] = {};
  for (int i = 0; i < 5 && n == 5; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  entry.rope = (decltype(entry.rope))p[0];
  entry.prompt = (decltype(entry.prompt))p[1];
  entry.write = (decltype(entry.write))p[2];
  entry.read = (decltype(entry.read))p[3];
  entry.attention = (decltype(entry.attention))p[4];
  Py_RETURN_NONE;
}

// (context, device, q, k, q_norm, k_norm, eps, cos, sin, pos, q_out, k_out, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 13, [&] {
    const int64_t dev = integer(a[1]);
    const Tensor &q = tensor("q", a[2], dev), &k = tensor("k", a[3], dev), &cos = tensor("cos", a[7], dev), &sin = tensor("sin", a[8], dev),
                 &pos = tensor("pos", a[9], dev), &q_out = tensor("q_out", a[10], dev), &k_out = tensor("k_out", a[11], dev);
    rank3("q", q);
    rank3("k", k);
    if (q.scalar_type() != k.scalar_type() || q_out.scalar_type() != k_out.scalar_type() || cos.dim() != 2 || cos.sizes() != sin.sizes())
      bad("q and k, q_out and k_out, cos and sin go together");
    const int64_t n = q.size(0), heads = q.size(1), hd = q.size(2), kv = k.size(1), table = cos.size(0), half = cos.size(1);
    ms_qk_rope r = {};
    r.n_tokens = as_int("the tokens", n); r.heads = as_int("the heads", heads); r.kv_heads = as_int("the heads", kv);
    r.head_dim = as_int("head_dim", hd); r.rot_dim = as_int("the rotated dims", 2 * half); r.interleaved = truth(a[12]);
    r.in_type = type_id(q); r.out_type = type_id(q_out);
    r.eps = number(a[6]);
    r.max_pos = as_int("the positions", table);
    r.q_stride = rows("q", q, n, heads, hd); r.k_stride = rows("k", k, n, kv, hd);
    r.q = q.data_ptr(); r.k = k.data_ptr();
    r.q_norm = floats("q_norm", a[4], hd, dev); r.k_norm = floats("k_norm", a[5], hd, dev);
    r.cos_t = floats("cos", a[7], table * half, dev); r.sin_t = floats("sin", a[8], table * half, dev);
    r.pos = index("pos", pos, n);
    r.q_out_stride = rows("q_out", q_out, n, heads, hd); r.k_out_stride = rows("k_out", k_out, n, kv, hd);
    r.q_out = q_out.data_ptr(); r.k_out = k_out.data_ptr();
    ms_ctx* ctx = (ms_ctx*)pointer(a[0]);
    return launched([&] { return entry.rope(ctx, &r); });
  });
}

// (context, device, q, k, v, cu_q, cu_k, out, window, sinks, scale)
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 11, [&] {
    const int64_t dev = integer(a[1]);
    const Tensor &q = tensor("q", a[2], dev), &k = tensor("k", a[3], dev), &v = tensor("v", a[4], dev), &cu_q = tensor("cu_q", a[5], dev),
                 &cu_k = tensor("cu_k", a[6], dev), &out = tensor("out", a[7], dev);
    rank3("q", q);
    rank3("k", k);
    const auto type = q.scalar_type();
    if (k.scalar_type() != type || v.scalar_type() != type || out.scalar_type() != type) bad("q, k, v and out must have one type");
    const int64_t n = q.size(0), heads = q.size(1), hd = q.size(2), m = k.size(0), kv = k.size(1), seqs = cu_q.numel() - 1;
    ms_prompt_attn p = {};
    p.n_seqs = as_int("the sequences", seqs); p.heads = as_int("the heads", heads); p.kv_heads = as_int("the heads", kv);
    p.head_dim = as_int("head_dim", hd); p.type = type_id(q); p.window = as_int("window", integer(a[8]));
    p.total_q = as_int("the queries", n); p.total_k = as_int("the keys", m);
    p.scale = number(a[10]);
    p.q_stride = rows("q", q, n, heads, hd); p.k_stride = rows("k", k, m, kv, hd); p.v_stride = rows("v", v, m, kv, hd);
    p.out_stride = rows("out", out, n, heads, hd);
    p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.out = out.data_ptr();
    p.cu_q = index("cu_q", cu_q, seqs + 1); p.cu_k = index("cu_k", cu_k, seqs + 1);
    p.sinks = floats("sinks", a[9], heads, dev);
    ms_ctx* ctx = (ms_ctx*)pointer(a[0]);
    return launched([&] { return entry.prompt(ctx, &p); });
  });
}

// (context, device, pages, the cache's struct, k, v, cu, start)
PyObject* cache_rows(PyObject* const* a, Py_ssize_t n_args, bool write) {
  return guarded(n_args, 8, [&] {
    const int64_t dev = integer(a[1]);
    tensor("the cache", a[2], dev);
    const ms_kv4_cache* c = (const ms_kv4_cache*)pointer(a[3]);
    const Tensor &k = tensor("k", a[4], dev), &v = tensor("v", a[5], dev), &cu = tensor("cu", a[6], dev), &start = tensor("start", a[7], dev);
    rank3("k", k);
    if (k.scalar_type() != v.scalar_type()) bad("k and v must have one type");
    const int64_t n = k.size(0);
    ms_kv4_rows r = {};
    r.type = type_id(k); r.total = as_int("the rows", n);
    r.cu = index("cu", cu, (int64_t)c->n_seqs + 1); r.start = index("start", start, c->n_seqs);
    r.k_stride = rows("k", k, n, c->kv_heads, c->head_dim); r.v_stride = rows("v", v, n, c->kv_heads, c->head_dim);
    r.k = k.data_ptr(); r.v = v.data_ptr();
    ms_ctx* ctx = (ms_ctx*)pointer(a[0]);
    return launched([&] { return (write ? entry.write : entry.read)(ctx, c, &r); });
  });
}
PyObject* kv4_write(PyObject*, PyObject* const* a, Py_ssize_t n) { return cache_rows(a, n, true); }
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) { return cache_rows(a, n, false); }

// (context, device, pages, the cache's struct, q, lens, out, work, window, sinks, scale)
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 11, [&] {
    const int64_t dev = integer(a[1]);
    tensor("the cache", a[2], dev);
    const ms_kv4_cache* c = (const ms_kv4_cache*)pointer(a[3]);
    const Tensor &q = tensor("q", a[4], dev), &lens = tensor("lens", a[5], dev), &out = tensor("out", a[6], dev), &work = tensor("work", a[7], dev);
    if (q.dim() != 4 || q.size(0) != c->n_seqs || q.size(3) != c->head_dim || q.sizes() != out.sizes() || q.scalar_type() != out.scalar_type())
      bad("q and out must be [" + std::to_string(c->n_seqs) + ", n_query, heads, " + std::to_string(c->head_dim) + "] of one type, got " + shape_of(q) + " and " + shape_of(out));
    if (!q.is_contiguous() || !out.is_contiguous() || !work.is_contiguous()) bad("q, out and work must be contiguous");
    ms_kv4_attn p = {};
    p.n_query = as_int("n_query", q.size(1)); p.heads = as_int("the heads", q.size(2)); p.type = type_id(q);
    p.window = as_int("window", integer(a[8]));
    p.scale = number(a[10]);
    p.q = q.data_ptr(); p.out = out.data_ptr(); p.work = work.data_ptr();
    p.work_bytes = (size_t)work.numel() * work.element_size();
    p.lens = index("lens", lens, c->n_seqs);
    p.sinks = floats("sinks", a[9], p.heads, dev);
    ms_ctx* ctx = (ms_ctx*)pointer(a[0]);
    return launched([&] { return entry.attention(ctx, c, &p); });
  });
}

PyMethodDef methods[] = {{"entries", (PyCFunction)(void (*)())entries, METH_FASTCALL, nullptr},
                         {"qk_norm_rope", (PyCFunction)(void (*)())qk_norm_rope, METH_FASTCALL, nullptr},
                         {"prompt_attention", (PyCFunction)(void (*)())prompt_attention, METH_FASTCALL, nullptr},
                         {"kv4_write", (PyCFunction)(void (*)())kv4_write, METH_FASTCALL, nullptr},
                         {"kv4_read", (PyCFunction)(void (*)())kv4_read, METH_FASTCALL, nullptr},
                         {"kv4_attention", (PyCFunction)(void (*)())kv4_attention, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
