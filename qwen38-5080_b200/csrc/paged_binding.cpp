// The three paged calls for Python: tensors in, checks of arguments, one call of the C-ABI.  A decode step makes two such calls per layer
// when it is not captured, and reading fourteen tensors' types, devices, shapes and addresses from Python took longer than the work on
// the device (append of one token: 18 us issued, 2.4 on the device).  Nothing is computed, allocated or kept here.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/b200attn.h"

namespace {

decltype(&b200attn_paged_rope_append) call_append;
decltype(&b200attn_paged_decode) call_decode;
decltype(&b200attn_paged_prefill) call_prefill;

using Tensor = const at::Tensor*;   // null: None, or refused

bool refuse(const char* what) {
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, what);
  return false;
}

// A tensor of `type`, contiguous, on CUDA device `dev`; None gives null.
bool take(PyObject* o, const char* name, int dev, at::ScalarType type, Tensor& t) {
  t = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    return false;
  }
  const at::Tensor& x = THPVariable_Unpack(o);
  if (dev < 0 || !x.is_cuda() || x.get_device() != dev) {
    PyErr_Format(PyExc_ValueError, "%s must be on the cache's CUDA device: there is no CPU path", name);
    return false;
  }
  if (x.scalar_type() != type || !x.is_contiguous()) {
    PyErr_Format(PyExc_ValueError, "%s must be contiguous %s, not %s%s", name, c10::toString(type), x.is_contiguous() ? "" : "strided ",
                 c10::toString(x.scalar_type()));
    return false;
  }
  t = &x;
  return true;
}
bool need(PyObject* o, const char* name, int dev, at::ScalarType type, Tensor& t) {
  if (!take(o, name, dev, type, t)) return false;
  if (t) return true;
  PyErr_Format(PyExc_ValueError, "%s is missing", name);
  return false;
}
void* address(Tensor t) { return t ? t->data_ptr() : nullptr; }
constexpr at::ScalarType kBf16 = at::kBFloat16, kF32 = at::kFloat, kI32 = at::kInt;

// The cache handles: pools (dense within a layer, any stride over layers), scales, table.
struct Cache {
  B200AttnPagedShape shape{};
  int dev = -1;
  Tensor k = nullptr, v = nullptr, ks = nullptr, vs = nullptr, table = nullptr;

  bool read(PyObject* const* a, int64_t h_q) {
    if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) {
      PyErr_SetString(PyExc_TypeError, "k_pages and v_pages must be tensors");
      return false;
    }
    k = &THPVariable_Unpack(a[0]);
    v = &THPVariable_Unpack(a[1]);
    const auto dims = k->sizes();
    const size_t nd = dims.size();
    if ((nd != 4 && nd != 5) || v->sizes() != dims)
      return refuse("k_pages and v_pages must have the same shape [n_layers, n_pages, h_kv, page_size, head_dim]");
    for (Tensor t : {k, v})
      if (t->scalar_type() != at::kByte && t->scalar_type() != at::kFloat8_e4m3fn) return refuse("the cache must be uint8 / float8_e4m3fn");
    const int64_t n = nd == 5 ? dims[0] : 1, n_pages = dims[nd - 4], h_kv = dims[nd - 3], page = dims[nd - 2], d = dims[nd - 1];
    for (Tensor t : {k, v}) {
      const auto st = t->strides();
      if (st[nd - 1] != 1 || st[nd - 2] != d || st[nd - 3] != page * d || st[nd - 4] != h_kv * page * d) return refuse("the cache must be dense within a layer");
    }
    dev = k->is_cuda() ? k->get_device() : -1;
    if (!need(a[2], "k_scale", dev, kF32, ks) || !need(a[3], "v_scale", dev, kF32, vs) || !need(a[4], "page_table", dev, kI32, table)) return false;
    if (!v->is_cuda() || v->get_device() != dev || vs->numel() != ks->numel()) return refuse("k_pages / v_pages and k_scale / v_scale must match");
    if (ks->numel() != n * n_pages * h_kv) return refuse("scales must be [n_layers, n_pages, h_kv]");
    if (table->dim() != 2) return refuse("page_table must be [batch, max_pages]");
    for (const int64_t x : {n, n_pages, h_kv, page, d, h_q, table->size(0), table->size(1)})
      if (x > 0x7fffffff) return refuse("a dimension does not fit");
    shape = B200AttnPagedShape{(int)n, (int)table->size(0), (int)h_q, (int)h_kv, (int)d, (int)page, (int)n_pages, (int)table->size(1),
                               n > 1 ? (long long)k->stride(0) : 0, n > 1 ? (long long)v->stride(0) : 0, 0, 0};
    return true;
  }
};

// Whether a tensor that names its layers has them first: [n_tokens, n_layers, ..] has as many elements.
bool layers_first(Tensor t, int64_t n_layers) { return !t || n_layers == 1 || t->dim() < 4 || t->size(0) == n_layers; }

bool args_ok(Py_ssize_t n, Py_ssize_t want) { return n == want || refuse("wrong number of arguments"); }

// q's heads: its last dimension but one; without q the kv heads.
bool heads_of(PyObject* q, PyObject* pages, int64_t& h_q) {
  PyObject* o = q != Py_None ? q : pages;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "q, k_pages must be tensors");
    return false;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() < 3) return refuse("q must be [n_layers, n_tokens, h_q, head_dim]");
  h_q = t.size(q != Py_None ? -2 : -3);
  return true;
}

// (q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale, page_table, seq_pos, q_start, positions, pair_axis, q_norm_weight,
//  k_norm_weight, eps, advance, status, q_out, stream) -> error code
bool append(PyObject* const* a, int& rc) {
  int64_t h_q = 0;
  Cache c;
  if (!heads_of(a[0], a[5], h_q) || !c.read(a + 5, h_q)) return false;
  Tensor q, k, v, cos, sin, pos, start, positions, axis, wq, wk, status, q_out;
  if (!take(a[0], "q", c.dev, kBf16, q) || !need(a[1], "k", c.dev, kBf16, k) || !need(a[2], "v", c.dev, kBf16, v) ||
      !take(a[3], "cos", c.dev, kF32, cos) || !take(a[4], "sin", c.dev, kF32, sin) || !need(a[10], "seq_pos", c.dev, kI32, pos) ||
      !take(a[11], "q_start", c.dev, kI32, start) || !take(a[12], "positions", c.dev, kI32, positions) ||
      !take(a[13], "pair_axis", c.dev, kI32, axis) || !take(a[14], "q_norm_weight", c.dev, kBf16, wq) ||
      !take(a[15], "k_norm_weight", c.dev, kBf16, wk) || !need(a[18], "status", c.dev, kI32, status) || !take(a[19], "q_out", c.dev, kBf16, q_out))
    return false;
  const double eps = PyFloat_AsDouble(a[16]);
  const int advance = PyObject_IsTrue(a[17]);
  void* stream = PyLong_AsVoidPtr(a[20]);
  if (PyErr_Occurred()) return false;
  const B200AttnPagedShape& s = c.shape;
  const int64_t n = s.n_layers, d = s.head_dim, row = n * s.h_kv * d;
  const int64_t n_tokens = row ? k->numel() / row : 0;
  if (n_tokens > 0x7fffffff || k->numel() != row * n_tokens || v->sizes() != k->sizes() || k->dim() < 2 || k->size(-2) != s.h_kv || k->size(-1) != d || !layers_first(k, n))
    return refuse("k and v must be [n_layers, n_tokens, h_kv, head_dim]");
  if (q && (q->numel() != n * n_tokens * h_q * d || q->size(-1) != d || !layers_first(q, n))) return refuse("q must be [n_layers, n_tokens, h_q, head_dim]");
  if (pos->numel() != s.batch) return refuse("seq_pos must be int32 [batch]");
  if (!start && n_tokens != s.batch) return refuse("without q_start there is one token per sequence");
  if (start && start->numel() != (int64_t)s.batch + 1) return refuse("q_start must be int32 [batch + 1]");
  for (Tensor w : {wq, wk})
    if (w && w->numel() != n * d) return refuse("norm weights must be [n_layers, head_dim]");
  B200AttnRope rope{};
  const bool turns = cos && cos->dim() > 0 && cos->size(-1) > 0;
  if (turns) {
    if (!sin || cos->dim() != 2 || sin->sizes() != cos->sizes() || cos->size(0) > 0x7fffffff || cos->size(1) > 0x3fffffff)
      return refuse("cos and sin must be [n_positions, rotary_dim / 2]");
    const int64_t axes = positions && positions->dim() != 1 ? (positions->dim() ? positions->size(0) : 0) : 1;
    if (positions && (axes > 0x7fffffff || positions->numel() != axes * n_tokens)) return refuse("positions must be [n_tokens] or [n_axes, n_tokens]");
    if (axis && axis->numel() != cos->size(1)) return refuse("pair_axis must be int32 [rotary_dim / 2]");
    rope = B200AttnRope{(const float*)address(cos), (const float*)address(sin), (const int*)address(positions), (const int*)address(axis),
                        (int)cos->size(0), (int)axes, (int)(2 * cos->size(1)), 0};
  }
  if (q && (!q_out || q_out->numel() != q->numel() || !layers_first(q_out, n))) return refuse("q_out must have q's shape");
  if (n_tokens == 0) return true;
  rc = call_append(&s, turns ? &rope : nullptr, (int)n_tokens, (const int*)address(start), address(q), address(k), address(v), address(wq), address(wk),
                   (float)eps, q ? address(q_out) : nullptr, address(c.k), address(c.v), (float*)address(c.ks), (float*)address(c.vs),
                   (const int*)address(c.table), (int*)address(pos), advance, (int*)address(status), stream);
  return true;
}

struct Scratch {   // buffer, bytes, status, longest sequence, softmax scale (None: head_dim^-1/2), out, stream
  Tensor buf = nullptr, status = nullptr, out = nullptr;
  size_t bytes = 0;
  long longest = 0;
  float scale = 0.f;
  void* stream = nullptr;
  bool read(PyObject* const* a, const Cache& c, Tensor q) {
    if (!THPVariable_Check(a[0]) || !THPVariable_Unpack(a[0]).is_cuda() || THPVariable_Unpack(a[0]).get_device() != c.dev)
      return refuse("the workspace must be on the cache's device");
    if (!need(a[0], "workspace", c.dev, at::kByte, buf) || !need(a[2], "status", c.dev, kI32, status) || !need(a[5], "out", c.dev, kBf16, out)) return false;
    bytes = PyLong_AsSize_t(a[1]);
    longest = PyLong_AsLong(a[3]);
    scale = a[4] == Py_None ? (float)(1.0 / std::sqrt((double)c.shape.head_dim)) : (float)PyFloat_AsDouble(a[4]);
    stream = PyLong_AsVoidPtr(a[6]);
    if (PyErr_Occurred()) return false;
    if (longest < 0 || longest > 0x7fffffff || bytes > (size_t)buf->numel()) return refuse("the workspace does not fit");
    if (out->numel() != q->numel() || !layers_first(out, c.shape.n_layers)) return refuse("out must have q's shape");
    return true;
  }
};

// (q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, seq_len_offset, scratch ..) -> error code
bool decode(PyObject* const* a, int& rc) {
  int64_t h_q = 0;
  Cache c;
  Tensor q, len;
  Scratch w;
  if (!heads_of(a[0], a[1], h_q) || !c.read(a + 1, h_q) || !need(a[0], "q", c.dev, kBf16, q) || !need(a[6], "seq_len", c.dev, kI32, len)) return false;
  const B200AttnPagedShape& s = c.shape;
  if (q->size(-1) != s.head_dim || q->numel() != (int64_t)s.n_layers * s.batch * h_q * s.head_dim || !layers_first(q, s.n_layers))
    return refuse("q must be [n_layers, batch, h_q, head_dim]");
  if (len->numel() != s.batch) return refuse("seq_len must be int32 [batch]");
  const long offset = PyLong_AsLong(a[7]);
  if (PyErr_Occurred()) return false;
  if (offset < -0x7fffffffL || offset > 0x7fffffffL) return refuse("seq_len_offset does not fit");
  if (!w.read(a + 8, c, q)) return false;
  rc = call_decode(&s, address(q), address(c.k), address(c.v), (const float*)address(c.ks), (const float*)address(c.vs), (const int*)address(c.table),
                   (const int*)address(len), (int)offset, (int)w.longest, w.scale, address(w.buf), w.bytes, address(w.out), (int*)address(w.status), w.stream);
  return true;
}

// (q, k_pages, v_pages, k_scale, v_scale, page_table, seq_len, q_start, most tokens, causal, scratch ..) -> error code
bool prefill(PyObject* const* a, int& rc) {
  int64_t h_q = 0;
  Cache c;
  Tensor q, len, start;
  Scratch w;
  if (!heads_of(a[0], a[1], h_q) || !c.read(a + 1, h_q) || !need(a[0], "q", c.dev, kBf16, q) || !need(a[6], "seq_len", c.dev, kI32, len) ||
      !need(a[7], "q_start", c.dev, kI32, start))
    return false;
  const B200AttnPagedShape& s = c.shape;
  const int64_t row = (int64_t)s.n_layers * h_q * s.head_dim, n_tokens = row ? q->numel() / row : 0;
  if (n_tokens > 0x7fffffff || q->size(-1) != s.head_dim || q->numel() != row * n_tokens || !layers_first(q, s.n_layers))
    return refuse("q must be [n_layers, n_tokens, h_q, head_dim]");
  if (len->numel() != s.batch || start->numel() != (int64_t)s.batch + 1) return refuse("seq_len must be int32 [batch], q_start int32 [batch + 1]");
  const long most = PyLong_AsLong(a[8]);
  const int causal = PyObject_IsTrue(a[9]);
  if (PyErr_Occurred()) return false;
  if (most < n_tokens) {
    PyErr_Format(PyExc_ValueError, "the workspace must be one for %lld query tokens, on the cache's device", (long long)n_tokens);
    return false;
  }
  if (!w.read(a + 10, c, q)) return false;
  if (n_tokens == 0) return true;
  rc = call_prefill(&s, (int)n_tokens, address(q), (const int*)address(start), address(c.k), address(c.v), (const float*)address(c.ks),
                    (const float*)address(c.vs), (const int*)address(c.table), (const int*)address(len), (int)w.longest, causal, w.scale, address(w.buf),
                    w.bytes, address(w.out), (int*)address(w.status), w.stream);
  return true;
}

template <bool (*F)(PyObject* const*, int&), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!args_ok(n, N)) return nullptr;
  try {
    int rc = 0;
    return F(args, rc) ? PyLong_FromLong(rc) : nullptr;
  } catch (const std::exception& e) {
    refuse(e.what());
  } catch (...) {
    refuse("not a tensor that can be read");
  }
  return nullptr;
}

// Addresses of the three functions in the loaded library.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!args_ok(n, 3)) return nullptr;
  call_append = (decltype(call_append))PyLong_AsVoidPtr(args[0]);
  call_decode = (decltype(call_decode))PyLong_AsVoidPtr(args[1]);
  call_prefill = (decltype(call_prefill))PyLong_AsVoidPtr(args[2]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void (*)(void))entry<append, 21>, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void (*)(void))entry<decode, 15>, METH_FASTCALL, nullptr},
    {"prefill", (PyCFunction)(void (*)(void))entry<prefill, 17>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "source_hash", B200ATTN_BINDING_HASH) < 0) Py_CLEAR(m);
  return m;
}
