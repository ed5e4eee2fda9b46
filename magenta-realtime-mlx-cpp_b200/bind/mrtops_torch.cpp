// _mrtops: the Python side of the operators on device buffers (include/mrtdf.h,
// "operators") for torch tensors. Checks shapes, types, devices and gradients,
// allocates what the caller did not give, and calls the C ABI on the current
// torch stream of the tensors' device. Written against the CPython API because
// the smallest calls take less GPU time than a ctypes call with its arguments
// checked in Python: one drafted tree of a CFG pair took 21 us of host time
// that way, 7 us of GPU time.
//
// mrtops.py holds the signatures, their documentation and the defaults; every
// function here takes all its arguments by position, None where one is left
// out.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/mrtdf.h"

namespace {

PyObject* g_error = nullptr;  // mrtdf.MrtdfError

struct Failure {
  int code;
  std::string msg;
};
[[noreturn]] void invalid(const std::string& msg) { throw Failure{MRTDF_ERR_INVALID, msg}; }

void check(int rc) {
  if (rc != MRTDF_OK) throw Failure{rc, mrtdf_last_error()};
}

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
std::string about(const at::Tensor& t) {
  return std::string(c10::toString(t.scalar_type())) + " " + shape_of(t.sizes()) + " on " + t.device().str();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) invalid(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

void no_gradient(const at::Tensor& t, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    invalid(std::string(name) + " requires a gradient, which the operators do not give");
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    invalid(std::string(name) + " has a forward-mode tangent, which the operators do not carry on");
}

// What a call has written counts as modified in place: a backward pass that saved
// it before reports that instead of using the new values.
void written(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

int dtype_of(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return MRTDF_DTYPE_FP32;
  if (t.scalar_type() == at::kBFloat16) return MRTDF_DTYPE_BF16;
  invalid(std::string(name) + " must be float32 or bfloat16, is " + about(t));
}

int32_t small(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) invalid(std::string(name) + " is out of range");
  return (int32_t)v;
}

// (..., n, head_dim) rows; `want` the whole shape.
mrtdf_rows rows(const at::Tensor& t, at::IntArrayRef want, const at::Tensor& like, const char* name) {
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device() || t.sizes() != want)
    invalid(std::string(name) + " must be " + c10::toString(like.scalar_type()) + " " + shape_of(want) + " on " +
            like.device().str() + ", is " + about(t));
  no_gradient(t, name);
  const auto s = t.strides();
  const size_t d = s.size();
  if (s[d - 1] != 1) invalid(std::string(name) + ": elements of a row must lie next to each other");
  mrtdf_rows r;
  r.ptr = t.data_ptr();
  r.stride_l = d == 5 ? s[0] : 0;
  r.stride_b = s[d - 4];
  r.stride_h = s[d - 3];
  r.stride_n = s[d - 2];
  return r;
}

// Pointer of a contiguous tensor.
template <typename T>
T* flat(const at::Tensor& t, at::IntArrayRef want, at::ScalarType type, at::Device device, const char* name) {
  if (t.scalar_type() != type || t.device() != device || t.sizes() != want)
    invalid(std::string(name) + " must be " + c10::toString(type) + " " + shape_of(want) + " on " + device.str() + ", is " +
            about(t));
  if (!t.is_contiguous()) invalid(std::string(name) + " must be contiguous");
  no_gradient(t, name);
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* flat_or_null(PyObject* o, at::IntArrayRef want, at::ScalarType type, at::Device device, const char* name) {
  return o == Py_None ? nullptr : flat<T>(tensor(o, name), want, type, device, name);
}

// A (layers, batch, kv_heads, capacity, head_dim) cache, or one layer's four
// dimensions.
mrtdf_cache cache_of(const at::Tensor& k, const at::Tensor* v, PyObject* lens, PyObject* pos, PyObject* next_pos, bool layered) {
  const int64_t nd = k.dim();
  if (nd != 4 && !(nd == 5 && layered))
    invalid(std::string("the cache must be (batch, kv_heads, capacity, head_dim)") +
            (layered ? ", with the layers in front where there are several" : ""));
  if (!k.is_cuda()) invalid("the cache must be on a CUDA device, is " + about(k));
  mrtdf_cache c{};
  c.struct_bytes = sizeof(c);
  c.dtype = dtype_of(k, "the cache");
  const auto n = k.sizes();
  const auto s = k.strides();
  if (s[nd - 1] != 1) invalid("the cache: elements of a row must lie next to each other");
  no_gradient(k, "the cache");
  c.k = k.data_ptr();
  if (v) {
    if (v->sizes() != n || v->scalar_type() != k.scalar_type() || v->device() != k.device())
      invalid("k_cache and v_cache must have the same shape, dtype and device: " + about(k) + " and " + about(*v));
    if (v->strides() != s) invalid("k_cache and v_cache must have the same strides");
    no_gradient(*v, "the cache");
    c.v = v->data_ptr();
  }
  const bool l = nd == 5;
  c.stride_l = l ? s[0] : 0;
  c.stride_b = s[nd - 4];
  c.stride_h = s[nd - 3];
  c.stride_t = s[nd - 2];
  c.layers = l ? small(n[0], "layers") : 1;
  c.batch = small(n[nd - 4], "batch");
  c.kv_heads = small(n[nd - 3], "kv_heads");
  c.capacity = small(n[nd - 2], "capacity");
  c.head_dim = small(n[nd - 1], "head_dim");
  c.device = k.device().index();
  const int64_t batch[1] = {c.batch};
  c.lens = flat<int32_t>(tensor(lens, "lens"), batch, at::kInt, k.device(), "lens");
  c.pos = flat_or_null<int32_t>(pos, n.slice(0, nd - 1), at::kInt, k.device(), "pos");
  c.next_pos = flat_or_null<int32_t>(next_pos, batch, at::kInt, k.device(), "next_pos");
  return c;
}

void* stream_of(at::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, at::Device d) {
  return at::detail::empty_cuda(shape, type, d, std::nullopt);
}

float number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    invalid(std::string(name) + " must be a number");
  }
  return (float)v;
}
int32_t whole(PyObject* o, const char* name) {
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    invalid(std::string(name) + " must be a whole number");
  }
  if (overflow || v < INT32_MIN || v > INT32_MAX) invalid(std::string(name) + " is out of range");
  return (int32_t)v;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* given(PyObject* o) {
  Py_INCREF(o);
  return o;
}
PyObject* pair(PyObject* a, PyObject* b) {
  if (!a || !b) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyObject* t = PyTuple_New(2);
  if (!t) {
    Py_DECREF(a);
    Py_DECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}

// Body of a Python function: `count` arguments, C++ exceptions to Python ones.
template <typename F>
PyObject* call(Py_ssize_t n, Py_ssize_t count, F&& f) {
  try {
    if (n != count) invalid("wrong number of arguments");
    return f();
  } catch (const Failure& e) {
    PyObject* args = Py_BuildValue("(is)", e.code, e.msg.c_str());
    if (args) {
      PyErr_SetObject(g_error ? g_error : PyExc_RuntimeError, args);
      Py_DECREF(args);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

struct Table {
  const float* ptr = nullptr;
  int32_t len = 0;
};
Table bias_table(PyObject* o, int64_t heads, at::Device d) {
  Table t;
  if (o == Py_None) return t;
  const at::Tensor& b = tensor(o, "rel_bias");
  if (b.dim() != 2) invalid("rel_bias must be (heads, rel_len), is " + about(b));
  const int64_t want[2] = {heads, b.size(1)};
  t.ptr = flat<float>(b, want, at::kFloat, d, "rel_bias");
  t.len = small(b.size(1), "rel_len");
  return t;
}

// q, k_new, v_new, k_cache, v_cache, lens, parents, scale, rel_bias, pos,
// next_pos, out, lse, workspace
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 14, [&]() -> PyObject* {
    const at::Tensor &q = tensor(a[0], "q"), &kn = tensor(a[1], "k_new"), &vn = tensor(a[2], "v_new");
    const at::Tensor &k = tensor(a[3], "k_cache"), &v = tensor(a[4], "v_cache");
    const mrtdf_cache c = cache_of(k, &v, a[5], a[9], a[10], false);
    if (q.dim() != 4) invalid("q must be (batch, heads, nodes, head_dim), is " + about(q));
    const at::Device d = k.device();
    const int64_t heads = q.size(1), nodes = q.size(2);
    const int64_t shape[4] = {c.batch, heads, nodes, c.head_dim}, fresh_rows[4] = {c.batch, c.kv_heads, nodes, c.head_dim};
    const int64_t two[2] = {c.batch, nodes};
    mrtdf_tree_args t{};
    t.struct_bytes = sizeof(t);
    t.q = rows(q, shape, k, "q");
    t.k_new = rows(kn, fresh_rows, k, "k_new");
    t.v_new = rows(vn, fresh_rows, k, "v_new");
    t.parents = flat_or_null<int32_t>(a[6], two, at::kInt, d, "parents");
    t.scale = number(a[7], "scale");
    const Table table = bias_table(a[8], heads, d);
    t.rel_bias = table.ptr;
    t.rel_len = table.len;
    t.heads = small(heads, "heads");
    t.nodes = small(nodes, "nodes");
    at::Tensor out, lse, ws;
    out = a[11] == Py_None ? fresh(shape, k.scalar_type(), d) : tensor(a[11], "out");
    t.out = rows(out, shape, k, "out");
    lse = a[12] == Py_None ? fresh(at::IntArrayRef(shape, 3), at::kFloat, d) : tensor(a[12], "lse");
    t.lse = flat<float>(lse, at::IntArrayRef(shape, 3), at::kFloat, d, "lse");
    size_t need = 0;
    check(mrtdf_tree_attention_workspace(&c, &t, &need));
    if (need) {
      if (a[13] == Py_None) {
        const int64_t bytes[1] = {(int64_t)need};
        ws = fresh(bytes, at::kByte, d);
      } else {
        ws = tensor(a[13], "workspace");
        if (ws.device() != d || !ws.is_contiguous()) invalid("workspace must be contiguous and on the cache's device");
      }
      t.workspace = ws.data_ptr();
      t.workspace_bytes = ws.nbytes();
    }
    check(mrtdf_tree_attention(&c, &t, stream_of(d)));
    written({&out, &lse});
    if (ws.defined()) written({&ws});
    return pair(a[11] == Py_None ? wrap(out) : given(a[11]), a[12] == Py_None ? wrap(lse) : given(a[12]));
  });
}

// The shape (leading dimensions of the cache, x, y, z) in `to`; z < 0: left out.
at::IntArrayRef lead(int64_t* to, const at::Tensor& k, int64_t x, int64_t y, int64_t z) {
  size_t n = 0;
  for (int64_t i = 0; i < k.dim() - 3; ++i) to[n++] = k.size(i);
  to[n++] = x;
  to[n++] = y;
  if (z >= 0) to[n++] = z;
  return at::IntArrayRef(to, n);
}

const at::Tensor& path_of(PyObject* o) {
  const at::Tensor& p = tensor(o, "path");
  if (p.dim() != 2) invalid("path must be (batch, path_len), is " + about(p));
  return p;
}

// q, lse, k_new, k_cache, lens, path, mass, scale, rel_bias, pos, next_pos,
// decay, mass_out
PyObject* cache_mass(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 13, [&]() -> PyObject* {
    const at::Tensor &q = tensor(a[0], "q"), &lse = tensor(a[1], "lse"), &kn = tensor(a[2], "k_new"), &k = tensor(a[3], "k_cache");
    const mrtdf_cache c = cache_of(k, nullptr, a[4], a[9], a[10], true);
    if (q.dim() != k.dim()) invalid("q must have the cache's number of dimensions, is " + about(q));
    const at::Device d = k.device();
    const int64_t heads = q.size(-3), nodes = q.size(-2);
    const at::Tensor& path = path_of(a[5]);
    const int64_t two[2] = {c.batch, path.size(1)};
    int64_t s[5];
    mrtdf_mass_args m{};
    m.struct_bytes = sizeof(m);
    m.q = rows(q, lead(s, k, heads, nodes, c.head_dim), k, "q");
    m.k_new = rows(kn, lead(s, k, c.kv_heads, nodes, c.head_dim), k, "k_new");
    m.lse = flat<float>(lse, lead(s, k, heads, nodes, -1), at::kFloat, d, "lse");
    m.path = flat<int32_t>(path, two, at::kInt, d, "path");
    const Table table = bias_table(a[8], heads, d);
    m.rel_bias = table.ptr;
    m.rel_len = table.len;
    m.mass = flat<float>(tensor(a[6], "mass"), lead(s, k, c.kv_heads, c.capacity, -1), at::kFloat, d, "mass");
    PyObject* to = a[12] == Py_None ? a[6] : a[12];
    m.mass_out = flat<float>(tensor(to, "mass_out"), lead(s, k, c.kv_heads, c.capacity, -1), at::kFloat, d, "mass_out");
    m.heads = small(heads, "heads");
    m.nodes = small(nodes, "nodes");
    m.path_len = small(path.size(1), "path_len");
    m.scale = number(a[7], "scale");
    m.decay = number(a[11], "decay");
    check(mrtdf_cache_mass(&c, &m, stream_of(d)));
    written({&tensor(to, "mass_out")});
    return given(to);
  });
}

// k_new, v_new, k_cache, v_cache, lens, path, pos, next_pos, lens_out,
// next_pos_out
PyObject* cache_commit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 10, [&]() -> PyObject* {
    const at::Tensor &kn = tensor(a[0], "k_new"), &vn = tensor(a[1], "v_new"), &k = tensor(a[2], "k_cache"), &v = tensor(a[3], "v_cache");
    const mrtdf_cache c = cache_of(k, &v, a[4], a[6], a[7], true);
    if (kn.dim() != k.dim()) invalid("k_new must have the cache's number of dimensions, is " + about(kn));
    const at::Device d = k.device();
    const int64_t nodes = kn.size(-2);
    const at::Tensor& path = path_of(a[5]);
    const int64_t two[2] = {c.batch, path.size(1)}, one[1] = {c.batch};
    int64_t s[5];
    mrtdf_commit_args m{};
    m.struct_bytes = sizeof(m);
    m.k_new = rows(kn, lead(s, k, c.kv_heads, nodes, c.head_dim), k, "k_new");
    m.v_new = rows(vn, lead(s, k, c.kv_heads, nodes, c.head_dim), k, "v_new");
    m.path = flat<int32_t>(path, two, at::kInt, d, "path");
    at::Tensor lens, next;
    lens = a[8] == Py_None ? fresh(one, at::kInt, d) : tensor(a[8], "lens_out");
    m.lens_out = flat<int32_t>(lens, one, at::kInt, d, "lens_out");
    const bool positions = a[9] != Py_None || a[7] != Py_None;
    if (positions) {
      next = a[9] == Py_None ? fresh(one, at::kInt, d) : tensor(a[9], "next_pos_out");
      m.next_pos_out = flat<int32_t>(next, one, at::kInt, d, "next_pos_out");
    }
    m.nodes = small(nodes, "nodes");
    m.path_len = small(path.size(1), "path_len");
    check(mrtdf_cache_commit(&c, &m, stream_of(d)));
    written({&k, &v, &lens});
    if (positions) written({&next});
    if (a[6] != Py_None) written({&tensor(a[6], "pos")});
    return pair(a[8] == Py_None ? wrap(lens) : given(a[8]),
                a[9] != Py_None || !positions ? given(a[9]) : wrap(next));
  });
}

// k_cache, v_cache, lens, mass, pos, next_pos, budget, recent, sinks, mass_out,
// pos_out, lens_out
PyObject* cache_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 12, [&]() -> PyObject* {
    const at::Tensor &k = tensor(a[0], "k_cache"), &v = tensor(a[1], "v_cache");
    const mrtdf_cache c = cache_of(k, &v, a[2], a[4], a[5], true);
    const at::Device d = k.device();
    const auto shape = k.sizes().slice(0, k.dim() - 1);
    const int64_t one[1] = {c.batch};
    mrtdf_evict_args m{};
    m.struct_bytes = sizeof(m);
    m.mass = flat<float>(tensor(a[3], "mass"), shape, at::kFloat, d, "mass");
    const at::Tensor &mass_out = tensor(a[9] == Py_None ? a[3] : a[9], "mass_out"), &pos_out = tensor(a[10] == Py_None ? a[4] : a[10], "pos_out");
    m.mass_out = flat<float>(mass_out, shape, at::kFloat, d, "mass_out");
    m.pos_out = flat<int32_t>(pos_out, shape, at::kInt, d, "pos_out");
    at::Tensor lens = a[11] == Py_None ? fresh(one, at::kInt, d) : tensor(a[11], "lens_out");
    m.lens_out = flat<int32_t>(lens, one, at::kInt, d, "lens_out");
    m.budget = whole(a[6], "budget");
    m.recent = whole(a[7], "recent");
    m.sinks = whole(a[8], "sinks");
    check(mrtdf_cache_evict(&c, &m, stream_of(d)));
    written({&k, &v, &mass_out, &pos_out, &lens});
    return a[11] == Py_None ? wrap(lens) : given(a[11]);
  });
}

// x, packed, scales, biases, out, float32 out (None: x's type)
PyObject* q4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 6, [&]() -> PyObject* {
    const at::Tensor &x = tensor(a[0], "x"), &packed = tensor(a[1], "packed"), &scales = tensor(a[2], "scales"), &biases = tensor(a[3], "biases");
    if (x.dim() != 2 || packed.dim() != 2 || scales.dim() != 2 || biases.dim() != 2)
      invalid("x, packed, scales and biases must have two dimensions");
    if (!x.is_cuda()) invalid("x must be on a CUDA device, is " + about(x));
    mrtdf_q4_args m{};
    m.struct_bytes = sizeof(m);
    m.dtype = dtype_of(x, "x");
    no_gradient(x, "x");
    const at::Device d = x.device();
    const int64_t rows_x = x.size(0), k = x.size(1), outs = scales.size(0), groups = scales.size(1);
    if (rows_x < 1 || k < 1 || groups < 1 || k % groups) invalid("k must be a multiple of the number of groups");
    if (x.stride(1) != 1) invalid("x: elements of a row must lie next to each other");
    const int64_t pk[2] = {outs, k / 2}, sc[2] = {outs, groups}, os[2] = {rows_x, outs};
    at::Tensor out = a[4] != Py_None ? tensor(a[4], "out") : fresh(os, a[5] == Py_True ? at::kFloat : x.scalar_type(), d);
    if (out.sizes() != at::IntArrayRef(os) || out.device() != d || (outs > 1 && out.stride(1) != 1))
      invalid("out must be " + shape_of(os) + " on " + d.str() + " with contiguous rows, is " + about(out));
    m.out_dtype = dtype_of(out, "out");
    no_gradient(out, "out");
    m.x = x.data_ptr();
    m.packed = flat<uint8_t>(packed, pk, at::kByte, d, "packed");
    m.scales = flat<void>(scales, sc, x.scalar_type(), d, "scales");
    m.biases = flat<void>(biases, sc, x.scalar_type(), d, "biases");
    m.out = out.data_ptr();
    m.x_stride = x.stride(0);
    m.out_stride = out.stride(0);
    m.m = small(rows_x, "m");
    m.n = small(outs, "n");
    m.k = small(k, "k");
    m.group = small(k / groups, "group");
    m.device = d.index();
    size_t need = 0;
    check(mrtdf_q4_linear_workspace(&m, &need));
    at::Tensor ws;
    if (need) {
      const int64_t bytes[1] = {(int64_t)need};
      ws = fresh(bytes, at::kByte, d);
      m.workspace = ws.data_ptr();
      m.workspace_bytes = need;
    }
    check(mrtdf_q4_linear(&m, stream_of(d)));
    written({&out});
    return a[4] == Py_None ? wrap(out) : given(a[4]);
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XDECREF(g_error);
  g_error = cls;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(F));
}

PyMethodDef g_methods[] = {
    {"tree_attention", fast<tree_attention>(), METH_FASTCALL, nullptr},
    {"cache_mass", fast<cache_mass>(), METH_FASTCALL, nullptr},
    {"cache_commit", fast<cache_commit>(), METH_FASTCALL, nullptr},
    {"cache_evict", fast<cache_evict>(), METH_FASTCALL, nullptr},
    {"q4_linear", fast<q4_linear>(), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_mrtops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mrtops() { return PyModule_Create(&g_module); }
