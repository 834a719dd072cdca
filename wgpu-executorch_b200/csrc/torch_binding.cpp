// Calls of the text-decoding operators on torch tensors (wgx.decode): reads the
// tensors' metadata, checks it, fills the C ABI's argument structs and calls
// the library. A Python binding by ctypes spends 6 to 12 us on this, as long as
// the kernels of a small step run; this takes about one.
//
// The library's entry points are handed over at init() by address, so that the
// library chosen by the ctypes loader (wgx/_lib.py) is the one that runs.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <string>

#include "wgx.h"

namespace {

decltype(&wgx_last_error) f_last_error;
decltype(&wgx_kv_append) f_append;
decltype(&wgx_paged_attention_scratch_bytes) f_attention_bytes;
decltype(&wgx_paged_attention) f_attention;
decltype(&wgx_cache_evict) f_evict;
decltype(&wgx_beam_search_scratch_bytes) f_beam_bytes;
decltype(&wgx_beam_search_step) f_beam;
PyObject *g_error;  // wgx.WgxError

struct Failure {
  int code;
  std::string msg;
};
struct PythonError {};  // a Python exception is set

// One call's arguments: Python objects by position.
struct Call {
  const char *op;
  PyObject *const *args;
  c10::DeviceIndex dev = -1;

  [[noreturn]] void fail(const std::string &msg) const {
    throw Failure{WGX_ERR_INVALID, std::string(op) + ": " + msg};
  }
  void check(int code) const {
    if (code != WGX_OK) throw Failure{code, f_last_error()};
  }
  static std::string list(c10::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
  }
  const at::Tensor &tensor(int i, const char *what) const {
    if (!THPVariable_Check(args[i])) fail(std::string(what) + " must be a torch.Tensor");
    return THPVariable_Unpack(args[i]);
  }
  bool none(int i) const { return args[i] == Py_None; }
  void on_device(const at::Tensor &t, const char *what) const {
    if (!t.is_cuda() || t.get_device() != dev) fail(std::string(what) + " must be on the cache's device");
  }
  // a dense tensor of a type and shape
  template <typename P>
  P *dense(int i, const char *what, at::ScalarType type, c10::IntArrayRef shape) const {
    const at::Tensor &t = tensor(i, what);
    if (t.scalar_type() != type)
      fail(std::string(what) + " must be " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
    if (t.sizes() != shape)
      fail(std::string(what) + " shape " + list(t.sizes()) + " !== expected " + list(shape));
    if (!t.is_contiguous()) fail(std::string(what) + " must be contiguous");
    on_device(t, what);
    return static_cast<P *>(t.data_ptr());
  }
  template <typename P>
  P *optional(int i, const char *what, at::ScalarType type, c10::IntArrayRef shape) const {
    return none(i) ? nullptr : dense<P>(i, what, type, shape);
  }
  // flags are bool or uint8
  uint8_t *flags(int i, const char *what, c10::IntArrayRef shape) const {
    return dense<uint8_t>(i, what, flag_type(tensor(i, what), what), shape);
  }
  at::ScalarType flag_type(const at::Tensor &t, const char *what) const {
    if (t.scalar_type() != at::kBool && t.scalar_type() != at::kByte)
      fail(std::string(what) + " must be bool or uint8, got " + c10::toString(t.scalar_type()));
    return t.scalar_type();
  }
  void rows(const at::Tensor &t, const char *what, at::ScalarType type) const {
    if (t.scalar_type() != type) fail("Tensors must have matching float32 or float16 dtype");
    on_device(t, what);
    if (t.dim() < 1 || (t.stride(-1) != 1 && t.size(-1) != 1)) fail(std::string(what) + " must have a unit last stride");
  }
  int32_t i32(int64_t v, const char *what) const {
    if (v < INT32_MIN || v > INT32_MAX) fail(std::string(what) + " out of range");
    return int32_t(v);
  }
  int32_t integer(int i, const char *what) const {
    const long long v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return i32(v, what);
  }
  // the device of tensor i: the call's
  void device_of(const at::Tensor &t) {
    if (!t.is_cuda()) fail("tensors must be on a CUDA device");
    dev = t.get_device();
  }

  static int dtype(at::ScalarType t) { return t == at::kFloat ? WGX_FLOAT32 : WGX_FLOAT16; }
  static bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kHalf; }

  void cache(wgx_kv_cache &c, int k_at, int v_at, int table_at, bool layered) {
    const at::Tensor &k = tensor(k_at, "k_cache"), &v = tensor(v_at, "v_cache"),
                     &t = tensor(table_at, "page_table");
    if (dev < 0) device_of(k);
    if (!is_float(k.scalar_type())) fail("Tensors must have matching float32 or float16 dtype");
    rows(v, "v_cache", k.scalar_type());
    rows(k, "k_cache", k.scalar_type());
    if (k.sizes() != v.sizes()) fail("v_cache shape " + list(v.sizes()) + " !== expected " + list(k.sizes()));
    const int o = layered && k.dim() == 5 ? 1 : 0;
    if (k.dim() != 4 + o) fail("a cache is [pages, kv_heads, page_size, head_dim]");
    if (t.dim() != 2 || t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev)
      fail("page_table must be a 2-D int32 tensor on the cache's device");
    if (t.stride(1) != 1 && t.size(1) != 1) fail("page_table must have a unit last stride");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.page_table = static_cast<const int32_t *>(t.data_ptr());
    c.k_layer_stride = o ? k.stride(0) : 0;
    c.v_layer_stride = o ? v.stride(0) : 0;
    c.layers = o ? i32(k.size(0), "layers") : 1;
    c.k_page_stride = k.stride(o);
    c.k_head_stride = k.stride(o + 1);
    c.k_slot_stride = k.stride(o + 2);
    c.v_page_stride = v.stride(o);
    c.v_head_stride = v.stride(o + 1);
    c.v_slot_stride = v.stride(o + 2);
    c.table_stride = t.stride(0);
    c.batch = i32(t.size(0), "batch");
    c.kv_heads = i32(k.size(o + 1), "kv_heads");
    c.head_dim = i32(k.size(o + 3), "head_dim");
    c.dtype = dtype(k.scalar_type());
    c.pages = i32(k.size(o), "pages");
    c.page_size = i32(k.size(o + 2), "page_size");
    c.table_width = i32(t.size(1), "page table width");
  }
  // scratch memory: the workspace given, or torch's (stream-ordered)
  at::Tensor workspace(int i, uint64_t bytes) const {
    if (none(i))
      return at::empty({int64_t(bytes)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev));
    const at::Tensor &t = tensor(i, "workspace");
    if (t.scalar_type() != at::kByte || !t.is_contiguous() || !t.is_cuda() || t.get_device() != dev)
      fail("workspace must be a contiguous uint8 tensor on the cache's device");
    return t;
  }
  // what a call has written counts as written for autograd: saved tensors that
  // were overwritten are noticed
  void written(std::initializer_list<int> at) const {
    for (int i : at) {
      if (none(i)) continue;
      const at::Tensor &t = THPVariable_Unpack(args[i]);
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
  }
  void *stream() const { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
};

template <typename F>
PyObject *call(const char *op, int want, PyObject *const *args, Py_ssize_t n, F &&body) {
  try {
    Call c{op, args};
    if (n != want) c.fail("expected " + std::to_string(want) + " args, got " + std::to_string(n));
    return body(c);
  } catch (const Failure &f) {
    PyObject *a = Py_BuildValue("(is)", f.code, f.msg.c_str());
    if (a) PyErr_SetObject(g_error, a);
    Py_XDECREF(a);
  } catch (const PythonError &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// k, v, k_cache, v_cache, page_table, lengths, lengths_out, seen, seen_out,
// positions, weights
PyObject *kv_append(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return call("kv_append", 11, args, n, [](Call &c) -> PyObject * {
    wgx_kv_append_args a{};
    c.cache(a.cache, 2, 3, 4, false);
    const int64_t B = a.cache.batch, H = a.cache.kv_heads, D = a.cache.head_dim;
    const at::ScalarType dt = c.tensor(2, "k_cache").scalar_type();
    const at::Tensor &k = c.tensor(0, "k"), &v = c.tensor(1, "v");
    c.rows(k, "k", dt);
    c.rows(v, "v", dt);
    if (k.dim() != 4 || k.size(0) != B || k.size(2) != H || k.size(3) != D || v.sizes() != k.sizes())
      c.fail("k and v must be [" + std::to_string(B) + ", tokens, " + std::to_string(H) + ", " +
             std::to_string(D) + "], got " + Call::list(k.sizes()) + " and " + Call::list(v.sizes()));
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.k_batch_stride = k.stride(0);
    a.k_token_stride = k.stride(1);
    a.k_head_stride = k.stride(2);
    a.v_batch_stride = v.stride(0);
    a.v_token_stride = v.stride(1);
    a.v_head_stride = v.stride(2);
    a.tokens = c.i32(k.size(1), "tokens");
    a.lengths = c.dense<int32_t>(5, "lengths", at::kInt, {B});
    a.lengths_out = c.dense<int32_t>(6, "lengths_out", at::kInt, {B});
    a.seen = c.optional<int32_t>(7, "seen", at::kInt, {B});
    a.seen_out = c.optional<int32_t>(8, "seen_out", at::kInt, {B});
    if (!c.none(9) || !c.none(10)) {
      const at::Tensor &t = c.none(9) ? c.tensor(10, "weights") : c.tensor(9, "positions");
      a.slots = t.dim() ? t.size(-1) : 0;
      a.positions = c.optional<int32_t>(9, "positions", at::kInt, {B, H, a.slots});
      a.weights = c.optional<float>(10, "weights", at::kFloat, {B, H, a.slots});
    }
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != c.dev) guard.set_index(c.dev);
    c.check(f_append(&a, c.stream()));
    c.written({2, 3, 6, 8, 9, 10});
    Py_RETURN_NONE;
  });
}

// q, k_cache, v_cache, page_table, lengths, out, scale, window, mask, weights,
// weights_out, workspace
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return call("paged_attention", 12, args, n, [](Call &c) -> PyObject * {
    wgx_paged_attention_args a{};
    c.cache(a.cache, 1, 2, 3, false);
    const int64_t B = a.cache.batch, H = a.cache.kv_heads, D = a.cache.head_dim;
    const at::ScalarType dt = c.tensor(1, "k_cache").scalar_type();
    const at::Tensor &q = c.tensor(0, "q");
    if (q.dim() != 3 || q.size(0) != B || q.size(2) != D)
      c.fail("q must be [" + std::to_string(B) + ", q_heads, " + std::to_string(D) + "], got " +
             Call::list(q.sizes()));
    c.rows(q, "q", dt);
    a.q = q.data_ptr();
    a.q_heads = c.i32(q.size(1), "q_heads");
    a.q_batch_stride = q.stride(0);
    a.q_head_stride = q.stride(1);
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != c.dev) guard.set_index(c.dev);
    at::Tensor out;
    if (c.none(5)) {
      out = at::empty(q.sizes(), q.options());
    } else {
      out = c.tensor(5, "out");
      c.rows(out, "out", dt);
      if (out.sizes() != q.sizes())
        c.fail("out shape " + Call::list(out.sizes()) + " !== expected " + Call::list(q.sizes()));
    }
    a.out = out.data_ptr();
    a.out_batch_stride = out.stride(0);
    a.out_head_stride = out.stride(1);
    a.lengths = c.dense<int32_t>(4, "lengths", at::kInt, {B});
    if (c.none(6)) {
      a.scale = float(1.0 / std::sqrt(double(D)));
    } else {
      const double s = PyFloat_AsDouble(c.args[6]);
      if (s == -1.0 && PyErr_Occurred()) throw PythonError{};
      a.scale = float(s);
    }
    a.window = c.integer(7, "window");
    if (!c.none(8)) {
      const at::Tensor &m = c.tensor(8, "mask");
      c.flag_type(m, "mask");
      if (m.dim() != 2 || m.size(0) != B || !m.is_cuda() || m.get_device() != c.dev ||
          (m.stride(1) != 1 && m.size(1) != 1))
        c.fail("mask must be [" + std::to_string(B) + ", slots] with a unit last stride");
      a.mask = static_cast<const uint8_t *>(m.data_ptr());
      a.mask_stride = m.stride(0);
      a.mask_width = c.i32(m.size(1), "mask width");
    }
    if (c.none(9) != c.none(10)) c.fail("weights and weights_out come together");
    if (!c.none(9)) {
      const at::Tensor &w = c.tensor(9, "weights");
      a.slots = w.dim() ? w.size(-1) : 0;
      a.weights = c.dense<float>(9, "weights", at::kFloat, {B, H, a.slots});
      a.weights_out = c.dense<float>(10, "weights_out", at::kFloat, {B, H, a.slots});
    }
    c.check(f_attention_bytes(&a, &a.scratch_bytes));
    const at::Tensor ws = c.workspace(11, a.scratch_bytes);
    a.scratch = ws.data_ptr();
    a.scratch_bytes = uint64_t(ws.numel());
    c.check(f_attention(&a, c.stream()));
    c.written({5, 10});
    return THPVariable_Wrap(out);
  });
}

// k_cache, v_cache, page_table, lengths, lengths_out, weights, weights_out,
// positions, positions_out, seen, budget, recent, sinks
PyObject *cache_evict(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return call("cache_evict", 13, args, n, [](Call &c) -> PyObject * {
    wgx_cache_evict_args a{};
    c.cache(a.cache, 0, 1, 2, false);
    const int64_t B = a.cache.batch, H = a.cache.kv_heads;
    a.lengths = c.dense<int32_t>(3, "lengths", at::kInt, {B});
    a.lengths_out = c.dense<int32_t>(4, "lengths_out", at::kInt, {B});
    const at::Tensor &w = c.tensor(5, "weights");
    a.slots = w.dim() ? w.size(-1) : 0;
    a.weights = c.dense<float>(5, "weights", at::kFloat, {B, H, a.slots});
    a.weights_out = c.dense<float>(6, "weights_out", at::kFloat, {B, H, a.slots});
    a.positions = c.dense<int32_t>(7, "positions", at::kInt, {B, H, a.slots});
    a.positions_out = c.dense<int32_t>(8, "positions_out", at::kInt, {B, H, a.slots});
    a.seen = c.dense<int32_t>(9, "seen", at::kInt, {B});
    a.budget = c.integer(10, "budget");
    a.recent = c.integer(11, "recent");
    a.sinks = c.integer(12, "sinks");
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != c.dev) guard.set_index(c.dev);
    c.check(f_evict(&a, c.stream()));
    c.written({0, 1, 4, 6, 8});
    Py_RETURN_NONE;
  });
}

// logits, scores, finished, scores_out, parents, tokens, finished_out, eos,
// k_cache, v_cache, page_table, lengths, spare, page_table_out, lengths_out,
// workspace
PyObject *beam_search_step(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return call("beam_search_step", 16, args, n, [](Call &c) -> PyObject * {
    wgx_beam_search_args a{};
    const at::Tensor &x = c.tensor(0, "logits");
    c.device_of(x);
    if (!Call::is_float(x.scalar_type()) || x.dim() != 3)
      c.fail("logits must be [batch, beams, vocab], float32 or float16");
    const int64_t B = x.size(0), W = x.size(1), V = x.size(2);
    if (x.stride(2) != 1 && V != 1) c.fail("logits must have a unit last stride");
    a.logits = x.data_ptr();
    a.logits_batch_stride = x.stride(0);
    a.logits_beam_stride = x.stride(1);
    a.batch = c.i32(B, "batch");
    a.beams = c.i32(W, "beams");
    a.vocab = c.i32(V, "vocabulary");
    a.dtype = Call::dtype(x.scalar_type());
    a.scores = c.dense<float>(1, "scores", at::kFloat, {B, W});
    a.finished = c.flags(2, "finished", {B, W});
    a.scores_out = c.dense<float>(3, "scores_out", at::kFloat, {B, W});
    a.parents = c.dense<int32_t>(4, "parents", at::kInt, {B, W});
    a.tokens = c.dense<int32_t>(5, "tokens", at::kInt, {B, W});
    a.finished_out = c.flags(6, "finished_out", {B, W});
    a.eos = c.integer(7, "eos");
    if (!c.none(8)) {
      for (int i = 9; i <= 14; ++i)
        if (c.none(i)) c.fail("the cache's arguments come together");
      c.cache(a.cache, 8, 9, 10, true);
      c.on_device(c.tensor(8, "k_cache"), "logits");
      a.lengths = c.dense<int32_t>(11, "lengths", at::kInt, {B * W});
      a.spare = c.dense<int32_t>(12, "spare", at::kInt, {B * W});
      a.page_table_out = c.dense<int32_t>(13, "page_table_out", at::kInt, {B * W, a.cache.table_width});
      a.lengths_out = c.dense<int32_t>(14, "lengths_out", at::kInt, {B * W});
    }
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != c.dev) guard.set_index(c.dev);
    c.check(f_beam_bytes(&a, &a.scratch_bytes));
    const at::Tensor ws = c.workspace(15, a.scratch_bytes);
    a.scratch = ws.data_ptr();
    a.scratch_bytes = uint64_t(ws.numel());
    c.check(f_beam(&a, c.stream()));
    c.written({3, 4, 5, 6, 8, 9, 13, 14});
    Py_RETURN_NONE;
  });
}

// init(error class, {entry point: address})
PyObject *init(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "init(error, addresses)");
    return nullptr;
  }
  auto get = [&](const char *name, auto &f) {
    PyObject *v = PyDict_GetItemString(args[1], name);
    void *p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ImportError, name);
      return false;
    }
    f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
    return true;
  };
  if (!get("wgx_last_error", f_last_error) || !get("wgx_kv_append", f_append) ||
      !get("wgx_paged_attention_scratch_bytes", f_attention_bytes) ||
      !get("wgx_paged_attention", f_attention) || !get("wgx_cache_evict", f_evict) ||
      !get("wgx_beam_search_scratch_bytes", f_beam_bytes) || !get("wgx_beam_search_step", f_beam))
    return nullptr;
  Py_INCREF(args[0]);
  Py_XSETREF(g_error, args[0]);
  Py_RETURN_NONE;
}

#define WGX_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {WGX_METHOD(init),        WGX_METHOD(kv_append),        WGX_METHOD(paged_attention),
                         WGX_METHOD(cache_evict), WGX_METHOD(beam_search_step), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&module); }
