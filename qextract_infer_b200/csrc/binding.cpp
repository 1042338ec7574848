// Python binding of the head norm + rotation and of the 4-bit ring's operators:
// argument checks, outputs and scratch from torch's allocator, the current
// stream of the tensors' device, then one call of the C ABI (include/qx_b200.h).
// These operators run once a layer and decode step, on a few microseconds of GPU
// work: through ctypes the host side of a call (checks, allocations, argument
// conversion) took 12 to 22 us, here 4 to 8.  The functions are called by the
// documented ones of the package's _C module, which forwards its arguments in order.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "qx_b200.h"

namespace {

PyObject* g_error = nullptr;  // the package's QXError: a C-ABI call returned a negative status

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  PyErr_SetString(PyExc_RuntimeError, msg);
  throw python_error();
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a CUDA tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse("%s must be a CUDA tensor", name);
  if (!t.is_contiguous()) refuse("%s must be contiguous", name);
  return t;
}

const at::Tensor& half(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kHalf) refuse("%s must be float16, got %s", name, c10::toString(t.scalar_type()));
  return t;
}

int64_t integer(PyObject* o) {
  if (PyLong_CheckExact(o)) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  PyObject* i = PyNumber_Index(o);
  if (!i) throw python_error();
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

int small(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v > INT32_MAX || v < INT32_MIN) refuse("%s=%lld is out of range", name, (long long)v);
  return int(v);
}

// sizes of tensors that reach the C ABI as int
int size32(const at::Tensor& t, int64_t d, const char* what) {
  const int64_t v = t.size(d);
  if (v > INT32_MAX) refuse("%s: a dimension of %lld is too large", what, (long long)v);
  return int(v);
}

float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return float(v);
}

float scale_of(PyObject* o) { return o == Py_None ? 0.f : real(o); }

void arguments(const char* what, Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("%s: %zd arguments, %zd expected", what, n, want);
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, at::Device dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, dev, std::nullopt));
}

void same_device(const char* what, at::Device dev, std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t->device() != dev) refuse("%s: tensors must be on one device", what);
}

void check(int64_t rc, const char* what) {
  if (rc >= 0) return;
  char msg[1200];
  snprintf(msg, sizeof(msg), "%s: %s (status %d)", what, qx_last_error(), int(rc));
  PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, msg);
  throw python_error();
}

qx_stream_t stream_of(at::Device dev) {
  return reinterpret_cast<qx_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

PyObject* wrap(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New(Py_ssize_t(ts.size()));
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

// a layer's 4-bit ring, checked
struct Ring {
  at::Device dev{at::kCUDA};
  int batch, kv_heads, head_dim, group, sink, window;
  int64_t count = 0;
  const int64_t* counts = nullptr;
  unsigned char *k_codes, *v_codes;
  char *k_params, *v_params;

  // o: codes, params, count, sink, window
  Ring(const char* what, PyObject* const* o) {
    const at::Tensor &codes = tensor(o[0], "codes"), &params = tensor(o[1], "params");
    if (codes.scalar_type() != at::kByte || params.scalar_type() != at::kShort || codes.dim() != 5 || params.dim() != 5 ||
        codes.size(0) != 2 || params.size(0) != 2)
      refuse("%s: codes must be uint8 [2, B, Hkv, slots, D / 2] and params int16 [2, B, Hkv, slots, D / group]", what);
    sink = small(o[3], "sink");
    window = small(o[4], "window");
    const int64_t slots = qx_ring_q4_slots(sink, window);
    check(slots, what);
    if (codes.size(3) != slots || params.size(1) != codes.size(1) || params.size(2) != codes.size(2) || params.size(3) != slots)
      refuse("%s: codes and params must have %lld slots (sink + window rounded up to 64), got %s and %s", what,
             (long long)slots, shape_of(codes).c_str(), shape_of(params).c_str());
    batch = size32(codes, 1, what);
    kv_heads = size32(codes, 2, what);
    const int64_t groups = params.size(4), d = 2 * codes.size(4);
    if (groups < 1 || d % groups || d > 65536) refuse("%s: %lld groups do not divide head_dim %lld", what, (long long)groups, (long long)d);
    head_dim = int(d);
    group = int(d / groups);
    dev = codes.device();
    same_device(what, dev, {&params});
    if (THPVariable_Check(o[2])) {
      const at::Tensor& c = tensor(o[2], "count");
      if (c.scalar_type() != at::kLong || c.dim() != 1 || c.size(0) != batch)
        refuse("%s: a count tensor must be int64 [%d]", what, batch);
      same_device(what, dev, {&c});
      counts = c.const_data_ptr<int64_t>();
    } else {
      count = integer(o[2]);
    }
    k_codes = static_cast<unsigned char*>(codes.data_ptr());
    v_codes = k_codes + codes.numel() / 2;
    k_params = static_cast<char*>(params.data_ptr());
    v_params = k_params + params.numel();  // half of the 16-bit words
  }

  // new keys and values [B, tokens, Hkv, D]
  void check_new(const char* what, const at::Tensor& k, const at::Tensor& v, int64_t tokens) const {
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.size(0) != batch || k.size(2) != kv_heads || k.size(3) != head_dim ||
        (tokens >= 0 && k.size(1) != tokens))
      refuse("%s: new keys and values must be [%d, %s, %d, %d], got %s and %s", what, batch,
             tokens < 0 ? "T" : std::to_string(tokens).c_str(), kv_heads, head_dim, shape_of(k).c_str(), shape_of(v).c_str());
    same_device(what, dev, {&k, &v});
  }
};

// qkv, q_heads, kv_heads, q_norm, k_norm, eps, cos, sin -> (q, k, v)
PyObject* qk_norm_rope(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("qk_norm_rope", n, 8);
  const at::Tensor &qkv = half(o[0], "qkv"), &qn = half(o[3], "q_norm"), &kn = half(o[4], "k_norm");
  const int hq = small(o[1], "q_heads"), hkv = small(o[2], "kv_heads");
  const int64_t d = qn.numel();
  if (hq < 1 || hkv < 1 || qkv.dim() != 3 || kn.numel() != d || d > 65536 || qkv.size(2) != (int64_t(hq) + 2 * int64_t(hkv)) * d)
    refuse("qk_norm_rope: qkv must be [B, T, (q_heads + 2 kv_heads) * head_dim]");
  const int64_t B = qkv.size(0), T = qkv.size(1);
  const at::Tensor &cos = tensor(o[6], "cos"), &sin = tensor(o[7], "sin");
  for (const at::Tensor* t : {&cos, &sin}) {
    const bool rows = (t->dim() == 2 && t->size(0) == T && t->size(1) == d) ||
                      (t->dim() == 3 && t->size(0) == B && t->size(1) == T && t->size(2) == d);
    if (t->scalar_type() != at::kFloat || !rows || t->dim() != cos.dim())
      refuse("%s must be float32 [%lld, %lld] or [%lld, %lld, %lld]", t == &cos ? "cos" : "sin", (long long)T, (long long)d,
             (long long)B, (long long)T, (long long)d);
  }
  const at::Device dev = qkv.device();
  same_device("qk_norm_rope", dev, {&qn, &kn, &cos, &sin});
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor q = empty({B, T, hq, d}, at::kHalf, dev), k = empty({B, T, hkv, d}, at::kHalf, dev),
             v = empty({B, T, hkv, d}, at::kHalf, dev);
  check(qx_qk_norm_rope(qkv.const_data_ptr(), B * T, hq, hkv, int(d), qn.const_data_ptr(), kn.const_data_ptr(), real(o[5]),
                        cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), std::max<int64_t>(1, cos.dim() == 2 ? T : B * T),
                        q.data_ptr(), k.data_ptr(), v.data_ptr(), stream_of(dev)),
        "qk_norm_rope");
  return wrap({q, k, v});
  END_HANDLE_TH_ERRORS
}

// new_k, new_v, codes, params, count, sink, window
PyObject* ring_append_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("ring_append_q4", n, 7);
  const at::Tensor &k = half(o[0], "new_k"), &v = half(o[1], "new_v");
  const Ring r("ring_append_q4", o + 2);
  r.check_new("ring_append_q4", k, v, -1);
  const c10::cuda::CUDAGuard guard(r.dev);
  check(qx_ring_append_q4(r.k_codes, r.k_params, r.v_codes, r.v_params, k.const_data_ptr(), v.const_data_ptr(), r.batch,
                          size32(k, 1, "ring_append_q4"), r.kv_heads, r.head_dim, r.group, r.sink, r.window, r.count,
                          r.counts, stream_of(r.dev)),
        "ring_append_q4");
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// codes, params, count, sink, window -> (k, v)
PyObject* ring_gather_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("ring_gather_q4", n, 5);
  if (THPVariable_Check(o[2])) refuse("ring_gather_q4: count must be a number (it gives the output's length)");
  const Ring r("ring_gather_q4", o);
  const int64_t valid =
      std::max<int64_t>(0, std::min<int64_t>(r.count, r.sink)) + std::max<int64_t>(0, std::min<int64_t>(r.count - r.sink, r.window));
  const c10::cuda::CUDAGuard guard(r.dev);
  at::Tensor k = empty({r.batch, valid, r.kv_heads, r.head_dim}, at::kHalf, r.dev),
             v = empty({r.batch, valid, r.kv_heads, r.head_dim}, at::kHalf, r.dev);
  check(qx_ring_gather_q4(r.k_codes, r.k_params, r.v_codes, r.v_params, k.data_ptr(), v.data_ptr(), r.batch, r.kv_heads,
                          r.head_dim, r.group, r.sink, r.window, r.count, stream_of(r.dev)),
        "ring_gather_q4");
  return wrap({k, v});
  END_HANDLE_TH_ERRORS
}

// Scratch comes from torch's allocator for each call: calls on different streams and
// captured graphs never share it.
// q, codes, params, count, sink, window, softmax_scale -> out
PyObject* decode_attention_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "decode_attention_q4";
  arguments(what, n, 7);
  const at::Tensor& q = half(o[0], "q");
  const Ring r(what, o + 1);
  if (q.dim() != 3 || q.size(0) != r.batch || q.size(2) != r.head_dim)
    refuse("%s: q must be [%d, Hq, %d], got %s", what, r.batch, r.head_dim, shape_of(q).c_str());
  same_device(what, r.dev, {&q});
  const int hq = size32(q, 1, what);
  const c10::cuda::CUDAGuard guard(r.dev);
  at::Tensor out = empty(q.sizes(), at::kHalf, r.dev), scratch;
  const size_t need = qx_decode_attention_q4_workspace_size(r.batch, hq, r.kv_heads, r.head_dim, r.sink, r.window);
  if (need) scratch = empty({int64_t(need)}, at::kByte, r.dev);
  check(qx_decode_attention_q4(q.const_data_ptr(), r.k_codes, r.k_params, r.v_codes, r.v_params, out.data_ptr(), r.batch, hq,
                               r.kv_heads, r.head_dim, r.group, r.sink, r.window, r.count, r.counts, scale_of(o[6]),
                               need ? scratch.data_ptr() : nullptr, need, stream_of(r.dev)),
        what);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// q, k_new, v_new, codes, params, count, sink, window, softmax_scale -> out
PyObject* prefill_attention_q4(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "prefill_attention_q4";
  arguments(what, n, 9);
  const at::Tensor &q = half(o[0], "q"), &k = half(o[1], "k_new"), &v = half(o[2], "v_new");
  const Ring r(what, o + 3);
  if (q.dim() != 4 || q.size(0) != r.batch || q.size(3) != r.head_dim)
    refuse("%s: q must be [%d, n, Hq, %d], got %s", what, r.batch, r.head_dim, shape_of(q).c_str());
  same_device(what, r.dev, {&q});
  r.check_new(what, k, v, q.size(1));
  const int tokens = size32(q, 1, what), hq = size32(q, 2, what);
  const c10::cuda::CUDAGuard guard(r.dev);
  at::Tensor out = empty(q.sizes(), at::kHalf, r.dev), scratch;
  const size_t need = qx_prefill_attention_q4_workspace_size(r.batch, tokens, hq, r.kv_heads, r.head_dim, r.sink, r.window);
  if (need) scratch = empty({int64_t(need)}, at::kByte, r.dev);
  check(qx_prefill_attention_q4(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), r.k_codes, r.k_params, r.v_codes,
                                r.v_params, out.data_ptr(), r.batch, tokens, hq, r.kv_heads, r.head_dim, r.group, r.sink,
                                r.window, r.count, r.counts, scale_of(o[8]), need ? scratch.data_ptr() : nullptr, need,
                                stream_of(r.dev)),
        what);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XDECREF(g_error);
  g_error = cls;
  Py_RETURN_NONE;
}

#define QX_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {QX_FAST(qk_norm_rope),        QX_FAST(ring_append_q4),       QX_FAST(ring_gather_q4),
                         QX_FAST(decode_attention_q4), QX_FAST(prefill_attention_q4), {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module); }
