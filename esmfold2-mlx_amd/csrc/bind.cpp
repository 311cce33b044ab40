// Short way from a Python call to the C ABI for the operators that are called with a few rows at a time, where a
// call costs more on the host than on the GPU: the checks of the ordinary case, the output's allocation and the launch
// in one native function (norm and rotation 12 -> 6 us a call, attention 10 -> 5, the e4m3 linear 9 -> 5).
//
// Each function takes its operands unchecked. It returns the result; or, where the call needs a workspace and was given
// none, its size as an int; or None for whatever is not the ordinary case (another device than the current one, tensor
// subclasses, layouts or values that are refused): the Python function then makes the call itself, with its checks
// and its messages. Nothing here refuses or changes anything.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/esmfold2_amd.h"

namespace {

// The C ABI's entry points, from the library that the package has loaded.
struct Entries {
  decltype(&qk_norm_rope) rope = nullptr;
  decltype(&packed_attention) attention = nullptr;
  decltype(&packed_attention_workspace_bytes) attention_ws = nullptr;
  decltype(&f8_linear) linear = nullptr;
  decltype(&f8_linear_workspace_bytes) linear_ws = nullptr;
} entry;

struct Other {};  // thrown where a call is not the ordinary case

void need(bool ok) {
  if (!ok) throw Other{};
}

const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_CheckExact(o));
  const at::Tensor& t = THPVariable_Unpack(o);
  need(t.is_cuda() && t.layout() == at::kStrided);
  return t;
}

int dtype_of(const at::Tensor& t) {
  need(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16);
  return t.scalar_type() == at::kHalf ? ESM_F16 : ESM_BF16;
}

int small(int64_t v) {
  need(v >= 0 && v < INT32_MAX);
  return (int)v;
}

// A 16-bit [rows, heads, d] operand: sizes, strides (one that nothing is reached by says nothing).
struct Rows {
  const void* p;
  int T, H, d;
  int64_t st, sh;
  explicit Rows(const at::Tensor& t) {
    need(t.dim() == 3 && t.numel() > 0);
    p = t.const_data_ptr();
    T = small(t.size(0)), H = small(t.size(1)), d = small(t.size(2));
    need(t.stride(2) == 1);
    st = T > 1 ? t.stride(0) : ((int64_t)H * d + 7) / 8 * 8;
    sh = H > 1 ? t.stride(1) : 0;
  }
};

bool same_kind(const at::Tensor& a, const at::Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.get_device() == b.get_device();
}

// A contiguous auxiliary tensor of one type on the operands' device.
const at::Tensor& aux(PyObject* o, at::ScalarType type, int device) {
  const at::Tensor& t = tensor(o);
  need(t.scalar_type() == type && t.get_device() == device && t.is_contiguous());
  return t;
}

const float* weight(PyObject* o, int heads, int d, int device, int& each) {
  each = 0;
  if (o == Py_None) return nullptr;
  const at::Tensor& t = aux(o, at::kFloat, device);
  need(t.numel() == d || t.numel() == (int64_t)heads * d);
  each = t.numel() != d;
  return (const float*)t.const_data_ptr();
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Other{};
  }
  return v;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Other{};
  }
  return v;
}
bool truth(PyObject* o) {
  need(o == Py_True || o == Py_False);
  return o == Py_True;
}

void* stream_on(int device) {
  need(device == c10::hip::current_device());
  return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
}

// The body of a function: its result, None for Other, torch's exceptions as Python's.
template <class F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Other&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// q, k, freq, positions or None, gain, interleaved, norm (0, 1, 2), over the row, q_w, k_w or None, eps -> (q', k')
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 11 && entry.rope);
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]);
    const int dtype = dtype_of(q), device = q.get_device();
    need(same_kind(q, k));
    const Rows rq(q), rk(k);
    need(rq.T == rk.T && rq.d == rk.d);
    const at::Tensor& freq = aux(a[2], at::kDouble, device);
    const void* pos = nullptr;
    bool wide = false;
    if (a[3] != Py_None) {
      const at::Tensor& t = tensor(a[3]);
      wide = t.scalar_type() == at::kLong;
      need((wide || t.scalar_type() == at::kInt) && t.get_device() == device && t.is_contiguous() && t.numel() == rq.T);
      pos = t.const_data_ptr();
    }
    int qe, ke;
    const float *qw = weight(a[8], rq.H, rq.d, device, qe), *kw = weight(a[9], rk.H, rk.d, device, ke);
    const double gain = number(a[4]), eps = number(a[10]);
    const int norm = small(whole(a[6]));
    const bool inter = truth(a[5]), row = truth(a[7]);
    void* stream = stream_on(device);
    at::Tensor qo = at::empty({rq.T, rq.H, rq.d}, q.options()), ko = at::empty({rk.T, rk.H, rk.d}, k.options());
    need(entry.rope(rq.p, rk.p, qo.data_ptr(), ko.data_ptr(), rq.st, rq.sh, rk.st, rk.sh, (int64_t)rq.H * rq.d, rq.d,
                    (int64_t)rk.H * rk.d, rk.d, qw, qe, kw, ke, (float)eps, pos, wide, (const double*)freq.const_data_ptr(),
                    (float)gain, rq.T, rq.H, rk.H, rq.d, small(2 * freq.numel()), norm, row, inter, dtype, stream) == ESM_OK);
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyObject *x = THPVariable_Wrap(std::move(qo)), *y = THPVariable_Wrap(std::move(ko));
    if (!x || !y) {
      Py_XDECREF(x);
      Py_XDECREF(y);
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, 0, x);
    PyTuple_SET_ITEM(out, 1, y);
    return out;
  });
}

// q, k, v, cu_q, cu_k or None, causal, scale or None, workspace address (0: none), its bytes -> o, or bytes needed
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 9 && entry.attention);
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    const int dtype = dtype_of(q), device = q.get_device();
    need(same_kind(q, k) && same_kind(q, v));
    const Rows rq(q), rk(k), rv(v);
    need(rk.T == rv.T && rk.H == rv.H && rk.d == rv.d && rk.d == rq.d && rq.H % rk.H == 0);
    const at::Tensor& cq = aux(a[3], at::kInt, device);
    const at::Tensor& ck = a[4] == Py_None ? cq : aux(a[4], at::kInt, device);
    need((a[4] != Py_None || rq.T == rk.T) && cq.numel() >= 1 && ck.numel() == cq.numel());
    const int seqs = small(cq.numel() - 1);
    const bool causal = truth(a[5]);
    const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)rq.d) : number(a[6]);
    void* ws = (void*)(uintptr_t)whole(a[7]);
    const int64_t have = whole(a[8]);
    void* stream = stream_on(device);
    const size_t bytes = entry.attention_ws(seqs, rq.T, rk.T, rq.H, rk.H, rq.d);
    if (bytes > 0 && !ws) return PyLong_FromSize_t(bytes);
    at::Tensor o = at::empty({rq.T, rq.H, rq.d}, q.options());
    need(entry.attention(rq.p, rk.p, rv.p, o.data_ptr(), rq.st, rq.sh, rk.st, rk.sh, rv.st, rv.sh, (int64_t)rq.H * rq.d,
                         rq.d, (const int*)cq.const_data_ptr(), (const int*)ck.const_data_ptr(), seqs, rq.T, rk.T, rq.H, rk.H, rq.d, causal,
                         (float)scale, dtype, bytes ? ws : nullptr, bytes ? (size_t)have : 0, stream) == ESM_OK);
    return THPVariable_Wrap(std::move(o));
  });
}

// x [M, K], packed codes, scales, N, workspace address (0: none), its bytes -> y, or bytes needed
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 6 && entry.linear);
    const at::Tensor& x = tensor(a[0]);
    const int dtype = dtype_of(x), device = x.get_device();
    need(x.dim() == 2 && x.numel() > 0 && x.stride(1) == 1);
    const int M = small(x.size(0)), K = small(x.size(1)), N = small(whole(a[3]));
    const int64_t st = M > 1 ? x.stride(0) : ((int64_t)K + 7) / 8 * 8;
    const at::Tensor &codes = aux(a[1], at::kByte, device), &scales = aux(a[2], at::kFloat, device);
    const int64_t kb = ((int64_t)K + 127) / 128;
    need(codes.numel() == ((int64_t)N + 63) / 64 * kb * 8192 && scales.numel() == ((int64_t)N + 127) / 128 * kb);
    void* ws = (void*)(uintptr_t)whole(a[4]);
    const int64_t have = whole(a[5]);
    void* stream = stream_on(device);
    const size_t bytes = entry.linear_ws(M, K, N);
    if (bytes > 0 && !ws) return PyLong_FromSize_t(bytes);
    at::Tensor y = at::empty({M, N}, x.options());
    need(entry.linear(x.const_data_ptr(), st, (const uint8_t*)codes.const_data_ptr(), (const float*)scales.const_data_ptr(), y.data_ptr(), M,
                      K, N, dtype, bytes ? ws : nullptr, bytes ? (size_t)have : 0, stream) == ESM_OK);
    return THPVariable_Wrap(std::move(y));
  });
}

// The addresses of the entry points, in the order of Entries.
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[5];
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "connect: five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; i++) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  entry.rope = (decltype(entry.rope))p[0];
  entry.attention = (decltype(entry.attention))p[1];
  entry.attention_ws = (decltype(entry.attention_ws))p[2];
  entry.linear = (decltype(entry.linear))p[3];
  entry.linear_ws = (decltype(entry.linear_ws))p[4];
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"qk_norm_rope", FAST(rope)},       {"packed_attention", FAST(attention)},
                         {"f8_linear", FAST(linear)},        {"connect", FAST(connect)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_esm_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Read back by the build to tell whether the module was compiled from the current sources and in this environment.
extern "C" __attribute__((used, visibility("default"))) const char esm_bind_tag[] = "ESMSRC:" ESM_SOURCE_HASH " ESMENV:" ESM_ENVIRONMENT;

PyMODINIT_FUNC PyInit__esm_bind(void) { return PyModule_Create(&module); }
