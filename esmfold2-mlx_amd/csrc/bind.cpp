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
#include <type_traits>

#include "../../include/esmfold2_amd.h"

namespace {

// The C ABI's entry points, from the library that the package has loaded.
struct Entries {
  decltype(&qk_norm_rope) rope = nullptr;
  decltype(&packed_attention) attention = nullptr;
  decltype(&packed_attention_workspace_bytes) attention_ws = nullptr;
  decltype(&f8_linear) linear = nullptr;
  decltype(&f8_linear_workspace_bytes) linear_ws = nullptr;
  decltype(&add_norm) norm = nullptr;
  decltype(&f8_rows_bytes) rows = nullptr;
  decltype(&f8_rows_scales_bytes) rows_scales = nullptr;
  decltype(&linear16) linear16_ = nullptr;
  decltype(&linear16_workspace_bytes) linear16_ws = nullptr;
  decltype(&linear16_packed_bytes) linear16_packed = nullptr;
  decltype(&f8_linear_end) end = nullptr;
  decltype(&f8_linear_end_workspace_bytes) end_ws = nullptr;
  decltype(&cache4_bytes) c4_bytes = nullptr;
  decltype(&cache4_append) c4_append = nullptr;
  decltype(&cache4_read) c4_read = nullptr;
  decltype(&cache4_attention) c4_attention = nullptr;
  decltype(&cache4_attention_workspace_bytes) c4_attention_ws = nullptr;
} entry;
constexpr int kEntries = sizeof(Entries) / sizeof(void*);

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

// A [rows, values] operand: its stride (one that nothing is reached by says nothing).
int64_t row_stride(const at::Tensor& t, int64_t rows, int64_t values) {
  need(t.dim() == 2 && t.size(0) == rows && t.size(1) == values && t.stride(1) == 1);
  return rows > 1 ? t.stride(0) : (values + 7) / 8 * 8;
}
// An optional fp32 parameter of n values.
const float* vector(PyObject* o, int64_t n, int device) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = aux(o, at::kFloat, device);
  need(t.numel() == n);
  return (const float*)t.const_data_ptr();
}
PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
  if (!x || !y) {
    Py_XDECREF(x);
    Py_XDECREF(y);
    Py_DECREF(out);
    return nullptr;
  }
  PyTuple_SET_ITEM(out, 0, x);
  PyTuple_SET_ITEM(out, 1, y);
  return out;
}

// x, y, w or None, b or None, alpha, norm (1, 2), eps, e4m3 -> (s, h), or (s, codes, scales); h of y's type
PyObject* norm_of_sum(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 8 && entry.norm);
    const at::Tensor &x = tensor(a[0]), &y = tensor(a[1]);
    const int dtype = dtype_of(y), device = x.get_device();
    const bool wide = x.scalar_type() == at::kFloat;
    need((wide || x.scalar_type() == y.scalar_type()) && y.get_device() == device && x.dim() == 2 && x.numel() > 0);
    const int T = small(x.size(0)), D = small(x.size(1));
    const int64_t x_st = row_stride(x, T, D), y_st = row_stride(y, T, D);
    const float *w = vector(a[2], D, device), *b = vector(a[3], D, device);
    const double alpha = number(a[4]), eps = number(a[6]);
    const int norm = small(whole(a[5]));
    const bool f8 = truth(a[7]);
    void* stream = stream_on(device);
    need(D % 16 == 0);
    at::Tensor s = at::empty({T, D}, x.options());
    if (!f8) {
      at::Tensor h = at::empty({T, D}, y.options());
      need(entry.norm(x.const_data_ptr(), wide, y.const_data_ptr(), (float)alpha, s.data_ptr(), h.data_ptr(), nullptr, nullptr, w, b,
                      (float)eps, norm, x_st, y_st, D, D, T, D, dtype, stream) == ESM_OK);
      return pair(std::move(s), std::move(h));
    }
    at::Tensor q = at::empty({(int64_t)entry.rows(T, D)}, x.options().dtype(at::kByte));
    at::Tensor c = at::empty({(int64_t)entry.rows_scales(T, D) / 4}, x.options().dtype(at::kFloat));
    need(entry.norm(x.const_data_ptr(), wide, y.const_data_ptr(), (float)alpha, s.data_ptr(), nullptr, (uint8_t*)q.data_ptr(), (float*)c.data_ptr(),
                    w, b, (float)eps, norm, x_st, y_st, D, 0, T, D, dtype, stream) == ESM_OK);
    PyObject* in = pair(std::move(q), std::move(c));
    PyObject* first = in ? THPVariable_Wrap(std::move(s)) : nullptr;
    PyObject* out = first ? PyTuple_New(2) : nullptr;
    if (!out) {
      Py_XDECREF(in);
      Py_XDECREF(first);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, 0, first);
    PyTuple_SET_ITEM(out, 1, in);
    return out;
  });
}

// What both linears' ends share: bias, gated, activation, residual, alpha, workspace address (0: none), its bytes.
struct End {
  const float* bias;
  const void* res = nullptr;
  int64_t r_st = 0;
  int gated, act, No;
  float alpha;
  void* ws;
  size_t have;
  End(PyObject* const* a, int M, int N, at::ScalarType type, int device) {
    bias = vector(a[0], N, device);
    gated = truth(a[1]);
    act = small(whole(a[2]));
    No = gated ? N / 2 : N;
    if (a[3] != Py_None) {
      const at::Tensor& r = tensor(a[3]);
      need(r.scalar_type() == type && r.get_device() == device);
      r_st = row_stride(r, M, No);
      res = r.const_data_ptr();
    }
    alpha = (float)number(a[4]);
    ws = (void*)(uintptr_t)whole(a[5]);
    have = (size_t)whole(a[6]);
  }
};

// x, packed, N, bias, gated, activation, residual, alpha, workspace address, its bytes -> y, or bytes needed
PyObject* lin16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 10 && entry.linear16_);
    const at::Tensor& x = tensor(a[0]);
    const int dtype = dtype_of(x), device = x.get_device();
    need(x.dim() == 2 && x.numel() > 0);
    const int M = small(x.size(0)), K = small(x.size(1)), N = small(whole(a[2]));
    const int64_t st = row_stride(x, M, K);
    const at::Tensor& packed = aux(a[1], at::kByte, device);
    const End e(a + 3, M, N, x.scalar_type(), device);
    need(packed.numel() > 0 && (size_t)packed.numel() == entry.linear16_packed(N, K, e.gated));
    void* stream = stream_on(device);
    const size_t bytes = entry.linear16_ws(M, K, N, e.gated);
    if (bytes > 0 && !e.ws) return PyLong_FromSize_t(bytes);
    at::Tensor y = at::empty({M, e.No}, x.options());
    need(entry.linear16_(x.const_data_ptr(), st, packed.const_data_ptr(), e.bias, e.res, e.r_st, e.alpha, e.act, e.gated, y.data_ptr(), M, K, N,
                         dtype, bytes ? e.ws : nullptr, bytes ? e.have : 0, stream) == ESM_OK);
    return THPVariable_Wrap(std::move(y));
  });
}

// codes and scales of the rows, M, K, whether y is bf16, packed codes, scales, N, then as above -> y, or bytes needed
PyObject* lin8_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 15 && entry.end);
    const at::Tensor& xq = tensor(a[0]);
    const int device = xq.get_device();
    const at::Tensor &q = aux(a[0], at::kByte, device), &sx = aux(a[1], at::kFloat, device);
    const int M = small(whole(a[2])), K = small(whole(a[3])), N = small(whole(a[7]));
    const bool bf16 = truth(a[4]);
    const at::Tensor &codes = aux(a[5], at::kByte, device), &scales = aux(a[6], at::kFloat, device);
    const int64_t kb = ((int64_t)K + 127) / 128;
    need(M > 0 && codes.numel() == ((int64_t)N + 63) / 64 * kb * 8192 && scales.numel() == ((int64_t)N + 127) / 128 * kb);
    need((size_t)q.numel() == entry.rows(M, K) && (size_t)sx.numel() * 4 == entry.rows_scales(M, K));
    const at::ScalarType type = bf16 ? at::kBFloat16 : at::kHalf;
    const End e(a + 8, M, N, type, device);
    void* stream = stream_on(device);
    const size_t bytes = entry.end_ws(M, K, N, e.gated, 1);
    if (bytes > 0 && !e.ws) return PyLong_FromSize_t(bytes);
    at::Tensor y = at::empty({M, e.No}, q.options().dtype(type));
    need(entry.end(nullptr, 0, (const uint8_t*)q.const_data_ptr(), (const float*)sx.const_data_ptr(), (const uint8_t*)codes.const_data_ptr(),
                   (const float*)scales.const_data_ptr(), e.bias, e.res, e.r_st, e.alpha, e.act, e.gated, y.data_ptr(), M, K, N, bf16 ? ESM_BF16 : ESM_F16,
                   bytes ? e.ws : nullptr, bytes ? e.have : 0, stream) == ESM_OK);
    return THPVariable_Wrap(std::move(y));
  });
}

// The cache, starts, lengths and table of a call.
struct Held {
  const at::Tensor &data, &cu, &lens, &table;
  int n, pages, width;
  Held(PyObject* d, PyObject* const* a, int heads, int dim, int device)
      : data(aux(d, at::kByte, device)), cu(aux(a[0], at::kInt, device)), lens(aux(a[1], at::kInt, device)), table(aux(a[2], at::kInt, device)) {
    n = small(lens.numel());
    const size_t each = heads > 0 && dim > 0 ? entry.c4_bytes(1, heads, dim) : 0;
    need(n > 0 && cu.numel() == (int64_t)n + 1 && table.dim() == 2 && table.size(0) == n && each > 0 && (size_t)data.numel() % each == 0);
    pages = small((int64_t)((size_t)data.numel() / each));
    width = small(table.size(1));
    need(pages > 0 && width > 0);
  }
  const int *c() const { return (const int*)cu.const_data_ptr(); }
  const int *l() const { return (const int*)lens.const_data_ptr(); }
  const int *t() const { return (const int*)table.const_data_ptr(); }
};

// data, k, v, cu, lens, table -> True
PyObject* c4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 6 && entry.c4_append);
    const at::Tensor &k = tensor(a[1]), &v = tensor(a[2]);
    const int dtype = dtype_of(k), device = k.get_device();
    need(same_kind(k, v));
    const Rows rk(k), rv(v);
    need(rk.T == rv.T && rk.H == rv.H && rk.d == rv.d);
    const Held h(a[0], a + 3, rk.H, rk.d, device);
    need(entry.c4_append(rk.p, rv.p, rk.st, rk.sh, rv.st, rv.sh, h.data.data_ptr(), h.c(), h.l(), h.t(), h.n, rk.T, rk.H, rk.d, h.pages, h.width, dtype,
                         stream_on(device)) == ESM_OK);
    Py_RETURN_TRUE;
  });
}

// data, rows, heads, head size, whether bf16, cu, lens, table -> (k, v)
PyObject* c4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 8 && entry.c4_read);
    const at::Tensor& data = tensor(a[0]);
    const int device = data.get_device(), T = small(whole(a[1])), H = small(whole(a[2])), d = small(whole(a[3]));
    const bool bf16 = truth(a[4]);
    const Held h(a[0], a + 5, H, d, device);
    need(T > 0);
    void* stream = stream_on(device);
    const auto type = data.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
    at::Tensor k = at::empty({T, H, d}, type), v = at::empty({T, H, d}, type);
    need(entry.c4_read(k.data_ptr(), v.data_ptr(), h.data.const_data_ptr(), h.c(), h.l(), h.t(), h.n, T, H, d, h.pages, h.width,
                       bf16 ? ESM_BF16 : ESM_F16, stream) == ESM_OK);
    return pair(std::move(k), std::move(v));
  });
}

// data, q, key heads, cu, lens, table, causal, scale or None, workspace address (0: none), its bytes -> o, or bytes needed
PyObject* c4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 10 && entry.c4_attention);
    const at::Tensor& q = tensor(a[1]);
    const int dtype = dtype_of(q), device = q.get_device(), Hk = small(whole(a[2]));
    const Rows r(q);
    need(Hk > 0 && r.H % Hk == 0);
    const Held h(a[0], a + 3, Hk, r.d, device);
    const bool causal = truth(a[6]);
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)r.d) : number(a[7]);
    void* ws = (void*)(uintptr_t)whole(a[8]);
    const int64_t have = whole(a[9]);
    void* stream = stream_on(device);
    const size_t bytes = entry.c4_attention_ws(h.n, r.T, h.width, r.H, Hk, r.d);
    if (bytes > 0 && !ws) return PyLong_FromSize_t(bytes);
    at::Tensor o = at::empty({r.T, r.H, r.d}, q.options());
    need(entry.c4_attention(r.p, o.data_ptr(), r.st, r.sh, (int64_t)r.H * r.d, r.d, h.data.const_data_ptr(), h.c(), h.l(), h.t(), h.n, r.T, r.H, Hk, r.d,
                            h.pages, h.width, causal, (float)scale, dtype, bytes ? ws : nullptr, bytes ? (size_t)have : 0, stream) == ESM_OK);
    return THPVariable_Wrap(std::move(o));
  });
}

// The addresses of the entry points, in the order of Entries.
PyObject* connect(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[kEntries];
  if (n != kEntries) {
    PyErr_Format(PyExc_TypeError, "connect: %d addresses", kEntries);
    return nullptr;
  }
  for (int i = 0; i < kEntries; i++) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  int i = 0;
  const auto set = [&](auto& f) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(p[i++]); };
  set(entry.rope), set(entry.attention), set(entry.attention_ws), set(entry.linear), set(entry.linear_ws);
  set(entry.norm), set(entry.rows), set(entry.rows_scales), set(entry.linear16_), set(entry.linear16_ws), set(entry.linear16_packed);
  set(entry.end), set(entry.end_ws), set(entry.c4_bytes), set(entry.c4_append), set(entry.c4_read), set(entry.c4_attention);
  set(entry.c4_attention_ws);
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"qk_norm_rope", FAST(rope)},       {"packed_attention", FAST(attention)},
                         {"f8_linear", FAST(linear)},        {"add_norm", FAST(norm_of_sum)},
                         {"linear16", FAST(lin16)},          {"f8_linear_rows", FAST(lin8_rows)},
                         {"cache4_append", FAST(c4_append)}, {"cache4_read", FAST(c4_read)},
                         {"cache4_attention", FAST(c4_attention)}, {"connect", FAST(connect)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_esm_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Read back by the build to tell whether the module was compiled from the current sources and in this environment.
extern "C" __attribute__((used, visibility("default"))) const char esm_bind_tag[] = "ESMSRC:" ESM_SOURCE_HASH " ESMENV:" ESM_ENVIRONMENT;

PyMODINIT_FUNC PyInit__esm_bind(void) { return PyModule_Create(&module); }
