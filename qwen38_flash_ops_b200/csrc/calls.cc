// The per-call part of ops.py in C++: argument checks, output allocation, the current stream, and the call into the C ABI.
// In Python that part took 10.6 us of an eager call (4.7 of them in the library and the launch), which was longer than the
// kernels of the small calls take.  Every function returns None where a call is not of the ordinary form - the Python code
// then makes its own checks and reports the error or goes its way - and an integer where the library refused it.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <vector>

#include "qfg.h"

namespace {

// addresses of the library's entry points, given by ops.py (which finds the library)
struct Entries {
  decltype(&qfg_skinny_gemm_compute) skinny_gemm;
  decltype(&qfg_argmax_rows) argmax_rows;
  decltype(&qfg_dequant_compute) dequant;
  decltype(&qfg_lmhead_compute) lmhead;
  decltype(&qfg_shared_expert_down_compute) shared_expert_down;
  decltype(&qfg_rmsnorm_quant) rmsnorm_quant;
  decltype(&qfg_row_quant) row_quant;
  decltype(&qfg_quant_gemm_compute) quant_gemm;
  decltype(&qfg_quant_mlp_workspace_bytes) quant_mlp_workspace_bytes;
  decltype(&qfg_quant_mlp) quant_mlp;
} g_lib;

// A plain CUDA tensor, or null: no subclass, no wrapper of a transform, nothing without memory of its own.
const at::Tensor* Plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet keys = t.key_set();
  if (!t.defined() || !keys.has(c10::DispatchKey::CUDA) || keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::FuncTorchBatched) ||
      keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Functionalize) || !t.has_storage())
    return nullptr;
  return &t;
}
const at::Tensor* Dense(PyObject* o) {  // a contiguous one
  const at::Tensor* t = Plain(o);
  return t != nullptr && t->is_contiguous() ? t : nullptr;
}
const at::Tensor* Bf16(PyObject* o) {
  const at::Tensor* t = Dense(o);
  return t != nullptr && t->scalar_type() == at::kBFloat16 ? t : nullptr;
}
bool Weight(PyObject* o, qfg_tensor2d* d) {
  const at::Tensor* t = Dense(o);
  if (t == nullptr || t->dim() != 2) return false;
  switch (t->scalar_type()) {
    case at::kBFloat16: d->dtype = QFG_BFLOAT16; break;
    case at::kHalf: d->dtype = QFG_FLOAT16; break;
    case at::kFloat: d->dtype = QFG_FLOAT; break;
    case at::kByte: d->dtype = QFG_UINT8; break;
    case at::kFloat8_e4m3fn: d->dtype = QFG_FLOAT8E4M3FN; break;
    default: return false;
  }
  d->data = t->data_ptr();
  d->rows = t->size(0);
  d->cols = t->size(1);
  return true;
}
void* Stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
PyObject* None() { Py_RETURN_NONE; }

// Neither a C++ exception (an allocation that failed, say) nor the error of a conversion crosses into Python with a None: the
// Python code meets it on its own way.
template <typename F>
PyObject* Guard(F&& f) {
  PyObject* r;
  try {
    r = f();
  } catch (...) {
    r = None();
  }
  if (r == Py_None) PyErr_Clear();
  return r;
}
template <typename F>
int Call(F&& f) {  // without the interpreter's lock, as a foreign call through ctypes
  int code;
  Py_BEGIN_ALLOW_THREADS;
  code = f();
  Py_END_ALLOW_THREADS;
  return code;
}

constexpr int kMaxTensors = 16;
// the elements of a list of widths
int Widths(PyObject* list, std::array<int64_t, kMaxTensors>* w) {
  if (!PyList_CheckExact(list) || PyList_GET_SIZE(list) > kMaxTensors) return -1;
  const int n = static_cast<int>(PyList_GET_SIZE(list));
  for (int i = 0; i < n; ++i) {
    (*w)[i] = PyLong_AsLongLong(PyList_GET_ITEM(list, i));
    if ((*w)[i] < 0) return -1;
  }
  return n;
}
PyObject* ListOf(const std::array<at::Tensor, kMaxTensors>& t, int n) {
  PyObject* list = PyList_New(n);
  for (int i = 0; list != nullptr && i < n; ++i) {
    PyObject* o = THPVariable_Wrap(t[i]);
    if (o == nullptr) {
      Py_DECREF(list);
      return nullptr;
    }
    PyList_SET_ITEM(list, i, o);
  }
  return list;
}
PyObject* TupleOf(std::initializer_list<at::Tensor> t) {
  PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(t.size()));
  Py_ssize_t i = 0;
  for (const at::Tensor& v : t) {
    PyObject* o = tuple != nullptr ? THPVariable_Wrap(v) : nullptr;
    if (o == nullptr) {
      Py_XDECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

// skinny_gemm(handle, x, weights, widths) -> [y, ...]
PyObject* SkinnyGemm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    if (n_args != 4 || !PyTuple_CheckExact(a[2])) return None();
    const void* op = PyLong_AsVoidPtr(a[0]);
    const at::Tensor* x = Bf16(a[1]);
    const Py_ssize_t n_weights = PyTuple_GET_SIZE(a[2]);
    std::array<int64_t, kMaxTensors> widths;
    const int n_out = Widths(a[3], &widths);
    if (op == nullptr || x == nullptr || x->dim() < 1 || x->size(-1) < 1 || n_weights > kMaxTensors || n_out < 1) return None();
    std::array<qfg_tensor2d, kMaxTensors> w;
    for (Py_ssize_t i = 0; i < n_weights; ++i) {
      if (!Weight(PyTuple_GET_ITEM(a[2], i), &w[i])) return None();
    }
    const int64_t k = x->size(-1), m = x->numel() / k;
    std::array<at::Tensor, kMaxTensors> out;
    std::array<void*, kMaxTensors> ptr;
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    const at::TensorOptions options = x->options();
    for (int i = 0; i < n_out; ++i) {
      shape.back() = widths[i];
      out[i] = at::empty(shape, options);
      ptr[i] = out[i].data_ptr();
    }
    const void* xp = x->data_ptr();
    void* const stream = Stream();
    const int code = Call([&] {
      return g_lib.skinny_gemm(static_cast<const qfg_skinny_gemm*>(op), xp, m, k, w.data(), static_cast<int>(n_weights), ptr.data(), n_out, stream);
    });
    return code != 0 ? PyLong_FromLong(code) : ListOf(out, n_out);
  });
}

// argmax_rows(x, with_val) -> (idx, val) or idx
PyObject* ArgmaxRows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    const at::Tensor* x = n_args == 2 ? Dense(a[0]) : nullptr;
    if (x == nullptr || (a[1] != Py_True && a[1] != Py_False) || x->dim() < 1 || x->size(-1) < 1) return None();
    int dtype;
    switch (x->scalar_type()) {
      case at::kBFloat16: dtype = QFG_BFLOAT16; break;
      case at::kHalf: dtype = QFG_FLOAT16; break;
      case at::kFloat: dtype = QFG_FLOAT; break;
      default: return None();
    }
    const int64_t vocab = x->size(-1), rows = x->numel() / vocab;
    const at::IntArrayRef lead = x->sizes().slice(0, x->dim() - 1);
    const at::Tensor idx = at::empty(lead, x->options().dtype(at::kLong));
    at::Tensor val;
    if (a[1] == Py_True) val = at::empty(lead, x->options().dtype(at::kFloat));
    const void* xp = x->data_ptr();
    int64_t* const ip = idx.data_ptr<int64_t>();
    float* const vp = val.defined() ? val.data_ptr<float>() : nullptr;
    void* const stream = Stream();
    const int code = Call([&] { return g_lib.argmax_rows(dtype, xp, rows, vocab, ip, vp, stream); });
    if (code != 0) return PyLong_FromLong(code);
    return val.defined() ? TupleOf({idx, val}) : THPVariable_Wrap(idx);
  });
}

// dequant(handle, w, widths) -> [out, ...]
PyObject* Dequant(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    qfg_tensor2d w;
    std::array<int64_t, kMaxTensors> widths;
    if (n_args != 3 || !Weight(a[1], &w)) return None();
    const void* op = PyLong_AsVoidPtr(a[0]);
    const int n_out = Widths(a[2], &widths);
    if (op == nullptr || n_out < 1) return None();
    std::array<at::Tensor, kMaxTensors> out;
    std::array<void*, kMaxTensors> ptr;
    const at::TensorOptions options = THPVariable_Unpack(a[1]).options().dtype(at::kBFloat16);
    for (int i = 0; i < n_out; ++i) {
      out[i] = at::empty({w.rows, widths[i]}, options);
      ptr[i] = out[i].data_ptr();
    }
    void* const stream = Stream();
    const int code = Call([&] { return g_lib.dequant(static_cast<const qfg_dequant*>(op), &w, ptr.data(), n_out, stream); });
    return code != 0 ? PyLong_FromLong(code) : ListOf(out, n_out);
  });
}

// lmhead(handle, workspace, x, w, n, col_offset) -> (idx, val, key)
PyObject* LmHead(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    qfg_tensor2d w;
    if (n_args != 6 || !Weight(a[3], &w)) return None();
    const void* op = PyLong_AsVoidPtr(a[0]);
    const at::Tensor *space = Dense(a[1]), *x = Bf16(a[2]);
    const int64_t n = PyLong_AsLongLong(a[4]), col_offset = PyLong_AsLongLong(a[5]);
    if (PyErr_Occurred() || op == nullptr || space == nullptr || x == nullptr || x->dim() < 1 || x->size(-1) < 1) return None();
    const int64_t k = x->size(-1), m = x->numel() / k;
    const at::Tensor idx = at::empty({m}, x->options().dtype(at::kLong)), val = at::empty({m}, x->options().dtype(at::kFloat)),
                     key = at::empty({m}, x->options().dtype(at::kLong));
    const void* xp = x->data_ptr();
    void *const sp = space->data_ptr(), *const stream = Stream();
    int64_t* const ip = idx.data_ptr<int64_t>();
    float* const vp = val.data_ptr<float>();
    uint64_t* const kp = reinterpret_cast<uint64_t*>(key.data_ptr<int64_t>());
    const int code = Call([&] { return g_lib.lmhead(static_cast<const qfg_lmhead*>(op), xp, m, k, &w, n, col_offset, sp, ip, vp, kp, nullptr, stream); });
    return code != 0 ? PyLong_FromLong(code) : TupleOf({idx, val, key});
  });
}

// shared_expert_down(handle, g, u, w, gx, gw, routed) -> out
PyObject* SharedExpertDown(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    qfg_tensor2d w;
    if (n_args != 7 || !Weight(a[3], &w)) return None();
    const void* op = PyLong_AsVoidPtr(a[0]);
    const at::Tensor *g = Bf16(a[1]), *u = Bf16(a[2]), *gx = Bf16(a[4]), *gw = Bf16(a[5]), *routed = Bf16(a[6]);
    if (op == nullptr || g == nullptr || u == nullptr || gx == nullptr || gw == nullptr || routed == nullptr || w.rows < 1 || routed->dim() < 1 ||
        gw->dim() < 1)
      return None();
    const int64_t k = w.rows, n = routed->size(-1), m = g->numel() / k, gk = gw->numel();
    if (m < 1 || g->numel() != m * k || u->numel() != m * k || routed->numel() != m * n || gx->numel() != m * gk || gw->size(-1) != 1) return None();
    if (w.dtype == QFG_UINT8 ? n % 16 != 0 || w.cols != n * 9 / 16 : w.cols != n) return None();
    const at::Tensor out = at::empty(routed->sizes(), routed->options());
    const void *gp = g->data_ptr(), *up = u->data_ptr(), *gxp = gx->data_ptr(), *gwp = gw->data_ptr(), *rp = routed->data_ptr();
    void *const op_out = out.data_ptr(), *const stream = Stream();
    const int code = Call([&] {
      return g_lib.shared_expert_down(static_cast<const qfg_shared_expert_down*>(op), gp, up, m, k, &w, gxp, gk, gwp, rp, n, op_out, stream);
    });
    return code != 0 ? PyLong_FromLong(code) : THPVariable_Wrap(out);
  });
}

// ---- eight-bit rows
int Code(at::ScalarType t) {  // 0: none of the types here
  switch (t) {
    case at::kBFloat16: return QFG_BFLOAT16;
    case at::kHalf: return QFG_FLOAT16;
    case at::kFloat: return QFG_FLOAT;
    case at::kChar: return QFG_INT8;
    case at::kFloat8_e4m3fn: return QFG_FLOAT8E4M3FN;
    default: return 0;
  }
}
bool Float(const at::Tensor& t) { return Code(t.scalar_type()) != 0 && t.element_size() > 1; }
bool EightBits(const at::Tensor& t) { return Code(t.scalar_type()) != 0 && t.element_size() == 1; }
bool OnCurrent(const at::Tensor& t) { return t.get_device() == c10::cuda::current_device(); }
// Rows that are evenly spaced, on the current device: contiguous, or a matrix whose rows are further apart.
struct Rows {
  const at::Tensor* t = nullptr;
  int64_t rows = 0, n = 0, ld = 0;
};
bool ToRows(PyObject* o, Rows* r) {
  r->t = Plain(o);
  if (r->t == nullptr || r->t->dim() < 1 || r->t->size(-1) < 1 || !OnCurrent(*r->t)) return false;
  r->n = r->t->size(-1);
  r->rows = r->t->numel() / r->n;
  r->ld = r->n;
  if (r->t->is_contiguous()) return true;
  r->ld = r->t->dim() == 2 ? r->t->stride(0) : 0;
  return r->ld >= r->n && (r->t->stride(1) == 1 || r->n == 1);
}

// at::empty on the current device without its way through the dispatcher: 0.3 us a tensor, of the 5 to 6 that these calls take on the host
at::Tensor New(c10::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, c10::nullopt);
}

// rmsnorm_quant(eps, weight_offset, fp8, x, weight, residual or None) -> (q, scale) or (q, scale, h)
PyObject* RmsNormQuant(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    Rows x, r;
    if (n_args != 6 || !PyFloat_CheckExact(a[0]) || !PyFloat_CheckExact(a[1]) || (a[2] != Py_True && a[2] != Py_False) || !ToRows(a[3], &x)) return None();
    const at::Tensor* w = Dense(a[4]);
    const bool added = a[5] != Py_None;
    if (w == nullptr || !Float(*x.t) || (w->scalar_type() != x.t->scalar_type() && w->scalar_type() != at::kFloat) || w->numel() != x.n || !OnCurrent(*w))
      return None();
    if (added && (!ToRows(a[5], &r) || r.t->scalar_type() != x.t->scalar_type() || r.t->sizes() != x.t->sizes())) return None();
    const bool fp8 = a[2] == Py_True;
    const at::Tensor q = New(x.t->sizes(), fp8 ? at::kFloat8_e4m3fn : at::kChar), scale = New(x.t->sizes().slice(0, x.t->dim() - 1), at::kFloat);
    at::Tensor h;
    if (added) h = New(x.t->sizes(), x.t->scalar_type());
    const int dtype = Code(x.t->scalar_type()), w_dtype = Code(w->scalar_type());
    const float offset = static_cast<float>(PyFloat_AS_DOUBLE(a[1])), eps = static_cast<float>(PyFloat_AS_DOUBLE(a[0]));
    const void *xp = x.t->data_ptr(), *rp = added ? r.t->data_ptr() : nullptr, *wp = w->data_ptr();
    void *const qp = q.data_ptr(), *const hp = added ? h.data_ptr() : nullptr, *const stream = Stream();
    float* const sp = scale.data_ptr<float>();
    const int code = Call([&] {
      return g_lib.rmsnorm_quant(dtype, xp, x.ld, rp, r.ld, wp, w_dtype, offset, eps, x.rows, x.n, fp8 ? QFG_FLOAT8E4M3FN : QFG_INT8, qp, sp, hp, stream);
    });
    return code != 0 ? PyLong_FromLong(code) : added ? TupleOf({q, scale, h}) : TupleOf({q, scale});
  });
}

// row_quant(fp8, x, u or None) -> (q, scale)
PyObject* RowQuant(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    Rows x, u;
    if (n_args != 3 || (a[0] != Py_True && a[0] != Py_False) || !ToRows(a[1], &x) || !Float(*x.t)) return None();
    const bool gated = a[2] != Py_None, fp8 = a[0] == Py_True;
    if (gated && (!ToRows(a[2], &u) || u.t->scalar_type() != x.t->scalar_type() || u.t->sizes() != x.t->sizes())) return None();
    const at::Tensor q = New(x.t->sizes(), fp8 ? at::kFloat8_e4m3fn : at::kChar), scale = New(x.t->sizes().slice(0, x.t->dim() - 1), at::kFloat);
    const int dtype = Code(x.t->scalar_type());
    const void *xp = x.t->data_ptr(), *up = gated ? u.t->data_ptr() : nullptr;
    void *const qp = q.data_ptr(), *const stream = Stream();
    float* const sp = scale.data_ptr<float>();
    const int code = Call([&] { return g_lib.row_quant(dtype, xp, x.ld, up, u.ld, x.rows, x.n, fp8 ? QFG_FLOAT8E4M3FN : QFG_INT8, qp, sp, stream); });
    return code != 0 ? PyLong_FromLong(code) : TupleOf({q, scale});
  });
}

// How a weight [k, n] is stored: with its columns beside one another, or its inner dimension.
bool Order(const at::Tensor& w, int* order, int64_t* ld) {
  if (w.stride(1) == 1 && w.stride(0) >= w.size(1)) {
    *order = QFG_ORDER_N, *ld = w.stride(0);
  } else if (w.stride(0) == 1 && w.stride(1) >= w.size(0)) {
    *order = QFG_ORDER_K, *ld = w.stride(1);
  } else {
    return false;
  }
  return true;
}

at::ScalarType Type(long out_dtype) { return out_dtype == QFG_BFLOAT16 ? at::kBFloat16 : out_dtype == QFG_FLOAT16 ? at::kHalf : at::kFloat; }

// quant_gemm(handle, output type, x, x_scale, w) -> out
PyObject* QuantGemm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    Rows x;
    if (n_args != 5 || !ToRows(a[2], &x) || !EightBits(*x.t)) return None();
    const void* op = PyLong_AsVoidPtr(a[0]);
    const long out_dtype = PyLong_AsLong(a[1]);
    const at::Tensor *xs = Dense(a[3]), *w = Plain(a[4]);
    if (PyErr_Occurred() || op == nullptr || xs == nullptr || w == nullptr || xs->scalar_type() != at::kFloat || xs->numel() != x.rows || !OnCurrent(*xs) ||
        w->dim() != 2 || w->scalar_type() != x.t->scalar_type() || w->size(0) != x.n || w->size(1) < 1 || !OnCurrent(*w))
      return None();
    const int64_t n = w->size(1), k = x.n;
    int order;
    int64_t ldw;
    if (!Order(*w, &order, &ldw)) return None();
    c10::SmallVector<int64_t, 6> shape(x.t->sizes().begin(), x.t->sizes().end());
    shape.back() = n;
    const at::Tensor out = New(shape, Type(out_dtype));
    const int dtype = Code(x.t->scalar_type());
    const void *xp = x.t->data_ptr(), *wp = w->data_ptr();
    const float* const sp = xs->data_ptr<float>();
    void *const yp = out.data_ptr(), *const stream = Stream();
    const int code =
        Call([&] { return g_lib.quant_gemm(static_cast<const qfg_quant_gemm*>(op), dtype, xp, x.ld, sp, x.rows, k, wp, ldw, order, n, yp, n, stream); });
    return code != 0 ? PyLong_FromLong(code) : THPVariable_Wrap(out);
  });
}

// quant_mlp(eps, weight_offset, norm weight, gate and up's handle, its weight, down's handle, its weight, output type of both, x, residual) -> (y, h)
PyObject* QuantMlp(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return Guard([&]() -> PyObject* {
    Rows x, r;
    if (n_args != 10 || !PyFloat_CheckExact(a[0]) || !PyFloat_CheckExact(a[1]) || !ToRows(a[8], &x) || !ToRows(a[9], &r)) return None();
    const void *up = PyLong_AsVoidPtr(a[3]), *down = PyLong_AsVoidPtr(a[5]);
    const at::ScalarType out_type = Type(PyLong_AsLong(a[7]));
    const at::Tensor *g = Dense(a[2]), *w1 = Plain(a[4]), *w2 = Plain(a[6]);
    if (PyErr_Occurred() || up == nullptr || down == nullptr || g == nullptr || w1 == nullptr || w2 == nullptr || !Float(*x.t) ||
        r.t->scalar_type() != x.t->scalar_type() || r.t->sizes() != x.t->sizes() || x.rows < 1 ||
        (g->scalar_type() != x.t->scalar_type() && g->scalar_type() != at::kFloat) || g->numel() != x.n || !OnCurrent(*g) || !OnCurrent(*w1) ||
        !OnCurrent(*w2) || w1->dim() != 2 || w2->dim() != 2 || !EightBits(*w1) || w2->scalar_type() != w1->scalar_type() || w1->size(0) != x.n ||
        w2->size(0) < 1 || w1->size(1) != 2 * w2->size(0) || w2->size(1) != x.n)
      return None();
    int order1, order2;
    int64_t ld1, ld2;
    if (!Order(*w1, &order1, &ld1) || !Order(*w2, &order2, &ld2)) return None();
    const auto *up_op = static_cast<const qfg_quant_gemm*>(up), *down_op = static_cast<const qfg_quant_gemm*>(down);
    const int64_t width = w2->size(0);
    const size_t bytes = g_lib.quant_mlp_workspace_bytes(up_op, x.rows, x.n, width);
    if (bytes == 0) return None();
    const at::Tensor workspace = New({static_cast<int64_t>(bytes)}, at::kByte), y = New(x.t->sizes(), out_type), h = New(x.t->sizes(), x.t->scalar_type());
    const int dtype = Code(x.t->scalar_type()), g_type = Code(g->scalar_type()), type = Code(w1->scalar_type());
    const float eps = static_cast<float>(PyFloat_AS_DOUBLE(a[0])), offset = static_cast<float>(PyFloat_AS_DOUBLE(a[1]));
    const void *xp = x.t->data_ptr(), *rp = r.t->data_ptr(), *gp = g->data_ptr(), *w1p = w1->data_ptr(), *w2p = w2->data_ptr();
    void *const wp = workspace.data_ptr(), *const yp = y.data_ptr(), *const hp = h.data_ptr(), *const stream = Stream();
    const int code = Call([&] {
      return g_lib.quant_mlp(dtype, xp, x.ld, rp, r.ld, gp, g_type, offset, eps, x.rows, x.n, width, type, up_op, w1p, ld1, order1, down_op, w2p, ld2, order2, wp,
                             yp, hp, stream);
    });
    return code != 0 ? PyLong_FromLong(code) : TupleOf({y, h});
  });
}

template <typename T>
bool Address(PyObject* o, T* fn) {
  void* p = PyLong_AsVoidPtr(o);
  if (p == nullptr && !PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
  *fn = reinterpret_cast<T>(p);
  return p != nullptr;
}
// bind_rows(address, ...): the entry points of eight-bit rows, in the order of Entries
PyObject* BindRows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 3) {
    PyErr_SetString(PyExc_TypeError, "bind_rows takes three addresses");
    return nullptr;
  }
  Entries e = g_lib;
  if (!Address(a[0], &e.rmsnorm_quant) || !Address(a[1], &e.row_quant) || !Address(a[2], &e.quant_gemm)) return nullptr;
  g_lib = e;
  Py_RETURN_NONE;
}
PyObject* BindMlp(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 2) {
    PyErr_SetString(PyExc_TypeError, "bind_mlp takes two addresses");
    return nullptr;
  }
  Entries e = g_lib;
  if (!Address(a[0], &e.quant_mlp_workspace_bytes) || !Address(a[1], &e.quant_mlp)) return nullptr;
  g_lib = e;
  Py_RETURN_NONE;
}

// bind(address, ...) in the order of Entries
PyObject* Bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  void* p[5];
  if (n_args != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  g_lib.skinny_gemm = reinterpret_cast<decltype(g_lib.skinny_gemm)>(p[0]);
  g_lib.argmax_rows = reinterpret_cast<decltype(g_lib.argmax_rows)>(p[1]);
  g_lib.dequant = reinterpret_cast<decltype(g_lib.dequant)>(p[2]);
  g_lib.lmhead = reinterpret_cast<decltype(g_lib.lmhead)>(p[3]);
  g_lib.shared_expert_down = reinterpret_cast<decltype(g_lib.shared_expert_down)>(p[4]);
  Py_RETURN_NONE;
}

#define QFG_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {QFG_METHOD("bind", Bind),
                           QFG_METHOD("skinny_gemm", SkinnyGemm),
                           QFG_METHOD("argmax_rows", ArgmaxRows),
                           QFG_METHOD("dequant", Dequant),
                           QFG_METHOD("lmhead", LmHead),
                           QFG_METHOD("shared_expert_down", SharedExpertDown),
                           QFG_METHOD("bind_rows", BindRows),
                           QFG_METHOD("bind_mlp", BindMlp),
                           QFG_METHOD("rmsnorm_quant", RmsNormQuant),
                           QFG_METHOD("row_quant", RowQuant),
                           QFG_METHOD("quant_gemm", QuantGemm),
                           QFG_METHOD("quant_mlp", QuantMlp),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
  PyObject* m = PyModule_Create(&g_module);
  // the torch whose headers this was compiled against: ops.py uses the module with no other
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", QFG_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
