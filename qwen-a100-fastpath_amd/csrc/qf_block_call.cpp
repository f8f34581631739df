// qf_block_call.cpp — the short way from Python to libqf_block.so for calls in their plain form (host code, CPython's C API).
//
// A call of one token takes the GPU 3 to 10 us and took the host 10 to 18: checks and address arithmetic in Python, a
// ctypes call of twenty arguments, an allocation or two through torch's Python bindings.  These functions check the same
// things on the tensors themselves, allocate through ATen and call the C ABI: a product of one row 9.0 -> 5.1 us on the host,
// the norms of one row 9.5 -> 4.9 us (a launch is 3 of them).  A function returns None, before it has launched anything,
// wherever something is not in the plain form (a stride or alignment that needs a copy, another device or type, a tensor
// subclass, nothing to do, an argument that is wrong); the caller in Python then takes the call from the start, with its
// copies and its errors.  A status other than QF_OK also ends there.
//
// `device` and `stream` are the current device and torch's current stream on it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "qf_block.h"

namespace {

constexpr int64_t kMaxStride = (int64_t)1 << 26;
constexpr int64_t kIntMax = 0x7fffffff;

bool unpack(PyObject* o, int64_t device, const at::Tensor** t) {
  if (!THPVariable_CheckExact(o)) return false;
  *t = &THPVariable_Unpack(o);
  return (*t)->is_cuda() && (*t)->get_device() == device && (*t)->layout() == at::kStrided;
}
bool unpack_or_none(PyObject* o, int64_t device, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || unpack(o, device, t);
}
bool aligned(const void* p, uintptr_t bytes = 16) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// A [M, N] matrix with unit column stride, 16-byte aligned, its row stride a multiple of `align`; *ld: that stride.
bool rows(const at::Tensor& t, at::ScalarType type, int64_t align, int64_t* ld) {
  if (t.dim() != 2 || t.scalar_type() != type || (t.size(1) > 1 && t.stride(1) != 1) || !aligned(t.data_ptr())) return false;
  *ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
  return *ld % align == 0;
}
bool vector(const at::Tensor* t, at::ScalarType type, int64_t n, uintptr_t bytes) {
  return t == nullptr || (t->dim() == 1 && t->scalar_type() == type && t->size(0) == n && t->is_contiguous() &&
                          aligned(t->data_ptr(), bytes));
}
template <typename T>
T* ptr(const at::Tensor* t) {
  return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr());
}
int64_t blocks(int64_t n) { return (n + QF_FP8_BLOCK - 1) / QF_FP8_BLOCK; }
int64_t tiled_bytes(int64_t n, int64_t k) { return (n + 15) / 16 * 16 * k; }

// product(x, w, w_scale, bias, out_f32, out_features, decode, workspace, device, stream) -> y or None.  out_features: -1
// where it is not given; decode: 1 bf16 activations, 0 e4m3, -1 by rows; workspace(x, bytes): the zeroed one of K splits.
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 10) {
    PyErr_SetString(PyExc_TypeError, "product takes 10 arguments");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[8]);
  const int64_t named = PyLong_AsLongLong(args[5]), decode = PyLong_AsLongLong(args[6]);
  const int out_f32 = args[4] == Py_True;
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *x, *w, *scale, *bias;
  int64_t ldx, ldw, N;
  if (!unpack(args[0], device, &x) || !unpack(args[1], device, &w) || !unpack(args[2], device, &scale) ||
      !unpack_or_none(args[3], device, &bias) || !rows(*x, at::kBFloat16, 8, &ldx) ||
      w->scalar_type() != at::kFloat8_e4m3fn || scale->scalar_type() != at::kFloat)
    Py_RETURN_NONE;
  const int64_t M = x->size(0), K = x->size(1);
  if (M < 1 || M > kIntMax || K < 64 || K % 64 || K > kIntMax || ldx < K || ldx > kMaxStride || !aligned(w->data_ptr()))
    Py_RETURN_NONE;
  int layout = QF_LAYOUT_TILED;
  if (w->dim() == 1) {
    N = named < 0 ? w->numel() / K : named;
    if (!w->is_contiguous() || w->numel() != tiled_bytes(N, K)) Py_RETURN_NONE;
    ldw = K;
  } else {
    if (w->dim() != 2 || w->size(0) != K || w->stride(0) != 1) Py_RETURN_NONE;
    layout = QF_LAYOUT_ROWMAJOR;
    N = w->size(1);
    ldw = N > 1 ? w->stride(1) : K;
    if ((named >= 0 && named != N) || ldw < K || ldw > kMaxStride || ldw % 16) Py_RETURN_NONE;
  }
  if (N < 1 || N > kIntMax || scale->dim() != 2 || scale->size(0) != blocks(N) || scale->size(1) != blocks(K) ||
      !scale->is_contiguous() || !vector(bias, at::kBFloat16, N, 2))
    Py_RETURN_NONE;
  const bool a16 = decode < 0 ? M <= QF_FP8_MAX_DECODE_M : decode != 0;
  const size_t bytes = a16 ? qf_fp8_w8a16_workspace_bytes((int)M, (int)N, (int)K, layout)
                           : qf_fp8_w8a8_workspace_bytes((int)M, (int)N, (int)K);
  if (!a16 && bytes == 0) Py_RETURN_NONE;
  at::Tensor ws;
  size_t ws_bytes = bytes;
  if (!a16) {
    ws = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
  } else if (bytes > 0) {
    PyObject* o = PyObject_CallFunction(args[7], "OK", args[0], (unsigned long long)bytes);
    if (o == nullptr) return nullptr;
    if (THPVariable_Check(o)) ws = THPVariable_Unpack(o);  // kept by its owner
    Py_DECREF(o);
    if (!ws.defined()) Py_RETURN_NONE;
    ws_bytes = (size_t)ws.numel();
  }
  at::Tensor y = at::empty({M, N}, x->options().dtype(out_f32 ? at::kFloat : at::kBFloat16));
  auto* const f = a16 ? &qf_fp8_w8a16_gemm : &qf_fp8_w8a8_linear;
  const int rc = f(ptr<const uint16_t>(x), ldx, ptr<const uint8_t>(w), ldw, layout, ptr<const float>(scale),
                   ptr<const uint16_t>(bias), y.data_ptr(), N, out_f32 ? QF_DTYPE_F32 : QF_DTYPE_BF16, (int)M, (int)N, (int)K,
                   bytes ? ws.data_ptr() : nullptr, ws_bytes, stream);
  if (rc != QF_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// norm(x, residual, post_weight, pre_weight, gate, act, alpha, eps, weight_offset, device, stream) -> (y, h) or None; act: 0
// or 1.
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 11) {
    PyErr_SetString(PyExc_TypeError, "norm takes 11 arguments");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[9]);
  const int act = (int)PyLong_AsLong(args[5]);
  const double alpha = PyFloat_AsDouble(args[6]), eps = PyFloat_AsDouble(args[7]), offset = PyFloat_AsDouble(args[8]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[10]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *x, *residual, *post, *pre, *gate;
  int64_t ldx, ldr, ldg = 0;
  if (!unpack(args[0], device, &x) || !unpack(args[1], device, &residual) || !unpack_or_none(args[2], device, &post) ||
      !unpack_or_none(args[3], device, &pre) || !unpack_or_none(args[4], device, &gate) || !rows(*x, at::kBFloat16, 8, &ldx))
    Py_RETURN_NONE;
  const bool wide = residual->scalar_type() == at::kFloat;
  const int64_t M = x->size(0), N = x->size(1);
  if (!rows(*residual, wide ? at::kFloat : at::kBFloat16, wide ? 4 : 8, &ldr) || residual->size(0) != M ||
      residual->size(1) != N || M < 1 || M > kIntMax || N < 8 || N % 8 || N > QF_BLOCK_NORM_MAX_N || !(eps >= 0) ||
      !vector(post, at::kBFloat16, N, 16) || !vector(pre, at::kBFloat16, N, 16))
    Py_RETURN_NONE;
  int kind = QF_GATE_NONE;
  if (gate != nullptr) {
    if (gate->scalar_type() != at::kBFloat16) Py_RETURN_NONE;
    if (gate->dim() == 1) {
      if (!vector(gate, at::kBFloat16, N, 16)) Py_RETURN_NONE;
      kind = QF_GATE_CHANNEL;
    } else if (gate->dim() == 2 && gate->size(0) == M && gate->size(1) == 1) {
      kind = QF_GATE_TOKEN;
      ldg = M > 1 ? gate->stride(0) : 0;
    } else {
      if (!rows(*gate, at::kBFloat16, 8, &ldg) || gate->size(0) != M || gate->size(1) != N) Py_RETURN_NONE;
      kind = QF_GATE_FULL;
    }
  }
  at::Tensor y = at::empty({M, N}, residual->options()), h = at::empty({M, N}, x->options());
  const int rc = qf_block_norm_rows(ptr<const uint16_t>(x), ldx, residual->data_ptr(), ldr, wide, ptr<const uint16_t>(post),
                                    ptr<const uint16_t>(pre), (float)offset, ptr<const uint16_t>(gate), ldg, kind, act,
                                    (float)alpha, (float)eps, (int)M, (int)N, y.data_ptr(), N, ptr<uint16_t>(&h), N, stream);
  if (rc != QF_OK) Py_RETURN_NONE;
  PyObject* a = THPVariable_Wrap(std::move(y));
  PyObject* b = a == nullptr ? nullptr : THPVariable_Wrap(std::move(h));
  PyObject* both = b == nullptr ? nullptr : PyTuple_Pack(2, a, b);
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
  END_HANDLE_TH_ERRORS
}

// moe(x, router_logits, w13, s13, w2, s2, top_k, renormalize, device, stream) -> y or None.
PyObject* moe(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 10) {
    PyErr_SetString(PyExc_TypeError, "moe takes 10 arguments");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[8]), k = PyLong_AsLongLong(args[6]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const int renormalize = PyObject_IsTrue(args[7]);
  if (renormalize < 0) return nullptr;
  const at::Tensor *x, *logits, *w13, *s13, *w2, *s2;
  int64_t ldx;
  if (!unpack(args[0], device, &x) || !unpack(args[1], device, &logits) || !unpack(args[2], device, &w13) ||
      !unpack(args[3], device, &s13) || !unpack(args[4], device, &w2) || !unpack(args[5], device, &s2) ||
      !rows(*x, at::kBFloat16, 8, &ldx))
    Py_RETURN_NONE;
  const int64_t T = x->size(0), H = x->size(1);
  const bool f32 = logits->scalar_type() == at::kFloat;
  if (T < 1 || T > QF_FP8_MAX_DECODE_M || H < 64 || H % 64 || H > kIntMax || ldx < H || ldx > kMaxStride ||
      (!f32 && logits->scalar_type() != at::kBFloat16) || logits->dim() != 2 || logits->size(0) != T)
    Py_RETURN_NONE;
  const int64_t E = logits->size(1);
  const int64_t ldl = T > 1 ? logits->stride(0) : E;
  if (E < 1 || E > QF_MOE_MAX_EXPERTS || (E > 1 && logits->stride(1) != 1) || ldl < E || k < 1 || k > E ||
      k > QF_MOE_MAX_TOP_K || w13->dim() != 1 || w2->dim() != 1 || w13->scalar_type() != at::kFloat8_e4m3fn ||
      w2->scalar_type() != at::kFloat8_e4m3fn || !w13->is_contiguous() || !w2->is_contiguous() || !aligned(w13->data_ptr()) ||
      !aligned(w2->data_ptr()))
    Py_RETURN_NONE;
  const int64_t I = w2->numel() / (E * H);
  if (I < 64 || I % 64 || I > kIntMax || w2->numel() != E * H * I || w13->numel() != 2 * E * I * H) Py_RETURN_NONE;
  const int64_t nb = blocks(I), kb = blocks(H);
  if (s13->scalar_type() != at::kFloat || s2->scalar_type() != at::kFloat || s13->dim() != 3 || s2->dim() != 3 ||
      s13->size(0) != E || s13->size(1) != 2 * nb || s13->size(2) != kb || s2->size(0) != E || s2->size(1) != kb ||
      s2->size(2) != nb || !s13->is_contiguous() || !s2->is_contiguous())
    Py_RETURN_NONE;
  const size_t bytes = qf_moe_few_workspace_bytes((int)T, (int)E, (int)k, (int)H, (int)I);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor y = at::empty({T, H}, x->options());
  at::Tensor ws = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
  const int rc = qf_moe_few_tokens(ptr<const uint16_t>(x), ldx, logits->data_ptr(), ldl, f32, ptr<const uint8_t>(w13),
                                   ptr<const float>(s13), ptr<const uint8_t>(w2), ptr<const float>(s2), ptr<uint16_t>(&y), H,
                                   (int)T, (int)E, (int)k, (int)H, (int)I, renormalize, ws.data_ptr(), bytes, stream);
  if (rc != QF_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"product", (PyCFunction)(void*)product, METH_FASTCALL, nullptr},
                         {"norm", (PyCFunction)(void*)norm, METH_FASTCALL, nullptr},
                         {"moe", (PyCFunction)(void*)moe, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qf_block_call", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__qf_block_call(void) { return PyModule_Create(&module); }
