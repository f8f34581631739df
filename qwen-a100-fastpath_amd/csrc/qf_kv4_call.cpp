// qf_kv4_call.cpp — the way from Python to libqf_kv4.so (host code, CPython's C API).
//
// The calls of a decode step take the GPU 3 to 20 us each; checks and address arithmetic in Python with a ctypes call would
// take the host as long.  These functions check the tensors themselves, allocate through ATen and call the C ABI.  A function
// returns None, before it has launched anything, wherever something is not as the kernels take it (a stride or alignment that
// needs a copy, another device or type, an argument that is wrong); the caller in Python then names the error, or makes
// the copy and calls again.  A status other than QF_OK is returned as a number.
//
// `device` and `stream` are the current device and torch's current stream on it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "qf_kv4.h"

namespace {

constexpr int64_t kIntMax = 0x7fffffff;
constexpr int64_t kFar = 0x7fffffffffffffff;  // past any stride

bool unpack(PyObject* o, int64_t device, const at::Tensor** t) {
  if (!THPVariable_CheckExact(o)) return false;
  *t = &THPVariable_Unpack(o);
  return (*t)->is_cuda() && (*t)->get_device() == device && (*t)->layout() == at::kStrided;
}
bool unpack_or_none(PyObject* o, int64_t device, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || unpack(o, device, t);
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// [T, H, D] bf16 with the last dimension contiguous and other strides of multiples of 8.
bool heads(const at::Tensor& t, int64_t T, int64_t H, int64_t D, qf_heads* out) {
  if (t.dim() != 3 || t.scalar_type() != at::kBFloat16 || t.size(0) != T || t.size(1) != H || t.size(2) != D || t.stride(2) != 1)
    return false;
  out->data = static_cast<uint16_t*>(t.data_ptr());
  out->stride_tok = T > 1 ? t.stride(0) : 0;
  out->stride_head = H > 1 ? t.stride(1) : 0;
  return aligned(out->data) && out->stride_tok >= 0 && out->stride_head >= 0 && out->stride_tok % 8 == 0 && out->stride_head % 8 == 0;
}
// A tensor that is written: no two of its heads may share memory.
bool separate(const qf_heads& h, int64_t T, int64_t H, int64_t D) {
  const int64_t t = T > 1 ? h.stride_tok : kFar, n = H > 1 ? h.stride_head : kFar;
  return n <= t ? n >= D && (T == 1 || t >= (H == 1 ? D : (H - 1) * n + D)) : t >= D && n >= (T - 1) * t + D;
}
bool pages(const at::Tensor& t, int64_t H, int64_t D, qf_pages* out) {
  if (t.dim() != 4 || t.scalar_type() != at::kBFloat16 || t.size(0) < 1 || t.size(1) < 1 || t.size(2) != H || t.size(3) != D ||
      t.stride(3) != 1)
    return false;
  *out = {static_cast<uint16_t*>(t.data_ptr()), t.stride(0), t.stride(1), t.stride(2)};
  // they are written: no two heads may share memory, in whichever order the dimensions stand
  int order[] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return t.stride(a) < t.stride(b); });
  int64_t room = D;
  for (int i : order) {
    if (t.size(i) == 1) continue;
    if (t.stride(i) < room) return false;
    room += (t.size(i) - 1) * t.stride(i);
  }
  return aligned(out->data) && out->stride_block >= 0 && out->stride_tok >= 0 && out->stride_head >= 0 &&
         out->stride_block % 8 == 0 && out->stride_tok % 8 == 0 && out->stride_head % 8 == 0;
}
// The 4-bit cache [num_blocks, H, page / 16, 17 D].
bool cache4(const at::Tensor& t, int64_t* H, int64_t* D, int64_t* page) {
  if (t.dim() != 4 || t.scalar_type() != at::kByte || t.size(0) < 1) return false;
  *H = t.size(1);
  *D = t.size(3) / 17;
  *page = t.size(2) * QF_KV4_TILE;
  const int64_t record = 17 * *D;
  return t.size(3) == record && (*D == 64 || *D == 128 || *D == 256) && *H >= 1 && *page >= 1 && *page <= kIntMax && t.stride(3) == 1 &&
         (t.size(2) == 1 || t.stride(2) == record) && (*H == 1 || t.stride(1) == t.size(2) * record) &&
         (t.size(0) == 1 || (t.stride(0) % 16 == 0 && t.stride(0) >= *H * t.size(2) * record)) && aligned(t.data_ptr());
}
int64_t block_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3); }
bool vec(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.dim() == 1 && t.scalar_type() == type && t.size(0) == n && (n < 2 || t.stride(0) == 1);
}
bool table(const at::Tensor& t, int64_t rows, int64_t* stride) {
  if (t.dim() != 2 || t.scalar_type() != at::kInt || t.size(0) < rows || t.size(1) < 1 || t.size(1) > kIntMax ||
      (t.size(1) > 1 && t.stride(1) != 1))
    return false;
  *stride = t.size(0) > 1 ? t.stride(0) : t.size(1);
  return *stride >= t.size(1);
}
template <typename T>
T* ptr(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
bool ready(Py_ssize_t got, Py_ssize_t want, const char* name) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  return false;
}

// tables(context, q_lens, held, block_table, free_blocks, free_count, page_size, num_tokens, device, stream) -> (cu_q, seq_lens,
// positions, slots, held, free_count, fits)
PyObject* tables(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!ready(n_args, 10, "tables")) return nullptr;
  const int64_t page = PyLong_AsLongLong(args[6]), T = PyLong_AsLongLong(args[7]), device = PyLong_AsLongLong(args[8]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *context, *q, *held, *bt, *stack, *count;
  int64_t bt_stride;
  if (!unpack(args[0], device, &context) || !unpack(args[1], device, &q) || !unpack(args[2], device, &held) ||
      !unpack(args[3], device, &bt) || !unpack(args[4], device, &stack) || !unpack(args[5], device, &count) || context->dim() != 1)
    Py_RETURN_NONE;
  const int64_t B = context->size(0);
  if (B < 1 || B > QF_STEP_MAX_REQS || !vec(*context, at::kInt, B) || !vec(*q, at::kInt, B) || !vec(*held, at::kInt, B) ||
      !table(*bt, B, &bt_stride) || bt->size(1) > QF_STEP_MAX_TOKENS || stack->dim() != 1 ||
      !vec(*stack, at::kInt, stack->size(0)) || stack->size(0) > QF_STEP_MAX_TOKENS || !vec(*count, at::kInt, 1) || page < 1 ||
      page > kIntMax || T < 0 || T > QF_STEP_MAX_TOKENS)
    Py_RETURN_NONE;
  // one allocation for the int32 outputs, one for the int64 ones; parts start on 16 bytes
  const auto room = [](int64_t n) { return (n + 3) / 4 * 4; };
  at::Tensor small = at::empty({room(B + 1) + 2 * room(B) + 8}, context->options());
  at::Tensor tokens = at::empty({2, T}, context->options().dtype(at::kLong));
  const int64_t at_seq = room(B + 1), at_held = at_seq + room(B), at_count = at_held + room(B), at_fits = at_count + 4;
  int32_t* const s = ptr<int32_t>(small);
  int64_t* const t = ptr<int64_t>(tokens);
  const int rc = qf_step_tables(ptr<int32_t>(*context), ptr<int32_t>(*q), ptr<int32_t>(*held), ptr<int32_t>(*bt), bt_stride,
                                (int)bt->size(1), ptr<int32_t>(*stack), ptr<int32_t>(*count), (int)stack->size(0), (int)B,
                                (int)page, (int)T, s, s + at_seq, t, t + T, s + at_held, s + at_count, s + at_fits, stream);
  if (rc != QF_OK) return PyLong_FromLong(rc);
  at::AutoDispatchBelowADInplaceOrView guard;  // views of fresh integer tensors: nothing for autograd
  const auto part = [](const at::Tensor& of, int64_t from, int64_t n) { return of.as_strided({n}, {1}, from); };
  at::Tensor out[] = {part(small, 0, B + 1), part(small, at_seq, B), part(tokens, 0, T), part(tokens, T, T),
                      part(small, at_held, B), part(small, at_count, 1), part(small, at_fits, 1)};
  PyObject* all = PyTuple_New(7);
  for (int i = 0; all != nullptr && i < 7; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(out[i]));
    if (o == nullptr) {
      Py_DECREF(all);
      return nullptr;
    }
    PyTuple_SET_ITEM(all, i, o);
  }
  return all;
  END_HANDLE_TH_ERRORS
}

// rope(query, key, value, positions, cos_sin, q_weight, k_weight, cache, slots, eps, weight_offset, interleaved, query_out,
// key_out, device, stream) -> (query_out or None, key_out or None).  cache: None, the 4-bit cache or a tuple of key and value
// pages; without a cache key_out is made where it is None.
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!ready(n_args, 16, "rope")) return nullptr;
  qf_qk_norm_rope_args u = {};
  u.eps = PyFloat_AsDouble(args[9]);
  u.weight_offset = PyFloat_AsDouble(args[10]);
  u.interleaved = PyObject_IsTrue(args[11]);
  const int64_t device = PyLong_AsLongLong(args[14]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[15]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *query, *key, *value, *positions, *cos_sin, *qw, *kw, *slots, *query_out, *key_out;
  if (!unpack_or_none(args[0], device, &query) || !unpack(args[1], device, &key) || !unpack_or_none(args[2], device, &value) ||
      !unpack_or_none(args[3], device, &positions) || !unpack_or_none(args[4], device, &cos_sin) ||
      !unpack_or_none(args[5], device, &qw) || !unpack_or_none(args[6], device, &kw) || !unpack_or_none(args[8], device, &slots) ||
      !unpack_or_none(args[12], device, &query_out) || !unpack_or_none(args[13], device, &key_out) || key->dim() != 3)
    Py_RETURN_NONE;
  const int64_t T = key->size(0), HK = key->size(1), D = key->size(2);
  if (T < 1 || T > kIntMax || HK < 1 || HK > kIntMax || (D != 64 && D != 128 && D != 256) || !(u.eps >= 0) ||
      !heads(*key, T, HK, D, &u.key))
    Py_RETURN_NONE;
  int64_t H = 0;
  if (query != nullptr) {
    if (query->dim() != 3) Py_RETURN_NONE;
    H = query->size(1);
    if (H < 1 || H > kIntMax || !heads(*query, T, H, D, &u.query)) Py_RETURN_NONE;
  }
  if ((qw != nullptr && (!vec(*qw, at::kBFloat16, D) || !aligned(qw->data_ptr()))) ||
      (kw != nullptr && (!vec(*kw, at::kBFloat16, D) || !aligned(kw->data_ptr()))) || (cos_sin == nullptr) != (positions == nullptr))
    Py_RETURN_NONE;
  u.q_weight = qw == nullptr ? nullptr : ptr<uint16_t>(*qw);
  u.k_weight = kw == nullptr ? nullptr : ptr<uint16_t>(*kw);
  if (cos_sin != nullptr) {
    u.cos_sin_f32 = cos_sin->scalar_type() == at::kFloat;
    if (cos_sin->dim() != 2 || (!u.cos_sin_f32 && cos_sin->scalar_type() != at::kBFloat16) || !cos_sin->is_contiguous() ||
        cos_sin->size(0) < 1 || cos_sin->size(1) > D || cos_sin->size(1) % 16 || cos_sin->size(1) < 16 ||
        !aligned(cos_sin->data_ptr()) ||
        !vec(*positions, at::kLong, T))
      Py_RETURN_NONE;
    u.rot = (int)cos_sin->size(1);
    u.num_positions = cos_sin->size(0);
    u.cos_sin = cos_sin->data_ptr();
    u.positions = ptr<int64_t>(*positions);
  }
  if (args[7] != Py_None) {
    if (value == nullptr || slots == nullptr || !heads(*value, T, HK, D, &u.value) || !vec(*slots, at::kLong, T)) Py_RETURN_NONE;
    u.slots = ptr<int64_t>(*slots);
    if (PyTuple_CheckExact(args[7])) {
      const at::Tensor *kp, *vp;
      if (PyTuple_GET_SIZE(args[7]) != 2 || !unpack(PyTuple_GET_ITEM(args[7], 0), device, &kp) ||
          !unpack(PyTuple_GET_ITEM(args[7], 1), device, &vp) || !pages(*kp, HK, D, &u.key_pages) ||
          !pages(*vp, HK, D, &u.value_pages) || vp->size(0) != kp->size(0) || vp->size(1) != kp->size(1) || kp->size(1) > kIntMax)
        Py_RETURN_NONE;
      u.cache_kind = QF_CACHE_PAGES;
      u.num_blocks = kp->size(0);
      u.page_size = (int)kp->size(1);
    } else {
      const at::Tensor* c;
      int64_t ch, cd, page;
      if (!unpack(args[7], device, &c) || !cache4(*c, &ch, &cd, &page) || ch != HK || cd != D) Py_RETURN_NONE;
      u.cache_kind = QF_CACHE_KV4;
      u.cache = c->data_ptr();
      u.cache_stride = block_stride(*c);
      u.num_blocks = c->size(0);
      u.page_size = (int)page;
    }
  } else if (value != nullptr || slots != nullptr) {
    Py_RETURN_NONE;
  }
  at::Tensor q_new, k_new;
  if (query != nullptr) {
    if (query_out == nullptr) {
      q_new = at::empty({T, H, D}, query->options());
      query_out = &q_new;
    }
    if (!heads(*query_out, T, H, D, &u.query_out) || !separate(u.query_out, T, H, D)) Py_RETURN_NONE;
  } else if (query_out != nullptr) {
    Py_RETURN_NONE;
  }
  if (key_out == nullptr && args[7] == Py_None) {
    k_new = at::empty({T, HK, D}, key->options());
    key_out = &k_new;
  }
  if (key_out != nullptr && (!heads(*key_out, T, HK, D, &u.key_out) || !separate(u.key_out, T, HK, D))) Py_RETURN_NONE;
  u.num_tokens = (int)T;
  u.num_heads = (int)H;
  u.num_kv_heads = (int)HK;
  u.head_size = (int)D;
  const int rc = qf_qk_norm_rope(&u, stream);
  if (rc != QF_OK) return PyLong_FromLong(rc);
  const auto wrap = [](const at::Tensor* given, at::Tensor& made, PyObject* from) -> PyObject* {
    if (made.defined()) return THPVariable_Wrap(std::move(made));
    Py_INCREF(from);
    return from;
  };
  PyObject* a = wrap(query_out, q_new, args[12]);
  PyObject* b = a == nullptr ? nullptr : wrap(key_out, k_new, args[13]);
  PyObject* both = b == nullptr ? nullptr : PyTuple_Pack(2, a, b);
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
  END_HANDLE_TH_ERRORS
}

// load(cache, slots, device, stream) -> (key, value) bf16 [T, H, D]
PyObject* load(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!ready(n_args, 4, "load")) return nullptr;
  const int64_t device = PyLong_AsLongLong(args[2]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *c, *slots;
  int64_t H, D, page;
  if (!unpack(args[0], device, &c) || !unpack(args[1], device, &slots) || !cache4(*c, &H, &D, &page) || slots->dim() != 1)
    Py_RETURN_NONE;
  const int64_t T = slots->size(0);
  if (T < 1 || T > kIntMax || H > kIntMax || !vec(*slots, at::kLong, T)) Py_RETURN_NONE;
  at::Tensor k = at::empty({T, H, D}, c->options().dtype(at::kBFloat16)), v = at::empty({T, H, D}, k.options());
  const int rc = qf_kv4_load(c->data_ptr(), block_stride(*c), c->size(0), (int)page, (int)H, (int)D, ptr<int64_t>(*slots), (int)T,
                             ptr<uint16_t>(k), ptr<uint16_t>(v), stream);
  if (rc != QF_OK) return PyLong_FromLong(rc);
  PyObject* a = THPVariable_Wrap(std::move(k));
  PyObject* b = a == nullptr ? nullptr : THPVariable_Wrap(std::move(v));
  PyObject* both = b == nullptr ? nullptr : PyTuple_Pack(2, a, b);
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
  END_HANDLE_TH_ERRORS
}

// attention(query, cache, seq_lens, block_table, scale, q_len, cu_q, out, device, stream) -> out.
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (!ready(n_args, 10, "attention")) return nullptr;
  qf_kv4_attention_args u = {};
  u.scale = (float)PyFloat_AsDouble(args[4]);
  const int64_t q_len = PyLong_AsLongLong(args[5]), device = PyLong_AsLongLong(args[8]);
  void* const stream = (void*)PyLong_AsUnsignedLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *query, *c, *seq, *bt, *cu, *out;
  int64_t HK, D, page;
  if (!unpack(args[0], device, &query) || !unpack(args[1], device, &c) || !unpack(args[2], device, &seq) ||
      !unpack(args[3], device, &bt) || !unpack_or_none(args[6], device, &cu) || !unpack_or_none(args[7], device, &out) ||
      !cache4(*c, &HK, &D, &page) || query->dim() != 3 || seq->dim() != 1 || bt->dim() != 2)
    Py_RETURN_NONE;
  const int64_t T = query->size(0), H = query->size(1), B = seq->size(0);
  if (T < 1 || T > kIntMax || B < 1 || B > kIntMax || H < 1 || H > kIntMax || HK > kIntMax || H % HK || q_len < 1 ||
      q_len > kIntMax || bt->size(1) * page > 0x7fffffc0 || !heads(*query, T, H, D, &u.query) || !vec(*seq, at::kInt, B) ||
      !table(*bt, B, &u.bt_stride) ||
      !(u.scale == u.scale) || (cu != nullptr ? !vec(*cu, at::kInt, B + 1) : B * q_len > T))
    Py_RETURN_NONE;
  u.cache = c->data_ptr();
  u.cache_stride = block_stride(*c);
  u.num_blocks = c->size(0);
  u.block_table = ptr<int32_t>(*bt);
  u.seq_lens = ptr<int32_t>(*seq);
  u.cu_q = cu == nullptr ? nullptr : ptr<int32_t>(*cu);
  u.max_blocks = (int)bt->size(1);
  u.num_tokens = (int)T;
  u.num_reqs = (int)B;
  u.q_len = (int)q_len;
  u.num_heads = (int)H;
  u.num_kv_heads = (int)HK;
  u.head_size = (int)D;
  u.page_size = (int)page;
  at::Tensor made;
  if (out == nullptr) {
    made = at::empty({T, H, D}, query->options());
    out = &made;
  }
  if (!heads(*out, T, H, D, &u.out) || !separate(u.out, T, H, D)) Py_RETURN_NONE;
  const size_t bytes = qf_kv4_attention_workspace_bytes(&u);
  at::Tensor ws;  // the caching allocator's: one a call, capture-safe
  if (bytes > 0) ws = at::empty({(int64_t)bytes}, c->options());
  const int rc = qf_kv4_attention(&u, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  if (rc != QF_OK) return PyLong_FromLong(rc);
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  Py_INCREF(args[7]);
  return args[7];
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"tables", (PyCFunction)(void*)tables, METH_FASTCALL, nullptr},
                         {"rope", (PyCFunction)(void*)rope, METH_FASTCALL, nullptr},
                         {"load", (PyCFunction)(void*)load, METH_FASTCALL, nullptr},
                         {"attention", (PyCFunction)(void*)attention, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qf_kv4_call", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__qf_kv4_call(void) { return PyModule_Create(&module); }
