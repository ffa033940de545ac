// The calls of the 8-bit rows, their product and the quantised cache as a
// CPython module over torch's tensors (no counterpart in the reference).
//
// Such a call takes a few microseconds on the GPU, and taking its tensors apart
// in Python and handing them over through ctypes takes as long or longer: 8 x
// 4096 to codes and back 19.3 us that way, 9.2 this way, the kernels 3.2.  So
// the usual call -- ordinary tensors of one device that is the current one, laid
// out as the C entries want them, outputs to be made -- is taken here.  For
// everything else, a mistaken argument too, these functions do nothing and
// return None, and the caller's Python path checks, converts, or says what is
// wrong.
#define PY_SSIZE_T_CLEAN
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "memboost_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

// The tensor behind an argument: CUDA and strided, of no subclass; or null.
const Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

bool all_of_current_device(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t == nullptr || t->get_device() != (*ts.begin())->get_device()) return false;
  return (*ts.begin())->get_device() == c10::cuda::current_device();
}

bool known(ScalarType t, bool fp32, mb_dtype* to) {
  switch (t) {
    case ScalarType::Half: *to = MB_FP16; return true;
    case ScalarType::BFloat16: *to = MB_BF16; return true;
    case ScalarType::Float: *to = MB_FP32; return fp32;
    default: return false;
  }
}

bool known_dtype(PyObject* o, ScalarType* type, mb_dtype* to) {
  if (!THPDtype_Check(o)) return false;
  *type = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return known(*type, true, to);
}

Tensor empty(at::IntArrayRef sizes, at::IntArrayRef strides, ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_strided_cuda(sizes, strides, type, like.device()));
}

Tensor empty(at::IntArrayRef sizes, ScalarType type, const Tensor& like) {
  at::DimVector strides(sizes.size());
  int64_t n = 1;
  for (size_t i = sizes.size(); i-- > 0; n *= sizes[i]) strides[i] = n;
  return empty(sizes, strides, type, like);
}

Tensor workspace(size_t bytes, const Tensor& like) {
  const int64_t n = (int64_t)bytes, one = 1;
  return empty(at::IntArrayRef(&n, 1), at::IntArrayRef(&one, 1), ScalarType::Byte, like);
}

mb_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<mb_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

// Runs an entry without the interpreter's lock; false with an exception set.
template <typename F>
bool run(F&& entry) {
  mb_status st;
  Py_BEGIN_ALLOW_THREADS
  st = entry();
  Py_END_ALLOW_THREADS
  if (st == MB_OK) return true;
  PyErr_SetString(PyExc_RuntimeError, mb_last_error());
  return false;
}

PyObject* pair(Tensor a, Tensor b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = x == nullptr ? nullptr : THPVariable_Wrap(std::move(b));
  PyObject* both = y == nullptr ? nullptr : PyTuple_Pack(2, x, y);
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

int64_t pitch_of(int64_t K) { return (K + 15) / 16 * 16; }

// x as rows of K values: contiguous, or two-dimensional with contiguous rows.
struct Rows {
  int64_t rows, K, stride;
};
bool rows_of(const Tensor& x, Rows* r) {
  const int64_t dims = x.dim();
  if (dims == 0 || x.numel() == 0) return false;
  r->K = x.size(dims - 1);
  r->rows = x.numel() / r->K;
  r->stride = r->K;
  if (x.is_contiguous()) return true;
  if (dims != 2 || x.stride(1) != 1 || x.stride(0) < r->K) return false;
  r->stride = x.stride(0);
  return true;
}

// codes [rows, K] int8 whose rows begin on 16-byte boundaries, scales [rows].
bool codes_of(const Tensor& codes, const Tensor& scales, Rows* r) {
  if (codes.scalar_type() != ScalarType::Char || codes.dim() != 2 || codes.numel() == 0 ||
      scales.scalar_type() != ScalarType::Float || scales.dim() != 1 ||
      scales.size(0) != codes.size(0) || !scales.is_contiguous())
    return false;
  *r = Rows{codes.size(0), codes.size(1), codes.stride(0)};
  if (r->rows == 1) r->stride = pitch_of(r->K);
  return (r->K == 1 || codes.stride(1) == 1) && r->stride % 16 == 0 && r->stride >= r->K &&
         reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0;
}

bool cache_of(const Tensor* const (&parts)[4], mb_kv_cache* c) {
  const Tensor &kc = *parts[0], &vc = *parts[1], &ks = *parts[2], &vs = *parts[3];
  const bool wide = kc.scalar_type() == ScalarType::Char;
  const ScalarType scale = wide ? ScalarType::Float : ScalarType::Half;
  if ((!wide && kc.scalar_type() != ScalarType::Byte) || vc.scalar_type() != kc.scalar_type() ||
      ks.scalar_type() != scale || vs.scalar_type() != scale || kc.dim() != 4 ||
      vc.sizes() != kc.sizes() || vs.sizes() != ks.sizes() || ks.dim() != (wide ? 3 : 5))
    return false;
  for (int i = 0; i < 3; ++i)
    if (ks.size(i) != kc.size(i)) return false;
  const int64_t dim = kc.size(3) * (wide ? 1 : 2);
  if (!wide && (ks.size(3) != dim / 32 || ks.size(4) != 2)) return false;
  for (const Tensor* t : parts)
    if (!t->is_contiguous()) return false;
  if (kc.size(1) > INT32_MAX || kc.size(2) > INT32_MAX || dim > INT32_MAX) return false;
  *c = mb_kv_cache{kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), kc.size(0),
                   (int32_t)kc.size(2), (int32_t)kc.size(1), (int32_t)dim, wide ? 8 : 4};
  return true;
}

bool slots_of(const Tensor& slots) {
  return slots.dim() == 1 && slots.scalar_type() == ScalarType::Long && slots.is_contiguous() &&
         slots.numel() > 0;
}

// (x) -> (codes, scales)
PyObject* quantize_int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Tensor* x = n == 1 ? tensor(args[0]) : nullptr;
  Rows r;
  mb_dtype type;
  if (!all_of_current_device({x}) || !known(x->scalar_type(), true, &type) || !rows_of(*x, &r))
    Py_RETURN_NONE;
  const int64_t pitch = pitch_of(r.K);
  Tensor codes = empty({r.rows, r.K}, {pitch, 1}, ScalarType::Char, *x);
  Tensor scales = empty({r.rows}, ScalarType::Float, *x);
  const mb_stream_t stream = stream_of(*x);
  if (!run([&] {
        return mb_int8_quantize(x->data_ptr(), type, r.rows, r.K, r.stride,
                                static_cast<int8_t*>(codes.data_ptr()), pitch,
                                static_cast<float*>(scales.data_ptr()), stream);
      }))
    return nullptr;
  return pair(std::move(codes), std::move(scales));
  END_HANDLE_TH_ERRORS
}

// (codes, scales, dtype) -> values
PyObject* dequantize_int8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  const Tensor *codes = tensor(args[0]), *scales = tensor(args[1]);
  Rows r;
  ScalarType to;
  mb_dtype type;
  if (!all_of_current_device({codes, scales}) || !known_dtype(args[2], &to, &type) ||
      !codes_of(*codes, *scales, &r))
    Py_RETURN_NONE;
  Tensor out = empty({r.rows, r.K}, to, *codes);
  const mb_stream_t stream = stream_of(*codes);
  if (!run([&] {
        return mb_int8_dequantize(static_cast<const int8_t*>(codes->data_ptr()), r.stride,
                                  static_cast<const float*>(scales->data_ptr()), r.rows, r.K,
                                  out.data_ptr(), type, r.K, stream);
      }))
    return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (x, its scales or None, codes of w, scales of w, bias or None, dtype or None)
// -> x W^T + bias
PyObject* int8_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const bool given = args[1] != Py_None, biased = args[4] != Py_None;
  const Tensor *x = tensor(args[0]), *wc = tensor(args[2]), *ws = tensor(args[3]);
  const Tensor* xs = given ? tensor(args[1]) : x;
  const Tensor* bias = biased ? tensor(args[4]) : x;
  Rows a, b;
  mb_dtype x_type = MB_FP16, bias_type = MB_FP16, type;
  if (!all_of_current_device({x, xs, wc, ws, bias}) || !codes_of(*wc, *ws, &b)) Py_RETURN_NONE;
  if (given ? !codes_of(*x, *xs, &a) : !known(x->scalar_type(), true, &x_type) || !rows_of(*x, &a))
    Py_RETURN_NONE;
  if (a.K != b.K || b.K > MB_INT8_MAX_K) Py_RETURN_NONE;
  if (biased && (bias->dim() != 1 || bias->size(0) != b.rows || !bias->is_contiguous() ||
                 !known(bias->scalar_type(), true, &bias_type)))
    Py_RETURN_NONE;
  ScalarType to = given ? ScalarType::Half : x->scalar_type();
  if (args[5] == Py_None ? !known(to, true, &type) : !known_dtype(args[5], &to, &type))
    Py_RETURN_NONE;
  at::DimVector sizes(x->sizes());
  sizes.back() = b.rows;
  Tensor out = empty(sizes, to, *x);
  const auto* w = static_cast<const int8_t*>(wc->data_ptr());
  const auto* w_scales = static_cast<const float*>(ws->data_ptr());
  const void* bias_data = biased ? bias->data_ptr() : nullptr;
  const mb_stream_t stream = stream_of(*x);
  if (given) {
    if (!run([&] {
          return mb_int8_matmul(static_cast<const int8_t*>(x->data_ptr()), a.stride,
                                static_cast<const float*>(xs->data_ptr()), a.rows, w, b.stride,
                                w_scales, b.rows, b.K, bias_data, bias_type, out.data_ptr(), type,
                                b.rows, stream);
        }))
      return nullptr;
  } else {
    const size_t bytes = mb_int8_linear_workspace_size(a.rows, a.K);
    const Tensor space = workspace(bytes, *x);
    if (!run([&] {
          return mb_int8_linear(x->data_ptr(), x_type, a.stride, a.rows, w, b.stride, w_scales,
                                b.rows, b.K, bias_data, bias_type, out.data_ptr(), type, b.rows,
                                space.data_ptr(), bytes, stream);
        }))
      return nullptr;
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (k_codes, v_codes, k_scales, v_scales, k, v, slots) -> True
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const Tensor* parts[4] = {tensor(args[0]), tensor(args[1]), tensor(args[2]), tensor(args[3])};
  const Tensor *k = tensor(args[4]), *v = tensor(args[5]), *slots = tensor(args[6]);
  mb_kv_cache c;
  mb_dtype type;
  if (!all_of_current_device({parts[0], parts[1], parts[2], parts[3], k, v, slots}) ||
      !cache_of(parts, &c) || !slots_of(*slots) || !known(k->scalar_type(), false, &type) ||
      v->scalar_type() != k->scalar_type() || k->dim() != 3 || k->sizes() != v->sizes() ||
      k->size(0) != slots->size(0) || k->size(1) != c.kv_heads || k->size(2) != c.head_dim ||
      k->stride(2) != 1 || v->stride(2) != 1)
    Py_RETURN_NONE;
  const size_t bytes = mb_cache_write_workspace_size(k->size(0));
  Tensor space;
  if (bytes > 0) space = workspace(bytes, *k);
  const mb_stream_t stream = stream_of(*k);
  if (!run([&] {
        return mb_cache_write(&c, k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(),
                              v->stride(0), v->stride(1), type, k->size(0),
                              static_cast<const int64_t*>(slots->data_ptr()),
                              bytes > 0 ? space.data_ptr() : nullptr, bytes, stream);
      }))
    return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (k_codes, v_codes, k_scales, v_scales, slots, dtype) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const Tensor* parts[4] = {tensor(args[0]), tensor(args[1]), tensor(args[2]), tensor(args[3])};
  const Tensor* slots = tensor(args[4]);
  mb_kv_cache c;
  ScalarType to;
  mb_dtype type;
  if (!all_of_current_device({parts[0], parts[1], parts[2], parts[3], slots}) ||
      !cache_of(parts, &c) || !slots_of(*slots) || !known_dtype(args[5], &to, &type))
    Py_RETURN_NONE;
  Tensor k = empty({slots->size(0), c.kv_heads, c.head_dim}, to, *slots);
  Tensor v = empty({slots->size(0), c.kv_heads, c.head_dim}, to, *slots);
  const mb_stream_t stream = stream_of(*slots);
  if (!run([&] {
        return mb_cache_read(&c, static_cast<const int64_t*>(slots->data_ptr()), slots->size(0),
                             k.data_ptr(), v.data_ptr(), type, stream);
      }))
    return nullptr;
  return pair(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// (k_codes, v_codes, k_scales, v_scales, q, page_table, lengths, scale) -> out
PyObject* cache_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !PyFloat_CheckExact(args[7])) Py_RETURN_NONE;
  const Tensor* parts[4] = {tensor(args[0]), tensor(args[1]), tensor(args[2]), tensor(args[3])};
  const Tensor *q = tensor(args[4]), *table = tensor(args[5]), *lengths = tensor(args[6]);
  mb_kv_cache c;
  mb_dtype type;
  if (!all_of_current_device({parts[0], parts[1], parts[2], parts[3], q, table, lengths}) ||
      !cache_of(parts, &c) || c.kv_heads == 0 || !known(q->scalar_type(), false, &type) ||
      q->dim() != 3 || q->numel() == 0 || q->size(1) % c.kv_heads != 0 ||
      q->size(2) != c.head_dim || q->stride(2) != 1 || table->dim() != 2 ||
      table->scalar_type() != ScalarType::Int || table->size(0) != q->size(0) ||
      (table->size(1) > 1 && table->stride(1) != 1) || lengths->dim() != 1 ||
      lengths->scalar_type() != ScalarType::Int || lengths->size(0) != q->size(0) ||
      !lengths->is_contiguous())
    Py_RETURN_NONE;
  const float scale = (float)PyFloat_AS_DOUBLE(args[7]);
  Tensor out = empty(q->sizes(), q->scalar_type(), *q);
  const size_t bytes =
      mb_cache_attention_workspace_size(&c, q->size(0), q->size(1), table->size(1));
  Tensor space;
  if (bytes > 0) space = workspace(bytes, *q);
  const mb_stream_t stream = stream_of(*q);
  if (!run([&] {
        return mb_cache_attention(&c, q->data_ptr(), q->stride(0), q->stride(1), type, q->size(0),
                                  q->size(1), static_cast<const int32_t*>(table->data_ptr()),
                                  table->stride(0), table->size(1),
                                  static_cast<const int32_t*>(lengths->data_ptr()), scale,
                                  out.data_ptr(), bytes > 0 ? space.data_ptr() : nullptr, bytes,
                                  stream);
      }))
    return nullptr;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL,
          nullptr};
}

PyMethodDef methods[] = {method<quantize_int8>("quantize_int8"),
                         method<dequantize_int8>("dequantize_int8"),
                         method<int8_matmul>("int8_matmul"),
                         method<cache_write>("cache_write"),
                         method<cache_read>("cache_read"),
                         method<cache_attention>("cache_attention"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", MB_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
