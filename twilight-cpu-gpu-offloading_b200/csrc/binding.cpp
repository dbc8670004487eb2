// Python calls of the paged-cache entry points with torch tensors, unpacked here:
// these calls are made for every step and layer, and through ctypes the host takes
// longer for one (16 us for an attention, 8.5 us for the others) than the device for a
// short one.  Each call checks its tensors in one expression.  What it returns:
//   None or the output tensor: done; an int > 0: the status of the C ABI;
//   an int < 0: a tensor is not as wanted (the caller works out which).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <map>

#include "../../include/twilight_b200.h"

namespace {

constexpr int kHeadDim = 128;

// A tensor argument; nullptr for None and for what is no tensor.
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}
// An argument that may be None; false: it is something else.
bool optional(PyObject* o, const at::Tensor*& t) {
  t = tensor(o);
  return t != nullptr || o == Py_None;
}

// The CUDA device of a call: that of `t`, which is the current one (-1: it is not).
int device_of(const at::Tensor* t) {
  if (!t || !t->is_cuda()) return -1;
  const int dev = t->get_device();
  return dev == c10::cuda::current_device() ? dev : -1;
}

// [n] or, with rows > 0, [rows, any] of one type with contiguous rows.
bool vec(const at::Tensor* t, int dev, at::ScalarType type, int64_t n) {
  return t && t->is_cuda() && t->get_device() == dev && t->scalar_type() == type &&
         t->dim() == 1 && (n < 0 || t->size(0) == n) && t->is_contiguous();
}
bool table(const at::Tensor* t, int dev, int64_t rows) {
  return t && t->is_cuda() && t->get_device() == dev && t->scalar_type() == at::kInt &&
         t->dim() == 2 && t->size(0) == rows && (t->stride(1) == 1 || t->size(1) == 1);
}
bool flag(const at::Tensor* t, int dev) {
  return !t || (t->is_cuda() && t->get_device() == dev && t->scalar_type() == at::kInt &&
                t->numel() >= 1);
}
template <typename T> T* ptr(const at::Tensor* t) { return t ? (T*)t->data_ptr() : nullptr; }

bool stride_ok(int64_t s) { return s > 0 && s % 8 == 0; }

// (token, head) strides of [tokens, heads, 128] rows; an extent of 1 has none of its own.
bool rows(const at::Tensor& t, int64_t& token, int64_t& head) {
  head = t.size(1) > 1 ? t.stride(1) : kHeadDim;
  token = t.size(0) > 1 ? t.stride(0) : head * std::max<int64_t>(t.size(1), 1);
  return t.stride(2) == 1 && stride_ok(token) && stride_ok(head) &&
         ((uintptr_t)t.data_ptr() & 15) == 0;
}

bool pool(const at::Tensor* k, const at::Tensor* v, int dev, tw_paged_pool& p) {
  if (!k || !v || !k->is_cuda() || !v->is_cuda() || k->get_device() != dev ||
      v->get_device() != dev || k->dim() != 4 || k->sizes() != v->sizes() ||
      k->scalar_type() != v->scalar_type() || k->size(3) != kHeadDim || k->numel() == 0 ||
      (k->scalar_type() != at::kHalf && k->scalar_type() != at::kBFloat16) || k->stride(3) != 1 ||
      v->stride(3) != 1)
    return false;
  int64_t s[3];
  for (int i = 0; i < 3; ++i) {
    s[i] = k->size(i) > 1 ? k->stride(i) : kHeadDim;
    if ((k->size(i) > 1 && k->stride(i) != v->stride(i)) || !stride_ok(s[i])) return false;
  }
  p = {k->data_ptr(), v->data_ptr(), s[0], s[1], s[2], k->size(0), (int32_t)k->size(2),
       (int32_t)k->size(1), kHeadDim, k->scalar_type() == at::kHalf ? TW_F16 : TW_BF16};
  return (((uintptr_t)p.k_pages | (uintptr_t)p.v_pages) & 15) == 0;
}

PyObject* status(int rc) {
  if (rc == TW_OK) Py_RETURN_NONE;
  return PyLong_FromLong(rc);
}
PyObject* unexpected() { return PyLong_FromLong(-1); }

// A whole number that fits the C ABI's int; false with a Python error otherwise.
bool whole(PyObject* o, int& x) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) return false;
  if (v < INT32_MIN || v > INT32_MAX) {
    PyErr_SetString(PyExc_ValueError, "an argument does not fit 32 bits");
    return false;
  }
  x = (int)v;
  return true;
}

template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments wanted, %zd given", want, n);
    return nullptr;
  }
  try {
    return f();
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

// lens, new_lens, block_table, free_pages, free_count, page_size, kv_lens, cu_q, slots,
// positions, free_count_out, error_flag
PyObject* paged_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const at::Tensor *lens = tensor(o[0]), *fresh = tensor(o[1]), *tab = tensor(o[2]),
                     *stack = tensor(o[3]), *count = tensor(o[4]), *kv = tensor(o[6]),
                     *cu = tensor(o[7]), *slots = tensor(o[8]), *pos = tensor(o[9]),
                     *left = tensor(o[10]), *err;
    int page_size;
    if (!whole(o[5], page_size)) return nullptr;
    const int dev = device_of(lens);
    if (dev < 0 || !vec(lens, dev, at::kInt, -1)) return unexpected();
    const int64_t B = lens->size(0);
    if (!vec(fresh, dev, at::kInt, B) || !table(tab, dev, B) || !vec(stack, dev, at::kInt, -1) ||
        !vec(count, dev, at::kInt, 1) || !vec(kv, dev, at::kInt, B) ||
        !vec(cu, dev, at::kInt, B + 1) || !vec(slots, dev, at::kLong, -1) ||
        !vec(pos, dev, at::kInt, slots->size(0)) || !vec(left, dev, at::kInt, 1) ||
        !optional(o[11], err) || !flag(err, dev) || B > INT32_MAX ||
        slots->size(0) > INT32_MAX || tab->size(1) > INT32_MAX)
      return unexpected();
    tw_paged_step_args a = {};
    a.lens = ptr<int32_t>(lens);
    a.new_lens = ptr<int32_t>(fresh);
    a.block_table = ptr<int32_t>(tab);
    a.table_width = (int32_t)tab->size(1);
    a.table_stride = B > 1 ? tab->stride(0) : a.table_width;
    a.requests = (int32_t)B;
    a.page_size = page_size;
    a.tokens_cap = (int32_t)slots->size(0);
    a.free_pages = ptr<int32_t>(stack);
    a.num_pages = stack->size(0);
    a.free_count = ptr<int32_t>(count);
    a.kv_lens = ptr<int32_t>(kv);
    a.cu_q = ptr<int32_t>(cu);
    a.slots = ptr<int64_t>(slots);
    a.positions = ptr<int32_t>(pos);
    a.free_count_out = ptr<int32_t>(left);
    a.error_flag = ptr<int32_t>(err);
    return status(tw_paged_step(&a, stream_of(dev)));
  });
}

// k, v, slots, k_pages, v_pages, error_flag
PyObject* paged_write(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const at::Tensor *k = tensor(o[0]), *v = tensor(o[1]), *slots = tensor(o[2]), *err;
    const int dev = device_of(k);
    tw_paged_pool p;
    int64_t kt, kh, vt, vh;
    if (dev < 0 || !pool(tensor(o[3]), tensor(o[4]), dev, p) || !v || !v->is_cuda() ||
        v->get_device() != dev || k->dim() != 3 || k->sizes() != v->sizes() ||
        k->size(1) != p.kv_heads || k->size(2) != kHeadDim ||
        k->scalar_type() != tensor(o[3])->scalar_type() || v->scalar_type() != k->scalar_type() ||
        !vec(slots, dev, at::kLong, k->size(0)) || !optional(o[5], err) || !flag(err, dev) ||
        !rows(*k, kt, kh) || !rows(*v, vt, vh))
      return unexpected();
    return status(tw_paged_write(&p, k->data_ptr(), kt, kh, v->data_ptr(), vt, vh,
                                 ptr<int64_t>(slots), k->size(0), ptr<int32_t>(err),
                                 stream_of(dev)));
  });
}

// The workspace of calls that brought none, kept per stream: calls on one stream
// follow one another, and a larger one takes the place of a smaller.  A graph under
// capture gets its own, and so does a call that needs much, which takes long enough for
// the allocator's time not to count: what stays is bounded.
constexpr size_t kKeptBytes = 32 << 20;
at::Tensor workspace_for(const at::Tensor& like, int dev, void* stream, size_t bytes) {
  const auto fresh = [&] {
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
  };
  if (bytes > kKeptBytes ||
      c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return fresh();
  // never destroyed: at exit the allocator may be gone first
  static auto* kept = new std::map<std::pair<int, void*>, at::Tensor>;
  at::Tensor& t = (*kept)[{dev, stream}];
  if (!t.defined() || (size_t)t.numel() < bytes) t = fresh();
  return t;
}

// q, k_pages, v_pages, block_table, cu_q, kv_lens, max_q_len, max_kv_len, window,
// softmax_scale, out, out_dtype, lse, workspace, error_flag
PyObject* paged_attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 15, [&]() -> PyObject* {
    const at::Tensor *q = tensor(o[0]), *tab = tensor(o[3]), *cu = tensor(o[4]),
                     *kv = tensor(o[5]), *out, *lse, *ws, *err;
    tw_paged_attention_args a = {};
    if (!whole(o[6], a.max_q_len) || !whole(o[7], a.max_kv_len) || !whole(o[8], a.window))
      return nullptr;
    a.softmax_scale = 0.08838834764831845f;  // 1 / sqrt(128)
    if (o[9] != Py_None) {
      const double s = PyFloat_AsDouble(o[9]);
      if (s == -1.0 && PyErr_Occurred()) return nullptr;
      a.softmax_scale = (float)s;
    }
    const int dev = device_of(q);
    if (dev < 0 || !pool(tensor(o[1]), tensor(o[2]), dev, a.pool) || q->dim() != 3 ||
        q->size(2) != kHeadDim || q->scalar_type() != tensor(o[1])->scalar_type() ||
        q->size(1) == 0 || q->size(1) % a.pool.kv_heads != 0 || q->size(0) > INT32_MAX ||
        q->size(1) > INT32_MAX || !vec(kv, dev, at::kInt, -1) ||
        !vec(cu, dev, at::kInt, kv->size(0) + 1) || !table(tab, dev, kv->size(0)) ||
        kv->size(0) > INT32_MAX || tab->size(1) > INT32_MAX || !optional(o[10], out) ||
        !optional(o[12], lse) || !optional(o[13], ws) || !optional(o[14], err) ||
        !flag(err, dev) || !rows(*q, a.q_token_stride, a.q_head_stride))
      return unexpected();
    const int64_t T = q->size(0), H = q->size(1), B = kv->size(0);
    if (lse && !(lse->is_cuda() && lse->get_device() == dev && lse->scalar_type() == at::kFloat &&
                 lse->dim() == 2 && lse->size(0) == T && lse->size(1) == H &&
                 lse->is_contiguous()))
      return unexpected();
    at::ScalarType type = out ? out->scalar_type() : q->scalar_type();
    if (o[11] != Py_None) {
      if (!THPDtype_Check(o[11])) return unexpected();
      const at::ScalarType asked = reinterpret_cast<THPDtype*>(o[11])->scalar_type;
      if (out && asked != type) return unexpected();
      type = asked;
    }
    if (type != q->scalar_type() && type != at::kFloat) return unexpected();
    at::Tensor made;
    if (!out) {
      made = at::empty({T, H, kHeadDim}, q->options().dtype(type));
      out = &made;
    }
    if (!out->is_cuda() || out->get_device() != dev || out->sizes() != q->sizes() ||
        !rows(*out, a.out_token_stride, a.out_head_stride))
      return unexpected();
    void* stream = stream_of(dev);
    at::Tensor kept;
    if (!ws) {
      const size_t need = tw_paged_attention_workspace_size((int)B, (int)T, (int)H, a.pool.kv_heads,
                                                            a.max_q_len, a.max_kv_len, a.window,
                                                            kHeadDim);
      if (need > 0) {
        kept = workspace_for(*q, dev, stream, need);
        ws = &kept;
      }
    } else if (!ws->is_cuda() || ws->get_device() != dev || !ws->is_contiguous()) {
      return unexpected();
    }
    a.q = q->data_ptr();
    a.block_table = ptr<int32_t>(tab);
    a.table_width = (int32_t)tab->size(1);
    a.table_stride = B > 1 ? tab->stride(0) : a.table_width;
    a.requests = (int32_t)B;
    a.cu_q = ptr<int32_t>(cu);
    a.kv_lens = ptr<int32_t>(kv);
    a.tokens = (int32_t)T;
    a.q_heads = (int32_t)H;
    a.out = out->data_ptr();
    a.out_dtype = type == at::kFloat ? TW_F32 : type == at::kHalf ? TW_F16 : TW_BF16;
    a.lse = ptr<float>(lse);
    a.error_flag = ptr<int32_t>(err);
    a.workspace = ptr<void>(ws);
    a.workspace_bytes = ws ? ws->nbytes() : 0;
    const int rc = tw_paged_attention(&a, stream);
    if (rc != TW_OK) return PyLong_FromLong(rc);
    if (!made.defined()) {
      Py_INCREF(o[10]);
      return o[10];
    }
    return THPVariable_Wrap(std::move(made));
  });
}

PyMethodDef kMethods[] = {
    {"paged_step", (PyCFunction)(void*)paged_step, METH_FASTCALL, nullptr},
    {"paged_write", (PyCFunction)(void*)paged_write, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void*)paged_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
