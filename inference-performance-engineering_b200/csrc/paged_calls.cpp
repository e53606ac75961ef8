// The Python functions of the paged operators, without an interpreter's cost per tensor: a call whose tensors are as
// the entry points of include/ipe_b200.h take them is launched here, any other is left to ipe_b200/paged.py, which
// says what is wrong with it. The kernels of a decode step take 3 to 6 us; the same checks and the call by way of
// ctypes took the host 10 to 13.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ipe_b200.h"

namespace {

constexpr int64_t kHead = 128;

// The tensors of a call: `device` is that of all of them, and the current one.
class Call {
 public:
  explicit Call(PyObject* pages) {
    const at::Tensor* t = tensor(pages);
    ok_ = t && t->is_cuda();
    if (!ok_) return;
    device_ = t->get_device();
    ok_ = device_ == c10::cuda::current_device();
  }

  // A contiguous tensor of the call's device, or one that is empty and makes the call none.
  const at::Tensor& take(PyObject* object, at::ScalarType type, int64_t dims) {
    const at::Tensor* t = tensor(object);
    if (!t || t->scalar_type() != type || t->dim() != dims || !t->is_cuda() || t->get_device() != device_ ||
        !t->is_contiguous()) {
      ok_ = false;
      return nothing_;
    }
    return *t;
  }
  const at::Tensor& take_bf16(PyObject* object, int64_t dims) { return take(object, at::kBFloat16, dims); }
  const at::Tensor& take_int(PyObject* object, int64_t dims) { return take(object, at::kInt, dims); }

  void need(bool condition) { ok_ = ok_ && condition; }
  bool ok() const { return ok_; }

  void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream(); }
  // the call's own: other streams and graphs have others
  at::Tensor workspace(size_t bytes) const {
    return at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(device_)));
  }

 private:
  static const at::Tensor* tensor(PyObject* object) {
    return THPVariable_CheckExact(object) ? &THPVariable_Unpack(object) : nullptr;
  }
  at::Tensor nothing_;
  int64_t device_ = -1;
  bool ok_ = false;
};

// The cache's tensors and their sizes.
struct Cache {
  const at::Tensor &k, &v, &table, &lengths;
  Cache(Call& call, PyObject* k_pages, PyObject* v_pages, PyObject* page_table, PyObject* lengths)
      : k(call.take_bf16(k_pages, 4)), v(call.take_bf16(v_pages, 4)), table(call.take_int(page_table, 2)),
        lengths(call.take_int(lengths, 1)) {
    if (call.ok()) call.need(k.size(3) == kHead && k.sizes() == v.sizes() && this->lengths.size(0) == table.size(0) &&
                             k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX && table.size(0) < INT32_MAX && table.size(1) <= INT32_MAX);
  }
  int kv_heads() const { return static_cast<int>(k.size(1)); }
  int page_size() const { return static_cast<int>(k.size(2)); }
  int sequences() const { return static_cast<int>(table.size(0)); }
  int width() const { return static_cast<int>(table.size(1)); }
};

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

template <typename Function>
PyObject* launched(Function&& function) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = function();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
}

// Every function: the entry point's status, or None where the call is not one that it takes.
template <typename Body>
PyObject* guarded(Py_ssize_t given, Py_ssize_t expected, Body&& body) {
  if (given != expected) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", expected, given);
    return nullptr;
  }
  HANDLE_TH_ERRORS  // what torch throws (a workspace that does not fit the device's memory) as torch raises it
  return body();
  END_HANDLE_TH_ERRORS
}

// (qkv, q_norm, k_norm, cos, sin, cu_tokens, lengths, page_table, eps, q_out, k_pages, v_pages)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const double eps = PyFloat_CheckExact(args[8]) ? PyFloat_AS_DOUBLE(args[8]) : -1.0;
    Call call(args[10]);
    if (!call.ok() || !PyFloat_CheckExact(args[8])) Py_RETURN_NONE;
    const Cache c(call, args[10], args[11], args[7], args[6]);
    const at::Tensor &qkv = call.take_bf16(args[0], 2), &q_norm = call.take_bf16(args[1], 1), &k_norm = call.take_bf16(args[2], 1),
                     &q_out = call.take_bf16(args[9], 3), &cu = call.take_int(args[5], 1);
    const bool fp32 = THPVariable_CheckExact(args[3]) && THPVariable_Unpack(args[3]).scalar_type() == at::kFloat;
    const at::Tensor &cos = call.take(args[3], fp32 ? at::kFloat : at::kBFloat16, 2), &sin = call.take(args[4], fp32 ? at::kFloat : at::kBFloat16, 2);
    if (!call.ok()) Py_RETURN_NONE;
    call.need(q_out.size(2) == kHead && q_out.size(1) <= INT32_MAX && qkv.size(0) == q_out.size(0) &&
              qkv.size(1) == (q_out.size(1) + 2 * c.k.size(1)) * kHead && q_norm.size(0) == kHead && k_norm.size(0) == kHead &&
              cos.size(1) == kHead && sin.sizes() == cos.sizes() && cu.size(0) == c.sequences() + 1);
    if (!call.ok()) Py_RETURN_NONE;
    void* stream = call.stream();
    return launched([&] {
      return ipe_paged_qk_norm_rope_append(
          qkv.const_data_ptr(), q_out.size(0), static_cast<int>(q_out.size(1)), c.kv_heads(), q_norm.const_data_ptr(),
          k_norm.const_data_ptr(), cos.const_data_ptr(), sin.const_data_ptr(), fp32, cos.size(0), ints(cu), ints(c.lengths),
          ints(c.table), c.sequences(), c.width(), q_out.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.k.size(0),
          c.page_size(), static_cast<float>(eps), stream);
    });
  });
}

// (q, k_pages, v_pages, page_table, lengths, out)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    Call call(args[1]);
    if (!call.ok()) Py_RETURN_NONE;
    const Cache c(call, args[1], args[2], args[3], args[4]);
    const at::Tensor &q = call.take_bf16(args[0], 3), &out = call.take_bf16(args[5], 2);
    if (!call.ok()) Py_RETURN_NONE;
    call.need(q.size(2) == kHead && q.size(0) == c.sequences() && q.size(1) <= INT32_MAX && out.size(0) == q.size(0) &&
              out.size(1) == q.size(1) * kHead);
    if (!call.ok()) Py_RETURN_NONE;
    const int q_heads = static_cast<int>(q.size(1));
    const size_t bytes = ipe_paged_decode_attention_workspace(c.sequences(), q_heads, c.kv_heads());
    at::Tensor workspace = call.workspace(bytes);
    void* stream = call.stream();
    return launched([&] {
      return ipe_paged_decode_attention(q.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), ints(c.table),
                                        ints(c.lengths), out.data_ptr(), c.sequences(), q_heads, c.kv_heads(), c.k.size(0),
                                        c.page_size(), c.width(), workspace.data_ptr(), bytes, stream);
    });
  });
}

// (q, k_pages, v_pages, page_table, cu_tokens, lengths, out)
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    Call call(args[1]);
    if (!call.ok()) Py_RETURN_NONE;
    const Cache c(call, args[1], args[2], args[3], args[5]);
    const at::Tensor &q = call.take_bf16(args[0], 3), &out = call.take_bf16(args[6], 2), &cu = call.take_int(args[4], 1);
    if (!call.ok()) Py_RETURN_NONE;
    call.need(q.size(2) == kHead && q.size(1) <= INT32_MAX && out.size(0) == q.size(0) && out.size(1) == q.size(1) * kHead &&
              cu.size(0) == c.sequences() + 1);
    if (!call.ok()) Py_RETURN_NONE;
    const int q_heads = static_cast<int>(q.size(1));
    const size_t bytes = ipe_paged_prefill_attention_workspace(q.size(0), c.sequences(), q_heads, c.kv_heads());
    at::Tensor workspace = call.workspace(bytes);
    void* stream = call.stream();
    return launched([&] {
      return ipe_paged_prefill_attention(q.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), ints(c.table), ints(cu),
                                         ints(c.lengths), out.data_ptr(), q.size(0), c.sequences(), q_heads, c.kv_heads(),
                                         c.k.size(0), c.page_size(), c.width(), workspace.data_ptr(), bytes, stream);
    });
  });
}

// (q, k_pages, v_pages, prefix_pages, page_table, lengths, out)
PyObject* shared(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    Call call(args[1]);
    if (!call.ok()) Py_RETURN_NONE;
    const Cache c(call, args[1], args[2], args[4], args[5]);
    const at::Tensor &q = call.take_bf16(args[0], 3), &out = call.take_bf16(args[6], 2), &prefix = call.take_int(args[3], 1);
    if (!call.ok()) Py_RETURN_NONE;
    call.need(q.size(2) == kHead && q.size(0) == c.sequences() && q.size(1) <= INT32_MAX && out.size(0) == q.size(0) &&
              out.size(1) == q.size(1) * kHead && prefix.size(0) <= c.width());
    if (!call.ok()) Py_RETURN_NONE;
    const int q_heads = static_cast<int>(q.size(1)), pages = static_cast<int>(prefix.size(0));
    const size_t bytes = ipe_shared_prefix_attention_workspace(c.sequences(), q_heads, c.kv_heads(), c.page_size(), pages);
    at::Tensor workspace = call.workspace(bytes);
    void* stream = call.stream();
    return launched([&] {
      return ipe_shared_prefix_attention(q.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), ints(prefix), pages,
                                         ints(c.table), ints(c.lengths), out.data_ptr(), c.sequences(), q_heads, c.kv_heads(),
                                         c.k.size(0), c.page_size(), c.width(), workspace.data_ptr(), bytes, stream);
    });
  });
}

template <typename Function>
PyCFunction as_method(Function f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)); }

PyMethodDef methods[] = {
    {"paged_qk_norm_rope_append", as_method(append), METH_FASTCALL, nullptr},
    {"paged_decode_attention", as_method(decode), METH_FASTCALL, nullptr},
    {"paged_prefill_attention", as_method(prefill), METH_FASTCALL, nullptr},
    {"shared_prefix_attention", as_method(shared), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_calls() { return PyModule_Create(&module); }
