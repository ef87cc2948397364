// The good case of the multi-request calls, decided in C++.
//
// A call of kernels.py on sixteen operands spends 9-12 us of host time on its
// checks and on ctypes' conversions, more than its two or three launches take
// (about 2 us each) and more than the kernels run at small batches: a server's
// eager calls would wait for Python.  The functions here take the same operands,
// look at each tensor through its C++ object and call the C entry directly.
//
// They decide nothing by themselves.  An operand that is not plainly right (not
// exactly a torch.Tensor, another type, shape, layout or device, a device that
// is not the current one, an integer that is not an int below 2^31) makes them
// return None before anything is enqueued, and the caller's own Python checks
// then name the fault or take the call.  Otherwise they return the output
// tensor, or the C entry's status as an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/headeronly/version.h>

#include <initializer_list>

#include "leanb200.h"

namespace {

// Reads one call's operands; `ok` turns false at the first one that is not plainly right.
struct Operands {
  bool ok = true;
  int dev = -1;

  int64_t integer(PyObject* o) {
    int overflow = 0;
    const long long v = PyLong_CheckExact(o) ? PyLong_AsLongLongAndOverflow(o, &overflow) : -1;
    if (overflow || v < 0 || v >= (1ll << 31)) ok = false;
    return ok ? v : 0;
  }
  bool flag(PyObject* o) {
    if (o != Py_True && o != Py_False) ok = false;
    return o == Py_True;
  }
  float real(PyObject* o) {
    if (!PyFloat_CheckExact(o)) ok = false;
    return ok ? static_cast<float>(PyFloat_AS_DOUBLE(o)) : 0.f;
  }
  const at::Tensor* tensor(PyObject* o) {
    const at::Tensor* t = ok && THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
    ok = t && t->defined() && t->is_cuda() && t->is_contiguous() && (dev < 0 || t->get_device() == dev);
    if (!ok) return nullptr;
    dev = t->get_device();  // the first operand's
    return t;
  }
  void* pointer(PyObject* o, at::ScalarType type, std::initializer_list<int64_t> shape) {
    const at::Tensor* t = tensor(o);
    ok = t && t->scalar_type() == type && t->sizes().equals(at::IntArrayRef(shape));
    return ok ? t->data_ptr() : nullptr;
  }
  void* optional(PyObject* o, at::ScalarType type, std::initializer_list<int64_t> shape) {
    return o == Py_None ? nullptr : pointer(o, type, shape);
  }
  // Given buffer, or a fresh one of `bytes`; `keep` holds the fresh one for the call (the allocator then hands its
  // memory out again in stream order).
  void* buffer(PyObject* o, int64_t bytes, at::Tensor& keep, int64_t& have) {
    if (!ok) return nullptr;
    if (o != Py_None) {
      const at::Tensor* t = tensor(o);
      ok = t && t->scalar_type() == at::kByte;
      if (!ok) return nullptr;
      have = t->numel();
      return t->data_ptr();
    }
    keep = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev));
    have = bytes;
    return keep.data_ptr();
  }
  // Given output, or a fresh one.  `out` holds it.
  void* output(PyObject* o, at::ScalarType type, std::initializer_list<int64_t> shape, at::Tensor& out) {
    if (!ok) return nullptr;
    if (o != Py_None) {
      void* p = pointer(o, type, shape);
      if (ok) out = THPVariable_Unpack(o);
      return p;
    }
    out = at::empty(at::IntArrayRef(shape), at::TensorOptions().dtype(type).device(at::kCUDA, dev));
    return out.data_ptr();
  }
  bool on_current_device() {
    if (ok && c10::cuda::current_device() != dev) ok = false;
    return ok;
  }
};

// The C entry's status, or the output tensor.
PyObject* result(int rc, at::Tensor out) { return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out)); }

template <class F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {  // a tensor without storage, an allocation that failed: the Python path meets it again and reports it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

ls_stream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

// (q, k_prefix, v_prefix, k_cache, v_cache, batch, q_len, num_heads, num_kv_heads, head_dim, prefix_len, max_seq,
//  scale, cache_pos, uniform_past, out, workspace)
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 17) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Operands o;
    const int64_t batch = o.integer(a[5]), q_len = o.integer(a[6]), hq = o.integer(a[7]), hkv = o.integer(a[8]);
    const int64_t d = o.integer(a[9]), prefix = o.integer(a[10]), max_seq = o.integer(a[11]);
    const int64_t past = o.integer(a[14]);
    const float scale = o.real(a[12]);
    const at::Tensor* q = o.tensor(a[0]);
    const at::Tensor* kp = o.tensor(a[1]);
    int64_t rows, per_row, elements;
    if (!o.ok || q->scalar_type() != at::kBFloat16 || kp->dim() != 3 || __builtin_mul_overflow(batch, q_len, &rows) ||
        __builtin_mul_overflow(hq, d, &per_row) || __builtin_mul_overflow(rows, per_row, &elements) ||
        q->numel() != elements)
      Py_RETURN_NONE;
    const int64_t cap = kp->size(1);
    const void* k_prefix = o.pointer(a[1], at::kBFloat16, {hkv, cap, d});
    const void* v_prefix = o.pointer(a[2], at::kBFloat16, {hkv, cap, d});
    const void* k_cache = o.pointer(a[3], at::kBFloat16, {batch, hkv, max_seq, d});
    const void* v_cache = o.pointer(a[4], at::kBFloat16, {batch, hkv, max_seq, d});
    const void* cursor = o.optional(a[13], at::kInt, {batch});
    int64_t need = 0, have = 0;
    if (!o.on_current_device() ||
        (a[16] == Py_None && ls_shared_prefix_attention_workspace_bytes(batch, q_len, hq, hkv, d, prefix, &need)))
      Py_RETURN_NONE;
    at::Tensor out, keep;
    void* to = o.output(a[15], at::kBFloat16, {rows, per_row}, out);
    void* ws = o.buffer(a[16], need < 256 ? 256 : need, keep, have);
    if (!o.ok) Py_RETURN_NONE;
    const void* from = q->data_ptr();
    const ls_stream_t stream = stream_of(o.dev);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = ls_shared_prefix_attention(
        from, k_prefix, v_prefix, prefix, cap, k_cache, v_cache, static_cast<const int32_t*>(cursor), past, batch,
        q_len, hq, hkv, d, max_seq, scale, to, ws, have, stream);
    Py_END_ALLOW_THREADS return result(rc, std::move(out));
  });
}

// (x, a, b, scaling, adapter_ids, q_len, accumulate, out, workspace)
PyObject* lora_delta(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Operands o;
    const int64_t q_len = o.integer(a[5]);
    const bool accumulate = o.flag(a[6]);
    const at::Tensor* x = o.tensor(a[0]);
    const at::Tensor* ta = o.tensor(a[1]);
    const at::Tensor* tb = o.tensor(a[2]);
    if (!o.ok || x->scalar_type() != at::kBFloat16 || x->dim() != 2 || ta->dim() != 3 || tb->dim() != 3 || q_len < 1 ||
        x->size(0) % q_len || (accumulate && a[7] == Py_None))
      Py_RETURN_NONE;
    const int64_t m = x->size(0), k = x->size(1), batch = m / q_len;
    const int64_t adapters = ta->size(0), rank = ta->size(1), width = tb->size(1);
    const void* pa = o.pointer(a[1], at::kBFloat16, {adapters, rank, k});
    const void* pb = o.pointer(a[2], at::kBFloat16, {adapters, width, rank});
    const void* scaling = o.pointer(a[3], at::kFloat, {adapters});
    const void* ids = o.pointer(a[4], at::kInt, {batch});
    int64_t need = 0, have = 0;
    if (!o.on_current_device() ||
        (a[8] == Py_None && ls_lora_delta_workspace_bytes(batch, q_len, k, width, rank, &need)))
      Py_RETURN_NONE;
    at::Tensor out, keep;
    void* to = o.output(a[7], at::kFloat, {m, width}, out);
    void* ws = o.buffer(a[8], need, keep, have);
    if (!o.ok) Py_RETURN_NONE;
    const void* from = x->data_ptr();
    const ls_stream_t stream = stream_of(o.dev);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc =
        ls_lora_delta(from, batch, q_len, k, pa, pb, static_cast<const float*>(scaling), adapters, width, rank,
                      static_cast<const int32_t*>(ids), accumulate, static_cast<float*>(to), ws, have, stream);
    Py_END_ALLOW_THREADS return result(rc, std::move(out));
  });
}

// (logits, counts, seen, repetition, frequency, presence, bias_ids, bias_values, allowed, record, out_ids, out_logits,
//  workspace)
PyObject* constrained_argmax(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Operands o;
    const bool record = o.flag(a[9]);
    const at::Tensor* t = o.tensor(a[0]);
    if (!o.ok || t->dim() != 2 || (t->scalar_type() != at::kBFloat16 && t->scalar_type() != at::kFloat) ||
        (a[6] == Py_None) != (a[7] == Py_None))
      Py_RETURN_NONE;
    const int64_t m = t->size(0), vocab = t->size(1), words = (vocab + 31) / 32;
    void* counts = o.optional(a[1], at::kInt, {m, vocab});
    void* seen = o.optional(a[2], at::kInt, {m, words});
    const void* repetition = o.optional(a[3], at::kFloat, {m});
    const void* frequency = o.optional(a[4], at::kFloat, {m});
    const void* presence = o.optional(a[5], at::kFloat, {m});
    const void *bias_ids = nullptr, *bias_values = nullptr;
    int64_t cap = 0;
    if (a[6] != Py_None) {
      const at::Tensor* b = o.tensor(a[6]);
      if (!o.ok || b->dim() != 2) Py_RETURN_NONE;
      cap = b->size(1);
      bias_ids = o.pointer(a[6], at::kInt, {m, cap});
      bias_values = o.pointer(a[7], at::kFloat, {m, cap});
      if (!cap) bias_ids = bias_values = nullptr;
    }
    const void* allowed = o.optional(a[8], at::kInt, {m, words});
    void* out_logits = o.optional(a[11], at::kFloat, {m, vocab});
    int64_t need = 0, have = 0;
    if (!o.on_current_device() || (a[12] == Py_None && ls_constrained_argmax_workspace_bytes(m, vocab, &need)))
      Py_RETURN_NONE;
    at::Tensor out, keep;
    void* ids = o.output(a[10], at::kLong, {m}, out);
    void* ws = o.buffer(a[12], need, keep, have);
    if (!o.ok) Py_RETURN_NONE;
    const void* from = t->data_ptr();
    const int is_f32 = t->scalar_type() == at::kFloat;
    const ls_stream_t stream = stream_of(o.dev);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = ls_constrained_argmax(
        from, is_f32, m, vocab, static_cast<int32_t*>(counts), static_cast<uint32_t*>(seen),
        static_cast<const float*>(repetition), static_cast<const float*>(frequency),
        static_cast<const float*>(presence), static_cast<const int32_t*>(bias_ids),
        static_cast<const float*>(bias_values), cap, static_cast<const uint32_t*>(allowed), record,
        static_cast<int64_t*>(ids), static_cast<float*>(out_logits), ws, have, stream);
    Py_END_ALLOW_THREADS return result(rc, std::move(out));
  });
}

PyMethodDef kMethods[] = {
    {"shared_prefix_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(shared_prefix_attention)),
     METH_FASTCALL, nullptr},
    {"lora_delta", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(lora_delta)), METH_FASTCALL, nullptr},
    {"constrained_argmax", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(constrained_argmax)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_front", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_front() {
  PyObject* m = PyModule_Create(&kModule);
  if (m) PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION);
  return m;
}
