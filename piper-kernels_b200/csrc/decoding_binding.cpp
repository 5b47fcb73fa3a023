// Direct binding of the decoding entry points for torch tensors.
//
// These operators run once per layer and token, often with a few microseconds
// of GPU work; argument checks in Python and a ctypes call cost 11 to 15 us, a
// call through here 4 to 7 (a launch alone is 3).
// Each function here checks its arguments in C++, allocates the outputs and
// calls the C ABI on the current stream.  It returns
//   the outputs   when the call was made,
//   a status      (int) when the C ABI refused or failed, and
//   None          when an argument is not what the operator takes, or the call
//                 is being traced: the Python layer then says what is wrong, or
//                 calls the registered operator.
// Nothing else is decided here, so that the Python path stays the whole
// contract.
#include <ATen/core/TensorBody.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <Python.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "piper_b200.h"

namespace {

using at::Tensor;

// What stands between a call and its kernels: modes and transforms that record
// or replace operators, and tensors whose memory is not their value.  Such calls
// belong to torch's dispatcher, which knows the operators by their registered names.
constexpr c10::DispatchKeySet kIntercepts({
    c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::PythonDispatcher,
    c10::DispatchKey::PreDispatch, c10::DispatchKey::Fake, c10::DispatchKey::Functionalize,
    c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
    c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Batched,
    c10::DispatchKey::VmapMode, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Tracer,
    c10::DispatchKey::DeferredInit, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
    c10::DispatchKey::ZeroTensor,
});

bool intercepted() {
  const c10::impl::LocalDispatchKeySet keys = c10::impl::tls_local_dispatch_key_set();
  return (keys.included_ - keys.excluded_).has_any(kIntercepts);
}

// A tensor that is nothing but one; nullptr for anything else, subclasses among it.
const Tensor* tensor_of(PyObject* x) {
  if (!THPVariable_CheckExact(x)) return nullptr;
  const Tensor& t = THPVariable_Unpack(x);
  return t.key_set().has_any(kIntercepts) ? nullptr : &t;
}
const Tensor* tensor_at(PyObject* const* args, Py_ssize_t i) { return tensor_of(args[i]); }

bool fits(const Tensor* t, std::initializer_list<int64_t> sizes, at::ScalarType type, c10::Device device) {
  if (t == nullptr || t->layout() != at::kStrided || t->dim() != static_cast<int64_t>(sizes.size()) ||
      t->scalar_type() != type || t->device() != device)
    return false;
  int64_t i = 0;
  for (const int64_t n : sizes)
    if (t->size(i++) != n) return false;
  return t->stride(-1) == 1 || t->size(-1) <= 1;
}

bool half_type(at::ScalarType type) { return type == at::kHalf || type == at::kBFloat16; }
int dtype_code(at::ScalarType type) { return type == at::kHalf ? PIPER_B200_FLOAT16 : PIPER_B200_BFLOAT16; }

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// The buffers of a handle (a tuple of four tensors and the key mean or None)
// with a batch's table and lengths.  Buffers can be resized or replaced in place
// after the handle was made, so that each call looks at all of them.
struct Cache {
  const Tensor* t[5] = {};
  piper_b200_kv_cache_t c{};
  c10::Device device{c10::kCPU};

  // `mean`: the call's result depends on the key mean.
  bool take(PyObject* buffers, const Tensor* table, const Tensor* lengths, int64_t batch, bool mean) {
    if (!PyTuple_Check(buffers) || PyTuple_GET_SIZE(buffers) != 5) return false;
    for (int i = 0; i < 5; ++i) {
      PyObject* item = PyTuple_GET_ITEM(buffers, i);
      if (i == 4 && item == Py_None) break;
      if ((t[i] = tensor_of(item)) == nullptr) return false;
    }
    device = t[0]->device();
    if (!device.is_cuda() || t[0]->dim() != 4 || batch <= 0 || table == nullptr || table->dim() != 2 ||
        table->size(1) <= 0 || table->size(1) > INT32_MAX || batch > INT32_MAX)
      return false;
    const int64_t pages = t[0]->size(0), heads = t[0]->size(1), page = t[0]->size(2), d = t[0]->size(3);
    if (pages <= 0 || heads <= 0 || heads > INT32_MAX || page <= 0 || page > INT32_MAX || (d != 64 && d != 128))
      return false;
    for (int i = 0; i < 4; ++i)
      if (!(i % 2 == 0 ? fits(t[i], {pages, heads, page, d}, at::kChar, device)
                       : fits(t[i], {pages, heads, page}, at::kFloat, device)) ||
          !t[i]->is_contiguous())
        return false;
    if (t[4] != nullptr && !(fits(t[4], {heads, d}, at::kFloat, device) && t[4]->is_contiguous())) return false;
    if (wants_grad(*t[1]) || wants_grad(*t[3]) || (mean && t[4] != nullptr && wants_grad(*t[4]))) return false;
    if (!fits(table, {batch, table->size(1)}, at::kInt, device) || !fits(lengths, {batch}, at::kInt, device))
      return false;
    c.key_codes = t[0]->data_ptr();
    c.key_scales = static_cast<float*>(t[1]->data_ptr());
    c.value_codes = t[2]->data_ptr();
    c.value_scales = static_cast<float*>(t[3]->data_ptr());
    c.key_mean = t[4] ? static_cast<const float*>(t[4]->data_ptr()) : nullptr;
    c.block_table = static_cast<const int32_t*>(table->data_ptr());
    c.lengths = static_cast<const int32_t*>(lengths->data_ptr());
    c.pages = pages;
    c.kv_heads = static_cast<int32_t>(heads);
    c.page_size = static_cast<int32_t>(page);
    c.head_dim = static_cast<int32_t>(d);
    c.batch = static_cast<int32_t>(batch);
    c.table_width = static_cast<int32_t>(table->size(1));
    c.table_stride = table->stride(0);
    return true;
  }

  // The rows have been written to: autograd, and whoever else saved a buffer, can tell.
  void written() const {
    for (int i = 0; i < 4; ++i)
      if (!t[i]->is_inference()) t[i]->unsafeGetTensorImpl()->bump_version();
  }
};

// counts: None, or int32 [batch].
bool take_counts(PyObject* arg, int64_t batch, c10::Device device, const int32_t** out) {
  *out = nullptr;
  if (arg == Py_None) return true;
  const Tensor* t = tensor_of(arg);
  if (!fits(t, {batch}, at::kInt, device)) return false;
  *out = static_cast<const int32_t*>(t->data_ptr());
  return true;
}

void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

PyObject* none() { Py_RETURN_NONE; }
PyObject* status(int rc) { return PyLong_FromLong(rc); }

// C++ exceptions become the Python ones that torch raises for them.
template <typename Body>
PyObject* guarded(Body body) {
  HANDLE_TH_ERRORS
  return body();
  END_HANDLE_TH_ERRORS
}

// attend(buffers, query, table, lengths, mask or None, scale or None)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || intercepted()) return none();
    const Tensor* q = tensor_at(args, 1);
    if (q == nullptr || q->dim() != 4 || !half_type(q->scalar_type()) || wants_grad(*q)) return none();
    const int64_t batch = q->size(0), heads = q->size(1), nodes = q->size(2);
    const Tensor *table = tensor_at(args, 2), *lengths = tensor_at(args, 3);
    Cache cache;
    if (!cache.take(args[0], table, lengths, batch, false)) return none();
    const int64_t d = cache.c.head_dim;
    if (!fits(q, {batch, heads, nodes, d}, q->scalar_type(), cache.device) || nodes < 1 || nodes > 64 || heads < 1 ||
        heads % cache.c.kv_heads != 0)
      return none();
    const int64_t* mask = nullptr;
    int64_t mask_stride = 0;
    if (args[4] != Py_None) {
      const Tensor* m = tensor_at(args, 4);
      if (m == nullptr || !(m->dim() == 1 ? fits(m, {nodes}, at::kLong, cache.device)
                                          : fits(m, {batch, nodes}, at::kLong, cache.device)))
        return none();
      mask = static_cast<const int64_t*>(m->data_ptr());
      mask_stride = m->dim() == 2 ? m->stride(0) : 0;
    }
    double scale = 0.0;
    if (args[5] == Py_None) {
      scale = d == 64 ? 0.125 : 0.08838834764831845;  // d ** -0.5
    } else {
      if (!PyFloat_Check(args[5])) return none();
      scale = PyFloat_AS_DOUBLE(args[5]);
      if (!(scale >= 0x1p-126 && scale <= 0x1p127)) return none();
    }
    const c10::cuda::OptionalCUDAGuard guard(cache.device);
    size_t bytes = 0;
    int rc = piper_b200_tree_attention_workspace_bytes(
        batch, heads, cache.c.kv_heads, nodes, d, static_cast<int64_t>(cache.c.table_width) * cache.c.page_size,
        &bytes);
    if (rc != PIPER_B200_OK) return status(rc);
    Tensor out = at::empty({batch, heads, nodes, d}, q->options());
    Tensor workspace;
    if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, q->options().dtype(at::kByte));
    const int64_t strides[3] = {q->stride(0), q->stride(1), q->stride(2)};
    rc = piper_b200_tree_attention(&cache.c, q->data_ptr(), strides, out.data_ptr(), dtype_code(q->scalar_type()),
                                   heads, nodes, mask, mask_stride, scale, bytes > 0 ? workspace.data_ptr() : nullptr,
                                   bytes, stream_of(cache.device));
    return rc != PIPER_B200_OK ? status(rc) : THPVariable_Wrap(std::move(out));
  });
}

// write(buffers, key, value, table, lengths, counts or None): True
PyObject* write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || intercepted()) return none();
    const Tensor *k = tensor_at(args, 1), *v = tensor_at(args, 2);
    if (k == nullptr || v == nullptr || k->dim() != 4 || !half_type(k->scalar_type()) || wants_grad(*k) ||
        wants_grad(*v))
      return none();
    const int64_t batch = k->size(0), tokens = k->size(2);
    Cache cache;
    if (!cache.take(args[0], tensor_at(args, 3), tensor_at(args, 4), batch, true) || tokens < 1) return none();
    const std::initializer_list<int64_t> sizes = {batch, cache.c.kv_heads, tokens, cache.c.head_dim};
    const int32_t* counts = nullptr;
    if (!fits(k, sizes, k->scalar_type(), cache.device) || !fits(v, sizes, k->scalar_type(), cache.device) ||
        !take_counts(args[5], batch, cache.device, &counts))
      return none();
    const c10::cuda::OptionalCUDAGuard guard(cache.device);
    const int64_t ks[3] = {k->stride(0), k->stride(1), k->stride(2)};
    const int64_t vs[3] = {v->stride(0), v->stride(1), v->stride(2)};
    const int rc = piper_b200_kv_cache_write(&cache.c, k->data_ptr(), ks, v->data_ptr(), vs,
                                             dtype_code(k->scalar_type()), tokens, counts, stream_of(cache.device));
    if (rc != PIPER_B200_OK) return status(rc);
    cache.written();
    Py_RETURN_TRUE;
  });
}

// read(buffers, table, lengths, counts or None, tokens, half precision?): (key, value)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || intercepted() || !PyLong_Check(args[4])) return none();
    const Tensor* lengths = tensor_at(args, 2);
    const int64_t tokens = PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
    if (lengths == nullptr || lengths->dim() != 1 || tokens < 1) return none();
    const int64_t batch = lengths->size(0);
    Cache cache;
    const int32_t* counts = nullptr;
    if (!cache.take(args[0], tensor_at(args, 1), lengths, batch, true) ||
        !take_counts(args[3], batch, cache.device, &counts))
      return none();
    const at::ScalarType type = args[5] == Py_True ? at::kHalf : at::kBFloat16;
    const c10::cuda::OptionalCUDAGuard guard(cache.device);
    const auto options = lengths->options().dtype(type);
    Tensor key = at::empty({batch, cache.c.kv_heads, tokens, cache.c.head_dim}, options);
    Tensor value = at::empty({batch, cache.c.kv_heads, tokens, cache.c.head_dim}, options);
    const int rc = piper_b200_kv_cache_read(&cache.c, key.data_ptr(), value.data_ptr(), dtype_code(type), tokens,
                                            counts, stream_of(cache.device));
    if (rc != PIPER_B200_OK) return status(rc);
    PyObject* pair = PyTuple_New(2);
    if (pair == nullptr) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(key)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(value)));
    return pair;
  });
}

// keep(buffers, table, lengths, path, counts): True
PyObject* keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 5 || intercepted()) return none();
    const Tensor* path = tensor_at(args, 3);
    if (path == nullptr || path->dim() != 2 || args[4] == Py_None) return none();
    const int64_t batch = path->size(0), nodes = path->size(1);
    Cache cache;
    const int32_t* counts = nullptr;
    if (nodes < 1 || nodes > 64 || !cache.take(args[0], tensor_at(args, 1), tensor_at(args, 2), batch, false) ||
        !fits(path, {batch, nodes}, at::kInt, cache.device) || !take_counts(args[4], batch, cache.device, &counts))
      return none();
    const c10::cuda::OptionalCUDAGuard guard(cache.device);
    const int rc = piper_b200_kv_cache_keep(&cache.c, static_cast<const int32_t*>(path->data_ptr()), path->stride(0),
                                            nodes, counts, stream_of(cache.device));
    if (rc != PIPER_B200_OK) return status(rc);
    cache.written();
    Py_RETURN_TRUE;
  });
}

// verify(target, draft, tokens, parents, uniform, noise): (path, count, next)
PyObject* verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || intercepted()) return none();
    const Tensor* t[6];
    for (int i = 0; i < 6; ++i)
      if ((t[i] = tensor_at(args, i)) == nullptr) return none();
    if (t[0]->dim() != 3 || !t[0]->is_cuda() || wants_grad(*t[0]) || wants_grad(*t[1])) return none();
    const int64_t batch = t[0]->size(0), nodes = t[0]->size(1), vocab = t[0]->size(2);
    const c10::Device device = t[0]->device();
    if (batch < 1 || vocab < 1 || nodes < 1 || nodes > 64 || !fits(t[0], {batch, nodes, vocab}, at::kFloat, device) ||
        !fits(t[1], {batch, nodes, vocab}, at::kFloat, device) || !fits(t[2], {batch, nodes}, at::kLong, device) ||
        !fits(t[3], {batch, nodes}, at::kInt, device) || !fits(t[4], {batch, nodes}, at::kFloat, device) ||
        !fits(t[5], {batch, vocab}, at::kFloat, device))
      return none();
    const c10::cuda::OptionalCUDAGuard guard(device);
    Tensor path = at::empty({batch, nodes}, t[3]->options());
    Tensor count = at::empty({batch}, t[3]->options());
    Tensor next = at::empty({batch}, t[2]->options());
    const int64_t ts[2] = {t[0]->stride(0), t[0]->stride(1)}, ds[2] = {t[1]->stride(0), t[1]->stride(1)};
    const int rc = piper_b200_verify_draft_tree(
        static_cast<const float*>(t[0]->data_ptr()), ts, static_cast<const float*>(t[1]->data_ptr()), ds,
        static_cast<const int64_t*>(t[2]->data_ptr()), t[2]->stride(0), static_cast<const int32_t*>(t[3]->data_ptr()),
        t[3]->stride(0), static_cast<const float*>(t[4]->data_ptr()), t[4]->stride(0),
        static_cast<const float*>(t[5]->data_ptr()), t[5]->stride(0), batch, nodes, vocab,
        static_cast<int32_t*>(path.data_ptr()), static_cast<int32_t*>(count.data_ptr()),
        static_cast<int64_t*>(next.data_ptr()), stream_of(device));
    if (rc != PIPER_B200_OK) return status(rc);
    PyObject* found = PyTuple_New(3);
    if (found == nullptr) return nullptr;
    PyTuple_SET_ITEM(found, 0, THPVariable_Wrap(std::move(path)));
    PyTuple_SET_ITEM(found, 1, THPVariable_Wrap(std::move(count)));
    PyTuple_SET_ITEM(found, 2, THPVariable_Wrap(std::move(next)));
    return found;
  });
}

PyMethodDef methods[] = {
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(write)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(read)), METH_FASTCALL, nullptr},
    {"keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(keep)), METH_FASTCALL, nullptr},
    {"verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(verify)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "decoding_binding", nullptr, -1, methods,
                          nullptr,               nullptr,            nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_decoding_binding() {
  return PyModule_Create(&module_def);
}
