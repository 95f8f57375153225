// Short way from the Python ops of the quantised cache to the C ABI (include/kvc.h).
//
// A call's own work is a few microseconds: one launch.  Asking some ten tensors in Python for
// their shapes, strides, types and devices and handing twenty arguments to ctypes costs as much
// again or more (host time of a write 7.9 us, a read 9.7, a decode 12.3; by this way 3.5, 3.8 and
// 5.1).  Each function here takes the op's arguments, checks what the op checks and calls the C
// entry.  It returns None for whatever is not an ordinary call (wrong or unusual arguments, a
// stream of its own, another device than the current one): the op then goes on in Python, which
// says what is wrong or does the unusual.  Otherwise it returns the entry's status (0 is KVC_OK),
// or the decode's result.  The checks here and in quantized.py are two copies of the same ones: a
// change of either side changes both.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

#include "kvc.h"

namespace {

decltype(&kvc_reshape_and_cache_quantized) write_entry;
decltype(&kvc_gather_quantized_kv) read_entry;
decltype(&kvc_quantized_decode) decode_entry;
PyObject* current_device;   // torch's queries, as the ops make them
PyObject* current_stream;

constexpr int64_t kPage = 16;

// A tensor argument on GPU `device` (the first one sets it); null: none of that kind.
const at::Tensor* tensor(PyObject* o, int64_t& device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda()) return nullptr;
  if (device < 0) device = t.get_device();
  return t.get_device() == device ? &t : nullptr;
}

struct Cache {
  const at::Tensor *key, *value, *scales;
  int64_t blocks, heads, dim, stride, scales_stride;
  int32_t code;

  bool take(PyObject* const* o, int64_t& device) {
    if (!(key = tensor(o[0], device)) || !(value = tensor(o[1], device)) ||
        !(scales = tensor(o[2], device)))
      return false;
    const auto type = key->scalar_type();
    if (type == at::kFloat8_e4m3fn)
      code = KVC_CODE_E4M3;
    else if (type == at::kChar)
      code = KVC_CODE_INT8;
    else
      return false;
    if (value->scalar_type() != type || scales->scalar_type() != at::kFloat || key->dim() != 4 ||
        scales->dim() != 4)
      return false;
    blocks = key->size(0);
    heads = key->size(1);
    dim = key->size(3);
    stride = key->stride(0);
    scales_stride = scales->stride(0);
    return key->size(2) == kPage && value->sizes() == key->sizes() &&
           value->strides() == key->strides() && blocks > 1 && key->stride(3) == 1 &&
           key->stride(2) == dim && key->stride(1) == kPage * dim && scales->size(0) == blocks &&
           scales->size(1) == heads && scales->size(2) == 2 && scales->size(3) == kPage &&
           scales->stride(3) == 1 && scales->stride(2) == kPage && scales->stride(1) == 2 * kPage;
  }
};

// [tokens, heads, dim] of bf16 or fp16, a token's heads contiguous: its dtype code, or -1.
int32_t tokens(const at::Tensor& t, int64_t heads, int64_t dim, int64_t& stride) {
  if (t.dim() != 3 || t.size(1) != heads || t.size(2) != dim || t.stride(2) != 1 ||
      (t.stride(1) != dim && heads > 1))
    return -1;
  stride = t.size(0) > 1 ? t.stride(0) : heads * dim;
  if (t.scalar_type() == at::kBFloat16) return KVC_DTYPE_BF16;
  return t.scalar_type() == at::kHalf ? KVC_DTYPE_FP16 : -1;
}

bool ints(const at::Tensor* t, int64_t n) {
  return t && t->scalar_type() == at::kInt && t->dim() == 1 && t->numel() >= n && t->is_contiguous();
}

// The optional counter: false if it is not one.
bool counter(PyObject* o, int64_t& device, int32_t*& p) {
  p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o, device);
  if (!t || t->scalar_type() != at::kInt || t->numel() < 1) return false;
  p = static_cast<int32_t*>(t->data_ptr());
  return true;
}

// The stream's handle if `device` is the current one.  `given`: the op's stream argument.
bool stream_of(PyObject* given, int64_t device, void*& stream) {
  if (given != Py_None) return false;
  PyObject* now = PyObject_CallNoArgs(current_device);
  if (!now) return false;
  const bool here = PyLong_AsLongLong(now) == device;
  if (here) {
    PyObject* s = PyObject_CallOneArg(current_stream, now);
    if (s) {
      stream = PyLong_AsVoidPtr(s);
      Py_DECREF(s);
    }
  }
  Py_DECREF(now);
  return here && !PyErr_Occurred();
}

// A C entry's status.  Other Python threads run meanwhile, as during a ctypes call: a launch
// waits while the stream's queue is full.
template <typename... P, typename... A>
int call(int (*entry)(P...), A... args) {
  struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
  } unlocked;
  return entry(args...);
}

// Runs f; what it cannot do, and every exception in it, is None.
template <typename F>
PyObject* attempt(F f) {
  PyObject* got = nullptr;
  try {
    got = f();
  } catch (...) {
    got = nullptr;
  }
  if (got) return got;
  PyErr_Clear();
  Py_RETURN_NONE;
}

// key, value, key_cache, value_cache, scales, slot_mapping, oob_count, stream
PyObject* write(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    int64_t device = -1, ks, vs;
    Cache c;
    if (n != 8 || !c.take(o + 2, device)) return nullptr;
    const at::Tensor *key = tensor(o[0], device), *value = tensor(o[1], device),
                     *slots = tensor(o[5], device);
    if (!key || !value || !slots) return nullptr;
    const int32_t dtype = tokens(*key, c.heads, c.dim, ks);
    int32_t* oob;
    void* stream;
    if (dtype < 0 || tokens(*value, c.heads, c.dim, vs) != dtype ||
        slots->scalar_type() != at::kLong || slots->dim() != 1 || !slots->is_contiguous() ||
        key->size(0) < slots->numel() || value->size(0) < slots->numel() ||
        !counter(o[6], device, oob) || !stream_of(o[7], device, stream))
      return nullptr;
    return PyLong_FromLong(call(
        write_entry, key->data_ptr(), value->data_ptr(), c.key->data_ptr(), c.value->data_ptr(),
        static_cast<float*>(c.scales->data_ptr()), static_cast<const int64_t*>(slots->data_ptr()),
        slots->numel(), int32_t(c.heads), int32_t(c.dim), kPage, c.blocks, dtype, c.code, ks, vs,
        c.stride, c.scales_stride, oob, stream));
  });
}

// key_cache, value_cache, scales, block_table, cu_seq_lens, max_seq_len, out_key, out_value,
// seq_starts, oob_count, stream
PyObject* read(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    int64_t device = -1, ks, vs;
    Cache c;
    if (n != 11 || !c.take(o, device) || !PyLong_Check(o[5])) return nullptr;
    const at::Tensor *table = tensor(o[3], device), *cu = tensor(o[4], device),
                     *key = tensor(o[6], device), *value = tensor(o[7], device), *starts = nullptr;
    const int64_t longest = PyLong_AsLongLong(o[5]);
    if (!table || !key || !value || !ints(cu, 1) || longest < 0 || longest >= int64_t(1) << 31)
      return nullptr;
    const int64_t batch = cu->numel() - 1;
    if (o[8] != Py_None && !ints(starts = tensor(o[8], device), batch)) return nullptr;
    const int32_t dtype = tokens(*key, c.heads, c.dim, ks);
    int32_t* oob;
    void* stream;
    if (table->scalar_type() != at::kInt || table->dim() != 2 || table->stride(1) != 1 ||
        batch > table->size(0) || dtype < 0 || tokens(*value, c.heads, c.dim, vs) != dtype ||
        key->size(0) < 1 || value->size(0) < 1 || ks != vs || !counter(o[9], device, oob) ||
        !stream_of(o[10], device, stream))
      return nullptr;
    return PyLong_FromLong(call(
        read_entry, c.key->data_ptr(), c.value->data_ptr(), static_cast<const float*>(c.scales->data_ptr()),
        static_cast<const int32_t*>(table->data_ptr()), table->stride(0), int32_t(table->size(1)),
        static_cast<const int32_t*>(cu->data_ptr()),
        starts ? static_cast<const int32_t*>(starts->data_ptr()) : nullptr, int32_t(batch),
        int32_t(longest), int32_t(c.heads), int32_t(c.dim), kPage, c.blocks, dtype, c.code, c.stride,
        c.scales_stride, key->data_ptr(), value->data_ptr(), ks,
        std::min(key->size(0), value->size(0)), oob, stream));
  });
}

// q, key_cache, value_cache, scales, indptr, indices, last_page_len, sm_scale, out, lse,
// return_lse, workspace, stream
PyObject* decode(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return attempt([&]() -> PyObject* {
    int64_t device = -1, qs, os;
    Cache c;
    if (n != 13 || !c.take(o + 1, device)) return nullptr;
    const at::Tensor *q = tensor(o[0], device), *indptr = tensor(o[4], device),
                     *indices = tensor(o[5], device), *lengths = tensor(o[6], device),
                     *workspace = tensor(o[11], device);
    if (!q || !workspace || !workspace->is_contiguous() || q->dim() != 3) return nullptr;
    const int64_t batch = q->size(0), hq = q->size(1);
    const int32_t dtype = tokens(*q, hq, c.dim, qs);
    if (dtype < 0 || hq == 0 || c.heads == 0 || hq % c.heads || !ints(indptr, batch + 1) ||
        !ints(indices, 0) || !ints(lengths, batch))
      return nullptr;
    double scale = 1.0 / std::sqrt(double(c.dim));
    if (o[7] != Py_None) {
      scale = PyFloat_AsDouble(o[7]);
      if (PyErr_Occurred()) return nullptr;
    }
    const int wants = PyObject_IsTrue(o[10]);
    at::Tensor out, lse;
    if (o[8] != Py_None) {
      const at::Tensor* t = tensor(o[8], device);
      if (!t || tokens(*t, hq, c.dim, os) != dtype || t->size(0) < batch) return nullptr;
      out = *t;
    }
    if (o[9] != Py_None) {
      const at::Tensor* t = tensor(o[9], device);
      if (!t || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() < batch * hq)
        return nullptr;
      lse = *t;
    }
    void* stream;
    if (!stream_of(o[12], device, stream)) return nullptr;
    if (!out.defined()) {
      out = at::empty({batch, hq, c.dim}, q->options());
      os = hq * c.dim;
    }
    if (wants && !lse.defined()) lse = at::empty({batch, hq}, q->options().dtype(at::kFloat));
    const int status = call(
        decode_entry, q->data_ptr(), qs, c.key->data_ptr(), c.value->data_ptr(),
        static_cast<const float*>(c.scales->data_ptr()), c.stride, c.scales_stride, c.blocks,
        static_cast<const int32_t*>(indptr->data_ptr()),
        static_cast<const int32_t*>(indices->data_ptr()), indices->numel(),
        static_cast<const int32_t*>(lengths->data_ptr()), int32_t(batch), int32_t(hq),
        int32_t(c.heads), int32_t(c.dim), kPage, dtype, c.code, float(scale), workspace->data_ptr(),
        int64_t(workspace->nbytes()), out.data_ptr(), os,
        lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr, stream);
    if (status != KVC_OK) return PyLong_FromLong(status);
    PyObject* got = THPVariable_Wrap(out);
    return wants ? Py_BuildValue("(NN)", got, THPVariable_Wrap(lse)) : got;
  });
}

// Addresses of the three entries, torch's current device and raw stream queries.
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes three addresses and two functions");
    return nullptr;
  }
  write_entry = reinterpret_cast<decltype(write_entry)>(PyLong_AsVoidPtr(o[0]));
  read_entry = reinterpret_cast<decltype(read_entry)>(PyLong_AsVoidPtr(o[1]));
  decode_entry = reinterpret_cast<decltype(decode_entry)>(PyLong_AsVoidPtr(o[2]));
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(o[3]);
  Py_INCREF(o[4]);
  Py_XDECREF(current_device);
  Py_XDECREF(current_stream);
  current_device = o[3];
  current_stream = o[4];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(write)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(read)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL,
     nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "kvc_bind", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kvc_bind() { return PyModule_Create(&module); }
