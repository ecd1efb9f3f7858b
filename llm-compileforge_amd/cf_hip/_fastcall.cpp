// CPython extension: the tensor entry points' call path in native code.
//
// A call through ctypes costs 15-20 us of host time (a descriptor per tensor
// built in Python, two foreign calls, an output allocation through the Python
// API), more than the kernels of a small step take; the same call from here
// costs the launches plus about 2 us.  Each function checks what its ops.py
// wrapper checks, fills the descriptors from the tensors, allocates outputs
// and calls the library with the GIL released.  It returns
//   - the result (or 0 for calls without one) when the library accepted it,
//   - the library's negative status otherwise (ops.py raises from it),
//   - None when an argument is not an ordinary tensor on the current device
//     (another type or device, a rank or dtype without a descriptor, a tensor
//     without storage, ...): ops.py then takes its own path, which raises or
//     handles the case.
// No C++ exception leaves a function: one thrown by torch ends in None.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <vector>

#include "cf_hip.h"

namespace {

struct Lib {
  decltype(&cf_paged_decode_workspace_bytes) decode_ws = nullptr;
  decltype(&cf_paged_decode_shared) decode = nullptr;
  decltype(&cf_prefill_chunk_workspace_bytes) prefill_ws = nullptr;
  decltype(&cf_prefill_chunk_fp8) prefill = nullptr;
  decltype(&cf_paged_write) paged_write = nullptr;
  decltype(&cf_paged_gather) paged_gather = nullptr;
  decltype(&cf_kv_write_fp8) kv_write = nullptr;
  decltype(&cf_fp8_scale_quantize) scale_quantize = nullptr;
  decltype(&cf_fp8_dequantize_kv) dequantize_kv = nullptr;
  decltype(&cf_stage_from_host) stage = nullptr;
  decltype(&cf_paged_decode_weights_workspace_bytes) decode_weights_ws = nullptr;
  decltype(&cf_paged_decode_weights) decode_weights = nullptr;
  decltype(&cf_chunk_weights_workspace_bytes) chunk_weights_ws = nullptr;
  decltype(&cf_chunk_weights) chunk_weights = nullptr;
  decltype(&cf_rotary) rotary = nullptr;
  decltype(&cf_rotary_cache_write) rotary_write = nullptr;
  decltype(&cf_evict_select) evict_select = nullptr;
  decltype(&cf_evict_move) evict_move = nullptr;
  decltype(&cf_kv_write_blocks) write_blocks = nullptr;
  decltype(&cf_move_blocks) move_blocks = nullptr;
};
Lib g_lib;
PyObject* g_raw_stream = nullptr;        // device index -> hipStream_t of the current stream
PyObject* g_current_device = nullptr;    // () -> current device index
PyObject* g_workspaces = nullptr;        // {(device index, stream): workspace tensor}, shared with ops.py
PyObject* g_cached_workspace = nullptr;  // (bytes, device) -> workspace tensor

// Thrown to leave a call for ops.py's own path.
struct Slow {};

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return CF_F32;
    case at::kHalf: return CF_F16;
    case at::kBFloat16: return CF_BF16;
    case at::kLong: return CF_I64;
    case at::kInt: return CF_I32;
    case at::kChar: return CF_I8;
    case at::kByte: return CF_U8;
    case at::kFloat8_e4m3fn: return CF_F8E4M3FN;
    default: throw Slow{};
  }
}

// The plain tensor in `o` (torch.Tensor or Parameter, strided).
const at::Tensor& tensor_of(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw Slow{};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) throw Slow{};
  return t;
}

CfTensor describe(const at::Tensor& t) {
  const int64_t rank = t.dim();
  if (rank < 1 || rank > 4) throw Slow{};
  CfTensor d{};
  d.t.device = SFA_ROCM;
  d.t.rank = (int32_t)rank;
  d.t.elem_size = (int32_t)t.element_size();
  const int64_t off = t.storage_offset();
  char* base = (char*)t.data_ptr() - off * t.element_size();
  SFATensorRaw4& r = d.t.r4;  // the union members share their first three fields
  r.allocated = base;
  r.aligned = base;
  r.offset = off;
  int64_t* sizes = &r.offset + 1;
  for (int64_t i = 0; i < rank; ++i) {
    sizes[i] = t.size(i);
    sizes[rank + i] = t.stride(i);
  }
  d.dtype = dtype_code(t.scalar_type());
  return d;
}

// The device of a call: every tensor must be on it and it must be current.
struct Call {
  int device = -1;
  void* stream = nullptr;

  explicit Call(const at::Tensor& first) {
    if (g_raw_stream == nullptr) throw Slow{};
    device = first.get_device();
    PyObject* cur = PyObject_CallNoArgs(g_current_device);
    if (cur == nullptr) throw Slow{};
    const long now = PyLong_AsLong(cur);
    Py_DECREF(cur);
    if (now != device) throw Slow{};
    PyObject* idx = PyLong_FromLong(device);
    if (idx == nullptr) throw Slow{};
    PyObject* s = PyObject_CallOneArg(g_raw_stream, idx);
    Py_DECREF(idx);
    if (s == nullptr) throw Slow{};
    stream = (void*)PyLong_AsUnsignedLongLong(s);
    Py_DECREF(s);
    if (PyErr_Occurred()) throw Slow{};
  }
  CfTensor in(PyObject* o) const {
    const at::Tensor& t = tensor_of(o);
    if (t.get_device() != device) throw Slow{};
    return describe(t);
  }
  // [n] view of a scale tensor of any shape
  CfTensor flat(PyObject* o) const {
    const at::Tensor& t = tensor_of(o);
    if (t.get_device() != device) throw Slow{};
    if (t.dim() == 1) return describe(t);
    if (!t.is_contiguous()) throw Slow{};
    CfTensor d{};
    d.t.device = SFA_ROCM;
    d.t.rank = 1;
    d.t.elem_size = (int32_t)t.element_size();
    d.t.r1.allocated = d.t.r1.aligned = t.data_ptr();
    d.t.r1.sizes[0] = t.numel();
    d.t.r1.strides[0] = 1;
    d.dtype = dtype_code(t.scalar_type());
    return d;
  }
};

int64_t as_int(PyObject* o) {
  if (!PyLong_CheckExact(o)) throw Slow{};
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Slow{};
  return v;
}

double as_float(PyObject* o) {
  if (!PyFloat_CheckExact(o)) throw Slow{};
  return PyFloat_AS_DOUBLE(o);
}

at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::empty(sizes, at::TensorOptions().dtype(dtype).device(like.device()));
}

// A workspace of `need` bytes for this device and stream: the caller's, or
// ops.py's cached one (held by a new reference while the call runs).  `any`: the
// caller's may be of another size, for the library to judge.
struct Workspace {
  PyObject* held = nullptr;
  void* ptr = nullptr;
  uint64_t bytes = 0;

  Workspace(PyObject* given, uint64_t need, const Call& call, PyObject* tensor_on_device, bool any = false) {
    if (need == 0) return;
    bytes = need;
    if (given != Py_None) {
      const at::Tensor& t = tensor_of(given);
      const uint64_t has = (uint64_t)(t.numel() * t.element_size());
      if (any) bytes = has;
      else if (has < need) throw Slow{};
      ptr = t.data_ptr();
      return;
    }
    PyObject* key = Py_BuildValue("(iK)", call.device, (unsigned long long)(uintptr_t)call.stream);
    if (key == nullptr) throw Slow{};
    PyObject* ws = PyDict_GetItem(g_workspaces, key);  // borrowed
    Py_DECREF(key);
    if (ws != nullptr && THPVariable_Check(ws) && (uint64_t)THPVariable_Unpack(ws).numel() >= need) {
      Py_INCREF(ws);
      held = ws;
    } else {
      PyObject* dev = PyObject_GetAttrString(tensor_on_device, "device");
      if (dev == nullptr) throw Slow{};
      held = PyObject_CallFunction(g_cached_workspace, "KO", (unsigned long long)need, dev);
      Py_DECREF(dev);
      if (held == nullptr) throw Slow{};
    }
    ptr = THPVariable_Unpack(held).data_ptr();
  }
  ~Workspace() { Py_XDECREF(held); }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
};

// Runs f with the GIL released; held again also where f throws.
template <class F>
int32_t without_gil(F f) {
  struct Release {
    PyThreadState* st = PyEval_SaveThread();
    ~Release() { PyEval_RestoreThread(st); }
  } release;
  return f();
}

// Runs a call body: Slow, torch's exceptions and Python errors become None.
template <class F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F f) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return nullptr;
  }
  try {
    return f(args);
  } catch (...) {
    PyErr_Clear();
  }
  Py_RETURN_NONE;
}

const CfTensor* opt(PyObject* o, const CfTensor& d) { return o == Py_None ? nullptr : &d; }

// (q, k_cache, v_cache, block_tables, seq_lens, scale, block_size, k_scale,
// v_scale, partition_tokens, out, workspace, shared_prefix_lens) -> out
PyObject* paged_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 13, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& q = tensor_of(a[0]);
    const at::Tensor& k = tensor_of(a[1]);
    const at::Tensor& bt = tensor_of(a[3]);
    if (q.dim() != 3 || k.dim() != 4 || bt.dim() != 2) throw Slow{};
    const Call call(q);
    const CfTensor dq = call.in(a[0]), dk = call.in(a[1]), dv = call.in(a[2]), dt = call.in(a[3]), dl = call.in(a[4]);
    const double scale = as_float(a[5]);
    const int64_t bs = as_int(a[6]), pt = as_int(a[9]);
    if (bs != (int32_t)bs || pt != (int32_t)pt) throw Slow{};
    CfTensor dks{}, dvs{}, dsh{};
    if (a[7] != Py_None) dks = call.in(a[7]);
    if (a[8] != Py_None) dvs = call.in(a[8]);
    if (a[12] != Py_None) dsh = call.in(a[12]);
    uint64_t need = 0;
    if (g_lib.decode_ws(q.size(0), q.size(1), k.size(2), q.size(2), bt.size(1), (int32_t)bs, (int32_t)pt, &need) !=
        CF_OK)
      throw Slow{};
    const Workspace ws(a[11], need, call, a[0]);
    at::Tensor fresh;
    CfTensor dout;
    if (a[10] == Py_None) {
      fresh = new_tensor(q.sizes(), q.scalar_type(), q);
      dout = describe(fresh);
    } else {
      dout = call.in(a[10]);
    }
    const int32_t rc = without_gil([&] {
      return g_lib.decode(&dq, &dk, &dv, &dt, &dl, opt(a[12], dsh), opt(a[7], dks), opt(a[8], dvs), (float)scale,
                          (int32_t)bs, (int32_t)pt, &dout, ws.ptr, need, call.stream);
    });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    if (a[10] == Py_None) return THPVariable_Wrap(fresh);
    Py_INCREF(a[10]);
    return a[10];
  });
}

// (q, k_cache, v_cache, block_tables, seq_lens, q_start, scale, block_size,
// k_scale, v_scale, out, workspace) -> out
PyObject* prefill_chunk(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 12, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& q = tensor_of(a[0]);
    const at::Tensor& k = tensor_of(a[1]);
    const at::Tensor& bt = tensor_of(a[3]);
    if (q.dim() != 3 || k.dim() != 4 || bt.dim() != 2) throw Slow{};
    const Call call(q);
    const CfTensor dq = call.in(a[0]), dk = call.in(a[1]), dv = call.in(a[2]), dt = call.in(a[3]), dl = call.in(a[4]),
                   ds = call.in(a[5]);
    const double scale = as_float(a[6]);
    const int64_t bs = as_int(a[7]);
    if (bs != (int32_t)bs) throw Slow{};
    CfTensor dks{}, dvs{};
    if (a[8] != Py_None) dks = call.in(a[8]);
    if (a[9] != Py_None) dvs = call.in(a[9]);
    uint64_t need = 0;
    if (g_lib.prefill_ws(q.size(0), bt.size(0), q.size(1), k.size(2), q.size(2), (int32_t)bs, &need) != CF_OK)
      throw Slow{};
    const Workspace ws(a[11], need, call, a[0], true);
    at::Tensor fresh;
    CfTensor dout;
    if (a[10] == Py_None) {
      fresh = new_tensor(q.sizes(), q.scalar_type(), q);
      dout = describe(fresh);
    } else {
      dout = call.in(a[10]);
    }
    const int32_t rc = without_gil([&] {
      return g_lib.prefill(&dq, &dk, &dv, &dt, &dl, &ds, opt(a[8], dks), opt(a[9], dvs), (float)scale, (int32_t)bs,
                           &dout, ws.ptr, ws.bytes, call.stream);
    });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    if (a[10] == Py_None) return THPVariable_Wrap(fresh);
    Py_INCREF(a[10]);
    return a[10];
  });
}

// (x_new, slot_mapping, cache, scale) -> 0
PyObject* paged_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject* const* a) -> PyObject* {
    const Call call(tensor_of(a[0]));
    const CfTensor dx = call.in(a[0]), ds = call.in(a[1]);
    CfTensor dc = call.in(a[2]), dsc{};
    if (a[3] != Py_None) dsc = call.flat(a[3]);
    return PyLong_FromLong(
        without_gil([&] { return g_lib.paged_write(&dx, &ds, &dc, opt(a[3], dsc), call.stream); }));
  });
}

// (cache, block_tables, seq_len, out_dtype, scale, out) -> out
PyObject* paged_gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 6, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& cache = tensor_of(a[0]);
    const at::Tensor& bt = tensor_of(a[1]);
    if (cache.dim() != 4 || bt.dim() != 2) throw Slow{};
    const Call call(cache);
    const CfTensor dc = call.in(a[0]), dt = call.in(a[1]);
    const int64_t seq = as_int(a[2]);
    if (seq < 0) throw Slow{};
    CfTensor dsc{}, dout;
    // (2-D: a scale for each block and head)
    if (a[4] != Py_None) {
      const at::Tensor& sc = tensor_of(a[4]);
      dsc = sc.dim() == 2 && sc.size(0) == cache.size(0) && sc.size(1) == cache.size(2) ? call.in(a[4]) : call.flat(a[4]);
    }
    at::Tensor fresh;
    if (a[5] == Py_None) {
      const bool codes = cache.scalar_type() == at::kFloat8_e4m3fn || cache.scalar_type() == at::kChar;
      at::ScalarType dtype = codes ? at::kFloat : cache.scalar_type();
      if (a[3] != Py_None) {
        if (!THPDtype_Check(a[3])) throw Slow{};
        dtype = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
      }
      fresh = new_tensor({bt.size(0), seq, cache.size(2), cache.size(3)}, dtype, cache);
      dout = describe(fresh);
    } else {
      dout = call.in(a[5]);
    }
    const int32_t rc =
        without_gil([&] { return g_lib.paged_gather(&dc, &dt, opt(a[4], dsc), &dout, call.stream); });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    if (a[5] == Py_None) return THPVariable_Wrap(fresh);
    Py_INCREF(a[5]);
    return a[5];
  });
}

// (k_new, v_new, slot_mapping, k_cache, v_cache, k_scale, v_scale) -> 0
PyObject* kv_write_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 7, [](PyObject* const* a) -> PyObject* {
    const Call call(tensor_of(a[0]));
    const CfTensor dk = call.in(a[0]), dv = call.in(a[1]), ds = call.in(a[2]);
    CfTensor dkc = call.in(a[3]), dvc = call.in(a[4]);
    const CfTensor dks = call.flat(a[5]), dvs = call.flat(a[6]);
    return PyLong_FromLong(
        without_gil([&] { return g_lib.kv_write(&dk, &dv, &ds, &dkc, &dvc, &dks, &dvs, call.stream); }));
  });
}

// A contiguous tensor of n elements as [n / (heads * row), heads, row].
CfTensor rows3(const at::Tensor& t, int64_t heads, int64_t row) {
  CfTensor d{};
  d.t.device = SFA_ROCM;
  d.t.rank = 3;
  d.t.elem_size = (int32_t)t.element_size();
  SFATensorRaw3& r = d.t.r3;
  r.allocated = r.aligned = t.data_ptr();
  r.sizes[0] = t.numel() / (heads * row);
  r.sizes[1] = heads;
  r.sizes[2] = row;
  r.strides[0] = heads * row;
  r.strides[1] = row;
  r.strides[2] = 1;
  d.dtype = dtype_code(t.scalar_type());
  return d;
}

// (x, y or None, per_head) -> ((codes, scales), ...) for contiguous tensors of
// one shape and dtype
PyObject* scale_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 3, [](PyObject* const* a) -> PyObject* {
    const int count = a[1] == Py_None ? 1 : 2;
    const bool per_head = a[2] == Py_True;
    const at::Tensor& x0 = tensor_of(a[0]);
    const int64_t total = x0.numel();
    if (total == 0 || total % 16 != 0) throw Slow{};
    // (2-D: one head; the library takes 64 heads, and its workspace grows with them)
    if (per_head && (x0.dim() < 3 || x0.size(-1) % 16 != 0 || x0.size(-2) > 64)) throw Slow{};
    const Call call(x0);
    const int64_t heads = per_head ? x0.size(-2) : 1, row = per_head ? x0.size(-1) : 16;
    at::Tensor codes[2], scales[2];
    CfTensor dx[2], dc[2], ds[2];
    for (int i = 0; i < count; ++i) {
      const at::Tensor& x = tensor_of(a[i]);
      if (x.get_device() != call.device || !x.is_contiguous() || x.scalar_type() != x0.scalar_type() ||
          x.sizes() != x0.sizes())
        throw Slow{};
      codes[i] = new_tensor(x.sizes(), at::kFloat8_e4m3fn, x);
      scales[i] = new_tensor({heads}, at::kFloat, x);
      dx[i] = rows3(x, heads, row);
      dc[i] = rows3(codes[i], heads, row);
      ds[i] = describe(scales[i]);
    }
    const at::Tensor ws = new_tensor({4096 * heads}, at::kByte, x0);
    const int32_t rc = without_gil([&] {
      return g_lib.scale_quantize(&dx[0], count == 2 ? &dx[1] : nullptr, &ds[0], count == 2 ? &ds[1] : nullptr, &dc[0],
                                  count == 2 ? &dc[1] : nullptr, ws.data_ptr(), (uint64_t)ws.numel(), call.stream);
    });
    if (rc == CF_ERR_UNSUPPORTED) throw Slow{};
    if (rc != CF_OK) return PyLong_FromLong(rc);
    PyObject* out = PyTuple_New(count);
    if (out == nullptr) throw Slow{};
    for (int i = 0; i < count; ++i)
      PyTuple_SET_ITEM(out, i, Py_BuildValue("(NN)", THPVariable_Wrap(codes[i]), THPVariable_Wrap(scales[i])));
    return out;
  });
}

// (k, v, k_scales, v_scales) -> (f32 k, f32 v) for contiguous tensors of one
// shape with one scale each
PyObject* dequantize_kv(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& k = tensor_of(a[0]);
    const at::Tensor& v = tensor_of(a[1]);
    const Call call(k);
    if (v.get_device() != call.device || k.sizes() != v.sizes() || !k.is_contiguous() || !v.is_contiguous() ||
        k.numel() % 16 != 0 || k.numel() == 0)
      throw Slow{};
    const CfTensor dks = call.flat(a[2]), dvs = call.flat(a[3]);
    if (dks.t.r1.sizes[0] != 1 || dvs.t.r1.sizes[0] != 1) throw Slow{};
    at::Tensor out[2] = {new_tensor(k.sizes(), at::kFloat, k), new_tensor(k.sizes(), at::kFloat, k)};
    const CfTensor dk = rows3(k, 1, 16), dv = rows3(v, 1, 16);
    CfTensor dko = rows3(out[0], 1, 16), dvo = rows3(out[1], 1, 16);
    const int32_t rc =
        without_gil([&] { return g_lib.dequantize_kv(&dk, &dv, &dks, &dvs, &dko, &dvo, call.stream); });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NN)", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
  });
}

// (pinned host int32, device int32, requests, blocks): uploads the packed
// tables [requests, blocks] | lengths [requests] | shared-prefix lengths
// [requests] and returns their views of the device buffer
PyObject* stage_tables(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 4, [](PyObject* const* a) -> PyObject* {
    if (!THPVariable_CheckExact(a[0])) throw Slow{};
    const at::Tensor& host = THPVariable_Unpack(a[0]);
    const at::Tensor& dev = tensor_of(a[1]);
    const Call call(dev);
    const int64_t reqs = as_int(a[2]), mb = as_int(a[3]), used = reqs * (mb + 2), words = (used + 3) / 4;
    if (!host.is_cpu() || host.scalar_type() != at::kInt || dev.scalar_type() != at::kInt || !host.is_contiguous() ||
        !dev.is_contiguous() || reqs < 1 || mb < 1 || host.numel() < 4 * words || dev.numel() < 4 * words)
      throw Slow{};
    const int32_t rc = without_gil(
        [&] { return g_lib.stage(host.data_ptr(), dev.data_ptr(), (uint64_t)words * 16, call.stream); });
    if (rc == CF_ERR_INVALID) throw Slow{};
    if (rc != CF_OK) return PyLong_FromLong(rc);
    const int64_t at = dev.storage_offset();
    return Py_BuildValue("(NNN)", THPVariable_Wrap(dev.as_strided({reqs, mb}, {mb, 1}, at)),
                         THPVariable_Wrap(dev.as_strided({reqs}, {1}, at + reqs * mb)),
                         THPVariable_Wrap(dev.as_strided({reqs}, {1}, at + reqs * (mb + 1))));
  });
}

// An output: the caller's tensor, or a new one of `sizes`.
struct Output {
  at::Tensor fresh;
  PyObject* given;
  CfTensor d;

  Output(PyObject* o, const Call& call, at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) : given(o) {
    if (o != Py_None) {
      d = call.in(o);
      return;
    }
    fresh = new_tensor(sizes, dtype, like);
    d = describe(fresh);
  }
  PyObject* result() const {
    if (given == Py_None) return THPVariable_Wrap(fresh);
    Py_INCREF(given);
    return given;
  }
};

// (q, k_cache, v_cache, block_tables, seq_lens, weights, scale, block_size,
// decay, k_scale, v_scale, out, workspace, shared_prefix_lens) -> out
PyObject* paged_decode_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 14, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& q = tensor_of(a[0]);
    const at::Tensor& k = tensor_of(a[1]);
    const at::Tensor& bt = tensor_of(a[3]);
    if (q.dim() != 3 || k.dim() != 4 || bt.dim() != 2) throw Slow{};
    const Call call(q);
    const CfTensor dq = call.in(a[0]), dk = call.in(a[1]), dv = call.in(a[2]), dt = call.in(a[3]), dl = call.in(a[4]);
    CfTensor dw = call.in(a[5]), dks{}, dvs{}, dsh{};
    const double scale = as_float(a[6]), decay = as_float(a[8]);
    const int64_t bs = as_int(a[7]);
    if (bs != (int32_t)bs) throw Slow{};
    if (a[9] != Py_None) dks = call.in(a[9]);
    if (a[10] != Py_None) dvs = call.in(a[10]);
    if (a[13] != Py_None) dsh = call.in(a[13]);
    uint64_t need = 0;
    if (g_lib.decode_weights_ws(q.size(0), q.size(1), k.size(2), q.size(2), bt.size(1), (int32_t)bs, &need) != CF_OK)
      throw Slow{};
    if (a[12] != Py_None && tensor_of(a[12]).get_device() != call.device) throw Slow{};
    const Workspace ws(a[12], need, call, a[0]);
    Output out(a[11], call, q.sizes(), q.scalar_type(), q);
    const int32_t rc = without_gil([&] {
      return g_lib.decode_weights(&dq, &dk, &dv, &dt, &dl, opt(a[13], dsh), opt(a[9], dks), opt(a[10], dvs),
                                  (float)scale, (int32_t)bs, &dw, (float)decay, &out.d, ws.ptr, need, call.stream);
    });
    return rc != CF_OK ? PyLong_FromLong(rc) : out.result();
  });
}

// (q, k_cache, block_tables, seq_lens, q_start, weights, scale, block_size,
// decay, observe, k_scale, workspace) -> weights
PyObject* chunk_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 12, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& q = tensor_of(a[0]);
    const at::Tensor& k = tensor_of(a[1]);
    const at::Tensor& bt = tensor_of(a[2]);
    if (q.dim() != 3 || k.dim() != 4 || bt.dim() != 2) throw Slow{};
    const Call call(q);
    const CfTensor dq = call.in(a[0]), dk = call.in(a[1]), dt = call.in(a[2]), dl = call.in(a[3]), ds = call.in(a[4]);
    CfTensor dw = call.in(a[5]), dks{};
    const double scale = as_float(a[6]), decay = as_float(a[8]);
    const int64_t bs = as_int(a[7]), observe = as_int(a[9]);
    if (bs != (int32_t)bs || observe != (int32_t)observe) throw Slow{};
    if (a[10] != Py_None) dks = call.in(a[10]);
    uint64_t need = 0;
    if (g_lib.chunk_weights_ws(q.size(0), bt.size(0), q.size(1), k.size(2), q.size(2), bt.size(1), (int32_t)bs,
                               (int32_t)observe, &need) != CF_OK)
      throw Slow{};
    if (a[11] != Py_None && tensor_of(a[11]).get_device() != call.device) throw Slow{};
    const Workspace ws(a[11], need, call, a[0]);
    const int32_t rc = without_gil([&] {
      return g_lib.chunk_weights(&dq, &dk, &dt, &dl, &ds, opt(a[10], dks), (float)scale, (int32_t)bs, (int32_t)observe,
                                 &dw, (float)decay, ws.ptr, need, call.stream);
    });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    Py_INCREF(a[5]);
    return a[5];
  });
}

// The axes of a rotary call: a tuple or list of the sections, or None.
struct Sections {
  int32_t n[CF_ROTARY_MAX_AXES] = {};
  const int32_t* ptr = nullptr;
  int32_t axes = 1;

  Sections(PyObject* o, const at::Tensor& positions) {
    const int64_t rows = positions.dim() == 2 ? positions.size(0) : 1;
    if (rows < 1 || rows > CF_ROTARY_MAX_AXES) throw Slow{};
    axes = (int32_t)rows;
    if (o == Py_None) return;
    const bool tuple = PyTuple_CheckExact(o);
    if (!tuple && !PyList_CheckExact(o)) throw Slow{};
    if ((tuple ? PyTuple_GET_SIZE(o) : PyList_GET_SIZE(o)) != axes) throw Slow{};
    for (int32_t i = 0; i < axes; ++i) {
      const int64_t v = as_int(tuple ? PyTuple_GET_ITEM(o, i) : PyList_GET_ITEM(o, i));
      if (v != (int32_t)v) throw Slow{};
      n[i] = (int32_t)v;
    }
    ptr = n;
  }
};

// (x, positions, inv_freq, sections, flags, rotary_scale, out) -> out
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 7, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& x = tensor_of(a[0]);
    const Call call(x);
    const CfTensor dx = call.in(a[0]), dp = call.in(a[1]), df = call.in(a[2]);
    const Sections sec(a[3], tensor_of(a[1]));
    const int32_t flags = (int32_t)as_int(a[4]);
    const double scale = as_float(a[5]);
    Output out(a[6], call, x.sizes(), x.scalar_type(), x);
    const int32_t rc = without_gil([&] {
      return g_lib.rotary(&dx, &dp, &df, sec.ptr, sec.axes, flags, (float)scale, &out.d, call.stream);
    });
    return rc != CF_OK ? PyLong_FromLong(rc) : out.result();
  });
}

// (q, k_new, v_new, positions, inv_freq, slot_mapping, k_cache, v_cache,
// sections, flags, rotary_scale, k_scale, v_scale, out) -> out
PyObject* rotary_cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 14, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& q = tensor_of(a[0]);
    const Call call(q);
    const CfTensor dq = call.in(a[0]), dk = call.in(a[1]), dv = call.in(a[2]), dp = call.in(a[3]), df = call.in(a[4]),
                   ds = call.in(a[5]);
    CfTensor dkc = call.in(a[6]), dvc = call.in(a[7]), dks{}, dvs{};
    const Sections sec(a[8], tensor_of(a[3]));
    const int32_t flags = (int32_t)as_int(a[9]);
    const double scale = as_float(a[10]);
    if (a[11] != Py_None) dks = call.flat(a[11]);
    if (a[12] != Py_None) dvs = call.flat(a[12]);
    Output out(a[13], call, q.sizes(), q.scalar_type(), q);
    const int32_t rc = without_gil([&] {
      return g_lib.rotary_write(&dq, &dk, &dv, &dp, &df, sec.ptr, sec.axes, flags, (float)scale, &ds, &dkc, &dvc,
                                opt(a[11], dks), opt(a[12], dvs), &out.d, call.stream);
    });
    return rc != CF_OK ? PyLong_FromLong(rc) : out.result();
  });
}

// (weights, seq_lens, budget, sink, recent, positions, kept, seen, keep,
// new_lens) -> (keep, new_lens)
PyObject* evict_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 10, [](PyObject* const* a) -> PyObject* {
    const at::Tensor& w = tensor_of(a[0]);
    if (w.dim() != 3) throw Slow{};
    const Call call(w);
    const CfTensor dw = call.in(a[0]), dl = call.in(a[1]);
    const int64_t budget = as_int(a[2]), sink = as_int(a[3]), recent = as_int(a[4]);
    if (budget < 1 || budget != (int32_t)budget || sink != (int32_t)sink || recent != (int32_t)recent) throw Slow{};
    CfTensor dp{}, dk{}, ds{};
    if (a[5] != Py_None) dp = call.in(a[5]);
    if (a[6] != Py_None) dk = call.in(a[6]);
    if (a[7] != Py_None) ds = call.in(a[7]);
    if (a[8] != Py_None && (tensor_of(a[8]).dim() != 3 || tensor_of(a[8]).size(2) != budget)) throw Slow{};
    Output keep(a[8], call, {w.size(0), w.size(1), budget}, at::kInt, w);
    Output lens(a[9], call, {w.size(0)}, at::kInt, w);
    const int32_t rc = without_gil([&] {
      return g_lib.evict_select(&dw, &dl, opt(a[5], dp), opt(a[6], dk), opt(a[7], ds), (int32_t)sink, (int32_t)recent,
                                &keep.d, &lens.d, call.stream);
    });
    if (rc != CF_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("(NN)", keep.result(), lens.result());
  });
}

// (keep, seq_lens, block_tables, k_cache, v_cache, weights, positions, kept,
// seen) -> 0
PyObject* evict_move(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](PyObject* const* a) -> PyObject* {
    const Call call(tensor_of(a[0]));
    const CfTensor dk = call.in(a[0]), dl = call.in(a[1]), dt = call.in(a[2]);
    CfTensor dkc = call.in(a[3]), dvc = call.in(a[4]), dw{}, dp{}, dkept{}, dseen{};
    if (a[5] != Py_None) dw = call.in(a[5]);
    if (a[6] != Py_None) dp = call.in(a[6]);
    if (a[7] != Py_None) dkept = call.in(a[7]);
    if (a[8] != Py_None) dseen = call.in(a[8]);
    return PyLong_FromLong(without_gil([&] {
      return g_lib.evict_move(&dk, &dl, &dt, &dkc, &dvc, a[5] == Py_None ? nullptr : &dw,
                              a[6] == Py_None ? nullptr : &dp, opt(a[7], dkept), opt(a[8], dseen), call.stream);
    }));
  });
}

// (k_new, v_new, block_tables, seq_lens, q_start, k_cache, v_cache, k_scale,
// v_scale) -> 0
PyObject* kv_write_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](PyObject* const* a) -> PyObject* {
    const Call call(tensor_of(a[0]));
    const CfTensor dk = call.in(a[0]), dv = call.in(a[1]), dt = call.in(a[2]), dl = call.in(a[3]);
    CfTensor dq{};
    if (a[4] != Py_None) dq = call.in(a[4]);
    CfTensor dkc = call.in(a[5]), dvc = call.in(a[6]), dks = call.in(a[7]), dvs = call.in(a[8]);
    return PyLong_FromLong(without_gil([&] {
      return g_lib.write_blocks(&dk, &dv, &dt, &dl, opt(a[4], dq), &dkc, &dvc, &dks, &dvs, call.stream);
    }));
  });
}

// [NB, bytes] of a paged tensor whose blocks are one contiguous span each.
CfTensor block_bytes(const at::Tensor& t) {
  if (t.dim() < 1) throw Slow{};
  int64_t span = 1, elems = 1;
  for (int64_t i = 1; i < t.dim(); ++i) {
    if (t.size(i) > 1) span += (t.size(i) - 1) * t.stride(i);
    if (t.size(i) != 1) elems *= t.size(i);
  }
  const int64_t nb = t.size(0), es = t.element_size();
  if (elems == 0 || span != elems || (nb > 1 && t.stride(0) < elems)) throw Slow{};
  CfTensor d{};
  d.t.device = SFA_ROCM;
  d.t.rank = 2;
  d.t.elem_size = 1;
  SFATensorRaw2& r = d.t.r2;
  r.allocated = r.aligned = t.data_ptr();
  r.sizes[0] = nb;
  r.sizes[1] = elems * es;
  r.strides[0] = (nb > 1 ? t.stride(0) : elems) * es;
  r.strides[1] = 1;
  d.dtype = CF_U8;
  return d;
}

// (caches: a list or tuple, moves: a contiguous int32 [n, 2] CPU tensor or buffer)
PyObject* move_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 2, [](PyObject* const* a) -> PyObject* {
    if (!PyList_CheckExact(a[0]) && !PyTuple_CheckExact(a[0])) throw Slow{};
    const Py_ssize_t caches = PySequence_Fast_GET_SIZE(a[0]);
    if (caches == 0 || caches > INT32_MAX) throw Slow{};
    PyObject** items = PySequence_Fast_ITEMS(a[0]);
    const Call call(tensor_of(items[0]));
    std::vector<CfTensor> d;
    d.reserve(caches);
    for (Py_ssize_t i = 0; i < caches; ++i) {
      const at::Tensor& t = tensor_of(items[i]);
      if (t.get_device() != call.device) throw Slow{};
      d.push_back(block_bytes(t));
    }
    std::vector<int32_t> moves;  // (its own copy: the GIL is released)
    if (THPVariable_CheckExact(a[1])) {
      const at::Tensor& m = THPVariable_Unpack(a[1]);
      if (!m.defined() || !m.is_cpu() || m.scalar_type() != at::kInt || m.dim() != 2 || m.size(1) != 2 || !m.is_contiguous())
        throw Slow{};
      const int32_t* at = (const int32_t*)m.data_ptr();
      moves.assign(at, at + m.numel());
    } else {
      struct View {
        Py_buffer b{};
        explicit View(PyObject* o) {
          if (PyObject_GetBuffer(o, &b, PyBUF_FORMAT | PyBUF_C_CONTIGUOUS) != 0) throw Slow{};
        }
        ~View() { PyBuffer_Release(&b); }
      } v(a[1]);
      if (v.b.ndim != 2 || v.b.shape[1] != 2 || v.b.itemsize != 4 || v.b.format == nullptr || v.b.format[0] != 'i' ||
          v.b.format[1] != 0)
        throw Slow{};
      const int32_t* at = (const int32_t*)v.b.buf;
      moves.assign(at, at + 2 * v.b.shape[0]);
    }
    return PyLong_FromLong(without_gil([&] {
      return g_lib.move_blocks(d.data(), (int32_t)caches, moves.data(), (int64_t)(moves.size() / 2), call.stream);
    }));
  });
}

template <class T>
bool take_address(PyObject* addrs, const char* name, T* fn) {
  PyObject* v = PyDict_GetItemString(addrs, name);
  if (v == nullptr) {
    PyErr_Format(PyExc_KeyError, "%s", name);
    return false;
  }
  *fn = (T)(uintptr_t)PyLong_AsUnsignedLongLong(v);
  return !PyErr_Occurred();
}

// bind({entry point: address}, raw_stream, current_device, workspaces, cached_workspace)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *addrs, *raw, *cur, *wss, *cached;
  if (!PyArg_ParseTuple(args, "O!OOO!O", &PyDict_Type, &addrs, &raw, &cur, &PyDict_Type, &wss, &cached)) return nullptr;
  Lib l;
  if (!take_address(addrs, "cf_paged_decode_workspace_bytes", &l.decode_ws) ||
      !take_address(addrs, "cf_paged_decode_shared", &l.decode) ||
      !take_address(addrs, "cf_prefill_chunk_workspace_bytes", &l.prefill_ws) ||
      !take_address(addrs, "cf_prefill_chunk_fp8", &l.prefill) ||
      !take_address(addrs, "cf_paged_write", &l.paged_write) ||
      !take_address(addrs, "cf_paged_gather", &l.paged_gather) ||
      !take_address(addrs, "cf_kv_write_fp8", &l.kv_write) ||
      !take_address(addrs, "cf_fp8_scale_quantize", &l.scale_quantize) ||
      !take_address(addrs, "cf_fp8_dequantize_kv", &l.dequantize_kv) ||
      !take_address(addrs, "cf_stage_from_host", &l.stage) ||
      !take_address(addrs, "cf_paged_decode_weights_workspace_bytes", &l.decode_weights_ws) ||
      !take_address(addrs, "cf_paged_decode_weights", &l.decode_weights) ||
      !take_address(addrs, "cf_chunk_weights_workspace_bytes", &l.chunk_weights_ws) ||
      !take_address(addrs, "cf_chunk_weights", &l.chunk_weights) ||
      !take_address(addrs, "cf_rotary", &l.rotary) ||
      !take_address(addrs, "cf_rotary_cache_write", &l.rotary_write) ||
      !take_address(addrs, "cf_evict_select", &l.evict_select) ||
      !take_address(addrs, "cf_evict_move", &l.evict_move) ||
      !take_address(addrs, "cf_kv_write_blocks", &l.write_blocks) ||
      !take_address(addrs, "cf_move_blocks", &l.move_blocks))
    return nullptr;
  g_lib = l;
  for (auto [slot, obj] : {std::pair{&g_raw_stream, raw}, std::pair{&g_current_device, cur},
                           std::pair{&g_workspaces, wss}, std::pair{&g_cached_workspace, cached}}) {
    Py_INCREF(obj);
    Py_XDECREF(*slot);
    *slot = obj;
  }
  Py_RETURN_NONE;
}

#define CF_FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    CF_FAST(paged_decode),
    CF_FAST(prefill_chunk),
    CF_FAST(paged_write),
    CF_FAST(paged_gather),
    CF_FAST(kv_write_fp8),
    CF_FAST(scale_quantize),
    CF_FAST(dequantize_kv),
    CF_FAST(stage_tables),
    CF_FAST(paged_decode_weights),
    CF_FAST(chunk_weights),
    CF_FAST(rotary),
    CF_FAST(rotary_cache_write),
    CF_FAST(evict_select),
    CF_FAST(evict_move),
    CF_FAST(kv_write_blocks),
    CF_FAST(move_blocks),
    {nullptr, nullptr, 0, nullptr},
};
#undef CF_FAST

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&kModule); }
