// Host side of the serving and training calls for PyTorch tensors: the checks and the collection of
// addresses that Python would do tensor by tensor (0.3 to 0.5 us a tensor; a step of 64 adapters over
// seven projections names 896), then the C ABI call.  Each function returns None when anything is out of the
// ordinary: the Python caller then takes its own path, which raises the error or makes the copy.  No
// arithmetic happens here, and the library itself stays free of torch types.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <memory>
#include <mutex>
#include <vector>

#include "../../include/lorafusion_b200.h"

namespace {

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? LF_F32 : t == at::kBFloat16 ? LF_BF16 : t == at::kHalf ? LF_F16 : -1;
}

// A dense tensor on a CUDA device (an exact torch.Tensor or a subclass), else null.
const at::Tensor* cuda_tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  return &t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

PyObject* fail(int rc, const char* what) {
  PyErr_Format(rc == LF_ERR_CUDA || rc == LF_ERR_DEVICE ? PyExc_RuntimeError : PyExc_ValueError, "%s: %s (status %d)",
               what, lf_status_string(rc), rc);
  return nullptr;
}

// What a kernel has written: the caches of b200_ops and autograd's check of saved tensors go by the version.
void bump(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// rows_forward(x, weight, bank_a, bank_b, ranks, scales, row_slot, out or None, the bank's padded rank, its output
// features, 1 if the weight is the data of one in 4 bits (its shape and dtype were checked)): the call of
// fused_lora_forward_rows on operands that need no copy.  None otherwise.
PyObject* rows_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) {
    PyErr_SetString(PyExc_TypeError, "rows_forward takes 11 arguments");
    return nullptr;
  }
  const at::Tensor* t[7];
  for (int i = 0; i < 7; ++i)
    if (!(t[i] = cuda_tensor(a[i]))) Py_RETURN_NONE;
  const at::Tensor &x = *t[0], &w = *t[1], &ba = *t[2], &bb = *t[3], &ranks = *t[4], &scales = *t[5], &slot = *t[6];
  const long r_pad = PyLong_AsLong(a[8]), features = PyLong_AsLong(a[9]);
  const bool mx4 = PyLong_AsLong(a[10]) == 1;
  if (PyErr_Occurred()) return nullptr;
  const int code = dtype_code(x.scalar_type());
  if (code < 0 || x.dim() != 2 || w.dim() != (mx4 ? 1 : 2) || slot.dim() != 1) Py_RETURN_NONE;
  const int64_t T = x.size(0), K = x.size(1), N = mx4 ? features : w.size(0);
  const auto dev = x.device();
  for (int i = 1; i < 7; ++i)
    if (t[i]->device() != dev) Py_RETURN_NONE;
  const bool wide = slot.scalar_type() == at::kLong;
  if (mx4 ? w.scalar_type() != at::kByte || code == LF_F32
          : w.scalar_type() != x.scalar_type() || w.size(1) != K || N != features)
    Py_RETURN_NONE;
  if (ba.scalar_type() != x.scalar_type() ||
      slot.size(0) != T || (!wide && slot.scalar_type() != at::kInt) || !slot.is_contiguous() || !w.is_contiguous() ||
      ba.size(2) != K || T == 0 || T > INT32_MAX || K > INT32_MAX || N > INT32_MAX)
    Py_RETURN_NONE;
  // one column or row makes any stride contiguous: take the row pitch from the shape then
  const int64_t ldx = x.is_contiguous() ? K : x.stride(0);
  if (!x.is_contiguous() && (x.stride(1) != 1 || ldx < K)) Py_RETURN_NONE;
  at::Tensor y;
  if (a[7] == Py_None) {
    y = at::detail::empty_cuda({T, N}, x.scalar_type(), dev, std::nullopt);
  } else {
    const at::Tensor* o = cuda_tensor(a[7]);
    if (!o || o->dim() != 2 || o->size(0) != T || o->size(1) != N || o->scalar_type() != x.scalar_type() ||
        o->device() != dev || !o->is_contiguous() || (o->requires_grad() && c10::GradMode::is_enabled()))
      Py_RETURN_NONE;
    y = *o;
  }
  const void *xp = x.const_data_ptr(), *wp = w.const_data_ptr(), *ap = ba.const_data_ptr(), *bp = bb.const_data_ptr();
  void* yp = y.data_ptr();
  if (code != LF_F32 && (K % 8 || N % 8 || ldx % 8 || !aligned16(xp) || !aligned16(wp) || !aligned16(ap) ||
                         !aligned16(bp) || !aligned16(yp)))
    Py_RETURN_NONE;
  lf_rows_problem p{};
  p.dtype = code;
  p.T = static_cast<int32_t>(T);
  p.K = static_cast<int32_t>(K);
  p.N = static_cast<int32_t>(N);
  p.n_slots = static_cast<int32_t>(ba.size(0));
  p.r_pad = static_cast<int32_t>(r_pad);
  p.row_slot_bytes = wide ? 8 : 4;
  p.weight_format = mx4 ? LF_WEIGHT_MX4 : LF_WEIGHT_DENSE;
  p.ldx = ldx;
  p.x_dev = xp;
  p.w_dev = wp;
  p.a_bank_dev = ap;
  p.b_bank_dev = bp;
  p.slot_rank_dev = static_cast<const int32_t*>(ranks.const_data_ptr());
  p.slot_scale_dev = static_cast<const float*>(scales.const_data_ptr());
  p.row_slot_dev = slot.const_data_ptr();
  const size_t bytes = lf_rows_workspace_bytes(p.T, p.N, p.r_pad, code);
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor ws = at::detail::empty_cuda({static_cast<int64_t>(bytes)}, at::kByte, dev, std::nullopt);
  const int rc = lf_rows_forward(&p, yp, ws.data_ptr(), bytes, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc != LF_OK) return fail(rc, "lf_rows_forward");
  if (a[7] != Py_None) {
    bump(y);
    return Py_NewRef(a[7]);
  }
  return THPVariable_Wrap(std::move(y));
}

// mx4_linear(x, data, out_features, in_features, dtype code, transpose): x V^T, or x V with transpose, on operands that
// need no copy; V the values of the weight in 4 bits whose data and shape these are.  None otherwise.
PyObject* mx4_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "mx4_linear takes 6 arguments");
    return nullptr;
  }
  const at::Tensor *xt = cuda_tensor(a[0]), *wt = cuda_tensor(a[1]);
  if (!xt || !wt) Py_RETURN_NONE;
  const at::Tensor &x = *xt, &w = *wt;
  lf_mx4_problem p{};
  p.N = static_cast<int32_t>(PyLong_AsLong(a[2]));
  p.K = static_cast<int32_t>(PyLong_AsLong(a[3]));
  p.dtype = static_cast<int32_t>(PyLong_AsLong(a[4]));
  p.transpose = static_cast<int32_t>(PyLong_AsLong(a[5]));
  if (PyErr_Occurred()) return nullptr;
  const int64_t in = p.transpose ? p.N : p.K, out = p.transpose ? p.K : p.N;
  if (dtype_code(x.scalar_type()) != p.dtype || x.dim() != 2 || x.size(1) != in || x.device() != w.device() ||
      x.size(0) == 0 || x.size(0) > INT32_MAX || p.K % 8 || p.N % 8)
    Py_RETURN_NONE;
  const int64_t ld = x.is_contiguous() ? in : x.stride(0);
  if (!x.is_contiguous() && (x.stride(1) != 1 || ld < in)) Py_RETURN_NONE;
  if (ld % 8 || !aligned16(x.const_data_ptr())) Py_RETURN_NONE;
  p.T = static_cast<int32_t>(x.size(0));
  p.ld = ld;
  p.in_dev = x.const_data_ptr();
  p.mx4_dev = w.const_data_ptr();
  const auto dev = x.device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor y = at::detail::empty_cuda({x.size(0), out}, x.scalar_type(), dev, std::nullopt);
  const int64_t bytes = static_cast<int64_t>(lf_mx4_linear_workspace_bytes(p.K, p.N));
  at::Tensor ws = at::detail::empty_cuda({bytes}, at::kByte, dev, std::nullopt);
  const int rc = lf_mx4_linear(&p, y.data_ptr(), ws.data_ptr(), static_cast<size_t>(bytes),
                               c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc != LF_OK) return fail(rc, "lf_mx4_linear");
  return THPVariable_Wrap(std::move(y));
}

// mx4_quantize(weight, dtype code): the data of a weight in 4 bits, on an operand that needs no copy.  None otherwise.
PyObject* mx4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "mx4_quantize takes 2 arguments");
    return nullptr;
  }
  const at::Tensor* wt = cuda_tensor(a[0]);
  const long code = PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if (!wt || wt->dim() != 2 || dtype_code(wt->scalar_type()) != code) Py_RETURN_NONE;
  const at::Tensor& w = *wt;
  const int64_t N = w.size(0), K = w.size(1), ld = w.is_contiguous() ? K : w.stride(0);
  if (N < 1 || K < 1 || N > (1 << 24) || K > (1 << 24) || (!w.is_contiguous() && (w.stride(1) != 1 || ld < K)))
    Py_RETURN_NONE;
  const auto dev = w.device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int64_t bytes = static_cast<int64_t>(lf_mx4_bytes(static_cast<int32_t>(N), static_cast<int32_t>(K)));
  at::Tensor data = at::detail::empty_cuda({bytes}, at::kByte, dev, std::nullopt);
  const int rc = lf_mx4_quantize(static_cast<int32_t>(code), w.const_data_ptr(), static_cast<int32_t>(N),
                                 static_cast<int32_t>(K), ld, data.data_ptr(),
                                 c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc != LF_OK) return fail(rc, "lf_mx4_quantize");
  return THPVariable_Wrap(std::move(data));
}

// mx4_dequantize(data, out_features, in_features, dtype code): the dense weight.
PyObject* mx4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "mx4_dequantize takes 4 arguments");
    return nullptr;
  }
  const at::Tensor* dt = cuda_tensor(a[0]);
  const long N = PyLong_AsLong(a[1]), K = PyLong_AsLong(a[2]), code = PyLong_AsLong(a[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!dt || (code != LF_BF16 && code != LF_F16)) {
    PyErr_SetString(PyExc_ValueError, "mx4_dequantize: not the data of a weight in 4 bits");
    return nullptr;
  }
  const auto dev = dt->device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor w = at::detail::empty_cuda({N, K}, code == LF_BF16 ? at::kBFloat16 : at::kHalf, dev, std::nullopt);
  const int rc = lf_mx4_dequantize(static_cast<int32_t>(code), dt->const_data_ptr(), static_cast<int32_t>(N),
                                   static_cast<int32_t>(K), w.data_ptr(),
                                   c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc != LF_OK) return fail(rc, "lf_mx4_dequantize");
  return THPVariable_Wrap(std::move(w));
}

// The capture into a CUDA graph that a stream is in, 0 for none.
unsigned long long capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();  // the legacy stream beside another one's capture: not captured itself
    status = cudaStreamCaptureStatusNone;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// at(device index): the device's current stream, and the id of the capture into a CUDA graph that it is in (0: none).
PyObject* at_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) {
    PyErr_SetString(PyExc_TypeError, "at takes 1 argument");
    return nullptr;
  }
  const long dev = PyLong_AsLong(a[0]);
  if (PyErr_Occurred()) return nullptr;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  return Py_BuildValue("(KK)", static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream)), capture_of(stream));
}

// Captures whose graphs are gone, until ended() takes them.  Never destroyed: graphs may outlive the module.
struct Ended {
  std::mutex lock;
  std::vector<unsigned long long> ids;
};
Ended& ended_captures() {
  static Ended* e = new Ended;
  return *e;
}
struct Token {
  unsigned long long id;
};
void CUDART_CB capture_ended(void* p) {  // on a thread of CUDA's, which must make no CUDA call
  Token* token = static_cast<Token*>(p);
  Ended& e = ended_captures();
  try {
    const std::lock_guard<std::mutex> hold(e.lock);
    e.ids.push_back(token->id);
  } catch (...) {  // what the capture held stays held
  }
  delete token;
}

// hold_capture(device index): the id of the capture that the device's current stream is in, for ended() to return once its
// graph, every graph instantiated from it and their launches are over.
PyObject* hold_capture(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) {
    PyErr_SetString(PyExc_TypeError, "hold_capture takes 1 argument");
    return nullptr;
  }
  const long dev = PyLong_AsLong(a[0]);
  if (PyErr_Occurred()) return nullptr;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  cudaError_t e = cudaStreamGetCaptureInfo(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(),
                                           &status, &id, &graph);
  if (e == cudaSuccess && status != cudaStreamCaptureStatusActive) e = cudaErrorIllegalState;
  if (e == cudaSuccess) {
    std::unique_ptr<Token> token(new Token{id});
    cudaUserObject_t object = nullptr;
    e = cudaUserObjectCreate(&object, token.get(), capture_ended, 1, cudaUserObjectNoDestructorSync);
    if (e == cudaSuccess) {
      token.release();  // the object's
      e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
      if (e != cudaSuccess) cudaUserObjectRelease(object, 1);
    }
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    PyErr_Format(PyExc_RuntimeError, "hold_capture: %s", cudaGetErrorString(e));
    return nullptr;
  }
  return PyLong_FromUnsignedLongLong(id);
}

// ended(): ids of captures that are over since the last call.
PyObject* ended(PyObject*, PyObject* const*, Py_ssize_t n) {
  if (n != 0) {
    PyErr_SetString(PyExc_TypeError, "ended takes no arguments");
    return nullptr;
  }
  std::vector<unsigned long long> ids;
  {
    Ended& e = ended_captures();
    const std::lock_guard<std::mutex> hold(e.lock);
    ids.swap(e.ids);
  }
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ids.size()));
  for (size_t i = 0; out && i < ids.size(); ++i) {
    PyObject* id = PyLong_FromUnsignedLongLong(ids[i]);
    if (!id) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, static_cast<Py_ssize_t>(i), id);
  }
  return out;
}

// wait_event(cudaEvent_t): the host waits for an event recorded outside the capture that this thread may be in.
PyObject* wait_event(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) {
    PyErr_SetString(PyExc_TypeError, "wait_event takes 1 argument");
    return nullptr;
  }
  void* event = PyLong_AsVoidPtr(a[0]);
  if (PyErr_Occurred()) return nullptr;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // a wait here is none of the captured work
  cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
  if (e == cudaSuccess) {
    Py_BEGIN_ALLOW_THREADS
    e = cudaEventSynchronize(static_cast<cudaEvent_t>(event));
    Py_END_ALLOW_THREADS
    cudaThreadExchangeStreamCaptureMode(&mode);
  }
  if (e != cudaSuccess) {
    PyErr_Format(PyExc_RuntimeError, "wait_event: %s", cudaGetErrorString(e));
    return nullptr;
  }
  Py_RETURN_NONE;
}

// bank_load(bank_a, bank_b, ranks, scales, slot, lora_a, lora_b, scaling): an adapter into its slot.  None unless its
// tensors have the bank's dtype and device and dense rows; shapes were checked by the caller.
PyObject* bank_load(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bank_load takes 8 arguments");
    return nullptr;
  }
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = cuda_tensor(a[i < 4 ? i : i + 1]))) Py_RETURN_NONE;
  const at::Tensor &ba = *t[0], &bb = *t[1], &la = *t[4], &lb = *t[5];
  const int64_t slot = PyLong_AsLongLong(a[4]);
  lf_bank_adapter p{};
  p.scale = static_cast<float>(PyFloat_AsDouble(a[7]));
  if (PyErr_Occurred()) return nullptr;
  p.dtype = dtype_code(ba.scalar_type());
  if (p.dtype < 0 || la.scalar_type() != ba.scalar_type() || lb.scalar_type() != ba.scalar_type() ||
      la.device() != ba.device() || lb.device() != ba.device() || la.dim() != 2 || lb.dim() != 2 ||
      (la.size(1) > 1 && la.stride(1) != 1) || (lb.size(1) > 1 && lb.stride(1) != 1) || la.size(0) > ba.size(1) ||
      la.size(1) != ba.size(2) || lb.size(0) != bb.size(2) || lb.size(1) != la.size(0) || slot < 0 || slot >= ba.size(0))
    Py_RETURN_NONE;
  p.K = static_cast<int32_t>(ba.size(2));
  p.N = static_cast<int32_t>(bb.size(2));
  p.r_pad = static_cast<int32_t>(ba.size(1));
  p.rank = static_cast<int32_t>(la.size(0));
  p.lda = la.stride(0);
  p.ldb = lb.stride(0);
  if ((p.rank > 1 && p.lda < p.K) || (p.N > 1 && p.ldb < p.rank)) Py_RETURN_NONE;  // rows that overlap
  const size_t es = ba.element_size();
  p.a_dev = la.const_data_ptr();
  p.b_dev = lb.const_data_ptr();
  p.slot_a_dev = static_cast<char*>(ba.data_ptr()) + static_cast<size_t>(slot) * p.r_pad * p.K * es;
  p.slot_b_dev = static_cast<char*>(bb.data_ptr()) + static_cast<size_t>(slot) * p.r_pad * p.N * es;
  p.slot_rank_dev = static_cast<int32_t*>(t[2]->data_ptr()) + slot;
  p.slot_scale_dev = static_cast<float*>(t[3]->data_ptr()) + slot;
  const c10::cuda::OptionalCUDAGuard guard(ba.device());
  const int rc = lf_bank_load(&p, c10::cuda::getCurrentCUDAStream(ba.device().index()).stream());
  if (rc == LF_ERR_INVALID_ARG) Py_RETURN_NONE;  // the adapter lies in the slot itself
  if (rc != LF_OK) return fail(rc, "lf_bank_load");
  for (int i = 0; i < 4; ++i) bump(*t[i]);
  Py_RETURN_TRUE;
}

// clip(grads, per_adapter, inf_norm, max_norm or None): norms of clip_adapter_grads, or None.
PyObject* clip(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "clip takes 4 arguments");
    return nullptr;
  }
  const int per_adapter = PyObject_IsTrue(a[1]), inf = PyObject_IsTrue(a[2]);
  const bool scale = a[3] != Py_None;
  const double max_norm = scale ? PyFloat_AsDouble(a[3]) : 0.0;
  if (per_adapter < 0 || inf < 0 || (scale && max_norm == -1.0 && PyErr_Occurred())) return nullptr;
  if (!PyList_CheckExact(a[0]) && !PyTuple_CheckExact(a[0])) Py_RETURN_NONE;
  std::vector<lf_grad_tensor> rec;
  std::vector<const at::Tensor*> tensors;
  PyObject* order = PyDict_New();  // adapter id -> group, in order of first appearance
  if (!order) return nullptr;
  struct Release {
    PyObject* o;
    ~Release() { Py_DECREF(o); }
  } release{order};
  int32_t groups = per_adapter ? 0 : 1;
  const Py_ssize_t n_dicts = PySequence_Fast_GET_SIZE(a[0]);
  c10::Device dev(c10::kCPU);
  for (Py_ssize_t j = 0; j < n_dicts; ++j) {
    PyObject* d = PySequence_Fast_GET_ITEM(a[0], j);
    if (!PyDict_CheckExact(d)) Py_RETURN_NONE;
    Py_ssize_t pos = 0;
    PyObject *key, *value;
    while (PyDict_Next(d, &pos, &key, &value)) {
      const at::Tensor* t = cuda_tensor(value);
      if (!t || !t->is_contiguous()) Py_RETURN_NONE;
      const int code = dtype_code(t->scalar_type());
      if (code < 0) Py_RETURN_NONE;
      if (tensors.empty()) dev = t->device();
      else if (t->device() != dev) Py_RETURN_NONE;
      int32_t group = 0;
      if (per_adapter) {
        PyObject* g = PyDict_GetItemWithError(order, key);
        if (g) {
          group = static_cast<int32_t>(PyLong_AsLong(g));
        } else {
          if (PyErr_Occurred()) return nullptr;
          group = groups++;
          PyObject* v = PyLong_FromLong(group);
          if (!v) return nullptr;
          const int set = PyDict_SetItem(order, key, v);
          Py_DECREF(v);
          if (set < 0) return nullptr;
        }
      }
      rec.push_back({reinterpret_cast<uint64_t>(t->const_data_ptr()), static_cast<uint64_t>(t->numel()), code, group});
      tensors.push_back(t);
    }
  }
  if (rec.empty()) Py_RETURN_NONE;
  const int32_t count = static_cast<int32_t>(rec.size());
  const size_t bytes = lf_grad_clip_workspace_bytes(rec.data(), count, groups);
  if (bytes == 0) Py_RETURN_NONE;
  const c10::cuda::OptionalCUDAGuard guard(dev);
  at::Tensor norms = per_adapter ? at::detail::empty_cuda({groups}, at::kFloat, dev, std::nullopt)
                                 : at::detail::empty_cuda({}, at::kFloat, dev, std::nullopt);
  at::Tensor ws = at::detail::empty_cuda({static_cast<int64_t>(bytes)}, at::kByte, dev, std::nullopt);
  const int rc = lf_grad_clip(rec.data(), count, groups, inf, scale, max_norm, static_cast<float*>(norms.data_ptr()),
                              ws.data_ptr(), bytes, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  if (rc == LF_ERR_INVALID_ARG) Py_RETURN_NONE;
  if (rc != LF_OK) return fail(rc, "lf_grad_clip");
  if (scale)
    for (const at::Tensor* t : tensors) bump(*t);
  return THPVariable_Wrap(std::move(norms));
}

// gather_step(grads, keys, weights, addresses, out): fills `out` (a writable buffer of one uint64 a weight) with the
// addresses of this step's gradients, 0 where a dict has none.  keys: the ids of each dict, weights: all weights in
// that order, addresses: where the optimizer last saw them.  Returns the gradients' dtype code, -1 without any, or
// None.
PyObject* gather_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "gather_step takes 5 arguments");
    return nullptr;
  }
  if (!PyList_CheckExact(a[0]) && !PyTuple_CheckExact(a[0])) Py_RETURN_NONE;
  Py_ssize_t n_dicts = PySequence_Fast_GET_SIZE(a[0]), at_weight = 0;
  if (!PyList_CheckExact(a[1]) || !PyList_CheckExact(a[2]) || PyList_GET_SIZE(a[1]) != n_dicts) Py_RETURN_NONE;
  Py_buffer seen, out;
  if (PyObject_GetBuffer(a[3], &seen, PyBUF_SIMPLE) < 0) return nullptr;
  struct Release {
    Py_buffer* b;
    ~Release() { PyBuffer_Release(b); }
  } release_seen{&seen};
  if (PyObject_GetBuffer(a[4], &out, PyBUF_WRITABLE) < 0) return nullptr;
  Release release_out{&out};
  const Py_ssize_t n_weights = PyList_GET_SIZE(a[2]);
  if (seen.len != n_weights * 8 || out.len != n_weights * 8) Py_RETURN_NONE;
  const uint64_t* addresses = static_cast<const uint64_t*>(seen.buf);
  uint64_t* ptrs = static_cast<uint64_t*>(out.buf);
  int dtype = -1;
  for (Py_ssize_t j = 0; j < n_dicts; ++j) {
    PyObject *d = PySequence_Fast_GET_ITEM(a[0], j), *keys = PyList_GET_ITEM(a[1], j);
    if (!PyDict_CheckExact(d) || !PyList_CheckExact(keys)) Py_RETURN_NONE;
    Py_ssize_t found = 0;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(keys); ++i, ++at_weight) {
      if (at_weight >= n_weights) Py_RETURN_NONE;
      const at::Tensor* w = cuda_tensor(PyList_GET_ITEM(a[2], at_weight));
      if (!w || reinterpret_cast<uint64_t>(w->const_data_ptr()) != addresses[at_weight]) Py_RETURN_NONE;
      PyObject* v = PyDict_GetItemWithError(d, PyList_GET_ITEM(keys, i));
      if (!v) {
        if (PyErr_Occurred()) return nullptr;
        ptrs[at_weight] = 0;
        continue;
      }
      const at::Tensor* g = cuda_tensor(v);
      if (!g || !g->is_contiguous() || g->device() != w->device() || g->sizes() != w->sizes()) Py_RETURN_NONE;
      const int code = dtype_code(g->scalar_type());
      if (code < 0 || (dtype >= 0 && code != dtype) || (code != LF_F32 && g->scalar_type() != w->scalar_type()))
        Py_RETURN_NONE;
      dtype = code;
      ptrs[at_weight] = reinterpret_cast<uint64_t>(g->const_data_ptr());
      ++found;
    }
    if (found != PyDict_GET_SIZE(d)) Py_RETURN_NONE;
  }
  if (at_weight != n_weights) Py_RETURN_NONE;
  return PyLong_FromLong(dtype);
}

struct Buffer {  // a contiguous buffer for the length of a call
  Py_buffer b{};
  bool ok;
  explicit Buffer(PyObject* o) : ok(PyObject_GetBuffer(o, &b, PyBUF_SIMPLE) == 0) {}
  ~Buffer() {
    if (ok) PyBuffer_Release(&b);
  }
};

// adamw_step(weights, addresses, records, device records, chunks, hyper, steps, exp_avg, exp_avg_sq, master or None,
// n_chunks, n_groups, workspace bytes, (beta1, beta2), eps, max_norm or None, skip_nonfinite, dtype codes of the
// weights and the gradients): lf_adamw_step, and the version counters of the state and of every weight that has a gradient.
// Returns the norms, or None when neither clipping nor skip_nonfinite asks for them.
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 19 || !PyList_CheckExact(a[0]) || !PyTuple_CheckExact(a[13]) || PyTuple_GET_SIZE(a[13]) != 2) {
    PyErr_SetString(PyExc_TypeError, "adamw_step takes a list of weights and 18 more arguments");
    return nullptr;
  }
  const at::Tensor* t[7];
  for (int i = 0; i < 7; ++i) {
    t[i] = a[3 + i] == Py_None && i == 6 ? nullptr : cuda_tensor(a[3 + i]);
    if (!t[i] && !(i == 6 && a[9] == Py_None)) {
      PyErr_SetString(PyExc_TypeError, "the optimizer's state must be CUDA tensors");
      return nullptr;
    }
  }
  const Buffer grads(a[1]), records(a[2]);
  if (!grads.ok || !records.ok) return nullptr;
  const Py_ssize_t count = PyList_GET_SIZE(a[0]);
  if (grads.b.len != count * 8 || records.b.len != count * static_cast<Py_ssize_t>(sizeof(lf_adamw_tensor))) {
    PyErr_SetString(PyExc_ValueError, "one address and one record a weight");
    return nullptr;
  }
  lf_adamw_args p{};
  p.tensors = static_cast<const lf_adamw_tensor*>(records.b.buf);
  p.tensors_dev = static_cast<const lf_adamw_tensor*>(t[0]->const_data_ptr());
  p.chunk_tensor_dev = static_cast<const int32_t*>(t[1]->const_data_ptr());
  p.grads = static_cast<const uint64_t*>(grads.b.buf);
  p.hyper_dev = static_cast<const double*>(t[2]->const_data_ptr());
  p.steps_dev = static_cast<int32_t*>(t[3]->data_ptr());
  p.exp_avg_dev = static_cast<float*>(t[4]->data_ptr());
  p.exp_avg_sq_dev = static_cast<float*>(t[5]->data_ptr());
  p.master_dev = t[6] ? static_cast<float*>(t[6]->data_ptr()) : nullptr;
  p.n_chunks = PyLong_AsLongLong(a[10]);
  p.n_groups = static_cast<int32_t>(PyLong_AsLong(a[11]));
  p.workspace_bytes = PyLong_AsSize_t(a[12]);
  p.beta1 = PyFloat_AsDouble(PyTuple_GET_ITEM(a[13], 0));
  p.beta2 = PyFloat_AsDouble(PyTuple_GET_ITEM(a[13], 1));
  p.eps = PyFloat_AsDouble(a[14]);
  p.max_norm = a[15] == Py_None ? -1.0 : PyFloat_AsDouble(a[15]);
  p.skip_nonfinite = PyObject_IsTrue(a[16]);
  p.param_dtype = static_cast<int32_t>(PyLong_AsLong(a[17]));
  p.grad_dtype = static_cast<int32_t>(PyLong_AsLong(a[18]));
  p.n_tensors = static_cast<int32_t>(count);
  if (PyErr_Occurred()) return nullptr;
  const auto dev = t[3]->device();
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  const cudaError_t asked = cudaStreamIsCapturing(stream, &capture);
  if (asked != cudaSuccess || capture != cudaStreamCaptureStatusNone) {
    if (asked != cudaSuccess) cudaGetLastError();  // the answer to the question, not an error of a later call
    PyErr_SetString(PyExc_RuntimeError,
                    "AdapterAdamW.step cannot be captured into a CUDA graph: replays would change weights whose packed "
                    "copies b200_ops keeps");
    return nullptr;
  }
  at::Tensor norms;
  if (p.max_norm >= 0.0 || p.skip_nonfinite) {
    norms = at::detail::empty_cuda({p.n_groups}, at::kFloat, dev, std::nullopt);
    p.norms_dev = static_cast<float*>(norms.data_ptr());
  }
  at::Tensor ws = at::detail::empty_cuda({static_cast<int64_t>(p.workspace_bytes)}, at::kByte, dev, std::nullopt);
  p.workspace_dev = ws.data_ptr();
  const int rc = lf_adamw_step(&p, stream);
  if (rc != LF_OK) return fail(rc, "lf_adamw_step");
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* o = PyList_GET_ITEM(a[0], i);
    if (p.grads[i] && THPVariable_Check(o)) bump(THPVariable_Unpack(o));
  }
  for (int i = 3; i < 7; ++i)  // steps, both moments, masters
    if (t[i]) bump(*t[i]);
  if (!norms.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(norms));
}

// C++ exceptions (an allocation that fails, a CUDA error in the allocator) as Python ones.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyMethodDef methods[] = {
    {"rows_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<rows_forward>)), METH_FASTCALL, nullptr},
    {"mx4_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<mx4_linear>)), METH_FASTCALL, nullptr},
    {"mx4_quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<mx4_quantize>)), METH_FASTCALL, nullptr},
    {"mx4_dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<mx4_dequantize>)), METH_FASTCALL, nullptr},
    {"at", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<at_stream>)), METH_FASTCALL, nullptr},
    {"hold_capture", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<hold_capture>)), METH_FASTCALL, nullptr},
    {"ended", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<ended>)), METH_FASTCALL, nullptr},
    {"wait_event", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<wait_event>)), METH_FASTCALL, nullptr},
    {"bank_load", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<bank_load>)), METH_FASTCALL, nullptr},
    {"clip", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<clip>)), METH_FASTCALL, nullptr},
    {"gather_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<gather_step>)), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(guarded<adamw_step>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "lf_pyglue", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lf_pyglue(void) { return PyModule_Create(&module_def); }
