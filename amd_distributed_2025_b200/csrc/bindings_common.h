// What the files that bind C++ to Python share: checks, the fp8 kernels' status words, arguments and results of the calls
// that are functions of the C API.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/stl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <atomic>
#include <cstring>
#include <string>
#include <vector>

#include "status.h"

namespace b200 {
namespace bind {

namespace py = pybind11;

// A number in a message.  (Where the extension carries a C++ library of its own, an integer that goes through one of its
// streams ends the process: the locales of the two libraries have different facets.)
inline std::string num(int64_t v) { return std::to_string(v); }

inline void cuda_check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

// A kernel can read device memory and pinned host memory; an ordinary host tensor would fault the GPU.
inline void check_reachable(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() || t.is_pinned(), what, " must be a CUDA tensor");
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return 0;
    case at::kBFloat16: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "unsupported dtype ", t, " (expected float16, bfloat16 or float32)");
  }
  return -1;
}

inline py::dict status_to_dict(const b200::StatusWord& w) {
  py::dict d;
  d["code"] = w.code;
  d["phase"] = w.phase;
  d["peer"] = w.peer;
  d["detail"] = w.detail;
  d["epoch"] = w.epoch;
  d["seen"] = w.seen;
  return d;
}

inline int device_sms(int device) {
  static const std::vector<int> sms = [] {
    std::vector<int> v;
    for (int d = 0; d < (int)at::cuda::device_count(); ++d)
      v.push_back(at::cuda::getDeviceProperties(d)->multiProcessorCount);
    return v;
  }();
  return sms.at((size_t)device);
}

// Where fp8_gemm leaves the record of an expired wait: one word per device, in mapped host memory, for the life of the
// process (the operation has no object of its own to hold it).
inline b200::StatusWord* fp8_status(int device) {
  constexpr int kDevices = 64;
  static b200::StatusWord* const words = [] {
    // (the first call may come while a stream is being captured, which an allocation would break off in any other mode)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cuda_check(cudaThreadExchangeStreamCaptureMode(&mode), "fp8_gemm status");
    void* w = nullptr;
    const cudaError_t e = cudaHostAlloc(&w, kDevices * sizeof(b200::StatusWord), cudaHostAllocMapped | cudaHostAllocPortable);
    cuda_check(cudaThreadExchangeStreamCaptureMode(&mode), "fp8_gemm status");
    cuda_check(e, "fp8_gemm status");
    std::memset(w, 0, kDevices * sizeof(b200::StatusWord));
    return static_cast<b200::StatusWord*>(w);
  }();
  TORCH_CHECK(device >= 0 && device < kDevices, "device index out of range");
  return words + device;
}

inline uint32_t fp8_status_code(int device) { return reinterpret_cast<const volatile b200::StatusWord*>(fp8_status(device))->code; }

// The record of a device, which is cleared: an expired wait leaves nothing behind that a later call could trip over.
inline py::dict fp8_gemm_take_status(int device) {
  b200::StatusWord* w = fp8_status(device);
  const uint32_t code = fp8_status_code(device);
  std::atomic_thread_fence(std::memory_order_acquire);
  b200::StatusWord copy = *w;
  copy.code = code;
  if (code != 0) std::memset(w, 0, sizeof(*w));
  return status_to_dict(copy);
}

inline const at::Tensor& tensor_arg(PyObject* o) {
  if (!THPVariable_Check(o)) throw py::type_error(std::string("expected a torch.Tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
inline void count_args(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw py::type_error("expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
}
inline double double_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw py::error_already_set();
  return v;
}
inline PyObject* wrap(const c10::optional<at::Tensor>& t) {
  if (!t.has_value()) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}
// Runs a call; a C++ exception becomes a Python one.
template <typename F>
inline PyObject* guarded(F&& call) {
  HANDLE_TH_ERRORS
  try {
    return call();
  } catch (py::error_already_set& e) {
    e.restore();
    return nullptr;
  } catch (py::builtin_exception& e) {
    e.set_error();
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
}  // namespace bind
}  // namespace b200
