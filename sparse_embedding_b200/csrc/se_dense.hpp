// Host-side helpers of the dense operators (layer normalisation, the Muon
// update): argument checks and dispatch on the value type.
#pragma once

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "se_common.cuh"
#include "se_host.hpp"

namespace se_gpu {

inline void check_value_dtype(int32_t t, const char *what) {
  if (t < SE_FLOAT32 || t > SE_BFLOAT16) throw std::invalid_argument(std::string("unsupported ") + what);
}

// The dense operators read and write their arrays in place: device memory of
// the call's device (managed memory included). A host pointer, or one of
// another device, is refused here instead of faulting in a kernel.
inline void check_device_ptr(const void *p, int device, const char *what, bool optional = false) {
  if (p == nullptr) {
    if (optional) return;
    throw std::invalid_argument(std::string(what) + " is null");
  }
  cudaPointerAttributes a{};
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    a.type = cudaMemoryTypeUnregistered;
  }
  if (a.type == cudaMemoryTypeManaged) return;
  if (a.type != cudaMemoryTypeDevice) throw std::invalid_argument(std::string(what) + " must be device memory");
  if (a.device != device)
    throw std::invalid_argument(std::string(what) + " is on cuda:" + std::to_string(a.device) + ", the call on cuda:" +
                                std::to_string(device));
}

// f with the value type's tag (F32, F16, BF16).
template <class F> void dispatch_value(int32_t t, F &&f) {
  if (t == SE_FLOAT32) f(F32{});
  else if (t == SE_FLOAT16) f(F16{});
  else f(BF16{});
}

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Multiprocessors of a device (read once per device).
inline int sm_count(int device) {
  static std::mutex mu;
  static std::map<int, int> known;
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find(device);
  if (it != known.end()) return it->second;
  int n = 0;
  cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device), "cudaDeviceGetAttribute");
  return known[device] = n;
}

}  // namespace se_gpu
