// Host-side helpers of the dense operators (layer normalisation, the Muon
// update): argument checks and dispatch on the value type.
#pragma once

#include <algorithm>
#include <atomic>
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

// Blocks of a kernel that run on a multiprocessor at once (asked once per
// device, block and shared memory).
template <class... KArgs>
inline int resident_blocks(void (*kernel)(KArgs...), int device, int threads, size_t smem) {
  using Key = std::pair<std::pair<const void *, int>, std::pair<int, size_t>>;
  static std::mutex mu;
  static std::map<Key, int> known;
  const Key key{{reinterpret_cast<const void *>(kernel), device}, {threads, smem}};
  std::lock_guard<std::mutex> lock(mu);
  auto it = known.find(key);
  if (it != known.end()) return it->second;
  int n = 0;
  cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem), "occupancy");
  return known[key] = n < 1 ? 1 : n;
}

// Clocks after which a wait inside the dense operators' kernels gives up
// (se_set_wait_limit).
constexpr long long kWaitClocks = 8000000000ll;
inline std::atomic<long long> &wait_limit() {
  static std::atomic<long long> clocks{kWaitClocks};
  return clocks;
}

// Words in host memory that a kernel sets when one of its waits gave up: one per
// device and stream, so that the report reaches who works on that stream, and
// not another thread or stream. They live as long as the process, as graphs do
// that hold their addresses. A report is taken by an exchange: one that comes
// while it is taken is seen then or the next time.
class WaitWords {
 public:
  static WaitWords &get() {
    static WaitWords words;
    return words;
  }
  // The word of a call on `stream`; throws where an earlier call's report is in it.
  // (Memory for words may be asked for under stream capture.)
  uint32_t *of(int device, cudaStream_t stream) {
    static thread_local char here;
    if (stream == cudaStreamLegacy) stream = nullptr;
    const Key key{{device, stream}, stream == cudaStreamPerThread ? &here : nullptr};
    std::lock_guard<std::mutex> lock(mu_);
    auto it = known_.find(key);
    if (it == known_.end()) it = known_.emplace(key, fresh()).first;
    if (taken(it->second))
      throw Error(SE_ERR_RUNTIME, "an earlier layer normalisation or Muon update on this stream of cuda:" +
                                      std::to_string(device) + kGaveUp);
    return it->second;
  }
  // All reports of a device.
  void check(int device) {
    std::lock_guard<std::mutex> lock(mu_);
    bool any = false;
    for (auto &k : known_)
      if (k.first.first.first == device) any |= taken(k.second);
    if (any) throw Error(SE_ERR_RUNTIME, "a layer normalisation or Muon update on cuda:" + std::to_string(device) + kGaveUp);
  }

 private:
  using Key = std::pair<std::pair<int, cudaStream_t>, const void *>;
  static constexpr const char *kGaveUp = " gave up waiting for its copies; its results are not valid";
  static constexpr int kPage = 1024;
  static bool taken(uint32_t *word) {
    return *static_cast<volatile uint32_t *>(word) != 0u && __atomic_exchange_n(word, 0u, __ATOMIC_ACQ_REL) != 0u;
  }
  uint32_t *fresh() {
    if (left_ == 0) {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cuda_check(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
      void *p = nullptr;
      const cudaError_t e = cudaHostAlloc(&p, kPage * sizeof(uint32_t), cudaHostAllocMapped | cudaHostAllocPortable);
      cudaThreadExchangeStreamCaptureMode(&mode);
      cuda_check(e, "cudaHostAlloc");
      page_ = static_cast<uint32_t *>(p);
      std::fill(page_, page_ + kPage, 0u);
      left_ = kPage;
    }
    return page_ + --left_;
  }
  std::mutex mu_;
  std::map<Key, uint32_t *> known_;
  uint32_t *page_ = nullptr;
  int left_ = 0;
};

}  // namespace se_gpu
