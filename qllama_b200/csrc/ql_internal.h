// ql_internal.h -- library-internal view of the context, shared by the
// attention API (ql_api.cu) and the model host (ql_model.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

struct ql_ctx {
  int device = 0;
  int num_sms = 0;
  cudaStream_t own = nullptr;
  cudaStream_t stream = nullptr;
  uint32_t* status = nullptr;  // device word raised by kernels
  void* ws = nullptr;          // workspace (staging, split partials, scratch)
  size_t ws_bytes = 0;
  int32_t* counters = nullptr;  // split-merge arrival counters, kept at zero
  size_t counters_n = 0;
  cudaEvent_t order[2] = {nullptr, nullptr};  // of ql_ctx_wait_stream and ql_ctx_join_stream
};

// Records the message of a failed call (ql_last_error) and returns `code`.
int ql_fail(int code, const char* fmt, ...);
// Reads and clears the context's device status word; QL_ERR_DEVICE with a
// message when a kernel raised a bit.
int ql_check_status(ql_ctx* c);
// The context's reusable device workspace, grown to at least `bytes`
// (growing synchronises the context's stream first).
int ql_ctx_workspace(ql_ctx* c, size_t bytes, void** out);

// Makes `device` current for one call and puts the caller's device back.
class ql_device_guard {
 public:
  explicit ql_device_guard(int device) {
    if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
    if (prev_ != device) {
      err_ = cudaSetDevice(device);
      moved_ = true;
    }
  }
  ~ql_device_guard() {
    if (moved_ && prev_ >= 0) cudaSetDevice(prev_);
  }
  ql_device_guard(const ql_device_guard&) = delete;
  ql_device_guard& operator=(const ql_device_guard&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int prev_ = -1;
  bool moved_ = false;
  cudaError_t err_ = cudaSuccess;
};

// Runs `set` once for each device (kernel attributes belong to a device's context).
// Two first calls at once both run it, with the same effect.
template <typename F>
cudaError_t ql_once_per_device(std::atomic<uint64_t>& done, F set) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = set();
  if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
  return e;
}
