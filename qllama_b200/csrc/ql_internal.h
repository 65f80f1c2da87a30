// ql_internal.h -- library-internal view of the context, shared by the
// attention API (ql_api.cu) and the model host (ql_model.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <vector>

struct ql_ctx {
  int device = 0;
  int num_sms = 0;
  cudaStream_t own = nullptr;
  cudaStream_t stream = nullptr;
  uint32_t* status = nullptr;  // device word raised by kernels
  void* ws = nullptr;          // workspace (staging, split partials, scratch)
  size_t ws_bytes = 0;
  bool ws_captured = false;     // a captured graph uses the workspace
  int32_t* counters = nullptr;  // split-merge arrival counters, kept at zero
  size_t counters_n = 0;
  bool counters_captured = false;  // a captured graph uses them
  std::vector<void*> retired;   // outgrown workspaces and counters of captured graphs
  cudaEvent_t order[2] = {nullptr, nullptr};  // of ql_ctx_wait_stream and ql_ctx_join_stream
  cudaStream_t aside = nullptr;  // for what has to happen at once while `stream` is captured
  std::atomic<int> users{1};     // its handle, and what has been made with it
};

// One user less; the last one's going frees the context.
void ql_ctx_release(ql_ctx* c);

// The context of a cache, a weight, a model or a communicator: it stays until the last of them
// has gone, in whatever order a caller (or Python's collector) destroys them and the context.
class ql_ctx_ref {
 public:
  ql_ctx_ref() = default;
  ql_ctx_ref(const ql_ctx_ref&) = delete;
  ql_ctx_ref& operator=(const ql_ctx_ref&) = delete;
  ~ql_ctx_ref() {
    if (c_) ql_ctx_release(c_);
  }
  ql_ctx_ref& operator=(ql_ctx* c) {
    if (c) c->users.fetch_add(1, std::memory_order_relaxed);
    if (c_) ql_ctx_release(c_);
    c_ = c;
    return *this;
  }
  operator ql_ctx*() const { return c_; }
  ql_ctx* operator->() const { return c_; }

 private:
  ql_ctx* c_ = nullptr;
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
