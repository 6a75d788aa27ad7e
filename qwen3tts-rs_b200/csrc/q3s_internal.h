// Internal helpers shared by the C ABI translation units (q3s_capi.cpp owns
// the context and the per-thread error text).  Not installed.
#pragma once

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <mutex>
#include <string>

#include <cuda_runtime.h>

#include "../../include/q3s_sampler.h"

namespace q3s {

struct ContextInfo {
  int device;
  int sm_count;
  size_t smem_optin;
  uint64_t test_wait_ns;  // testing hooks (q3s_context_set_test_hooks); 0: the default
  bool test_hold_refill;
};

ContextInfo context_info(const q3s_context* ctx);

// Records `msg` as the calling thread's q3s_last_error() and returns `code`.
int record_error(int code, const std::string& msg);

// Records a CUDA failure of `what` and returns Q3S_E_CUDA (Q3S_E_OUT_OF_MEMORY
// for an allocation failure).
int record_cuda_error(cudaError_t e, const char* what);

// A device workspace of at least `need` bytes that belongs to the context and
// the stream: launches on one stream are ordered, so they share it.  Those of one
// call must follow one another, whatever thread launches on the stream too: `busy`
// is locked for that and has to stay so until the call's last launch.  It
// grows on demand.  Calls that are captured get a workspace of their own, which no
// other call is given while the graph or anything instantiated from it exists: a
// replay may run beside direct calls and other graphs.  Its contents are undefined.
int stream_scratch(q3s_context* ctx, void* stream, size_t need, unsigned char** scratch,
                   std::unique_lock<std::mutex>* busy);

// Makes `device` current for the scope and restores the caller's device.
struct DeviceScope {
  int prev = -1, device;
  cudaError_t err;
  explicit DeviceScope(int d) : device(d) {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
  }
  ~DeviceScope() {
    if (err == cudaSuccess && prev != device) cudaSetDevice(prev);
  }
};

// Lets a kernel have `bytes` of dynamic shared memory; once per device and
// call site (`done`, a static there).
inline cudaError_t allow_smem(const void* kernel, int bytes, int device,
                              std::atomic<uint64_t>& done) {
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// A C entry's body: a C++ exception (an allocation that failed) must not
// cross the C boundary.
template <class Body>
int no_throw(Body&& body) {
  try {
    return body();
  } catch (...) {
    return Q3S_E_OUT_OF_MEMORY;
  }
}

}  // namespace q3s
