// Statuses of the C entry points outside the engine: what a failed call
// throws inside the library, the message that specdec_last_error(NULL)
// returns, and the launch helper that reports its own launch's error.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <exception>
#include <new>
#include <string>

#include "specdec.h"

namespace specdec {

// The calling thread's message of the last failed call that has no handle.
extern thread_local std::string g_thread_err;

struct OpError {
  int code;
  std::string msg;
};

[[noreturn]] inline void op_fail(int code, const std::string &msg) { throw OpError{code, msg}; }
inline void op_check(bool ok, const char *msg) {
  if (!ok) op_fail(SPECDEC_ERR_INVALID, msg);
}
inline void op_cuda(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return;
  cudaGetLastError();  // a failed call's error stays with this call
  op_fail(e == cudaErrorMemoryAllocation ? SPECDEC_ERR_OOM : SPECDEC_ERR_CUDA,
          std::string(what) + ": " + cudaGetErrorString(e));
}

// Runs `body` and turns what it throws into a status and a message: no C++
// exception leaves a C entry point.
template <typename F>
int op_guard(std::string &err, F &&body) {
  try {
    body();
    return SPECDEC_OK;
  } catch (const OpError &e) {
    try {
      err = e.msg;
    } catch (...) {
    }
    return e.code;
  } catch (const std::bad_alloc &) {
    return SPECDEC_ERR_OOM;
  } catch (...) {
    return SPECDEC_ERR_CUDA;
  }
}

// The device a call works on, made current for the call and put back after it.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    op_cuda(cudaGetDevice(&prev_), "cudaGetDevice");
    if (prev_ != device) {
      op_cuda(cudaSetDevice(device), "cudaSetDevice");
      changed_ = true;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;

 private:
  int prev_ = 0;
  bool changed_ = false;
};

// Launches `fn` over `grid` blocks (clusters of `cluster` along x when it is
// above 1) on `stream`.
template <typename... P, typename... A>
void op_launch(const char *what, void (*fn)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
               int cluster, A &&...args) {
  cudaLaunchConfig_t lc{};
  lc.gridDim = grid;
  lc.blockDim = dim3(threads);
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute at[1];
  if (cluster > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
  }
  op_cuda(cudaLaunchKernelEx(&lc, fn, P(args)...), what);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace specdec
