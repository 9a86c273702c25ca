// The 8-bit paged cache with a scale per block of tokens and kv head
// (specdec_kv8): geometry, the buffers of a layer and of a batch as the
// kernels take them, and the per-request prefix sums that the kernels share.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "common.cuh"
#include "status.cuh"

namespace specdec {

constexpr int kKv8MaxBatch = 4096;  // requests of a batch: their prefix sums fit in shared memory

// P positions a page, t positions a scale, codes [page][Hkv][P][D], scales [page][Hkv][P / t].
struct Kv8Geom {
  int H, Hkv, G, D, P, t;
};

struct Kv8Layer {
  int8_t *k, *v;
  float *ks, *vs;
  int n_pages;
};

struct Kv8Batch {
  int32_t *table;  // [B][cols]
  int B, cols;
  int32_t *kv_len, *cu_q;
  int T;  // rows of the call's row arrays
};

// Exclusive prefix sums of units(b), b < B, into pre[0 .. B] by the whole
// block; red holds one value per warp.  Every thread owns a run of
// consecutive requests, so the sums come out in request order.
template <typename T, typename F>
__device__ __forceinline__ void request_prefix(int B, T *pre, T *red, F &&units) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int per = (B + blockDim.x - 1) / blockDim.x;
  const int b0 = min(B, static_cast<int>(threadIdx.x) * per), b1 = min(B, b0 + per);
  T sum = 0;
  for (int b = b0; b < b1; ++b) {
    const T n = units(b);
    pre[b] = n;
    sum += n;
  }
  T inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) red[wid] = inc;
  __syncthreads();
  T run = inc - sum;
  for (int w = 0; w < wid; ++w) run += red[w];
  for (int b = b0; b < b1; ++b) {
    const T n = pre[b];
    pre[b] = run;
    run += n;
  }
  if (threadIdx.x == 0) {
    T total = 0;
    for (int w = 0; w < nw; ++w) total += red[w];
    pre[B] = total;
  }
  __syncthreads();
}

// The request whose run [pre[b], pre[b + 1]) holds unit u.
template <typename T>
__device__ __forceinline__ int request_of(const T *pre, int B, T u) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The rows [q0, q0 + q) of request b in the call's row arrays and its cached
// length, held inside the arrays whatever the batch's own arrays say.
struct Kv8Req {
  int q0, q, len;
};
__device__ __forceinline__ Kv8Req kv8_req(const Kv8Batch &a, int P, int b) {
  Kv8Req r;
  const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1];
  r.q0 = max(0, min(c0, a.T));
  r.q = max(r.q0, min(c1, a.T)) - r.q0;
  const long long cap = static_cast<long long>(a.cols) * P;
  r.len = static_cast<int>(max(0ll, min(static_cast<long long>(a.kv_len[b]), min(cap, 0x7fffff00ll))));
  return r;
}

}  // namespace specdec

struct specdec_kv8 {
  specdec_kv8_config cfg{};
  specdec::Kv8Geom g{};
  int device = 0;
  int num_sms = 0;
  std::string err;
  float *part = nullptr;  // attention: partial results of split items
  int *ticket = nullptr;  // attention: arrivals per split item, 0 between launches
  int *err_word = nullptr;  // attention: set by a bounded wait that gave up (part of ticket's allocation)
};
