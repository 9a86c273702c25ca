// Attention over the 8-bit paged cache: arguments and helpers that its kernels
// share, and what the handle keeps for them.
#pragma once

#include <cuda_fp16.h>

#include "kv8.cuh"

namespace specdec {

struct AttendArgs {
  Kv8Geom g;
  Kv8Layer c;
  Kv8Batch b;
  const void *q;
  long long q_row, q_head;  // strides in elements
  void *out;
  long long o_row, o_head;
  float *lse;
  float scale;
  int window;
  float *part;
  int *ticket;
  int p_shift, t_shift;  // log2 of page and block positions
  int g_shift;           // log2 of the query heads of a kv head, -1 where that is no power of two
  int q_vec, o_vec;      // query / output rows start at 4-element boundaries
  int q_vec8, o_vec8;    // ... at 8-element boundaries
  int *err;              // set to 1 by a bounded wait that gave up
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNone = -1e30f;                  // the running maximum before anything was seen
constexpr float kLazy = 8.f;                     // weights may grow by 2^8 before the maximum is moved
// The running maximum is held this many binades below the largest weight x value scale, so that those products are f16
// values of 2^6 and up to 2^15 (65,504 is the last): f16 has no step below 2^-24, and from 1 upwards all weights under
// 2^-25 of the largest would be lost, which over a long tail adds up (131,071 positions, one 17 nats above the others, by
// arithmetic: 4e-4 of the largest value; 9e-6 with the room).
constexpr float kRoom = 6.f;
// What fp32 rows add to such an f16 value, w - f16(w), enters 2^12 times larger against codes 2^-12 as large (both exact):
// 22 bits of every weight down to 2^-25, steps of 2^-36 below (2e-9 of the largest value in the case above).
constexpr float kLowUp = 4096.f;
constexpr int kScaleFloor = -84;                 // exponents of value scales count from here: 2^(kLazy + kRoom + 84) stays
                                                 // far enough below 2^127 for sums of weights

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bytes 0x64 u as f16 are 1024 + u; u = code + 128, so minus 1152 leaves the code, exactly.
__device__ __forceinline__ uint32_t f16_codes(uint32_t biased) {
  __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&biased), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t scale_f16(uint32_t pair, float by) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&pair), __float2half2_rn(by));
  return *reinterpret_cast<const uint32_t *>(&h);
}
// Row r of a kv head's rows of a request: new token r / G, query head r % G.
struct RowAt {
  int i, h;
};
__device__ __forceinline__ RowAt row_at(const AttendArgs &a, int r) {
  if (a.g_shift >= 0) return {r >> a.g_shift, r & (a.g.G - 1)};
  const int i = r / a.g.G;
  return {i, r - i * a.g.G};
}

// A value that is the same in the whole warp, as the compiler can see it.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// a / b where both mostly fit 32 bits.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The batch in shared memory: per request its rows, its length and the units before it.
struct DecBatch {
  long long *pre;  // [B + 1]
  int *q0, *q, *len;
};

__device__ __forceinline__ void store4(float *p, bool vec, float4 v) {
  if (vec) {
    *reinterpret_cast<float4 *>(p) = v;
  } else {
    p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, bool vec, float4 v) {
  if (vec) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
  } else {
    p[0] = from_f32<__nv_bfloat16>(v.x);
    p[1] = from_f32<__nv_bfloat16>(v.y);
    p[2] = from_f32<__nv_bfloat16>(v.z);
    p[3] = from_f32<__nv_bfloat16>(v.w);
  }
}

// Four adjacent values of a row as loaded (vec: at a 4-element boundary), zeros unless live.
template <typename XT>
struct Quad;
template <>
struct Quad<float> {
  float x[4];
  __device__ __forceinline__ void load(const float *p, bool vec, bool live) {
    if (vec) {
      const float4 v = live ? *reinterpret_cast<const float4 *>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live ? p[j] : 0.f;
    }
  }
  __device__ __forceinline__ float get(int j) const { return x[j]; }
};
template <>
struct Quad<__nv_bfloat16> {
  uint2 x;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p, bool vec, bool live) {
    if (vec) {
      x = live ? *reinterpret_cast<const uint2 *>(p) : make_uint2(0, 0);
    } else {
      const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
      x = live ? make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16) : make_uint2(0, 0);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = j < 2 ? x.x : x.y;
    return __uint_as_float((j & 1) ? w & 0xffff0000u : w << 16);
  }
};

// Workspaces and kernel attributes of a handle's attention (its device current).
void kv8_attn_create(specdec_kv8 *h);
void kv8_attn_destroy(specdec_kv8 *h);

// Row tiles of 256 rows on tcgen05 (kv8_chunk.cu): bf16 rows, head_dim 64 or 128, batches of at most
// kChunkMaxBatch requests.
constexpr int kChunkMaxBatch = 1024;
void kv8_chunk_create(specdec_kv8 *h);
size_t kv8_chunk_part_bytes(const specdec_kv8 *h);
void kv8_chunk_launch(const specdec_kv8 *h, const AttendArgs &a, cudaStream_t st);

// Checked views of the caller's records (throw OpError).
Kv8Layer kv8_layer(const specdec_kv8 *h, const specdec_kv8_layer *l);
Kv8Batch kv8_batch(const specdec_kv8 *h, const specdec_kv8_batch *b, int n_tokens);

}  // namespace specdec
