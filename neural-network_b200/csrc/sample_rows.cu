// Sampling of logit rows with per-row temperature, top-k, top-p and min-p
// from given uniforms (specdec_sample).
//
// The distribution is held in whole numbers, so that no sum depends on the
// order of its terms: z = l / T, e = exp(z - max z) (1 at the maximum),
// w = floor(2^31 e) < 2^32, sums in 64 bits.  A token below 2^-31 of the
// likeliest one has weight 0; the uniforms have 24 bits, so it could hardly be
// drawn.  A cut (top-k by count, top-p by mass) is a pair (key, ties): tokens
// with a larger z, and the first `ties` tokens in index order with that z.
#include <math.h>

#include "common.cuh"
#include "status.cuh"

namespace specdec {

namespace {

constexpr int kSampleThreads = 1024;

struct SampleArgs {
  const void *logits;
  long long row_stride;
  int rows, V;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p, *u;
  int32_t *tokens;
  float *probs;
};

using u64 = unsigned long long;

// Order-preserving key of a float: a < b as numbers exactly when key(a) < key(b)
// (-0 and +0 are brought together by adding +0).
__device__ __forceinline__ uint32_t float_key(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// floor(f * total / 2^24), f <= 2^24, without a product over 64 bits.
__device__ __forceinline__ u64 part_of(u64 f, u64 total) { return f * (total >> 24) + ((f * (total & 0xffffffu)) >> 24); }

__device__ __forceinline__ float weight_e(float z, float zmax) { return z == zmax ? 1.f : expf(__fsub_rn(z, zmax)); }
__device__ __forceinline__ uint32_t weight_w(float e) { return static_cast<uint32_t>(e * 2147483648.f); }

// Exclusive prefix of v over the block; *total gets the sum.
__device__ __forceinline__ u64 block_scan(u64 v, u64 *red, u64 *total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) red[wid] = inc;
  __syncthreads();
  u64 run = inc - v, all = 0;
  for (int w = 0; w < kSampleThreads / 32; ++w) {
    if (w < wid) run += red[w];
    all += red[w];
  }
  *total = all;
  return run;
}

template <typename XT>
__global__ void __launch_bounds__(kSampleThreads) sample_rows_kernel(const SampleArgs a) {
  __shared__ float redf[32];
  __shared__ int redi[32];
  __shared__ u64 red[32];
  __shared__ u64 hist[256];
  __shared__ uint32_t s_key;
  __shared__ u64 s_left;
  const int b = blockIdx.x, V = a.V;
  const XT *x = static_cast<const XT *>(a.logits) + b * a.row_stride;
  const float T = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(T > 0.f);
  auto zat = [&](int i) {
    const float l = to_f32(x[i]);
    return isnan(l) ? -INFINITY : greedy ? l : __fdiv_rn(l, T);
  };
  ArgMax am{-INFINITY, 0x7fffffff};
  for (int i = threadIdx.x; i < V; i += kSampleThreads) am = argmax_merge(am, {zat(i), i});
  am = block_argmax(am, redf, redi);
  const float zmax = am.v;
  if (zmax == -INFINITY || greedy) {
    if (threadIdx.x == 0) {
      a.tokens[b] = zmax == -INFINITY ? -1 : am.i;
      if (a.probs) a.probs[b] = zmax == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  const int k = a.top_k ? a.top_k[b] : 0;
  const float top_p = a.top_p ? a.top_p[b] : 1.f;
  const float min_e = a.min_p ? fminf(a.min_p[b], 1.f) : 0.f;
  // the cut so far: every token
  uint32_t cut = 0;
  int ties = V;
  // Finds the key at which the running sum of f over descending keys of the
  // kept tokens reaches `want` (the sum over larger keys is below it), 8 bits
  // a pass; `left` = want minus the sum over larger keys.
  auto select = [&](u64 want, auto &&f) {
    uint32_t key = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSampleThreads) hist[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < V; i += kSampleThreads) {
        const float z = zat(i);
        const uint32_t kk = float_key(z);
        if (shift == 24 || (kk >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(kk >> shift) & 255], f(z, kk));
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        u64 run = 0;
        int bin = 255;
        for (; bin > 0; --bin) {
          if (run + hist[bin] >= want) break;
          run += hist[bin];
        }
        s_key = key | static_cast<uint32_t>(bin) << shift;
        s_left = want - run;
      }
      __syncthreads();
      key = s_key;
      want = s_left;
      __syncthreads();
    }
    return key;
  };
  if (k > 0 && k < V) {
    cut = select(k, [&](float, uint32_t) { return u64(1); });
    ties = static_cast<int>(s_left);
  }
  auto sum_kept = [&]() {
    u64 s = 0, total;
    for (int i = threadIdx.x; i < V; i += kSampleThreads) {
      const float z = zat(i);
      if (float_key(z) > cut) s += weight_w(weight_e(z, zmax));
    }
    block_scan(s, red, &total);
    return total;
  };
  if (top_p < 1.f) {
    const u64 cw = weight_w(weight_e(key_float(cut), zmax));
    u64 mass = sum_kept();
    if (cut == 0) ties = 0;  // no token has key 0
    mass += static_cast<u64>(ties) * cw;
    const u64 p24 = static_cast<u64>(rintf(fmaxf(top_p, 0.f) * 16777216.f));
    u64 most = part_of(p24, mass);
    if (most < 1) most = 1;
    // the mass over larger keys reaches `most`: inside the top-k set
    const uint32_t kc = cut;
    const int kt = ties;
    const uint32_t pc = select(most, [&](float z, uint32_t kk) {
      return kk >= kc ? static_cast<u64>(weight_w(weight_e(z, zmax))) : 0ull;
    });
    const u64 w = weight_w(weight_e(key_float(pc), zmax));
    const u64 n = w ? (s_left + w - 1) / w : 0;
    ties = static_cast<int>(min(n, static_cast<u64>(pc == kc ? kt : V)));
    cut = pc;
  }
  // running sums in index order, one run of tokens a thread
  const int per = (V + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(V, static_cast<int>(threadIdx.x) * per), i1 = min(V, i0 + per);
  u64 nt = 0, total;
  for (int i = i0; i < i1; ++i) nt += float_key(zat(i)) == cut;
  const u64 t0 = block_scan(nt, red, &total);
  auto run_over = [&](u64 sum, auto &&at) {
    u64 tie = t0;
    for (int i = i0; i < i1; ++i) {
      const float z = zat(i);
      const uint32_t kk = float_key(z);
      bool keep = kk > cut;
      if (kk == cut) keep = tie++ < static_cast<u64>(ties);
      const float e = weight_e(z, zmax);
      if (!keep || !(e >= min_e)) continue;
      const u64 w = weight_w(e);
      if (at(i, sum, w)) return sum;
      sum += w;
    }
    return sum;
  };
  const u64 mine = run_over(0, [](int, u64, u64) { return false; });
  const u64 before = block_scan(mine, red, &total);
  const float uu = a.u[b];
  const u64 u24 = static_cast<u64>(fminf(fmaxf(uu * 16777216.f, 0.f), 16777215.f));
  const u64 target = part_of(u24, total);
  if (target >= before && target < before + mine)
    run_over(before, [&](int i, u64 sum, u64 w) {
      if (target >= sum + w) return false;
      a.tokens[b] = i;
      if (a.probs) a.probs[b] = __fdiv_rn(static_cast<float>(w), static_cast<float>(total));
      return true;
    });
}

}  // namespace

}  // namespace specdec

using namespace specdec;

extern "C" int specdec_sample(const void *logits, int dtype, int rows, int vocab, int64_t row_stride,
                              const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                              const float *u, int32_t *tokens, float *probs, void *stream) {
  return op_guard(g_thread_err, [&] {
    op_check(dtype == SPECDEC_F32 || dtype == SPECDEC_BF16, "logits must be SPECDEC_F32 or SPECDEC_BF16");
    op_check(rows >= 0 && vocab > 0 && vocab <= (1 << 20), "rows must not be negative, vocab in [1, 2^20]");
    op_check(row_stride >= vocab || rows <= 1, "row_stride must be at least vocab");
    if (rows == 0) return;
    op_check(logits && u && tokens, "null sampling buffer");
    const SampleArgs a{logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, u, tokens, probs};
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == SPECDEC_F32)
      op_launch("specdec_sample", sample_rows_kernel<float>, dim3(rows), kSampleThreads, 0, st, 1, a);
    else
      op_launch("specdec_sample", sample_rows_kernel<__nv_bfloat16>, dim3(rows), kSampleThreads, 0, st, 1, a);
  });
}
