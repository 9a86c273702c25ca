// Sampling of logit rows with per-row temperature, top-k, top-p and min-p
// from given uniforms (specdec_sample).
//
// The distribution is held in whole numbers, so that no sum depends on the
// order of its terms: z = l / T, e = exp(z - max z) (1 at the maximum),
// w = floor(2^31 e) < 2^32, sums in 64 bits.  A token below 2^-31 of the
// likeliest one has weight 0; the uniforms have 24 bits, so it could hardly be
// drawn.  A cut (top-k by count, top-p by mass) is a pair (key, ties): tokens
// with a larger z, and the first `ties` tokens in index order with that z.
//
// HBM would let 256 rows of 128,259 bf16 logits (66 MB) take 10 us; latency and
// issue slots bound it.  Measured, rows with a mix of all filters: that batch
// 175 to 191 us, 160 rows of 32,000 fp32 47 to 52 us, a single one 8 to 27 us.  A
// cut among more than 1,024 equal weights goes to one block and global memory:
// rows of 52,000 with 30,000 equal logits take 1.9 to 4.2 ms.  Alone in the
// large batch: arg max 54 us, top-k 50 121, no filter 119, top-p 0.9 246 (435
// on flat rows).  A pass over the tokens that takes the exponential costs 60 us
// there (about 50 instructions a token with the division by the temperature).
// A block per row that reads it again from L2 in every pass takes 58 us for
// top-k but 352 for top-p, and 324 for the mix: its exponentials cannot stay in
// shared memory, and the slowest row decides.  Bins that hold exact 64-bit sums
// need no estimate of their edges but two additions a token: 200 us for the mix.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "status.cuh"

namespace specdec {

namespace {

constexpr int kThreads = 512;        // of a block; a cluster of blocks takes a row
constexpr int kSlice = 16384;        // tokens of a block where the row count gives enough blocks: two blocks' fit an SM
                                     // (160 rows of 32,000: 49 us with 8,192, 51 so, 62 with 32,768; 512 rows: 129, 103)
constexpr int kMaxSlice = 40960;     // tokens that a block's shared memory holds
constexpr int kMaxCluster = 8;
constexpr int kBins = 128;
constexpr int kCap = 1024;           // tokens that are sorted to settle a cut exactly
constexpr float kFar = 22.2f;        // nats below the maximum from which the weight is 0: 2^31 exp(-22.2) < 1
constexpr int kLevels = 4;           // of finer bins for a top-k cut
constexpr int kNarrow = 8;           // of finer bins for a top-p cut: 2^28 bit patterns at most, down by 64 or so each time
constexpr int kFewHighs = kThreads / 2;  // k a block up to which the threads' maxima bound the k-th token well

struct SampleArgs {
  const void *logits;
  long long row_stride;
  int rows, V;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p, *u;
  int32_t *tokens;
  float *probs;
  int slice;  // tokens of a block (a multiple of 8)
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

// A logit's z: NaN counts as -infinity.
struct Scale {
  float T, inv;  // temperature and its reciprocal (the latter for estimates only)
  __device__ __forceinline__ float z(float l) const { return T == 1.f ? l : __fdiv_rn(l, T); }
};
__device__ __forceinline__ float no_nan(float l) { return fmaxf(l, -INFINITY); }

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, v, o);
    if (static_cast<int>(threadIdx.x & 31) >= o) v += n;
  }
  return v;
}
// Sum over the block, in every thread; red holds a value per warp.
__device__ __forceinline__ u64 block_sum_u64(u64 v, u64 *red) {
  v = warp_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 all = 0;
  for (int w = 0; w < kThreads / 32; ++w) all += red[w];
  return all;
}
// Exclusive prefix over the block; *total gets the sum.
__device__ __forceinline__ u64 block_scan_u64(u64 v, u64 *red, u64 *total) {
  const u64 inc = warp_scan_u64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 31) red[threadIdx.x >> 5] = inc;
  __syncthreads();
  u64 run = inc - v, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) run += red[w];
    all += red[w];
  }
  *total = all;
  return run;
}

// Radix selection, 8 bits a pass, by the whole block.  each(f) calls
// f(value, weight) for every entry; returns the value v at which the sum of
// weights over descending values first reaches `want` (at least 1), and in
// *left want minus the sum over values above v, in *at the weight at v.
template <typename Each>
__device__ uint32_t radix_select(u64 want, Each &&each, u64 *hist, u64 *out, u64 *left, u64 *at) {
  uint32_t value = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    each([&](uint32_t v, u64 w) {
      if (shift == 24 || (v >> (shift + 8)) == (value >> (shift + 8))) atomicAdd(&hist[(v >> shift) & 255], w);
    });
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l holds bins 255 - 8 l .. 248 - 8 l, in descending order
      const int lane = threadIdx.x;
      u64 mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += hist[255 - 8 * lane - i];
      const u64 inc = warp_scan_u64(mine);
      const uint32_t reach = __ballot_sync(0xffffffffu, inc >= want);
      const int who = reach ? __ffs(reach) - 1 : 31;
      if (lane == who) {
        u64 run = inc - mine;
        int bin = 255 - 8 * lane;
        for (int i = 0; i < 7 && run + hist[bin] < want; ++i) run += hist[bin--];
        out[0] = bin;
        out[1] = want - run;
        out[2] = hist[bin];
      }
    }
    __syncthreads();
    value |= static_cast<uint32_t>(out[0]) << shift;
    want = out[1];
  }
  *left = want;
  *at = out[2];
  __syncthreads();
  return value;
}

// Sorts the n <= 2 kThreads distinct values of v in descending order, by the
// whole block; spare holds as many.  Few values find their places by counting
// the larger ones (two threads a value), more go through a bitonic network.
__device__ void sort_down(u64 *v, u64 *spare, int n) {
  if (n <= kThreads / 2) {
    const int i = threadIdx.x >> 1;
    const u64 mine = i < n ? v[i] : 0;
    int larger = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 1; j < n; j += 2) larger += v[j] > mine;
    larger += __shfl_xor_sync(0xffffffffu, larger, 1);
    if (i < n && (threadIdx.x & 1) == 0) spare[larger] = mine;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n) v[threadIdx.x] = spare[threadIdx.x];
    __syncthreads();
    return;
  }
  int size = kThreads;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += kThreads) v[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int p = threadIdx.x; p < size / 2; p += kThreads) {
        const int i = 2 * p - (p & (j - 1)), o = i + j;  // the pair (i, i + j)
        const u64 x = v[i], y = v[o];
        if ((x < y) == ((i & k) == 0)) {
          v[i] = y;
          v[o] = x;
        }
      }
      __syncthreads();
    }
}

// The tokens that a filter keeps: those with a larger key, and those with this
// key up to index idx.  Values (logits, or bits of e) above hi have a larger
// key for sure, those below lo a smaller one; between them the key decides.
template <typename T>
struct Cut {
  uint32_t key;
  int idx;
  T lo, hi;
};
__device__ __forceinline__ bool keeps(uint32_t key, int idx, const Scale &sc, float l, int i) {
  const uint32_t k = float_key(sc.z(l));
  return k > key || (k == key && i <= idx);
}

// The whole row by one block, straight from global memory: for rows whose cut
// the estimates below cannot settle (over kCap equal logits at the cut, scaled
// logits outside the normal range) and for vocabularies that do not fit the
// cluster's shared memory.
template <typename XT>
__device__ void sample_whole_row(const SampleArgs &a, int b, u64 *hist, u64 *red, u64 *out) {
  const XT *x = static_cast<const XT *>(a.logits) + b * a.row_stride;
  const float T = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(T > 0.f);
  const int V = a.V;
  auto zat = [&](int i) {
    const float l = no_nan(to_f32(x[i]));
    const float z = greedy ? l : __fdiv_rn(l, T);
    return isnan(z) ? l : z;  // an infinite logit stays one at an infinite T
  };
  __shared__ float redf[32];
  __shared__ int redi[32];
  ArgMax am{-INFINITY, 0x7fffffff};
  for (int i = threadIdx.x; i < V; i += kThreads) am = argmax_merge(am, {zat(i), i});
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
  uint32_t cut = 0;  // no key is 0
  u64 ties = 0, left, at;
  if (k > 0 && k < V) {
    cut = radix_select(k, [&](auto &&f) { for (int i = threadIdx.x; i < V; i += kThreads) f(float_key(zat(i)), u64(1)); },
                       hist, out, &left, &at);
    ties = left;
  }
  if (top_p < 1.f) {
    u64 mass = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float z = zat(i);
      if (float_key(z) > cut) mass += weight_w(weight_e(z, zmax));
    }
    mass = block_sum_u64(mass, red) + ties * (cut ? weight_w(weight_e(key_float(cut), zmax)) : 0);
    u64 most = part_of(static_cast<u64>(rintf(fmaxf(top_p, 0.f) * 16777216.f)), mass);
    if (most < 1) most = 1;
    const uint32_t kc = cut;
    const u64 kt = ties;
    cut = radix_select(most, [&](auto &&f) {
      for (int i = threadIdx.x; i < V; i += kThreads) {
        const float z = zat(i);
        const uint32_t kk = float_key(z);
        if (kk >= kc) f(kk, static_cast<u64>(weight_w(weight_e(z, zmax))));
      }
    }, hist, out, &left, &at);
    const u64 w = weight_w(weight_e(key_float(cut), zmax));
    ties = w ? (left + w - 1) / w : 0;
    if (cut == kc) ties = min(ties, kt);
  }
  // running sums in index order, one run of tokens a thread
  const int per = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, static_cast<int>(threadIdx.x) * per), i1 = min(V, i0 + per);
  u64 nt = 0, total;
  for (int i = i0; i < i1; ++i) nt += float_key(zat(i)) == cut;
  const u64 t0 = block_scan_u64(nt, red, &total);
  auto run_over = [&](u64 sum, auto &&stop) {
    u64 tie = t0;
    for (int i = i0; i < i1; ++i) {
      const float z = zat(i);
      const uint32_t kk = float_key(z);
      if (!(kk > cut || (kk == cut && tie++ < ties))) continue;
      const float e = weight_e(z, zmax);
      if (!(e >= min_e)) continue;
      const u64 w = weight_w(e);
      if (stop(i, sum, w)) return sum;
      sum += w;
    }
    return sum;
  };
  const u64 mine = run_over(0, [](int, u64, u64) { return false; });
  const u64 before = block_scan_u64(mine, red, &total);
  const u64 u24 = static_cast<u64>(fminf(fmaxf(a.u[b] * 16777216.f, 0.f), 16777215.f));
  const u64 target = part_of(u24, total);
  if (target >= before && target < before + mine)
    run_over(before, [&](int i, u64 sum, u64 w) {
      if (target >= sum + w) return false;
      a.tokens[b] = i;
      if (a.probs) a.probs[b] = __fdiv_rn(static_cast<float>(w), static_cast<float>(total));
      return true;
    });
}

template <typename XT>
__global__ void __launch_bounds__(kThreads) sample_whole_kernel(const SampleArgs a) {
  __shared__ u64 hist[256], red[32], out[3];
  sample_whole_row<XT>(a, blockIdx.x, hist, red, out);
}

// What the blocks of a cluster tell each other: every block writes its own
// entry in every block's copy, then the cluster meets.
struct alignas(16) Shared {
  float high[kMaxCluster];
  int first[kMaxCluster];
  u64 counts[kMaxCluster][kBins];
  u64 mass[kMaxCluster], above[kMaxCluster];
  int n[kMaxCluster], n_top[kMaxCluster];
  float min_above[kMaxCluster], max_below[kMaxCluster];
  // of this block alone
  uint4 part[kThreads / 32];
  u64 hist[256], red[32], out[3];
  float redf[32];
  int redi[32], n_local, n_local_top, band[2], at;
};

// Eight logits from a 16- or 32-byte run.
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// One row per cluster, its logits read once and held in the blocks' shared
// memory.  A cut is found from the outside in: the tokens (for top-k), or their
// weights (for top-p, in 32 bits with a shift), are added up in 128 bins of
// their distance to the maximum, or of the bits of e; each lane of a warp adds
// to a column of its own, so no two lanes meet in a bank or a word.  Where the
// tokens down to the bins that hold the cut are few, they are listed and
// sorted, and every filter and the draw are settled on that list.  Else only
// the bins' tokens are listed, or binned again by finer bins where they are too
// many, the exact cut is taken from their sorted list, and the draw passes over
// the row.  Top-p works on e, which takes the logits' place in shared memory
// (the exponential is taken once a token); e orders tokens as z does but for
// the last bits, and within 8 units of them z decides, read again.  A list of
// logits is checked to hold its cut: what lies outside it is strictly above or
// below.  A row that fails, and one that never narrows, is done by
// sample_whole_row.
template <typename XT>
__global__ void __launch_bounds__(kThreads, 2) sample_cluster_kernel(const SampleArgs a) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // every block says that it has started, and waits for the others before it first writes to one: the loads lie between
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  extern __shared__ __align__(16) unsigned char sample_smem[];
  Shared &sh = *reinterpret_cast<Shared *>(sample_smem);
  uint32_t *columns = reinterpret_cast<uint32_t *>(sample_smem + sizeof(Shared));  // [kBins][32]; also sorting's spare room
  uint2 *list = reinterpret_cast<uint2 *>(columns + kBins * 32);  // [kCap] (logit, index) of this block
  int *list_top = reinterpret_cast<int *>(list), *list_band = list_top + kCap;  // or [kCap] indexes each
  u64 *sorted = reinterpret_cast<u64 *>(list + kCap);             // [kCap] of the cluster
  float *row = reinterpret_cast<float *>(sorted + kCap);          // [slice + 16]
  auto meet = [&]() { cluster.sync(); };
  auto tell = [&](auto *p, auto v) {  // writes *p in every block; called by whole warps with a uniform v
    if (lane < C) *cluster.map_shared_rank(p, lane) = v;
  };

  // ---- the slice, its maximum ------------------------------------------------
  const int V = a.V, i_begin = min(V, rank * a.slice), i_end = min(V, i_begin + a.slice), n = i_end - i_begin;
  const XT *x = static_cast<const XT *>(a.logits) + b * a.row_stride + i_begin;
  // the first `head` tokens come before a 16-byte boundary; token i lies at row[i + 8 - head], so that runs of eight
  // are aligned in shared memory too
  constexpr int kAlign = 16 / sizeof(XT);
  const int head = min(n, static_cast<int>((kAlign - reinterpret_cast<uintptr_t>(x) / sizeof(XT) % kAlign) % kAlign));
  const int off = 8 - head, n4 = (n + off + 3) / 4;  // float4s of the row, its edges filled with -infinity
  const float T = a.temperature ? a.temperature[b] : 1.f;
  const bool greedy = !(T > 0.f);
  float high = -INFINITY, second = -INFINITY;  // of this thread's tokens: the largest of half of them, and of the others
  for (int i = tid; i < off; i += kThreads) row[i] = -INFINITY;
  for (int i = n + off + tid; i < 4 * n4; i += kThreads) row[i] = -INFINITY;
  for (int i = tid; i < head; i += kThreads) {
    const float l = no_nan(to_f32(x[i]));
    row[i + off] = l;
    high = fmaxf(high, l);
  }
  const int runs = (n - head) / 8;
#pragma unroll 4
  for (int i = tid; i < runs; i += kThreads) {
    float v[8];
    load8(x + head + 8 * i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = no_nan(v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      high = fmaxf(high, v[j]);
      second = fmaxf(second, v[j + 4]);
    }
    *reinterpret_cast<float4 *>(row + 8 + 8 * i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(row + 12 + 8 * i) = make_float4(v[4], v[5], v[6], v[7]);
  }
  for (int i = head + 8 * runs + tid; i < n; i += kThreads) {
    const float l = no_nan(to_f32(x[i]));
    row[i + off] = l;
    high = fmaxf(high, l);
  }
  const float my_high[2] = {high, second};
  high = block_max(fmaxf(high, second), sh.redf);
  asm volatile("barrier.cluster.wait;" ::: "memory");
  if (warp == 0) tell(&sh.high[rank], high);
  meet();
  high = -INFINITY;
  for (int r = 0; r < C; ++r) high = fmaxf(high, sh.high[r]);
  // a pass over the slice by whole warps: f(four values, index of the first in the row), `none` where there is no token
  const float4 *row4 = reinterpret_cast<const float4 *>(row);
  auto each4 = [&](float none, auto &&f) {
    for (int q = tid; q - lane < n4; q += kThreads) {
      const float4 x = q < n4 ? row4[q] : make_float4(none, none, none, none);
      const float v[4] = {x.x, x.y, x.z, x.w};
      f(v, i_begin + 4 * q - off);
    }
  };
  // put(place, j) for those of a thread's four tokens j for which `is` holds, places counted up in `count`; by whole warps.
  auto append4 = [&](const bool (&is)[4], int *count, auto &&put) {
    if (!__any_sync(0xffffffffu, is[0] || is[1] || is[2] || is[3])) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t who = __ballot_sync(0xffffffffu, is[j]);
      if (!who) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(count, __popc(who));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
      if (is[j] && at < kCap) put(at, j);
    }
  };
  if (high == -INFINITY || greedy) {
    int first = 0x7fffffff;
    if (greedy && high != -INFINITY)
      each4(-INFINITY, [&](const float (&l)[4], int i) {
        for (int j = 3; j >= 0; --j)
          if (l[j] == high) first = min(first, i + j);
      });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.redi[warp] = first;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kThreads / 32; ++w) first = min(first, sh.redi[w]);
      *cluster.map_shared_rank(&sh.first[rank], 0) = first;
    }
    meet();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < C; ++r) first = min(first, sh.first[r]);
      a.tokens[b] = high == -INFINITY ? -1 : first;
      if (a.probs) a.probs[b] = high == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  const Scale sc{T, 1.f / T};
  const float zmax = sc.z(high);
  const int k = a.top_k ? a.top_k[b] : 0;
  const float top_p = a.top_p ? a.top_p[b] : 1.f;
  const float min_e = a.min_p ? fminf(a.min_p[b], 1.f) : 0.f;
  const bool has_k = k > 0 && k < V, has_p = top_p < 1.f;
  const u64 p24 = static_cast<u64>(rintf(fminf(fmaxf(top_p, 0.f), 1.f) * 16777216.f));
  auto most_of = [&](u64 mass) { return max(part_of(p24, mass), u64(1)); };
  const u64 u24 = static_cast<u64>(fminf(fmaxf(a.u[b] * 16777216.f, 0.f), 16777215.f));
  // temperatures and logits for which equal z means nearly equal logits
  bool slow = !(T >= 9.1e-13f && T <= 1.1e12f && fabsf(high) < 1.2e24f);
  auto far_of = [&](float l) { return (high - l) * sc.inv; };  // the distance to the maximum, falling with l
  const XT *whole = static_cast<const XT *>(a.logits) + b * a.row_stride;
  auto logit = [&](int i) { return no_nan(to_f32(whole[i])); };
  auto w_of = [&](uint32_t bits) { return weight_w(__uint_as_float(bits)); };
  auto key_w = [&](u64 e) { return weight_w(weight_e(key_float(static_cast<uint32_t>(e >> 32)), zmax)); };
  // (key, ~index): descending order is by descending key, then by ascending index
  auto entry = [&](float l, int i) { return static_cast<u64>(float_key(sc.z(l))) << 32 | static_cast<uint32_t>(~i); };
  auto entry_key = [&](u64 e) { return static_cast<uint32_t>(e >> 32); };
  auto entry_index = [&](u64 e) { return static_cast<int>(~static_cast<uint32_t>(e)); };
  u64 *spare = reinterpret_cast<u64 *>(columns);

  // The first place of `sorted` at which the running sum of f reaches want; n where it does not.
  auto reach = [&](int n, u64 want, auto &&f) {
    if (tid == 0) sh.at = n;
    const int i = 2 * tid;
    const u64 w0 = i < n ? f(i) : 0, w1 = i + 1 < n ? f(i + 1) : 0;
    u64 all;
    const u64 before = block_scan_u64(w0 + w1, sh.red, &all);
    if (before < want && want <= before + w0 + w1) sh.at = before + w0 >= want ? i : i + 1;
    __syncthreads();
    const int at = sh.at;
    __syncthreads();
    return at;
  };
  // A weight's shift in a column leaves less than 2^(22 - extra) of it, so that the slice's tokens fit 32 bits.
  const int extra = 32 - __clz((a.slice + 255) >> 15);
  // The columns' sums to every block's counts, `mine` to every block's mass; then the first bin in which the running sum
  // of all blocks' counts may reach want(), and in `must` the first in which it does; scale(bin) is the bin's shift.
  auto settle = [&](u64 mine, u64 base, auto &&want, auto &&scale, int &must) {
    __syncthreads();
#pragma unroll
    for (int j = warp; j < kBins; j += kThreads / 32) {
      const uint32_t c = columns[j * 32 + lane];  // 32 columns of up to 32 bits: the sum in two halves
      const uint32_t low = __reduce_add_sync(0xffffffffu, c & 0xffffu), high16 = __reduce_add_sync(0xffffffffu, c >> 16);
      tell(&sh.counts[rank][j], (static_cast<u64>(high16) << 16) + low);
    }
    mine = block_sum_u64(mine, sh.red);
    if (warp == 0) tell(&sh.mass[rank], mine);
    meet();
    if (warp == 0) {  // lane l: bins 4 l .. 4 l + 3
      const u64 target = want();
      u64 some[4], most[4], sum_some = 0, sum_most = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u64 c = 0;
        for (int r = 0; r < C; ++r) c += sh.counts[r][4 * lane + j];
        const int shift = scale(4 * lane + j);  // it leaves at least 2^(19 - extra) of a weight, so drops less than that part
        sum_some += some[j] = c << shift;
        sum_most += most[j] = some[j] + (shift ? some[j] >> (18 - extra) : 0);
      }
      u64 run_some = base + warp_scan_u64(sum_some) - sum_some, run_most = base + warp_scan_u64(sum_most) - sum_most;
      int first = kBins, sure = kBins;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        run_some += some[j];
        run_most += most[j];
        if (run_most >= target) first = min(first, 4 * lane + j);
        if (run_some >= target) sure = min(sure, 4 * lane + j);
      }
      first = __reduce_min_sync(0xffffffffu, first);
      sure = __reduce_min_sync(0xffffffffu, sure);
      if (lane == 0) {
        sh.band[0] = first;
        sh.band[1] = sure;
      }
    }
    __syncthreads();
    must = sh.band[1];
    return sh.band[0];
  };
  auto clear_columns = [&]() {
    for (int i = tid; i < kBins * 8; i += kThreads) reinterpret_cast<uint4 *>(columns)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  };
  auto no_shift = [](int) { return 0; };
  auto sum_told = [&](const u64 *v) {
    u64 sum = 0;
    for (int r = 0; r < C; ++r) sum += v[r];
    return sum;
  };

  // ---- top-k: bins of the distance to the maximum --------------------------------
  // The k-th largest of the threads' own maxima is no larger than the k-th largest token, and little smaller while k is
  // well below the number of threads: two values a thread in place of a pass over the row.
  // 256 rows of 128,259 bf16 logits: 136 us with that pass, 123 without at k = 20, 179 and 165 at k = 400; 160 rows of
  // 32,000: 31 and 27 us at k = 20, no difference at 400.
  auto count_highs = [&](u64 want, int &must) {
    clear_columns();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float d = far_of(my_high[j]);
      if (d < kFar) atomicAdd(&columns[min(kBins - 1, static_cast<int>(d * (kBins / kFar))) * 32 + lane], 1u);
    }
    return settle(0, 0, [&]() { return want; }, no_shift, must);
  };
  auto count_bins = [&](float lo, float hi, u64 base, u64 want, int &must) {
    const float per = kBins / (hi - lo);
    clear_columns();
    for (int q = tid; q < n4; q += kThreads) {
      const float4 v = row4[q];
      const float d[4] = {far_of(v.x), far_of(v.y), far_of(v.z), far_of(v.w)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (d[j] >= lo && d[j] < hi) atomicAdd(&columns[min(kBins - 1, static_cast<int>((d[j] - lo) * per)) * 32 + lane], 1u);
    }
    return settle(0, base, [&]() { return want; }, no_shift, must);
  };
  // Lists the tokens between lo and hi and counts those above lo, to every block; returns the number listed.
  auto collect = [&](float lo, float hi, u64 &above, float &min_above, float &max_below) {
    if (tid == 0) sh.n_local = 0;
    __syncthreads();
    uint32_t mine = 0;
    min_above = INFINITY;
    max_below = -INFINITY;
    each4(-INFINITY, [&](const float (&l)[4], int i) {
      bool is[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = far_of(l[j]);
        is[j] = d >= lo && d < hi;
        if (d < lo) {
          ++mine;
          min_above = fminf(min_above, l[j]);
        } else if (!is[j]) {
          max_below = fmaxf(max_below, l[j]);
        }
      }
      append4(is, &sh.n_local, [&](int at, int j) { list[at] = make_uint2(__float_as_uint(l[j]), i + j); });
    });
    __syncthreads();
    {  // the block's three results at once: the floats as keys, which integers compare
      const uint32_t n_warp = __reduce_add_sync(0xffffffffu, mine), low_key = __reduce_min_sync(0xffffffffu, float_key(min_above)),
                     high_key = __reduce_max_sync(0xffffffffu, float_key(max_below));
      if (lane == 0) sh.part[warp] = make_uint4(n_warp, low_key, high_key, 0);
      __syncthreads();
      if (warp == 0) {
        const uint4 p = sh.part[lane & (kThreads / 32 - 1)];
        const uint32_t n_all = __reduce_add_sync(0xffffffffu, lane < kThreads / 32 ? p.x : 0u);
        const float lowest = key_float(__reduce_min_sync(0xffffffffu, p.y)), highest = key_float(__reduce_max_sync(0xffffffffu, p.z));
        tell(&sh.above[rank], static_cast<u64>(n_all));
        tell(&sh.n[rank], sh.n_local);
        tell(&sh.min_above[rank], lowest);
        tell(&sh.max_below[rank], highest);
      }
    }
    meet();
    above = sum_told(sh.above);
    int n_all = 0;
    for (int r = 0; r < C; ++r) {
      n_all += sh.n[r];
      min_above = fminf(min_above, sh.min_above[r]);
      max_below = fmaxf(max_below, sh.max_below[r]);
    }
    return n_all;
  };
  // Place p of the blocks' lists of n[r] entries one after the other: the block, p becoming the place in its list.
  auto block_of = [&](const int *n, int &p) {
    int r = 0;
    while (p >= n[r]) p -= n[r++];
    return r;
  };
  auto merge = [&](int n_all) {  // all blocks' listed tokens
    for (int i = tid; i < n_all; i += kThreads) {
      int p = i;
      const int r = block_of(sh.n, p);
      const uint2 e = cluster.map_shared_rank(list, r)[p];
      sorted[i] = entry(__uint_as_float(e.x), static_cast<int>(e.y));
    }
    __syncthreads();
  };
  // This block's listed tokens to their place in block 0's `sorted`; the other blocks are done then, and make room.
  auto put_in_first = [&](u64 e, int at) { *cluster.map_shared_rank(sorted + at, 0) = e; };
  auto hand_over = [&]() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (rank == 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  };
  auto send_lists = [&]() {
    int at = 0;
    for (int r = 0; r < rank; ++r) at += sh.n[r];
    for (int i = tid; i < sh.n[rank]; i += kThreads)
      put_in_first(entry(__uint_as_float(list[i].x), static_cast<int>(list[i].y)), at + i);
    hand_over();
  };
  auto outside = [&](u64 e, float min_above, float max_below) {  // whether these lie strictly above and below the entry
    const uint32_t key = entry_key(e);
    return (min_above == INFINITY || float_key(sc.z(min_above)) > key) && (max_below == -INFINITY || float_key(sc.z(max_below)) < key);
  };

  // ---- the kept tokens of a sorted list: min-p, then the draw (by one block) --------
  auto draw_from = [&](int n) {
    const int i = 2 * tid;
    u64 e[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      e[j] = 0;
      if (i + j < n) {
        const float w_e = weight_e(key_float(entry_key(sorted[i + j])), zmax);
        e[j] = sorted[i + j] << 32 | (w_e >= min_e ? weight_w(w_e) : 0u);  // (~index, weight)
      }
    }
    const u64 total = block_sum_u64((e[0] & 0xffffffffu) + (e[1] & 0xffffffffu), sh.red);
    const u64 target = part_of(u24, total);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (i + j < n) sorted[i + j] = e[j];
    __syncthreads();
    auto write = [&](u64 x) {
      a.tokens[b] = static_cast<int>(~static_cast<uint32_t>(x >> 32));
      if (a.probs) a.probs[b] = __fdiv_rn(static_cast<float>(x & 0xffffffffu), static_cast<float>(total));
    };
    if (n <= kThreads / 2) {  // two threads a token add up the weights before it
      const u64 mine = (tid >> 1) < n ? sorted[tid >> 1] : 0;
      u64 before = 0;
#pragma unroll 4
      for (int j = tid & 1; j < n; j += 2) {
        const u64 x = sorted[j];
        before += x > mine ? x & 0xffffffffu : 0;  // a larger ~index: a smaller index
      }
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      if ((tid >> 1) < n && (tid & 1) == 0 && before <= target && target < before + (mine & 0xffffffffu)) write(mine);
      return;
    }
    sort_down(sorted, spare, n);
    const int at = reach(n, target + 1, [&](int j) { return sorted[j] & 0xffffffffu; });
    if (tid == 0) write(sorted[at]);
  };

  Cut<float> top{0, -1, -INFINITY, -INFINITY};  // top-k's cut, over logits
  if (!slow && has_k) {
    int b1, b0 = kBins;
    const bool few = k <= min(kFewHighs * C, kCap / 2);
    if (few) b0 = count_highs(k, b1);
    bool by_highs = b0 < kBins;
    if (!by_highs) {
      if (few) meet();  // what the blocks told each other has been read
      b0 = count_bins(0.f, kFar, 0, k, b1);
    }
    bool all = b0 >= kBins;  // fewer than k tokens have a weight above 0: all of them are kept
    float lo = 0.f, hi = all ? kFar : (b0 + 1.02f) * (kFar / kBins), min_above, max_below;
    u64 above;
    int n_all = collect(lo, hi, above, min_above, max_below);
    if (n_all > kCap && by_highs) {
      meet();
      b0 = count_bins(0.f, kFar, 0, k, b1);
      hi = (b0 + 1.02f) * (kFar / kBins);
      n_all = collect(lo, hi, above, min_above, max_below);
    }
    if (n_all <= kCap) {
      send_lists();
      if (rank != 0) return;
      sort_down(sorted, spare, n_all);
      int n = all ? n_all : k;
      const bool bad = !all && (n > n_all || !outside(sorted[min(n, n_all) - 1], INFINITY, max_below));
      if (!bad && has_p) {
        const int i = 2 * tid;
        const u64 mass = block_sum_u64((i < n ? key_w(sorted[i]) : 0u) + static_cast<u64>(i + 1 < n ? key_w(sorted[i + 1]) : 0u), sh.red);
        n = reach(n, most_of(mass), [&](int j) { return static_cast<u64>(key_w(sorted[j])); }) + 1;
      }
      if (bad) sample_whole_row<XT>(a, b, sh.hist, sh.red, sh.out);
      else draw_from(n);
      return;
    } else if (!all) {
      float width = kFar / kBins;
      for (int level = 0;; ++level) {
        const float new_lo = b0 == 0 ? lo : lo + (b0 - 0.02f) * width;
        hi = b0 == kBins - 1 ? hi : lo + (b0 + 1.02f) * width;
        lo = new_lo;
        meet();  // what the blocks told each other has been read
        n_all = collect(lo, hi, above, min_above, max_below);
        if (n_all <= kCap) {
          merge(n_all);
          sort_down(sorted, spare, n_all);
          const u64 want = k - above;  // the cut's place in the list
          slow = above >= static_cast<u64>(k) || want > static_cast<u64>(n_all);
          if (!slow) {
            const u64 e = sorted[want - 1];
            const float l = key_float(entry_key(e)) * T, margin = fabsf(l) * 1e-6f + 8.3e-25f;
            top = {entry_key(e), entry_index(e), l - margin, l + margin};
            slow = !outside(e, min_above, max_below);
          }
          meet();  // the lists have been read
          break;
        }
        if (level + 1 == kLevels) {
          slow = true;
          break;
        }
        meet();
        width = (hi - lo) / kBins;
        b0 = count_bins(lo, hi, above, k, b1);
        if (b0 >= kBins) {
          slow = true;
          break;
        }
      }
    } else {
      meet();
    }
  }
  auto in_top = [&](float l, int i) { return l > top.hi || (l >= top.lo && keeps(top.key, top.idx, sc, l, i)); };
  auto e_of = [&](float l, int i) {  // zmax is finite here, so that exp(0) needs no case of its own
    const float e = expf(__fsub_rn(sc.z(l), zmax));
    return has_k && !in_top(l, i) ? 0.f : e;
  };

  Cut<uint32_t> nucleus{0, -1, 0, 0};  // top-p's cut, over the bits of e
  if (!slow && has_p) {
    // e takes the logits' place; bins of its exponent and two bits more, 0 for e in 1 .. 1/2 and up
    constexpr int kTop = 0x3f800000 >> 21;
    auto shift_of = [&](uint32_t bits) { return max(0, static_cast<int>(bits >> 23) - 117 + extra); };
    clear_columns();
    u64 mine = 0;
    for (int q = tid; q < n4; q += kThreads) {
      const float4 v = row4[q];
      const int i = i_begin + 4 * q - off;
      const float e[4] = {e_of(v.x, i), e_of(v.y, i + 1), e_of(v.z, i + 2), e_of(v.w, i + 3)};
      reinterpret_cast<float4 *>(row)[q] = make_float4(e[0], e[1], e[2], e[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = weight_w(e[j]), bits = __float_as_uint(e[j]);
        mine += w;
        if (w) atomicAdd(&columns[(kTop - (bits >> 21)) * 32 + lane], w >> shift_of(bits));
      }
    }
    int b1, b0 = settle(mine, 0, [&]() { return most_of(sum_told(sh.mass)); },
                        [&](int j) { return shift_of(static_cast<uint32_t>(kTop - j) << 21); }, b1);
    const u64 most = most_of(sum_told(sh.mass));
    slow = b0 >= kBins || b1 >= kBins;
    uint32_t lo = 0, hi = 0;  // the bits of e between which the cut lies
    if (!slow) {
      lo = static_cast<uint32_t>(kTop - b1) << 21;
      hi = static_cast<uint32_t>(kTop - b0 + 1) << 21;
    }
    for (int level = 0; !slow; ++level) {
      const uint32_t from = lo - 8, to = hi + 8;  // beyond them z is strictly smaller or larger
      // every token above the band is listed too where they may be few: there are at most most / w(band) of them
      const bool list_all = level == 0 && most < static_cast<u64>(4 * kCap) * w_of(lo);
      if (tid == 0) sh.n_local = sh.n_local_top = 0;
      __syncthreads();
      u64 sum = 0;
      each4(0.f, [&](const float (&e)[4], int i) {
        bool up[4], band[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t bits = __float_as_uint(e[j]);
          up[j] = bits >= to;
          band[j] = !up[j] && bits >= from;
          if (up[j]) sum += w_of(bits);
        }
        append4(band, &sh.n_local, [&](int at, int j) { list_band[at] = i + j; });
        if (list_all) append4(up, &sh.n_local_top, [&](int at, int j) { list_top[at] = i + j; });
      });
      __syncthreads();
      sum = block_sum_u64(sum, sh.red);
      if (warp == 0) {
        tell(&sh.above[rank], sum);
        tell(&sh.n[rank], sh.n_local);
        tell(&sh.n_top[rank], sh.n_local_top);
      }
      meet();
      const u64 above = sum_told(sh.above);
      int n_band = 0, n_top = 0;
      for (int r = 0; r < C; ++r) {
        n_band += sh.n[r];
        n_top += sh.n_top[r];
      }
      if (list_all && n_band + n_top <= kCap) {  // the listed tokens with their z, read again
        int at = 0;
        for (int r = 0; r < rank; ++r) at += sh.n[r] + sh.n_top[r];
        for (int i = tid; i < sh.n[rank] + sh.n_top[rank]; i += kThreads) {
          const int idx = i < sh.n[rank] ? list_band[i] : list_top[i - sh.n[rank]];
          put_in_first(entry(logit(idx), idx), at + i);
        }
        hand_over();
        if (rank != 0) return;
        const int n_all = n_band + n_top;
        sort_down(sorted, spare, n_all);
        const int place = reach(n_all, most, [&](int j) { return static_cast<u64>(key_w(sorted[j])); });
        if (place < n_all) draw_from(place + 1);
        else sample_whole_row<XT>(a, b, sh.hist, sh.red, sh.out);
        return;
      }
      if (n_band <= kCap) {
        for (int i = tid; i < n_band; i += kThreads) {
          int p = i;
          const int r = block_of(sh.n, p);
          const int idx = cluster.map_shared_rank(list_band, r)[p];
          sorted[i] = entry(logit(idx), idx);
        }
        __syncthreads();
        sort_down(sorted, spare, n_band);
        const int place = reach(n_band, most - above, [&](int j) { return static_cast<u64>(key_w(sorted[j])); });
        slow = place == n_band || above >= most;  // above < most: the cut lies below
        if (!slow) {
          const u64 e = sorted[place];
          const uint32_t bits = __float_as_uint(weight_e(key_float(entry_key(e)), zmax));
          nucleus = {entry_key(e), entry_index(e), bits - 8, bits + 8};
        }
        meet();  // the lists have been read
        break;
      }
      if (hi - lo == 1 || level + 1 == kNarrow) {  // that many equal weights
        slow = true;
        break;
      }
      // too many: 128 finer bins from hi down
      const int step = max(0, 25 - __clz(hi - lo - 1));  // (hi - lo - 1) >> step < 128
      const uint32_t top_bits = hi - 1, low_bits = lo;
      const int shift = shift_of(top_bits);  // one for all: it leaves 2^(19 - extra) of the lowest weight
      meet();  // what the blocks told each other has been read
      clear_columns();
      mine = 0;
      each4(0.f, [&](const float (&e)[4], int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t bits = __float_as_uint(e[j]);
          if (bits > top_bits) mine += w_of(bits);
          else if (bits >= low_bits) atomicAdd(&columns[((top_bits - bits) >> step) * 32 + lane], w_of(bits) >> shift);
        }
      });
      // what lies above the bins comes with the masses
      b0 = settle(mine, 0, [&]() {
        const u64 base = sum_told(sh.mass);
        return most > base ? most - base : u64(1);
      }, [&](int) { return shift; }, b1);
      slow = b0 >= kBins || b1 >= kBins;
      hi = top_bits + 1 - (static_cast<uint32_t>(b0) << step);
      lo = max(low_bits, top_bits + 1 - (static_cast<uint32_t>(b1 + 1) << step));
      // A cut at the edge of many equal weights: the shifted sums leave it open whether it lies among them or at the next
      // lower weight, which may be the lowest of the band, and finer bins tell no more.
      if (hi == top_bits + 1 && lo == low_bits) slow = true;
    }
  }
  if (slow) {
    if (rank == 0) sample_whole_row<XT>(a, b, sh.hist, sh.red, sh.out);
    return;
  }

  // ---- the draw over the row: running sums in index order, a run of float4s a warp ---
  const int seg = (n4 + kThreads / 32 - 1) / (kThreads / 32);
  const int q0 = min(n4, warp * seg), q1 = min(n4, q0 + seg);
  // a logit below this one has e < min_p, or weight 0, for sure
  const float low = fmaxf(min_e > 0.f ? high + T * (logf(min_e) - 1e-3f) - fabsf(high) * 1e-5f : -INFINITY, high - T * kFar - fabsf(high) * 1e-5f);
  auto weight_at = [&](float v, int i) -> uint32_t {
    float e;
    if (has_p) {
      e = v;
      const uint32_t bits = __float_as_uint(e);
      if (bits < nucleus.hi && (bits < nucleus.lo || !keeps(nucleus.key, nucleus.idx, sc, logit(i), i))) e = 0.f;
    } else {
      e = v >= low ? e_of(v, i) : 0.f;
    }
    return e >= min_e ? weight_w(e) : 0u;
  };
  u64 mine = 0;
  for (int q = q0 + lane; q < q1; q += 32) {
    const float4 v = row4[q];
    const int i = i_begin + 4 * q - off;
    const uint32_t w[4] = {weight_at(v.x, i), weight_at(v.y, i + 1), weight_at(v.z, i + 2), weight_at(v.w, i + 3)};
    mine += static_cast<u64>(w[0]) + w[1] + static_cast<u64>(w[2]) + w[3];
  }
  mine = warp_sum_u64(mine);
  __syncthreads();
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  u64 before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.red[w];
    total += sh.red[w];
  }
  if (warp == 0) tell(&sh.above[rank], total);
  meet();
  total = 0;
  for (int r = 0; r < C; ++r) {
    if (r < rank) before += sh.above[r];
    total += sh.above[r];
  }
  const u64 target = part_of(u24, total);
  if (target < before || target >= before + mine) return;
  for (int q = q0; q < q1; q += 32) {
    uint32_t w[4] = {0, 0, 0, 0};
    const int i = i_begin + 4 * (q + lane) - off;
    if (q + lane < q1) {
      const float4 v = row4[q + lane];
      w[0] = weight_at(v.x, i);
      w[1] = weight_at(v.y, i + 1);
      w[2] = weight_at(v.z, i + 2);
      w[3] = weight_at(v.w, i + 3);
    }
    const u64 sum = static_cast<u64>(w[0]) + w[1] + static_cast<u64>(w[2]) + w[3], inc = warp_scan_u64(sum);
    const u64 all = __shfl_sync(0xffffffffu, inc, 31);
    if (target < before + all) {
      u64 run = before + inc - sum;
      if (target >= run && target < run + sum) {
        int j = 0;
        while (target >= run + w[j]) run += w[j++];
        a.tokens[b] = i + j;
        if (a.probs) a.probs[b] = __fdiv_rn(static_cast<float>(w[j]), static_cast<float>(total));
      }
      return;
    }
    before += all;
  }
}

size_t cluster_smem(int slice) {
  return sizeof(Shared) + kBins * 32 * sizeof(uint32_t) + 2 * kCap * sizeof(u64) + (static_cast<size_t>(slice) + 16) * sizeof(float);
}

template <typename XT>
void launch(const SampleArgs &args, cudaStream_t st) {
  SampleArgs a = args;
  int device = 0, sms = 0;
  op_cuda(cudaGetDevice(&device), "cudaGetDevice");
  op_cuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "device attributes");
  // a block for every kSlice tokens; more where the rows alone would leave multiprocessors idle, down to 2,048 tokens a
  // block, below which the meetings cost more than the passes (a row of 32,000: 16.5 us, 18 with 8,192 a block; 4 rows 23 and
  // 26)
  int c = 1;
  while (c < kMaxCluster && (a.V > c * kSlice || (static_cast<long long>(a.rows) * c < sms && a.V > c * 2048))) c *= 2;
  a.slice = ((a.V + c - 1) / c + 7) / 8 * 8;
  if (a.slice > kMaxSlice) {
    op_launch("specdec_sample", sample_whole_kernel<XT>, dim3(a.rows), kThreads, 0, st, 1, a);
    return;
  }
  const size_t smem = cluster_smem(a.slice);
  static std::atomic<unsigned long long> ready{0};  // devices whose kernel has its shared memory limit
  const unsigned long long bit = 1ull << (device & 63);
  if (!(ready.load() & bit)) {
    op_cuda(cudaFuncSetAttribute(sample_cluster_kernel<XT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(cluster_smem(kMaxSlice))),
            "cudaFuncSetAttribute");
    ready.fetch_or(bit);
  }
  op_launch("specdec_sample", sample_cluster_kernel<XT>, dim3(static_cast<unsigned>(a.rows) * c), kThreads, smem, st, c, a);
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
    op_check(rows <= (1 << 24), "rows must be at most 2^24");
    cudaPointerAttributes at{};
    op_cuda(cudaPointerGetAttributes(&at, logits), "specdec_sample");
    op_check(at.type != cudaMemoryTypeUnregistered, "logits must be device memory");
    DeviceScope scope(at.device);
    const SampleArgs a{logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, u, tokens, probs, 0};
    const auto st = static_cast<cudaStream_t>(stream);
    dtype == SPECDEC_F32 ? launch<float>(a, st) : launch<__nv_bfloat16>(a, st);
  });
}
