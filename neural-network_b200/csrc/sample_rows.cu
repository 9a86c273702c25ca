// Sampling of logit rows with per-row temperature, top-k, top-p and min-p
// from given uniforms (specdec_sample).
//
// The distribution is held in whole numbers, so that no sum depends on the
// order of its terms: z = l / T, e = exp(z - max z) (1 at the maximum),
// w = floor(2^31 e) < 2^32, sums in 64 bits.  A token below 2^-31 of the
// likeliest one has weight 0; the uniforms have 24 bits, so it could hardly be
// drawn.  A cut (top-k by count, top-p by mass) is a pair (key, ties): tokens
// with a larger z, and the first `ties` tokens in index order with that z.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "status.cuh"

namespace specdec {

namespace {

constexpr int kThreads = 512;        // of a block; a cluster of blocks takes a row
constexpr int kSlice = 16384;        // tokens of a block where the row count gives enough blocks
constexpr int kMaxSlice = 40960;     // tokens that a block's shared memory holds
constexpr int kMaxCluster = 8;
constexpr int kBins = 128;
constexpr int kCap = 1024;           // tokens that are sorted to settle a cut exactly
constexpr float kFar = 22.2f;        // nats below the maximum from which the weight is 0: 2^31 exp(-22.2) < 1
constexpr int kLevels = 4;

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
__device__ __forceinline__ float no_nan(float l) { return isnan(l) ? -INFINITY : l; }

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

// Bitonic sort of `size` values (a power of two, at most 2 kThreads) in
// descending order, by the whole block.
__device__ void sort_down(u64 *v, int size) {
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

// The tokens kept so far: those with a larger key, and those with this key up
// to index idx.  Logits above hi have a larger key for sure, those below lo a
// smaller one; between them the key decides.
struct Cut {
  uint32_t key;
  int idx;
  float lo, hi;
};
__device__ __forceinline__ bool kept_by(const Cut &c, const Scale &sc, float l, int idx) {
  if (l > c.hi) return true;
  if (!(l >= c.lo)) return false;
  const uint32_t k = float_key(sc.z(l));
  return k > c.key || (k == c.key && idx <= c.idx);
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
    return greedy ? l : __fdiv_rn(l, T);
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
  int n[kMaxCluster];
  float min_above[kMaxCluster], max_below[kMaxCluster];
  // of this block alone
  u64 hist[256], red[32], out[3];
  float redf[32];
  int redi[32], n_local, band[2], at;
  unsigned char shift[kBins];
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
// memory.  A cut (top-k by count, top-p by mass) is found from the outside in:
// the counts (or the masses, in 32 bits with a shift per bin) of the tokens in
// 128 bins of their distance to the maximum give the bins in which the cut
// lies; each lane of a warp adds to a column of its own, so no two lanes meet
// in a bank or a word.  Where the tokens down to those bins are few, they are
// listed and sorted, and every filter and the draw are settled on that list.
// Else the tokens of the bins alone are listed, or binned again where they are
// too many, the exact cut is taken from their sorted list, and the draw passes
// over the row.  A list is checked to hold its cut: what lies outside it is
// strictly above or below; a row that fails, and one that never narrows, is
// done by sample_whole_row.
template <typename XT>
__global__ void __launch_bounds__(kThreads) sample_cluster_kernel(const SampleArgs a) {
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ __align__(16) unsigned char sample_smem[];
  Shared &sh = *reinterpret_cast<Shared *>(sample_smem);
  uint32_t *columns = reinterpret_cast<uint32_t *>(sample_smem + sizeof(Shared));  // [kBins][32]
  uint2 *list = reinterpret_cast<uint2 *>(columns + kBins * 32);                  // [kCap] (logit, index) of this block
  u64 *sorted = reinterpret_cast<u64 *>(list + kCap);                             // [kCap] of the cluster
  float *row = reinterpret_cast<float *>(sorted + kCap);                          // [slice + 16]
  auto meet = [&]() { cluster.sync(); };
  auto tell = [&](auto *p, auto v) {  // writes *p in every block
    for (int r = 0; r < C; ++r) *cluster.map_shared_rank(p, r) = v;
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
  float high = -INFINITY;
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
    for (int j = 0; j < 8; ++j) {
      v[j] = no_nan(v[j]);
      high = fmaxf(high, v[j]);
    }
    *reinterpret_cast<float4 *>(row + 8 + 8 * i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(row + 12 + 8 * i) = make_float4(v[4], v[5], v[6], v[7]);
  }
  for (int i = head + 8 * runs + tid; i < n; i += kThreads) {
    const float l = no_nan(to_f32(x[i]));
    row[i + off] = l;
    high = fmaxf(high, l);
  }
  high = block_max(high, sh.redf);
  if (tid == 0) tell(&sh.high[rank], high);
  meet();
  high = -INFINITY;
  for (int r = 0; r < C; ++r) high = fmaxf(high, sh.high[r]);
  // every pass: f(logit, index in the row)
  auto each = [&](auto &&f) {
    for (int q = tid; q < n4; q += kThreads) {
      const float4 v = reinterpret_cast<const float4 *>(row)[q];
      const int i = i_begin + 4 * q - off;
      f(v.x, i);
      f(v.y, i + 1);
      f(v.z, i + 2);
      f(v.w, i + 3);
    }
  };
  if (high == -INFINITY || greedy) {
    int first = 0x7fffffff;
    if (greedy && high != -INFINITY)
      each([&](float l, int i) { if (l == high) first = min(first, i); });
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
  // temperatures and logits for which equal z means nearly equal logits
  bool slow = !(T >= 9.1e-13f && T <= 1.1e12f && fabsf(high) < 1.2e24f);
  Cut cut{0, -1, -INFINITY, -INFINITY};
  auto far_of = [&](float l) { return (high - l) * sc.inv; };  // the distance to the maximum, falling with l

  // The tokens of all blocks' lists in `sorted`, by descending key and ascending index (key above, ~index below), filled
  // with zeros to a power of two.  The caller has met after the lists' end.
  auto merge = [&](int n_all) {
    int size = 32;
    while (size < n_all) size *= 2;
    for (int i = n_all + tid; i < size; i += kThreads) sorted[i] = 0;
    for (int r = 0, at = 0; r < C; at += sh.n[r++]) {
      const uint2 *src = cluster.map_shared_rank(list, r);
      for (int i = tid; i < sh.n[r]; i += kThreads) {
        const uint2 e = src[i];
        sorted[at + i] = static_cast<u64>(float_key(sc.z(__uint_as_float(e.x)))) << 32 | static_cast<uint32_t>(~e.y);
      }
    }
    __syncthreads();
    sort_down(sorted, size);
  };
  auto sorted_w = [&](int i) { return weight_w(weight_e(key_float(static_cast<uint32_t>(sorted[i] >> 32)), zmax)); };
  // The first place of `sorted` at which the running sum of f reaches want; n_all where it does not.
  auto reach = [&](int n_all, u64 want, auto &&f) {
    if (tid == 0) sh.at = n_all;
    const int i = 2 * tid;
    const u64 w0 = i < n_all ? f(i) : 0, w1 = i + 1 < n_all ? f(i + 1) : 0;
    u64 all;
    const u64 before = block_scan_u64(w0 + w1, sh.red, &all);
    if (before < want && want <= before + w0 + w1) sh.at = before + w0 >= want ? i : i + 1;
    __syncthreads();
    const int at = sh.at;
    __syncthreads();
    return at;
  };
  auto cut_at = [&](int i) {
    const u64 e = sorted[i];
    Cut c;
    c.key = static_cast<uint32_t>(e >> 32);
    c.idx = static_cast<int>(~static_cast<uint32_t>(e));
    const float l = key_float(c.key) * T, margin = fabsf(l) * 1e-6f + 8.3e-25f;
    c.lo = l - margin;
    c.hi = l + margin;
    return c;
  };

  // Counts (or masses) of the tokens kept by `in` in bins between lo and hi, to every block; a mass's sum goes to sh.mass.
  // Returns the first bin in which the running sum may reach want(), and in sure the first in which it must.
  auto bins = [&](bool by_mass, float lo, float hi, u64 base, const Cut in, auto &&want, int &sure) {
    const float width = (hi - lo) * (1.f / kBins), per = 1.f / width;
    for (int i = tid; i < kBins * 32; i += kThreads) columns[i] = 0;
    if (by_mass && tid < kBins)  // a column's sum of up to slice / 32 weights of the bin fits 32 bits
      sh.shift[tid] = max(0, static_cast<int>((__float_as_uint(expf(-(lo + tid * width)) * 1.01f * 2147483648.f * (a.slice / 32 + 4)) >> 23)) - 127 - 31);
    __syncthreads();
    u64 mine = 0;
    if (by_mass) {
      each([&](float l, int i) {
        const float d = far_of(l);
        if (!(d >= lo && d < hi) || !kept_by(in, sc, l, i)) return;
        const uint32_t w = weight_w(weight_e(sc.z(l), zmax));
        const int j = min(kBins - 1, static_cast<int>((d - lo) * per));
        mine += w;
        atomicAdd(&columns[j * 32 + lane], w >> sh.shift[j]);
      });
      mine = block_sum_u64(mine, sh.red);
    } else {
      each([&](float l, int i) {
        const float d = far_of(l);
        if (d >= lo && d < hi && kept_by(in, sc, l, i))
          atomicAdd(&columns[min(kBins - 1, static_cast<int>((d - lo) * per)) * 32 + lane], 1u);
      });
    }
    __syncthreads();
    for (int j = warp; j < kBins; j += kThreads / 32) {
      // 32 columns of up to 31 bits: the sum in two halves
      const uint32_t c = columns[j * 32 + lane];
      const uint32_t low = __reduce_add_sync(0xffffffffu, c & 0xffffu), high16 = __reduce_add_sync(0xffffffffu, c >> 16);
      const u64 sum = (static_cast<u64>(high16) << 16) + low;
      if (lane == 0) tell(&sh.counts[rank][j], sum);
    }
    if (tid == 0) tell(&sh.mass[rank], mine);
    meet();
    if (warp == 0) {  // lane l: bins 4 l .. 4 l + 3
      const u64 target = want();
      u64 some[4], most[4], sum_some = 0, sum_most = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u64 c = 0;
        for (int r = 0; r < C; ++r) c += sh.counts[r][4 * lane + j];
        some[j] = most[j] = c;
        if (by_mass) {  // a shift leaves at least 2^20 of a weight, so it drops less than 2^-20 of the sum
          some[j] = c << sh.shift[4 * lane + j];
          most[j] = some[j] + (sh.shift[4 * lane + j] ? some[j] >> 18 : 0);
        }
        sum_some += some[j];
        sum_most += most[j];
      }
      u64 run_some = base + warp_scan_u64(sum_some) - sum_some, run_most = base + warp_scan_u64(sum_most) - sum_most;
      int first = kBins, must = kBins;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        u64 s = run_some, m = run_most;
        for (int i = 0; i <= j; ++i) {
          s += some[i];
          m += most[i];
        }
        if (m >= target) first = 4 * lane + j;
        if (s >= target) must = 4 * lane + j;
      }
      first = __reduce_min_sync(0xffffffffu, first);
      must = __reduce_min_sync(0xffffffffu, must);
      if (lane == 0) {
        sh.band[0] = first;
        sh.band[1] = must;
      }
    }
    __syncthreads();
    sure = sh.band[1];
    return sh.band[0];
  };
  // Lists the tokens kept by `in` between lo and hi; counts (or sums) those above lo; all to every block.  Returns the
  // number listed by all blocks; above and the nearest logits outside come back too.
  auto collect = [&](bool by_mass, float lo, float hi, const Cut in, u64 &above, float &min_above, float &max_below) {
    if (tid == 0) sh.n_local = 0;
    __syncthreads();
    above = 0;
    min_above = INFINITY;
    max_below = -INFINITY;
    each([&](float l, int i) {
      const float d = far_of(l);
      if (!(d < hi)) {
        max_below = fmaxf(max_below, l);
        return;
      }
      if (!kept_by(in, sc, l, i)) return;
      if (d < lo) {
        above += by_mass ? weight_w(weight_e(sc.z(l), zmax)) : 1u;
        min_above = fminf(min_above, l);
      } else {
        const int at = atomicAdd(&sh.n_local, 1);
        if (at < kCap) list[at] = make_uint2(__float_as_uint(l), i);
      }
    });
    above = block_sum_u64(above, sh.red);
    min_above = -block_max(-min_above, sh.redf);
    max_below = block_max(max_below, sh.redf);
    if (tid == 0) {
      tell(&sh.above[rank], above);
      tell(&sh.n[rank], sh.n_local);
      tell(&sh.min_above[rank], min_above);
      tell(&sh.max_below[rank], max_below);
    }
    meet();
    above = 0;
    int n_all = 0;
    for (int r = 0; r < C; ++r) {
      above += sh.above[r];
      n_all += sh.n[r];
      min_above = fminf(min_above, sh.min_above[r]);
      max_below = fmaxf(max_below, sh.max_below[r]);
    }
    return n_all;
  };
  auto below_cut = [&](float l, const Cut &c) { return l == -INFINITY || float_key(sc.z(l)) < c.key; };
  auto above_cut = [&](float l, const Cut &c) { return l == INFINITY || float_key(sc.z(l)) > c.key; };
  const u64 p24 = static_cast<u64>(rintf(fminf(fmaxf(top_p, 0.f), 1.f) * 16777216.f));
  auto most_of = [&](u64 mass) { return max(part_of(p24, mass), u64(1)); };
  const u64 u24 = static_cast<u64>(fminf(fmaxf(a.u[b] * 16777216.f, 0.f), 16777215.f));

  // The cut at which the count (or mass) over descending z first reaches its target, among the tokens that `in` keeps.
  // b0, b1: the bins of the first level, already found.
  auto search = [&](bool by_mass, u64 want, const Cut in, int b0, int b1) {
    float lo = 0.f, hi = kFar;
    for (int level = 0; level < kLevels && !slow; ++level) {
      const float width = (hi - lo) * (1.f / kBins);
      if (b0 >= kBins) break;
      b1 = min(b1, kBins - 1);
      const float new_lo = b0 == 0 ? lo : lo + (b0 - 0.02f) * width, new_hi = b1 == kBins - 1 ? hi : lo + (b1 + 1.02f) * width;
      u64 above;
      float min_above, max_below;
      const int n_all = collect(by_mass, new_lo, new_hi, in, above, min_above, max_below);
      if (n_all <= kCap) {
        merge(n_all);
        const int at = above < want ? reach(n_all, want - above, [&](int i) { return by_mass ? static_cast<u64>(sorted_w(i)) : u64(1); }) : n_all;
        Cut c = in;
        if (at < n_all) c = cut_at(at);
        slow = at == n_all || !above_cut(min_above, c) || !below_cut(max_below, c);
        meet();  // the lists have been read
        return c;
      }
      lo = new_lo;
      hi = new_hi;
      meet();  // what the blocks told each other has been read
      b0 = bins(by_mass, lo, hi, above, in, [&]() { return want; }, b1);
    }
    slow = true;
    return in;
  };

  if (!slow && (has_k || has_p)) {
    // the bins of the first cut, and the list of everything down to it
    int b1, b0 = bins(!has_k, 0.f, kFar, 0, cut, [&]() {
      if (has_k) return static_cast<u64>(k);
      u64 mass = 0;
      for (int r = 0; r < C; ++r) mass += sh.mass[r];
      return most_of(mass);
    }, b1);
    u64 mass_all = 0;
    for (int r = 0; r < C; ++r) mass_all += sh.mass[r];
    // has_k and no bin: fewer than k tokens have a weight above 0, and all of them are kept
    u64 above = 0;
    float min_above = INFINITY, max_below = -INFINITY;
    const float hi = b0 >= kBins || b1 >= kBins - 1 ? kFar : (b1 + 1.02f) * (kFar / kBins);
    const int n_all = collect(false, 0.f, hi, cut, above, min_above, max_below);
    if (n_all <= kCap) {
      if (rank == 0) {
        merge(n_all);
        // how many of the list the filters keep
        int n = n_all;
        bool bad = false;
        if (has_k && b0 < kBins) {
          n = k;
          bad = n > n_all || !below_cut(max_below, cut_at(max(0, min(n, n_all) - 1)));
          n = min(n, n_all);
        }
        u64 mass = mass_all;
        const int i = 2 * tid;
        if (has_p) {
          if (has_k) mass = block_sum_u64((i < n ? sorted_w(i) : 0u) + static_cast<u64>(i + 1 < n ? sorted_w(i + 1) : 0u), sh.red);
          const int at = reach(n, most_of(mass), [&](int j) { return static_cast<u64>(sorted_w(j)); });
          bad = bad || at == n;
          if (at < n) {
            if (!has_k) bad = bad || !below_cut(max_below, cut_at(at));
            n = at + 1;
          }
        }
        if (!bad) {
          // the kept tokens by index: (index, weight) sorted again; min-p leaves its tokens with weight 0
          __syncthreads();
          u64 e[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            e[j] = 0;
            if (i + j < n) {
              const float w_e = weight_e(key_float(static_cast<uint32_t>(sorted[i + j] >> 32)), zmax);
              const uint32_t w = w_e >= min_e ? weight_w(w_e) : 0u;
              e[j] = sorted[i + j] << 32 | w;  // ~index above: descending is by ascending index
            }
          }
          __syncthreads();
          int size = 32;
          while (size < n) size *= 2;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (i + j < size) sorted[i + j] = e[j];
          __syncthreads();
          sort_down(sorted, size);
          const u64 total = block_sum_u64((i < n ? sorted[i] & 0xffffffffu : 0) + (i + 1 < n ? sorted[i + 1] & 0xffffffffu : 0), sh.red);
          const int at = reach(n, part_of(u24, total) + 1, [&](int j) { return sorted[j] & 0xffffffffu; });
          if (tid == 0) {
            a.tokens[b] = static_cast<int>(~static_cast<uint32_t>(sorted[at] >> 32));
            if (a.probs) a.probs[b] = __fdiv_rn(static_cast<float>(sorted[at] & 0xffffffffu), static_cast<float>(total));
          }
        }
        if (tid == 0) tell(&sh.first[0], bad ? 1 : 0);
      }
      meet();  // the lists have been read
      if (!sh.first[0]) return;
      slow = true;
    } else {
      meet();  // what the blocks told each other has been read
      if (has_k && b0 < kBins) cut = search(false, k, cut, b0, b1);
      if (has_p && !slow) {
        u64 most = 0;
        if (has_k) {
          b0 = bins(true, 0.f, kFar, 0, cut, [&]() {
            u64 mass = 0;
            for (int r = 0; r < C; ++r) mass += sh.mass[r];
            return most_of(mass);
          }, b1);
          mass_all = 0;
          for (int r = 0; r < C; ++r) mass_all += sh.mass[r];
        }
        most = most_of(mass_all);
        cut = search(true, most, cut, b0, b1);
      }
    }
  }
  if (slow) {
    if (rank == 0) sample_whole_row<XT>(a, b, sh.hist, sh.red, sh.out);
    return;
  }

  // ---- the draw: running sums in index order, a run of float4s a warp -----------
  const int seg = (n4 + kThreads / 32 - 1) / (kThreads / 32);
  const int q0 = min(n4, warp * seg), q1 = min(n4, q0 + seg);
  // a logit below this one has e < min_p for sure
  const float low = min_e > 0.f ? high + T * (logf(min_e) - 1e-3f) - fabsf(high) * 1e-5f : -INFINITY;
  auto weight_at = [&](float l, int i) -> u64 {
    if (!(far_of(l) < kFar) || l < low || !kept_by(cut, sc, l, i)) return 0;
    const float e = weight_e(sc.z(l), zmax);
    return e >= min_e ? weight_w(e) : 0u;
  };
  u64 mine = 0;
  for (int q = q0 + lane; q < q1; q += 32) {
    const float4 v = reinterpret_cast<const float4 *>(row)[q];
    const int i = i_begin + 4 * q - off;
    mine += weight_at(v.x, i) + weight_at(v.y, i + 1) + weight_at(v.z, i + 2) + weight_at(v.w, i + 3);
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
  if (tid == 0) tell(&sh.mass[rank], total);
  meet();
  total = 0;
  for (int r = 0; r < C; ++r) {
    if (r < rank) before += sh.mass[r];
    total += sh.mass[r];
  }
  const u64 target = part_of(u24, total);
  if (target < before || target >= before + mine) return;
  for (int q = q0; q < q1; q += 32) {
    u64 w[4] = {0, 0, 0, 0};
    const int i = i_begin + 4 * (q + lane) - off;
    if (q + lane < q1) {
      const float4 v = reinterpret_cast<const float4 *>(row)[q + lane];
      w[0] = weight_at(v.x, i);
      w[1] = weight_at(v.y, i + 1);
      w[2] = weight_at(v.z, i + 2);
      w[3] = weight_at(v.w, i + 3);
    }
    const u64 sum = w[0] + w[1] + w[2] + w[3], inc = warp_scan_u64(sum);
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
  // a block for every kSlice tokens; more where the rows alone would leave multiprocessors idle (148 of them), down to
  // 2,048 tokens a block, below which the meetings cost more than the passes
  int c = 1;
  while (c < kMaxCluster && (a.V > c * kSlice || (a.rows * c < 148 && a.V > c * 2048))) c *= 2;
  a.slice = ((a.V + c - 1) / c + 7) / 8 * 8;
  if (a.slice > kMaxSlice) {
    op_launch("specdec_sample", sample_whole_kernel<XT>, dim3(a.rows), kThreads, 0, st, 1, a);
    return;
  }
  const size_t smem = cluster_smem(a.slice);
  static std::atomic<unsigned long long> ready{0};  // devices whose kernel has its shared memory limit
  int device = 0;
  op_cuda(cudaGetDevice(&device), "cudaGetDevice");
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
    const SampleArgs a{logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, u, tokens, probs, 0};
    const auto st = static_cast<cudaStream_t>(stream);
    dtype == SPECDEC_F32 ? launch<float>(a, st) : launch<__nv_bfloat16>(a, st);
  });
}
