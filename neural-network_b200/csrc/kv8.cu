// The 8-bit paged cache (specdec_kv8): its handle, the block tables and slot
// maps of a batch, and writing and reading cache rows.
#include "kv8.cuh"

#include <memory>

#include "kv8_attn.cuh"

namespace specdec {

namespace {

// ---------------------------------------------------------------------------
// Block tables and slot maps.  Per request: pages held = ceil(held / P),
// pages needed = ceil((keep + q) / P); requests in order take what they lack
// from the head of the ring of free pages and give back what they no longer
// need at its tail.  The ring's two regions do not overlap (free pages plus
// returned pages are at most all pages, and the ring holds all of them), so
// every block reads the old ring and table while others write the new parts.
//
// Bound by latency: three dependent reads and a scan.  Every block does the
// whole scan over the requests (12 bytes each, from L2 after the first) so
// that one launch is enough; the blocks then share tokens, moved pages and
// requests.  Both scans in one pass of 512 threads, one packed into the other:
// 6.7 us for 32 requests (an empty launch takes about 3), 8.4 us for 2,048
// requests with 65,000 rows (1.1 MB, 0.2 us of HBM); with two passes of 1,024
// threads 8.9 and 16.4 us.
struct PlanArgs {
  const int32_t *held, *keep, *q_len;
  int32_t *table;
  int B, cols, P;
  int32_t *ring;
  int ring_cap;
  const int32_t *ring_state;
  int32_t *ring_out;
  int32_t *kv_len, *cu_q, *tok_req, *tok_pos;
  int64_t *slots;
  int T;
  int32_t *status;
};

constexpr int kPlanThreads = 512;
constexpr int kPlanBytes = 2 * 8 + 2 * 4;  // shared memory of a request

__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const PlanArgs a) {
  extern __shared__ long long plan_smem[];
  long long *cu = plan_smem;                            // [B + 1] first row of a request
  long long *mv = cu + a.B + 1;                         // [B + 1] pages taken (low half) and given back (high) before it
  int *keeps = reinterpret_cast<int *>(mv + a.B + 1);   // [B] positions kept
  int *haves = keeps + a.B;                             // [B] pages held
  __shared__ long long red[2][kPlanThreads / 32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int p_shift = 31 - __clz(a.P);
  const long long cap = static_cast<long long>(a.cols) << p_shift;
  auto pages = [&](long long n) { return (n + a.P - 1) >> p_shift; };

  // Both prefix sums at once; a thread owns a run of consecutive requests.
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(a.B, static_cast<int>(threadIdx.x) * per), b1 = min(a.B, b0 + per);
  long long rows = 0, moves = 0;
  int bad = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    const long long held = a.held[b], keep = a.keep[b], q = a.q_len[b];
    const bool ok = held >= 0 && keep >= 0 && keep <= held && q >= 0 && held <= cap && keep + q <= cap;
    const long long more = ok ? pages(keep + q) - pages(held) : 0;
    const long long m = more >= 0 ? more : -more << 32;
    cu[b] = ok ? q : 0;
    mv[b] = m;
    keeps[b] = static_cast<int>(keep);
    haves[b] = static_cast<int>(pages(held));
    rows += cu[b];
    moves += m;
    bad |= !ok;
  }
  long long inc_r = rows, inc_m = moves;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long r = __shfl_up_sync(0xffffffffu, inc_r, o), m = __shfl_up_sync(0xffffffffu, inc_m, o);
    if (lane >= o) {
      inc_r += r;
      inc_m += m;
    }
  }
  if (lane == 31) {
    red[0][wid] = inc_r;
    red[1][wid] = inc_m;
  }
  const long long head = a.ring_state[0], count = a.ring_state[1];
  bad = __syncthreads_or(bad);
  long long run_r = inc_r - rows, run_m = inc_m - moves;
  for (int w = 0; w < wid; ++w) {
    run_r += red[0][w];
    run_m += red[1][w];
  }
  for (int b = b0; b < b1; ++b) {
    const long long r = cu[b], m = mv[b];
    cu[b] = run_r;
    mv[b] = run_m;
    run_r += r;
    run_m += m;
  }
  if (threadIdx.x == kPlanThreads - 1) {
    cu[a.B] = run_r;
    mv[a.B] = run_m;
  }
  __syncthreads();

  const long long takes = mv[a.B] & 0xffffffffll, gives = mv[a.B] >> 32;
  // the tail's writes must not reach places that the head's reads come from, whose pages leave only with this step
  const bool ring_ok = head >= 0 && head < a.ring_cap && count >= 0 && count + gives <= a.ring_cap;
  const int status = ((ring_ok && takes > count) ? 1 : 0) | (bad || !ring_ok ? 2 : 0) | (cu[a.B] > a.T ? 4 : 0);
  const bool fine = status == 0;
  // ring places wrap at most twice: head, count and the moves are each at most ring_cap
  auto place = [&](long long i) {
    if (i >= a.ring_cap) i -= a.ring_cap;
    return i >= a.ring_cap ? i - a.ring_cap : i;
  };
  const long long tid = static_cast<long long>(blockIdx.x) * kPlanThreads + threadIdx.x;
  const long long stride = static_cast<long long>(gridDim.x) * kPlanThreads;
  if (tid == 0) {
    *a.status = status;
    a.ring_out[0] = static_cast<int>(fine ? place(head + takes) : head);
    a.ring_out[1] = static_cast<int>(fine ? count - takes + gives : count);
  }
  for (long long b = tid; b <= a.B; b += stride) {
    a.cu_q[b] = fine ? static_cast<int>(cu[b]) : 0;
    if (b < a.B) a.kv_len[b] = fine ? keeps[b] + static_cast<int>(cu[b + 1] - cu[b]) : a.held[b];
  }
  if (fine) {
    auto find = [&](long long u, auto &&at) {  // the last request with at(b) <= u
      int lo = 0, hi = a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at(mid) <= u) lo = mid;
        else hi = mid - 1;
      }
      return lo;
    };
    auto low = [&](int b) { return mv[b] & 0xffffffffll; };
    auto high = [&](int b) { return mv[b] >> 32; };
    for (long long i = tid; i < takes; i += stride) {
      const int b = find(i, low);
      a.table[static_cast<long long>(b) * a.cols + haves[b] + (i - low(b))] = a.ring[place(head + i)];
    }
    for (long long i = tid; i < gives; i += stride) {
      const int b = find(i, high);
      const long long need = pages(keeps[b] + (cu[b + 1] - cu[b]));
      a.ring[place(head + count + i)] = a.table[static_cast<long long>(b) * a.cols + need + (i - high(b))];
    }
  }
  for (long long t = tid; t < a.T; t += stride) {
    int req = -1, pos = -1;
    long long slot = -1;
    if (fine && t < cu[a.B]) {
      req = request_of(cu, a.B, t);
      pos = keeps[req] + static_cast<int>(t - cu[req]);
      const int col = pos >> p_shift, have = haves[req];
      // a page taken in this call is read from the ring: its table entry is being written
      const long long page = col < have ? a.table[static_cast<long long>(req) * a.cols + col]
                                        : a.ring[place(head + (mv[req] & 0xffffffffll) + col - have)];
      slot = (page << p_shift) + (pos & (a.P - 1));
    }
    a.tok_req[t] = req;
    a.tok_pos[t] = pos;
    a.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------
// Cache write.  One unit = the new rows of one scale block and kv head, K then
// V: a = max |x| over the finite new values, scale' = max(|scale| if the block
// has older rows, a x (1 / 127)); older rows are brought to scale', new rows
// become rint(x x (1 / scale')).  A scale below the smallest normal number is
// 0 (its codes are 0), so 1 / scale' is finite.
//
// Bound by HBM: every value is read once and its code written once.  A unit's
// values stay in registers between the maximum and the codes, up to eight runs
// of eight adjacent values a lane (all of them in flight at once), so a block
// of 16 x 128 takes one warp and no barrier, one of 128 x 128 eight warps.
// 4 prompts of 2,048 bf16 rows, 32 heads of 128, written and read back (403 MB,
// 61.5 us at the measured 6.55 TB/s): 81 us, 5.0 TB/s; half of what is moved are
// stores.  What that took: 738 us with a thread per value, 149 with a warp per
// block, 128 with rounding by an addition, 110 with K and V together and heads
// read in one piece, 103 with whole sectors written, 92 without branches between
// a unit's loads, 84 with the read's places found once, 81 with three blocks a
// multiprocessor.  A verify step (160 rows; 10 MB) takes 13 us for the two
// launches: latency.
constexpr float kInv127 = 1.f / 127.f;
constexpr int kRun = 8;  // adjacent values that a lane handles together

// rint(x) of |x| < 2^22 in the low bits: adding 1.5 x 2^23 rounds to whole numbers, to even on a tie, as rint does.
__device__ __forceinline__ uint32_t rint_bits(float x) { return __float_as_uint(__fadd_rn(x, 12582912.f)); }
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The code of any value: a NaN is 0, what is beyond 127 (infinities) stays there.
__device__ __forceinline__ uint32_t any_code(float x, float inv) {
  return isnan(x) ? 0u : rint_bits(fminf(fmaxf(__fmul_rn(x, inv), -127.f), 127.f));
}

// Eight adjacent values (vec: at a 16-byte boundary).
template <typename XT>
struct Run;
template <>
struct Run<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p, bool vec) {
    if (vec) {
      v = __ldg(reinterpret_cast<const uint4 *>(p));
    } else {
      const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
      v = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
    }
  }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  // bits of the largest |x|, those of an infinity or a NaN where there is one
  __device__ __forceinline__ uint32_t top() const {
    auto mag = [](uint32_t w) {
      w &= 0x7fff7fffu;
      return *reinterpret_cast<const __nv_bfloat162 *>(&w);
    };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(mag(v.x), mag(v.y)), __hmax2_nan(mag(v.z), mag(v.w)));
    const uint32_t w = *reinterpret_cast<const uint32_t *>(&m);
    return max(w << 16, w & 0xffff0000u);
  }
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    return __uint_as_float((j & 1) ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&f)[kRun], bool vec) {
    if (vec) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&t);
      }
      *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int j = 0; j < kRun; ++j) p[j] = __float2bfloat16_rn(f[j]);
    }
  }
};
template <>
struct Run<float> {
  float v[kRun];
  __device__ __forceinline__ void load(const float *p, bool vec) {
    if (vec) {
      const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      for (int j = 0; j < kRun; ++j) v[j] = p[j];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < kRun; ++j) v[j] = 0.f;
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ float get(int j) const { return v[j]; }
  static __device__ __forceinline__ void store(float *p, const float (&f)[kRun], bool vec) {
    if (vec) {
      *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
      *(reinterpret_cast<float4 *>(p) + 1) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      for (int j = 0; j < kRun; ++j) p[j] = f[j];
    }
  }
};

struct AppendArgs {
  Kv8Geom g;
  Kv8Layer c;
  Kv8Batch b;
  const void *x[2];                         // K and V rows
  long long row_stride[2], head_stride[2];  // elements
  int vec[2];                               // rows and heads start at 16-byte boundaries
};

constexpr int kAppendThreads = 256;
// blocks per SM: registers (bf16 rows: 84 us for the case above with two, 81 with three; 4 x 1,024 fp32 rows, blocks of 128:
// 99 us with one, 85 with two)
template <typename XT>
constexpr int append_ctas() {
  return sizeof(XT) == 2 ? 3 : 2;
}

// RUNS runs a lane, WARPS warps a unit: RUNS x WARPS x 256 values = block_tokens x head_dim.
template <typename XT, int RUNS, int WARPS>
__global__ void __launch_bounds__(kAppendThreads, append_ctas<XT>()) kv8_append_kernel(const AppendArgs a) {
  extern __shared__ int append_smem[];
  int *pre = append_smem;  // [B + 1] blocks touched before a request
  __shared__ int red[kAppendThreads / 32];
  __shared__ uint32_t tops[kAppendThreads / 32];
  const Kv8Geom &g = a.g;
  request_prefix(a.b.B, pre, red, [&](int b) {
    const Kv8Req r = kv8_req(a.b, g.P, b);
    return (r.q > 0 && r.len >= r.q) ? (r.len - 1) / g.t - (r.len - r.q) / g.t + 1 : 0;
  });
  constexpr int kGroups = kAppendThreads / 32 / WARPS;  // units a block works on at a time
  const int warp = threadIdx.x >> 5, group = warp / WARPS, lane = threadIdx.x % (32 * WARPS);
  const int per_row_shift = 31 - __clz(g.D / kRun), t_shift = 31 - __clz(g.t), p_shift = 31 - __clz(g.P);
  const long long units = static_cast<long long>(pre[a.b.B]) * g.Hkv;
  for (long long u = static_cast<long long>(blockIdx.x) * kGroups + group; u < units; u += static_cast<long long>(gridDim.x) * kGroups) {
    const uint32_t blk = static_cast<uint32_t>((u >> 32) ? u / g.Hkv : static_cast<uint32_t>(u) / static_cast<uint32_t>(g.Hkv));
    const uint32_t h = static_cast<uint32_t>(u - static_cast<long long>(blk) * g.Hkv);
    const int b = request_of(pre, a.b.B, static_cast<int>(blk));
    const Kv8Req r = kv8_req(a.b, g.P, b);
    const int start = r.len - r.q;
    const int p0 = ((start >> t_shift) + static_cast<int>(blk) - pre[b]) << t_shift;  // the block's first position
    const int n_old = max(0, start - p0), n = min(g.t, r.len - p0);  // older rows, rows in all
    const int page = a.b.table[static_cast<long long>(b) * a.b.cols + (p0 >> p_shift)];
    if (page < 0 || page >= a.c.n_pages) continue;
    const long long ph = static_cast<long long>(page) * g.Hkv + h;
    const int in = p0 & (g.P - 1);
    const long long code_at = ((ph << p_shift) + in) * g.D, scale_at = (ph << (p_shift - t_shift)) + (in >> t_shift);
#pragma unroll 1
    for (int kv = 0; kv < 2; ++kv) {
    int8_t *code = (kv ? a.c.v : a.c.k) + code_at;
    float *sc = (kv ? a.c.vs : a.c.ks) + scale_at;
    const XT *x = static_cast<const XT *>(a.x[kv]) + (r.q0 + p0 - start) * a.row_stride[kv] + h * a.head_stride[kv];
    // all runs are asked for at once: no branch stands between the loads, those of rows that are not new read one that is
    Run<XT> v[RUNS];
    int row[RUNS];
    auto load = [&](bool vec) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        const int e = lane + 32 * WARPS * i;
        row[i] = e >> per_row_shift;
        v[i].load(x + min(max(row[i], n_old), n - 1) * a.row_stride[kv] + (e - (row[i] << per_row_shift)) * kRun, vec);
      }
    };
    if (a.vec[kv]) load(true);
    else load(false);
    const bool full = n_old == 0 && n == g.t;
    if (!full) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i)
        if (row[i] < n_old || row[i] >= n) v[i].zero();
    }
    const float old = n_old ? *sc : 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) top = max(top, v[i].top());
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (WARPS > 1) {  // the group's own barrier: groups may have different numbers of units left
      if ((threadIdx.x & 31) == 0) tops[warp] = top;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WARPS) : "memory");
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = max(top, tops[group * WARPS + w]);
    }
    float m = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    if (!finite) {  // the largest finite value
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < RUNS; ++i)
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          const uint32_t f = __float_as_uint(v[i].get(j)) & 0x7fffffffu;
          t = max(t, f < 0x7f800000u ? f : 0u);
        }
      t = __reduce_max_sync(0xffffffffu, t);
      if constexpr (WARPS > 1) {
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WARPS) : "memory");
        if ((threadIdx.x & 31) == 0) tops[warp] = t;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WARPS) : "memory");
#pragma unroll
        for (int w = 0; w < WARPS; ++w) t = max(t, tops[group * WARPS + w]);
      }
      m = __uint_as_float(t);
    }
    float s = fmaxf(fabsf(old), __fmul_rn(m, kInv127));  // a block that came with a scale below 0 gets one above
    if (s < 1.17549435e-38f) s = 0.f;
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    const float factor = s > old && s > 0.f ? __fdiv_rn(old, s) : 1.f;  // -1 .. 1
    if constexpr (WARPS > 1)  // every warp of the group has read the scale and the maxima
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WARPS) : "memory");
    else
      __syncwarp();
    if (lane == 0) *sc = s;
    if (full && finite) {  // the loop below without its cases
#pragma unroll
      for (int i = 0; i < RUNS; ++i) {
        uint32_t c[kRun];
#pragma unroll
        for (int j = 0; j < kRun; ++j) c[j] = rint_bits(__fmul_rn(v[i].get(j), inv));
        *reinterpret_cast<uint2 *>(code + (lane + 32 * WARPS * i) * kRun) =
            make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      uint2 *to = reinterpret_cast<uint2 *>(code + (lane + 32 * WARPS * i) * kRun);
      if (row[i] < n_old) {
        if (factor == 1.f) continue;
        const uint2 w = *to;
        uint32_t o[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          const int c = static_cast<int8_t>(((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 255u);
          const int d = static_cast<int>(rintf(__fmul_rn(static_cast<float>(c), factor)));
          o[j >> 2] |= (static_cast<uint32_t>(d) & 255u) << (8 * (j & 3));
        }
        *to = make_uint2(o[0], o[1]);
      } else if (row[i] < n) {
        uint32_t c[kRun];
        if (finite) {  // |x / scale'| <= 127 (1 + 2^-22): rint needs no bounds; 1 / scale' is 0 where scale' is
#pragma unroll
          for (int j = 0; j < kRun; ++j) c[j] = rint_bits(__fmul_rn(v[i].get(j), inv));
        } else {
#pragma unroll
          for (int j = 0; j < kRun; ++j) c[j] = s > 0.f ? any_code(v[i].get(j), inv) : 0u;
        }
        *to = make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
      }
    }
    }
  }
}

template <typename XT, int RUNS, int WARPS>
void append_launch(const specdec_kv8 *h, const AppendArgs &a, cudaStream_t st) {
  const long long units = (static_cast<long long>(a.b.T) / h->g.t + 2ll * a.b.B) * h->g.Hkv;
  const int groups = kAppendThreads / 32 / WARPS;
  const int grid = static_cast<int>(std::min((units + groups - 1) / groups, 8ll * h->num_sms));
  op_launch("specdec_kv8_append", kv8_append_kernel<XT, RUNS, WARPS>, dim3(grid), kAppendThreads, (a.b.B + 1) * sizeof(int), st, 1, a);
}
template <typename XT>
void append_any(const specdec_kv8 *h, const AppendArgs &a, cudaStream_t st) {
  switch (h->g.t * h->g.D / 256) {
    case 1: return append_launch<XT, 1, 1>(h, a, st);
    case 2: return append_launch<XT, 2, 1>(h, a, st);
    case 4: return append_launch<XT, 4, 1>(h, a, st);
    case 8: return append_launch<XT, 8, 1>(h, a, st);
    case 16: return append_launch<XT, 8, 2>(h, a, st);
    case 32: return append_launch<XT, 8, 4>(h, a, st);
    default: return append_launch<XT, 8, 8>(h, a, st);
  }
}

// Cache read: the values code * scale of given rows, [n][Hkv][D].  A warp takes
// one head of a group of rows (8 at D = 128), so that rows that follow each
// other in the cache are read in one piece; K and V, four runs of 8 codes a lane in
// flight each (16 codes would leave every store with half-written sectors).  A code byte c + 128 in the low bits of 2^23 is
// 2^23 + 128 + c as a float: one subtraction leaves c.
struct GatherArgs {
  Kv8Geom g;
  Kv8Layer c;
  const int64_t *rows;
  int n;
  void *out[2];
  int vec;
};

constexpr int kGatherThreads = 256;
constexpr int kGatherAhead = 4;

template <typename XT>
__global__ void __launch_bounds__(kGatherThreads, 4) kv8_gather_kernel(const GatherArgs a) {
  const Kv8Geom &g = a.g;
  const int lanes = g.D / kRun, at_once = 32 / lanes, lane = threadIdx.x & 31;  // lanes of a row, rows a load
  const int p_shift = 31 - __clz(g.P), scale_shift = 31 - __clz(g.t) + 31 - __clz(g.D);
  const int d = lane % lanes * kRun, mine = lane / lanes;
  const long long slots = static_cast<long long>(a.c.n_pages) << p_shift;
  const long long tasks = (static_cast<long long>(a.n) + at_once * kGatherAhead - 1) / (at_once * kGatherAhead) * g.Hkv;
  for (long long task = (static_cast<long long>(blockIdx.x) * kGatherThreads + threadIdx.x) >> 5; task < tasks;
       task += static_cast<long long>(gridDim.x) * (kGatherThreads / 32)) {
    const long long group = (task >> 32) ? task / g.Hkv : static_cast<uint32_t>(task) / static_cast<uint32_t>(g.Hkv);
    const int h = static_cast<int>(task - group * g.Hkv);
    const long long n0 = group * (at_once * kGatherAhead) + mine;
    long long at[kGatherAhead];  // code places; -1: no such slot
#pragma unroll
    for (int k = 0; k < kGatherAhead; ++k) {
      const long long n = n0 + k * at_once;
      const int64_t slot = n < a.n ? a.rows[n] : -1;
      at[k] = -1;
      if (slot >= 0 && slot < slots) {
        const long long ph = (slot >> p_shift) * g.Hkv + h;
        const int off = static_cast<int>(slot & (g.P - 1));
        at[k] = ((ph << p_shift) + off) * g.D + d;
      }
    }
    uint2 w[2][kGatherAhead];
    float s[2][kGatherAhead];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int k = 0; k < kGatherAhead; ++k) {
        w[kv][k] = make_uint2(0, 0);
        s[kv][k] = 0.f;
        if (at[k] >= 0 && a.out[kv]) {
          w[kv][k] = __ldg(reinterpret_cast<const uint2 *>((kv ? a.c.v : a.c.k) + at[k]));
          s[kv][k] = __ldg((kv ? a.c.vs : a.c.ks) + (at[k] >> scale_shift));
        }
      }
    const long long step = static_cast<long long>(at_once) * g.Hkv * g.D;  // between two of a lane's rows
    const int rows_left = static_cast<int>(min(static_cast<long long>(kGatherAhead * at_once), a.n - n0));
    auto store = [&](bool vec) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (!a.out[kv]) continue;
        XT *to = static_cast<XT *>(a.out[kv]) + (n0 * g.Hkv + h) * g.D + d;
#pragma unroll
        for (int k = 0; k < kGatherAhead; ++k, to += step) {
          if (k * at_once >= rows_left) break;
          float f[kRun];
#pragma unroll
          for (int j = 0; j < kRun; ++j) {
            const uint32_t x = (j < 4 ? w[kv][k].x : w[kv][k].y) ^ 0x80808080u;
            f[j] = __fmul_rn(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440 | (j & 3))) - 8388736.f, s[kv][k]);
          }
          Run<XT>::store(to, f, vec);
        }
      }
    };
    if (a.vec) store(true);
    else store(false);
  }
}

bool is_pow2_in(int v, int lo, int hi) { return v >= lo && v <= hi && (v & (v - 1)) == 0; }

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

}  // namespace

Kv8Layer kv8_layer(const specdec_kv8 *h, const specdec_kv8_layer *l) {
  op_check(l && l->k && l->v && l->k_scale && l->v_scale && l->n_pages > 0, "null cache layer buffer, or no pages");
  op_check(aligned16(l->k) && aligned16(l->v), "cache code buffers must be 16-byte aligned");
  op_check(static_cast<long long>(l->n_pages) * h->g.Hkv * (h->g.P / h->g.t) <= 0x7fffffffll,
           "n_pages x n_kv_heads x blocks of a page must be below 2^31");
  return {l->k, l->v, l->k_scale, l->v_scale, l->n_pages};
}

Kv8Batch kv8_batch(const specdec_kv8 *h, const specdec_kv8_batch *b, int n_tokens) {
  op_check(b && b->n_requests >= 0 && b->n_requests <= h->cfg.max_batch, "n_requests must be in [0, max_batch]");
  op_check(b->n_requests == 0 || (b->table && b->kv_len && b->cu_q), "null batch buffer");
  op_check(b->table_cols > 0 && static_cast<long long>(b->table_cols) * h->g.P <= 0x7fffff00ll,
           "table_cols x page_tokens must be in [1, 2^31 - 256]");
  op_check(n_tokens >= 0, "negative row count");
  return {b->table, b->n_requests, b->table_cols, b->kv_len, b->cu_q, n_tokens};
}

}  // namespace specdec

using namespace specdec;

extern "C" {

int specdec_kv8_create(const specdec_kv8_config *cfg, int device, specdec_kv8 **out) {
  return op_guard(g_thread_err, [&] {
    op_check(out, "null output");
    *out = nullptr;
    op_check(cfg, "null config");
    const specdec_kv8_config &c = *cfg;
    op_check(c.n_heads > 0 && c.n_kv_heads > 0 && c.n_heads % c.n_kv_heads == 0,
             "n_heads must be a positive multiple of n_kv_heads");
    op_check(c.n_heads <= 65536, "n_heads must be at most 65536");
    op_check(is_pow2_in(c.head_dim, 16, 128), "head_dim must be 16, 32, 64 or 128");
    op_check(is_pow2_in(c.page_tokens, 16, 128), "page_tokens must be 16, 32, 64 or 128");
    op_check(is_pow2_in(c.block_tokens, 16, c.page_tokens), "block_tokens must be 16, 32, 64 or 128 and divide page_tokens");
    op_check(c.max_batch > 0 && c.max_batch <= kKv8MaxBatch, "max_batch must be in [1, 4096]");
    DeviceScope scope(device);
    auto h = std::make_unique<specdec_kv8>();
    h->cfg = c;
    h->g = {c.n_heads, c.n_kv_heads, c.n_heads / c.n_kv_heads, c.head_dim, c.page_tokens, c.block_tokens};
    h->device = device;
    op_cuda(cudaDeviceGetAttribute(&h->num_sms, cudaDevAttrMultiProcessorCount, device), "device attributes");
    op_cuda(cudaFuncSetAttribute(kv8_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (kKv8MaxBatch + 1) * kPlanBytes),
            "cudaFuncSetAttribute");
    kv8_attn_create(h.get());
    *out = h.release();
  });
}

int specdec_kv8_destroy(specdec_kv8 *h) {
  if (!h) return SPECDEC_OK;
  std::string err;
  const int rc = op_guard(err, [&] {
    DeviceScope scope(h->device);
    kv8_attn_destroy(h);
  });
  delete h;
  return rc;
}

const char *specdec_kv8_last_error(const specdec_kv8 *h) { return h ? h->err.c_str() : g_thread_err.c_str(); }

int specdec_kv8_plan(specdec_kv8 *h, const specdec_kv8_batch *batch, const int32_t *held, const int32_t *keep,
                     const int32_t *q_len, int32_t *ring, int ring_cap, const int32_t *ring_state, int32_t *ring_state_out,
                     void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    const Kv8Batch b = kv8_batch(h, batch, batch ? batch->max_tokens : 0);
    op_check((b.B == 0 || (held && keep && q_len)) && ring && ring_state && ring_state_out && ring_cap > 0,
             "null plan buffer, or an empty ring");
    op_check(b.cu_q, "null batch buffer");
    op_check(batch->status && (b.T == 0 || (batch->tok_req && batch->tok_pos && batch->slots)), "null batch buffer");
    const size_t n = sizeof(int32_t) * b.B, two = 2 * sizeof(int32_t);
    for (const int32_t *in : {held, keep, q_len})
      op_check(!overlap(in, n, b.kv_len, n) && !overlap(in, n, b.cu_q, n + 4), "plan inputs must not overlap its outputs");
    op_check(!overlap(ring_state, two, ring_state_out, two), "ring_state_out must not overlap ring_state");
    DeviceScope scope(h->device);
    const PlanArgs a{held, keep, q_len, b.table, b.B, b.cols, h->g.P, ring, ring_cap, ring_state, ring_state_out,
                     b.kv_len, b.cu_q, batch->tok_req, batch->tok_pos, batch->slots, b.T, batch->status};
    // a thread per row, in at most two blocks per multiprocessor: each repeats the scan
    const int work = std::max(b.T, b.B);
    const int grid = std::max(1, std::min(2 * h->num_sms, (work + kPlanThreads - 1) / kPlanThreads));
    op_launch("specdec_kv8_plan", kv8_plan_kernel, dim3(grid), kPlanThreads, (b.B + 1) * kPlanBytes,
              static_cast<cudaStream_t>(stream), 1, a);
  });
}

int specdec_kv8_append(specdec_kv8 *h, const specdec_kv8_layer *layer, const specdec_kv8_batch *batch, const void *k,
                       int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                       int64_t v_head_stride, int dtype, int n_tokens, void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    const Kv8Layer c = kv8_layer(h, layer);
    const Kv8Batch b = kv8_batch(h, batch, n_tokens);
    op_check(dtype == SPECDEC_F32 || dtype == SPECDEC_BF16, "rows must be SPECDEC_F32 or SPECDEC_BF16");
    if (b.B == 0 || b.T == 0) return;
    op_check(k && v, "null row buffer");
    DeviceScope scope(h->device);
    const int size = dtype == SPECDEC_F32 ? 4 : 2;
    auto vec = [&](const void *p, int64_t row, int64_t head) { return aligned16(p) && row * size % 16 == 0 && head * size % 16 == 0; };
    const AppendArgs a{h->g, c, b, {k, v}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride},
                       {vec(k, k_row_stride, k_head_stride), vec(v, v_row_stride, v_head_stride)}};
    const auto st = static_cast<cudaStream_t>(stream);
    dtype == SPECDEC_F32 ? append_any<float>(h, a, st) : append_any<__nv_bfloat16>(h, a, st);
  });
}

int specdec_kv8_gather(specdec_kv8 *h, const specdec_kv8_layer *layer, const int64_t *rows, int n, void *out_k,
                       void *out_v, int dtype, void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    const Kv8Layer c = kv8_layer(h, layer);
    op_check(dtype == SPECDEC_F32 || dtype == SPECDEC_BF16, "outputs must be SPECDEC_F32 or SPECDEC_BF16");
    op_check(n >= 0, "negative row count");
    if (n == 0 || (!out_k && !out_v)) return;
    op_check(rows, "null row list");
    DeviceScope scope(h->device);
    const GatherArgs a{h->g, c, rows, n, {out_k, out_v}, (!out_k || aligned16(out_k)) && (!out_v || aligned16(out_v))};
    const long long rows_a_warp = 32 / (h->g.D / kRun) * kGatherAhead;
    const long long warps = (n + rows_a_warp - 1) / rows_a_warp * h->g.Hkv;
    const int grid = static_cast<int>(std::min((warps + 7) / 8, 16ll * h->num_sms));
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == SPECDEC_F32)
      op_launch("specdec_kv8_gather", kv8_gather_kernel<float>, dim3(grid), kGatherThreads, 0, st, 1, a);
    else
      op_launch("specdec_kv8_gather", kv8_gather_kernel<__nv_bfloat16>, dim3(grid), kGatherThreads, 0, st, 1, a);
  });
}

}  // extern "C"
