// Attention over the 8-bit paged cache for many rows per kv head (chunks of a
// prompt, wide verify blocks): the formulas of kv8_attn.cu on tcgen05.
//
// With 128 and more rows every cached code meets all of them and the call is
// bound by its products and exponentials, not by HBM: a tile of 128 rows x 128
// positions x 128 dims is 256 tensor cycles a product, 1,024 cycles of
// exponentials (16 a cycle and SM) and about as many issue slots for the rest
// of the softmax.  One persistent block per SM takes 256 rows of a (request, kv
// head) at a time:
//   4 converter warps   codes from global memory through registers (one tile
//                       ahead) into f16 tiles of K and V in shared memory, two
//                       buffers each, 128-byte swizzle: once for 256 rows
//   1 issuing thread    S = Q K^T (M = 128 rows, N = 128 positions) and
//                       O += P V (A = P from tensor memory, N = D) for each of
//                       the two row tiles in turn
//   2 x 4 softmax warps one per row tile, thread = row = tensor memory lane:
//                       the maximum, then weights p = 2^(s - m) whose f16
//                       products with the value scales go back to tensor
//                       memory in the place of the scores
// The products of one row tile run while the other tile's warps are in their
// softmax.  Tensor memory: scores 2 x 128 columns, outputs 2 x D.  A row's
// maximum is moved (and its output rescaled) only when a weight would grow by
// 2^8.  The queries are scaled by a power of two per row: bf16 values down to
// 2^-17 of the row's largest are exact in f16, smaller ones off by up to 2^-25 of
// it; codes are whole numbers, exact too.
// Units (tiles of 128 positions) of all items are shared out evenly, as in
// kv8_attn.cu; partial results of an item meet in the workspace.  Every wait
// is bounded; one that gives up sets the handle's error word and ends the
// block after the products in flight.
//
// Measured (32 / 8 heads of 128): 4 requests of up to 509 rows over up to 4,096
// positions 119 us (52 GFLOP, 31 us at the measured 1,661 TFLOP/s), 512 rows
// over 8,192 in 116 us, 572 TFLOP/s; 8 x 2,048 rows over themselves with 32 / 32
// heads 524 us, 525 TFLOP/s.  The softmax bounds long items: of a unit's cycles
// a row's maximum takes 1,400 and its weights 2,900, on two warps a scheduler,
// and part of each wait for the products between them shows, in halves of 64
// positions (whole tiles: 188 us for the first).  Short items are bound by their
// start (7,000 cycles: queries in, a first score tile) and end (8,000: outputs
// out): 64 prompts of 128 rows over themselves 97 us.  There it took loads
// without a branch around each (166 us before), rows copied as they are and
// converted by their own thread, addresses without products.  Slower: 64
// columns of scores in registers at once (its loops outgrow the instruction
// cache), registers for the softmax taken from the converters (512 threads then
// share the same file: 152 us for the first where it was 140), a maximum over
// all of a half's scores at once (143).
#include <algorithm>

#include "gemm.cuh"
#include "kv8_attn.cuh"

namespace specdec {

namespace {

constexpr int kTileRows = 128;    // rows of a softmax warpgroup, lanes of tensor memory
constexpr int kItemRows = 256;
constexpr int kTilePos = 128;     // positions of a unit
constexpr int kSlices = kTilePos / 16;
constexpr int kSoftmaxThreads = 256;
constexpr int kConverterWarps = 4;
constexpr int kChunkThreads = kSoftmaxThreads + 32 * kConverterWarps + 32;
constexpr int kScaleSlots = 4;    // the scales of a tile stay until both softmax groups are past it
constexpr int kMergeParts = 8;

template <int D>
struct ChunkGeom {
  static constexpr int kAtom = kTilePos * 128;          // 64 dims of 128 rows, two bytes each
  static constexpr int kTile = D / 64 * kAtom;
  static constexpr int kTiles = 6 * kTile;              // Q of both row tiles, K and V twice
  static constexpr int kScales = kScaleSlots * (2 * kSlices + 4) * 4;
  static constexpr int kFixed = kTiles + kScales;
  static constexpr int kPart = kItemRows * (D + 2);     // floats of a partial result
};

constexpr int kHalfPos = kTilePos / 2;  // positions of a step of the softmax

// kind::f16, D fp32, A and B f16, M = 128.  S: A and B K-major, N = 64.  O: A from tensor memory, B (V) MN-major, N = D.
constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(kHalfPos >> 3) << 17) | (8u << 24);
template <int D>
constexpr uint32_t idesc_o() {
  return (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (8u << 24);
}

// MN-major operand of atoms of 64 columns (kAtom bytes apart), 128-byte swizzle; along K rows are 128 bytes apart,
// groups of 8 rows 1024 bytes.
__device__ __forceinline__ uint64_t desc_mn128(uint32_t saddr, int atom_bytes) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(atom_bytes >> 4) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}

// One lane of a converged warp.
__device__ __forceinline__ bool one_lane() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// D[tmem] (+)= A[tmem] B
__device__ __forceinline__ void tc_mma_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}

// 32 columns of the warp's 32 lanes: asked for (valid after tmem_wait_ld), and waited for.
__device__ __forceinline__ void tmem_ask32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ask16(uint32_t addr, uint32_t (&r)[16]) { tmem_ld16_nowait(addr, r); }
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  tmem_ask32(addr, r);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A phase of an mbarrier, for at most about two seconds; false: gave up, or another role did.
__device__ __forceinline__ bool chunk_wait(uint64_t *bar, uint32_t phase, volatile int *stop) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(addr), "r"(phase)
        : "memory");
    if (done) return true;
    if ((it & 63) == 63) {
      if (*stop) return false;
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > 2000000000ull) return false;
    }
  }
}
__device__ __forceinline__ void chunk_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A row tile pair of a request: 256 rows from row0, n of them there; its first unit along the cache and its units.
struct ChunkTile {
  int row0, n, t0, nt;
};
__device__ __forceinline__ ChunkTile chunk_tile(const AttendArgs &a, int q, int len, int rt) {
  ChunkTile t;
  t.row0 = rt * kItemRows;
  t.n = min(kItemRows, q * a.g.G - t.row0);
  const int first = len - q + row_at(a, t.row0).i, last = len - q + row_at(a, t.row0 + t.n - 1).i;  // positions of the rows
  t.t0 = a.window > 0 ? max(0, first - a.window + 1) / kTilePos : 0;
  t.nt = max(1, (last < 0 ? 0 : last / kTilePos + 1) - t.t0);
  return t;
}

// Walks consecutive units: request, kv head, row tile pair, unit.
struct ChunkCursor {
  int b, q0, q, len, nr, h, rt, unit;
  ChunkTile t;
  __device__ __forceinline__ void enter(const AttendArgs &a, const DecBatch &s, int req) {
    b = req;
    q0 = s.q0[b];
    q = s.q[b];
    len = s.len[b];
    nr = (q * a.g.G + kItemRows - 1) / kItemRows;
  }
  __device__ __forceinline__ void seek(const AttendArgs &a, const DecBatch &s, long long u) {
    enter(a, s, request_of(s.pre, a.b.B, u));
    const long long in = u - s.pre[b], per_head = (s.pre[b + 1] - s.pre[b]) / a.g.Hkv;
    h = static_cast<int>(in / per_head);
    long long left = in - h * per_head;
    for (rt = 0;; ++rt) {
      t = chunk_tile(a, q, len, rt);
      if (left < t.nt) break;
      left -= t.nt;
    }
    unit = static_cast<int>(left);
  }
  __device__ __forceinline__ void next(const AttendArgs &a, const DecBatch &s) {
    if (++unit < t.nt) return;
    unit = 0;
    if (++rt == nr) {
      rt = 0;
      if (++h == a.g.Hkv) {
        h = 0;
        int n = b + 1;
        while (n < a.b.B && s.pre[n + 1] == s.pre[n]) ++n;
        if (n == a.b.B) return;  // past the last unit
        enter(a, s, n);
      }
    }
    t = chunk_tile(a, q, len, rt);
  }
  __device__ __forceinline__ int pos() const { return (t.t0 + unit) * kTilePos; }
  // rows of row tile w, the positions of its first and last row
  __device__ __forceinline__ int rows(int w) const { return max(0, min(kTileRows, t.n - w * kTileRows)); }
  __device__ __forceinline__ int first(const AttendArgs &a, int w) const { return len - q + row_at(a, t.row0 + w * kTileRows).i; }
  __device__ __forceinline__ int last(const AttendArgs &a, int w) const {
    return len - q + row_at(a, t.row0 + w * kTileRows + rows(w) - 1).i;
  }
  // of the next `units` units, the first of which row tile w sees anything and the one after the last: equal if none
  __device__ __forceinline__ int2 sees(const AttendArgs &a, int w, int units) const {
    if (rows(w) == 0) return make_int2(0, 0);
    const int end = last(a, w), here = t.t0 + unit;
    const int lo = a.window > 0 ? max(0, max(0, first(a, w) - a.window + 1) / kTilePos - here) : 0;
    const int hi = min(units, end < 0 ? 0 : end / kTilePos + 1 - here);
    return hi > lo ? make_int2(lo, hi) : make_int2(0, 0);
  }
  // over the next `units` units, which end the item or the block's share
  __device__ __forceinline__ void skip(const AttendArgs &a, const DecBatch &s, int units) {
    unit += units - 1;
    next(a, s);
  }
};

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1) kv8_chunk_kernel(const __grid_constant__ AttendArgs a) {
  using Geo = ChunkGeom<D>;
  using XT = __nv_bfloat16;
  constexpr int kAtoms = D / 64;
  extern __shared__ unsigned char chunk_smem[];
  unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(chunk_smem) + 1023) & ~uintptr_t(1023));
  unsigned char *q_smem = base, *k_smem = base + 2 * Geo::kTile, *v_smem = base + 4 * Geo::kTile;
  float *scales = reinterpret_cast<float *>(base + Geo::kTiles);  // per slot: key scales, value scales, a byte for two slices
  DecBatch bt;
  bt.pre = reinterpret_cast<long long *>(base + Geo::kFixed);
  bt.q0 = reinterpret_cast<int *>(bt.pre + a.b.B + 1);
  bt.q = bt.q0 + a.b.B;
  bt.len = bt.q + a.b.B;
  __shared__ long long red[kChunkThreads / 32];
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], pv_done[2],
      q_full[2], o_full[2], mma_done;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_stop;
  __shared__ int s_last;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  constexpr int kIssuer = (kSoftmaxThreads >> 5) + kConverterWarps;

  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], kConverterWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kConverterWarps);
      mbar_init(&v_empty[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s_full[i][h], 1);
        mbar_init(&p_full[i][h], 4);
      }
      mbar_init(&pv_done[i], 1);
      mbar_init(&q_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(&mma_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_stop = 0;
  }
  request_prefix(a.b.B, bt.pre, red, [&](int b) {
    const Kv8Req r = kv8_req(a.b, a.g.P, b);
    bt.q0[b] = r.q0;
    bt.q[b] = r.q;
    bt.len[b] = r.len;
    long long n = 0;
    const int nr = (r.q * a.g.G + kItemRows - 1) / kItemRows;
    for (int rt = 0; rt < nr; ++rt) n += chunk_tile(a, r.q, r.len, rt).nt;
    return n * a.g.Hkv;
  });
  const long long total = bt.pre[a.b.B];
  const long long share = quotient(total + gridDim.x - 1, gridDim.x);
  const long long u0 = min(total, share * blockIdx.x), u1 = min(total, u0 + share);
  const int n_units = uniform(static_cast<int>(u1 - u0));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto give_up = [&]() {
    if (!s_stop) {
      s_stop = 1;
      if (a.err) atomicOr(a.err, 1);
    }
  };

  if (warp >= (kSoftmaxThreads >> 5) && warp < kIssuer) {
    // ---- converters ----------------------------------------------------------
    // A warp has 32 positions of a tile: of 8 positions at a time 4 lanes read 64 codes each, one 64-dim atom after the other.
    const int w = warp - (kSoftmaxThreads >> 5), row_in = lane >> 2, c16 = lane & 3;
    constexpr int kLoads = 4 * kAtoms;
    uint4 rk[kLoads], rv[kLoads];
    float sc = 0.f;
    uint32_t there = 0;
    ChunkCursor cur;
    int left = n_units;
    if (left > 0) cur.seek(a, bt, u0);
    int pages[4];
    auto find_pages = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = cur.pos() + 32 * w + 8 * i;
        const int page = p < cur.len ? a.b.table[static_cast<long long>(cur.b) * a.b.cols + (p >> a.p_shift)] : -1;
        pages[i] = page >= 0 && page < a.c.n_pages ? page : -1;
      }
    };
    auto load = [&](const int8_t *src, uint4 (&r)[kLoads]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = cur.pos() + 32 * w + 8 * i + row_in;
        const long long ph = static_cast<long long>(pages[i]) * a.g.Hkv + cur.h;
        const long long at = ((ph << a.p_shift) + (p & (a.g.P - 1))) * D + 16 * c16;
#pragma unroll
        for (int t = 0; t < kAtoms; ++t)
          r[i * kAtoms + t] = pages[i] >= 0 ? __ldg(reinterpret_cast<const uint4 *>(src + at + 64 * t)) : make_uint4(0, 0, 0, 0);
      }
    };
    auto put = [&](unsigned char *dst, const uint4 (&r)[kLoads]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 32 * w + 8 * i + row_in;
#pragma unroll
        for (int t = 0; t < kAtoms; ++t) {
          const uint4 v = r[i * kAtoms + t];
          const uint32_t x[4] = {v.x, v.y, v.z, v.w};
          uint32_t f[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t y = x[j] ^ 0x80808080u;
            f[2 * j] = f16_codes(__byte_perm(y, 0x64646464u, 0x4140));
            f[2 * j + 1] = f16_codes(__byte_perm(y, 0x64646464u, 0x4342));
          }
          unsigned char *line = dst + t * Geo::kAtom + row * 128;
          *reinterpret_cast<uint4 *>(line + (((2 * c16) ^ (row & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
          *reinterpret_cast<uint4 *>(line + (((2 * c16 + 1) ^ (row & 7)) << 4)) = make_uint4(f[4], f[5], f[6], f[7]);
        }
      }
    };
    // lanes 0 .. 3 of a warp: key and value scales of its two slices
    auto load_scales = [&]() {
      const int slice = 2 * w + (lane >> 1 & 1), p = cur.pos() + 16 * slice;
      const int page = (lane & 2) ? pages[2] : pages[0];
      sc = 0.f;
      if (lane < 4 && page >= 0) {
        const long long ph = static_cast<long long>(page) * a.g.Hkv + cur.h;
        sc = ((lane & 1) ? a.c.vs : a.c.ks)[(ph << (a.p_shift - a.t_shift)) + ((p & (a.g.P - 1)) >> a.t_shift)];
      }
      there = __ballot_sync(0xffffffffu, lane < 2 && (lane ? pages[2] : pages[0]) >= 0);
    };
    auto publish = [&](uint64_t *bar) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) chunk_arrive(bar);
    };
    if (left > 0) {
      find_pages();
      load(a.c.k, rk);
      load(a.c.v, rv);
      load_scales();
    }
    bool ok = true;
    for (int n = 0; left > 0 && ok; ++n, --left) {
      const int buf = n & 1;
      const uint32_t ph = (n >> 1) & 1;
      ok = chunk_wait(&k_empty[buf], ph ^ 1, &s_stop);
      if (!ok) break;
      put(k_smem + buf * Geo::kTile, rk);
      float *slot = scales + (n % kScaleSlots) * (2 * kSlices + 4);
      if (lane < 4) slot[(lane & 1) * kSlices + 2 * w + (lane >> 1)] = sc;
      const uint32_t below = __ballot_sync(0xffffffffu, lane < 4 && sc < 0.f);  // of bits 0 and 2: key scales below 0
      if (lane == 0)
        reinterpret_cast<unsigned char *>(slot + 2 * kSlices)[w] =
            static_cast<unsigned char>(there | (below & 1) << 2 | (below & 4) << 1);
      publish(&k_full[buf]);
      uint4 keep[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) keep[i] = rv[i];
      if (left > 1) {
        cur.next(a, bt);
        find_pages();
        load(a.c.k, rk);
        load(a.c.v, rv);
        load_scales();
      }
      ok = chunk_wait(&v_empty[buf], ph ^ 1, &s_stop);
      if (!ok) break;
      put(v_smem + buf * Geo::kTile, keep);
      publish(&v_full[buf]);
    }
    if (!ok) give_up();
  } else if (warp == kIssuer) {
    // ---- products --------------------------------------------------------------
    // The whole warp walks and waits, so that what describes the products is uniform; one lane issues them.
    if (n_units > 0) {
      const bool leader = one_lane();
      bool ok = true;
      uint32_t acts[2] = {0, 0}, segs[2] = {0, 0};  // units and segments of each row tile so far
      ChunkCursor cur;
      cur.seek(a, bt, u0);
      // descriptors hold addresses in 16-byte units in their low bits: offsets are added there
      const uint64_t q_desc = umma_desc_k128(smem_u32(q_smem)), k_desc = umma_desc_k128(smem_u32(k_smem));
      const uint64_t v_desc = desc_mn128(smem_u32(v_smem), Geo::kAtom);
      auto scores = [&](int w, int h, int n) {  // of half h of unit n
        const uint64_t qd = q_desc + (w * Geo::kTile >> 4), kd = k_desc + (((n & 1) * Geo::kTile + h * kHalfPos * 128) >> 4);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t at = ((kk >> 2) * Geo::kAtom + 32 * (kk & 3)) >> 4;
            tc_mma(tmem + 128 * w + kHalfPos * h, qd + at, kd + at, kIdescS, kk ? 1u : 0u);
          }
          tc_commit(&s_full[w][h]);
        }
      };
      auto commit = [&](uint64_t *bar) {
        if (leader) tc_commit(bar);
      };
      auto wait = [&](uint64_t *bar, uint32_t phase) { return __all_sync(0xffffffffu, chunk_wait(bar, phase, &s_stop)) != 0; };
      for (int n = 0; n < n_units && ok;) {
        const int units = min(cur.t.nt - cur.unit, n_units - n);
        const int2 see[2] = {cur.sees(a, 0, units), cur.sees(a, 1, units)};
        // A new segment's scores wait for its queries, which come after both groups have their outputs: not before both
        // groups' products are issued.  K and V of every unit are waited for: phases are told apart by parity
        ok = wait(&k_full[n & 1], (n >> 1) & 1);
#pragma unroll 1
        for (int w = 0; w < 2; ++w)
          if (ok && (w ? see[1].x : see[0].x) == 0 && (w ? see[1].y : see[0].y) > 0) {
            ok = wait(&q_full[w], (w ? segs[1]++ : segs[0]++) & 1);
            tc_fence_after();
            if (ok) {
              scores(w, 0, n);
              scores(w, 1, n);
            }
          }
        commit(&k_empty[n & 1]);
        for (int i = 0; i < units && ok; ++i, ++n) {
          const bool more = i + 1 < units;
          ok = wait(&v_full[n & 1], (n >> 1) & 1);
          if (ok && more) ok = wait(&k_full[(n + 1) & 1], ((n + 1) >> 1) & 1);
#pragma unroll 1
          for (int h = 0; h < 2; ++h)
#pragma unroll 1
            for (int w = 0; w < 2; ++w) {
              const bool here = i >= (w ? see[1].x : see[0].x) && i < (w ? see[1].y : see[0].y);
              const bool then = more && i + 1 >= (w ? see[1].x : see[0].x) && i + 1 < (w ? see[1].y : see[0].y);
              if (ok && here) {
                ok = wait(&p_full[w][h], (w ? acts[1] : acts[0]) & 1);
                tc_fence_after();
                const uint64_t vd = v_desc + (((n & 1) * Geo::kTile + h * kHalfPos * 128) >> 4);
                const uint32_t later = h == 1 || i > (w ? see[1].x : see[0].x);
                if (ok && leader) {
#pragma unroll
                  for (int kk = 0; kk < kHalfPos / 16; ++kk)
                    tc_mma_ta(tmem + 256 + 128 * w, tmem + 128 * w + kHalfPos * h + 8 * kk, vd + (2048 * kk >> 4), idesc_o<D>(), kk ? 1u : later);
                  tc_commit(&pv_done[w]);
                }
              }
              if (ok && then) {
                if (h == 0 && !here) ok = wait(&q_full[w], (w ? segs[1]++ : segs[0]++) & 1);
                tc_fence_after();
                if (ok) scores(w, h, n + 1);
              }
            }
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (i >= see[w].x && i < see[w].y) ++acts[w];
            if (!more && ok && see[w].y > 0) commit(&o_full[w]);
          }
          commit(&v_empty[n & 1]);
          if (more) commit(&k_empty[(n + 1) & 1]);
        }
        cur.skip(a, bt, units);
      }
      if (!ok) give_up();
      commit(&mma_done);  // every product has ended before the block moves on
      if (!chunk_wait(&mma_done, 0, &s_stop) && !mbar_wait(&mma_done, 0)) give_up();
    }
  } else if (warp < (kSoftmaxThreads >> 5)) {
    // ---- softmax and output: thread = row -------------------------------------------
    const int w = warp >> 2, r = threadIdx.x & 127, r_item = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t s_at = tmem + lanes + 128 * w, o_at = tmem + lanes + 256 + 128 * w;
    constexpr int kRowLanes = D / 8;  // lanes of a row where a warp goes through its 32 rows together
    // the row that a lane has in such a pass: its place in a row array, and on to the next without a product or a division
    struct RowWalk {
      const XT *p;
      long long step, wrap;
      int h;
      __device__ __forceinline__ void next(int G) {
        h += 32 / kRowLanes;
        p += step;
        while (h >= G) {
          h -= G;
          p += wrap;
        }
      }
    };
    auto walk = [&](const ChunkCursor &c, int w, const XT *base, long long row, long long head) {
      const RowAt of = row_at(a, c.t.row0 + kTileRows * w + 32 * (warp & 3) + lane / kRowLanes);
      return RowWalk{base + (c.q0 + of.i) * row + (c.h * a.g.G + of.h) * head, 32 / kRowLanes * head, row - a.g.G * head, of.h};
    };
    ChunkCursor cur;
    if (n_units > 0) cur.seek(a, bt, u0);
    bool ok = true;
    int n_act = 0, n_seg = 0, n_pv = 0;
    for (int n = 0; n < n_units;) {
      // the segment: units of the item within this block's share
      const int units = min(cur.t.nt - cur.unit, n_units - n);
      const int rows = cur.rows(w), first_pos = rows > 0 ? cur.first(a, w) : 0, last_pos = rows > 0 ? cur.last(a, w) : -1;
      const int p_begin = cur.pos();
      const int2 see = cur.sees(a, w, units);
      const bool any = see.y > 0;
      const RowAt at_row = row_at(a, cur.t.row0 + r_item);
      const bool live = r < rows;
      const int lim = live ? cur.len - cur.q + at_row.i : -1;
      const long long token = cur.q0 + at_row.i;
      const int head = cur.h * a.g.G + at_row.h;
      float m = kNone, l = 0.f, l_err = 0.f, cs = 0.f;  // l_err: what the last additions to l were too much by
      // eight dims of a row in the query tile, for its queries and later for its outputs: a warp's rows are its own, so
      // that a warp that is through with its outputs may bring in the next segment's queries
      unsigned char *tile = q_smem + w * Geo::kTile;
      auto place = [&](int row, int run) { return tile + (run >> 3) * Geo::kAtom + row * 128 + (((run & 7) ^ (row & 7)) << 4); };
      if (any && ok) {
        // the warp's 32 query rows to their places as they are, neighbouring lanes along a row; then each thread brings its
        // row to a power of two times f16 (NaN where the row has a value that is not finite)
        const int run = lane % kRowLanes;
        RowWalk at = walk(cur, w, static_cast<const XT *>(a.q) + 8 * run, a.q_row, a.q_head);
#pragma unroll 2
        for (int it = 0; it < kRowLanes; ++it, at.next(a.g.G)) {
          const int rr = 32 * (warp & 3) + it * (32 / kRowLanes) + lane / kRowLanes;
          const XT *src = rr < rows ? at.p : static_cast<const XT *>(a.q);
          if (a.q_vec8) {  // zeros past the last row
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(place(rr, run))), "l"(src), "r"(rr < rows ? 16 : 0)
                         : "memory");
          } else {
            const unsigned short *u = reinterpret_cast<const unsigned short *>(src);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (rr < rows) v = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
            *reinterpret_cast<uint4 *>(place(rr, run)) = v;
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        // bits of the row's largest |x|; those of an infinity or a NaN are the largest there are
        uint32_t top2 = 0;
#pragma unroll 4
        for (int run = 0; run < kRowLanes; ++run) {
          const uint4 v = *reinterpret_cast<const uint4 *>(place(r, run));
          auto mag = [](uint32_t v) {
            v &= 0x7fff7fffu;
            return *reinterpret_cast<const __nv_bfloat162 *>(&v);
          };
          const __nv_bfloat162 m2 = __hmax2_nan(__hmax2_nan(__hmax2_nan(mag(v.x), mag(v.y)), __hmax2_nan(mag(v.z), mag(v.w))), mag(top2));
          top2 = *reinterpret_cast<const uint32_t *>(&m2);
        }
        const uint32_t big = max(top2 << 16, top2 & 0xffff0000u);
        const float bad = big < 0x7f800000u ? 0.f : __uint_as_float(0x7fc00000u);
        const int e = min(max(static_cast<int>(big >> 23) - 127, -100), 126);
        const float down = __uint_as_float((127 - e) << 23) * (a.scale < 0.f ? -1.f : 1.f);
        cs = (__uint_as_float((127 + e) << 23) + bad) * (fabsf(a.scale) * kLog2e);
#pragma unroll 4
        for (int run = 0; run < kRowLanes; ++run) {
          const uint4 v = *reinterpret_cast<const uint4 *>(place(r, run));
          auto halves = [&](uint32_t v) { return pack_f16(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xffff0000u) * down); };
          *reinterpret_cast<uint4 *>(place(r, run)) = make_uint4(halves(v.x), halves(v.y), halves(v.z), halves(v.w));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) chunk_arrive(&q_full[w]);
      }
      bool opened = false;
      for (int i = 0; i < units; ++i, ++n) {
        const int p0 = p_begin + i * kTilePos;
        if (!ok || i < see.x || i >= see.y) continue;
#pragma unroll 1
        for (int half = 0; half < 2 && ok; ++half) {
        const int c_half = half * (kSlices / 2);                     // the half's first slice
        const uint32_t h_at = s_at + kHalfPos * half;
        ok = chunk_wait(&s_full[w][half], n_act & 1, &s_stop);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const float *slot = scales + (n % kScaleSlots) * (2 * kSlices + 4);
        const uint32_t there4 = *reinterpret_cast<const uint32_t *>(slot + 2 * kSlices);  // a byte for two slices: bits 0, 1 there,
                                                                                          // bits 2, 3 a key scale below 0
        const bool whole = p0 + kTilePos - 1 <= first_pos && (a.window <= 0 || p0 > last_pos - a.window) && there4 == 0x03030303u;
        // bit j: whether this row sees column 16 c + j
        auto seen = [&](int c) -> uint32_t {
          const int n = lim - (p0 + 16 * c) + 1;  // columns up to the row's own position
          uint32_t v = n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1;
          if (a.window > 0) {
            const int k = n - a.window;  // columns before the window
            v = k <= 0 ? v : k >= 16 ? 0u : v & (~0u << k);
          }
          return (there4 >> (8 * (c >> 1) + (c & 1)) & 1) ? v : 0u;
        };
        // the largest weight x value scale, by exponent
        float top = kNone;
        auto top_of = [&](const float (&s)[16], int c) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fmaxf(s[j], s[j + 8]);
          const float m4 = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
          const float ev = static_cast<float>(max(static_cast<int>(__float_as_uint(slot[kSlices + c]) >> 23 & 0xff) - 127, kScaleFloor));
          if (m4 != -INFINITY) top = fmaxf(top, fmaf(m4, cs * fabsf(slot[c]), ev));
        };
        if (whole) {  // a slice's scores are asked for while the one before is worked on
          uint32_t x[2][16];
          tmem_ask16(h_at, x[0]);
#pragma unroll
          for (int c = 0; c < kSlices / 2; ++c) {
            tmem_wait_ld();
            if (c + 1 < kSlices / 2) tmem_ask16(h_at + 16 * (c + 1), x[(c + 1) & 1]);
            float s[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = __uint_as_float(x[c & 1][j]);
            top_of(s, c_half + c);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kSlices / 2; ++c) {
            float s[16];
            tmem_ld16(h_at + 16 * c, s);
            const uint32_t v = seen(c_half + c);
            const int slice = c_half + c;
            const float sign = there4 >> (8 * (slice >> 1) + 2 + (slice & 1)) & 1 ? -1.f : 1.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] = (v >> j & 1) ? s[j] * sign : -INFINITY;
            top_of(s, slice);
          }
        }
        if (__any_sync(0xffffffffu, top > m + (kLazy + kRoom))) {
          const float nm = top > m + (kLazy + kRoom) ? top - kRoom : m;
          const float al = exp2_fast(m - nm);
          m = nm;
          l *= al;
          l_err *= al;
          if (opened) {  // once the last step's product has ended (those before it have: these scores were issued after them)
            ok = chunk_wait(&pv_done[w], (n_pv - 1) & 1, &s_stop);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              uint32_t x[16];
              tmem_ld32(o_at + 32 * c, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(o[j] * al);
              tmem_st16(o_at + 32 * c, x);
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(o[16 + j] * al);
              tmem_st16(o_at + 32 * c + 16, x);
            }
          }
        }
        // The weights take the place of scores that have been read: 8 columns a slice, the scores 16 columns ahead of them.
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (whole) {
          uint32_t x[2][16];
          tmem_ask16(h_at, x[0]);
#pragma unroll
          for (int c = 0; c < kSlices / 2; ++c) {
            tmem_wait_ld();
            if (c + 1 < kSlices / 2) tmem_ask16(h_at + 16 * (c + 1), x[(c + 1) & 1]);
            const float k = cs * slot[c_half + c], vsc = slot[kSlices + c_half + c];
            uint32_t f[8];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float p = exp2_fast(fmaf(__uint_as_float(x[c & 1][j]), k, -m));
              const float q = exp2_fast(fmaf(__uint_as_float(x[c & 1][j + 1]), k, -m));
              sum[j & 2] += p;
              sum[(j & 2) + 1] += q;
              f[j / 2] = pack_f16(p * vsc, q * vsc);
            }
            tmem_st8(h_at + 8 * c, f);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kSlices / 2; ++c) {
            float s[16];
            tmem_ld16(h_at + 16 * c, s);
            const float k = cs * slot[c_half + c], vsc = slot[kSlices + c_half + c];
            const uint32_t v = seen(c_half + c);
            uint32_t f[8];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {  // a scale that a row does not see may be anything
              const float p = (v >> j & 1) ? exp2_fast(fmaf(s[j], k, -m)) : 0.f;
              const float q = (v >> j & 2) ? exp2_fast(fmaf(s[j + 1], k, -m)) : 0.f;
              sum[0] += p;
              sum[1] += q;
              f[j / 2] = pack_f16((v >> j & 1) ? p * vsc : 0.f, (v >> j & 2) ? q * vsc : 0.f);
            }
            tmem_st8(h_at + 8 * c, f);
          }
        }
        // compensated: halves of a long tail must not vanish beside one large weight (2,048 halves of 131,072 positions
        // could lose 6e-5 of the sum)
        const float add = ((sum[0] + sum[1]) + (sum[2] + sum[3])) - l_err, grown = l + add;
        l_err = (grown - l) - add;
        l = grown;
        opened = true;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) chunk_arrive(&p_full[w][half]);
        ++n_pv;
        }
        ++n_act;
      }
      // ---- end of the segment -------------------------------------------------------
      if (any && ok) {
        ok = chunk_wait(&o_full[w], n_seg++ & 1, &s_stop);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      uint32_t all_ok;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                   : "=r"(all_ok)
                   : "r"(static_cast<uint32_t>(ok))
                   : "memory");
      if (!all_ok) {
        ok = false;
        break;
      }
      const long long i0 = u0 + (n - units) - cur.unit, i1 = i0 + cur.t.nt;
      const bool all = i0 >= u0 && i1 <= u1;
      // outputs leave through the query tile of the warp's rows, whose products have ended, so that a row is written by
      // neighbouring lanes
      auto put = [&](int run, const float (&v)[8]) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          x[j] = *reinterpret_cast<const uint32_t *>(&t);
        }
        *reinterpret_cast<uint4 *>(place(r, run)) = make_uint4(x[0], x[1], x[2], x[3]);
      };
      auto flush = [&]() {
        __syncwarp();
        const int run = lane % kRowLanes;
        auto row_in = [&](int it) { return 32 * (warp & 3) + it * (32 / kRowLanes) + lane / kRowLanes; };
        RowWalk at = walk(cur, w, static_cast<const XT *>(a.out) + 8 * run, a.o_row, a.o_head);
        auto staged = [&](int rr) { return *reinterpret_cast<const uint4 *>(place(rr, run)); };
        if (a.o_vec8) {
#pragma unroll 4
          for (int it = 0; it < kRowLanes; ++it, at.next(a.g.G)) {
            const uint4 v = staged(row_in(it));
            if (row_in(it) < rows) *reinterpret_cast<uint4 *>(const_cast<XT *>(at.p)) = v;
          }
        } else {
#pragma unroll 1
          for (int it = 0; it < kRowLanes; ++it, at.next(a.g.G)) {
            if (row_in(it) >= rows) continue;
            const uint4 v = staged(row_in(it));
            unsigned short *dst = reinterpret_cast<unsigned short *>(const_cast<XT *>(at.p));
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = static_cast<unsigned short>(x[j >> 1] >> (16 * (j & 1)));
          }
        }
        __syncwarp();
      };
      auto finish = [&](float lsum, float top) {
        if (live && a.lse) a.lse[token * a.g.H + head] = lsum == 0.f ? -INFINITY : logf(lsum) + top * kLn2;
        return lsum == 0.f ? 0.f : __fdividef(1.f, lsum);  // 0: the row saw nothing
      };
      float4 *part = reinterpret_cast<float4 *>(a.part + (2 * static_cast<long long>(blockIdx.x) + (i0 >= u0 ? 1 : 0)) * Geo::kPart);
      const float inv = all ? finish(l, m) : 1.f;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        if (any) {
          tmem_ld32(o_at + 32 * c, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = o[j + k] * inv;
          if (all) {
            put(4 * c + j / 8, v);
          } else {
            part[(8 * c + j / 4) * kItemRows + r_item] = make_float4(v[0], v[1], v[2], v[3]);
            part[(8 * c + j / 4 + 1) * kItemRows + r_item] = make_float4(v[4], v[5], v[6], v[7]);
          }
        }
      }
      if (all) flush();
      if (!all) {
        float *ml = reinterpret_cast<float *>(part) + kItemRows * D;
        ml[r_item] = m;
        ml[kItemRows + r_item] = l;
        const int c0 = static_cast<int>(quotient(i0, share)), c1 = static_cast<int>(quotient(i1 - 1, share));
        __threadfence();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (threadIdx.x == 0) s_last = atomicAdd(a.ticket + c0, 1) == c1 - c0;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s_last) {
          __threadfence();
          auto part_of_block = [&](int c) { return a.part + (2ll * c + (c == c0)) * Geo::kPart; };
          float top = kNone, lsum = 0.f;
          for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(part_of_block(c) + kItemRows * D + r_item));
          for (int c = c0; c <= c1; ++c) {
            const float *pm = part_of_block(c) + kItemRows * D + r_item;
            lsum += __ldcg(pm + kItemRows) * exp2_fast(__ldcg(pm) - top);
          }
          const float inv_all = finish(lsum, top);
#pragma unroll 1
          for (int d = 0; d < D / 4; d += kMergeParts) {
            float4 v[kMergeParts];
#pragma unroll
            for (int j = 0; j < kMergeParts; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = c0; c <= c1; ++c) {
              const float *p = part_of_block(c);
              const float f = exp2_fast(__ldcg(p + kItemRows * D + r_item) - top) * inv_all;
#pragma unroll
              for (int j = 0; j < kMergeParts; ++j) {
                const float4 y = __ldcg(reinterpret_cast<const float4 *>(p) + (d + j) * kItemRows + r_item);
                v[j].x += y.x * f; v[j].y += y.y * f; v[j].z += y.z * f; v[j].w += y.w * f;
              }
            }
#pragma unroll
            for (int j = 0; j < kMergeParts; j += 2) {
              const float y[8] = {v[j].x, v[j].y, v[j].z, v[j].w, v[j + 1].x, v[j + 1].y, v[j + 1].z, v[j + 1].w};
              put((d + j) / 2, y);
            }
          }
          flush();
          asm volatile("bar.sync 1, 256;" ::: "memory");
          if (threadIdx.x == 0) a.ticket[c0] = 0;
        }
      }
      tc_fence_before();
      cur.skip(a, bt, units);
    }
    if (!ok) give_up();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssuer)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D>
int chunk_smem_bytes(int B) {
  return 1024 + ChunkGeom<D>::kFixed + (B + 1) * static_cast<int>(sizeof(long long)) + 3 * B * static_cast<int>(sizeof(int));
}

}  // namespace

void kv8_chunk_create(specdec_kv8 *h) {
  if (h->g.D < 64) return;
  if (h->g.D == 64)
    op_cuda(cudaFuncSetAttribute(kv8_chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, chunk_smem_bytes<64>(kChunkMaxBatch)),
            "cudaFuncSetAttribute");
  else
    op_cuda(cudaFuncSetAttribute(kv8_chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, chunk_smem_bytes<128>(kChunkMaxBatch)),
            "cudaFuncSetAttribute");
}

size_t kv8_chunk_part_bytes(const specdec_kv8 *h) {
  if (h->g.D < 64) return 0;
  return static_cast<size_t>(h->num_sms) * 2 * (kItemRows * (h->g.D + 2)) * sizeof(float);
}

void kv8_chunk_launch(const specdec_kv8 *h, const AttendArgs &a, cudaStream_t st) {
  if (h->g.D == 64)
    op_launch("specdec_kv8_attend", kv8_chunk_kernel<64>, dim3(h->num_sms), kChunkThreads, chunk_smem_bytes<64>(a.b.B), st, 1, a);
  else
    op_launch("specdec_kv8_attend", kv8_chunk_kernel<128>, dim3(h->num_sms), kChunkThreads, chunk_smem_bytes<128>(a.b.B), st, 1, a);
}

}  // namespace specdec
