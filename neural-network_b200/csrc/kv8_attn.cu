// Attention over the 8-bit paged cache (specdec_kv8_attend).
//
// Per query row and head: s_j = scale sk(j) (q . ck_j), p_j = exp(s_j - m),
// out = sum p_j sv(j) cv_j / sum p_j, with one scale pair per block of
// positions.  Both products run on the tensor cores over the codes
// themselves (whole numbers up to 127, exact in f16 too) and the scales enter
// the scores and the weights.
//
// Few rows per kv head (decode steps, verify blocks): kv8_decode_kernel.  The
// cache is read once and every byte meets at most 16 rows, so HBM bounds it.
// The cache is the products' A operand (16 positions or 16 dims a tile), the
// rows are their N side (8 or 16 columns), which wastes nothing of the tensor
// cores that a 128-row tile would need:
//   S^T [16 positions][8 rows]  = K codes [16][D] x Q^T      8-bit products
//   O^T [16 dims][8 rows]      += V^T codes [16 dims][16 positions] x P^T   f16
// The queries enter as whole numbers of three bytes (22 bits of the row's
// largest value), so the K codes need no conversion and the scores' sums are
// exact; the weights span too many binades for that and enter as f16 (11 bits;
// for fp32 rows a second f16 of what is left, 22 bits), a few binades above 1 at
// the largest weight x value scale (kRoom, kLowUp).
// A slice of 16 positions lies in one page and has one scale pair.  Every
// warp takes two slices a step from a ring in shared memory that it fills
// itself with 16-byte asynchronous copies (no barrier between warps until the
// end of an item), converts V codes to f16 in registers, and keeps its running
// maximum, sum and output; the block's warps take steps in turn and merge at
// the end of a (request, kv head, row tile) item.  A row's maximum moves only
// when a weight would grow by 2^8: most steps rescale nothing.
//
// Work is split evenly whatever the lengths are: all items' 128-position units
// in a row, an equal share of consecutive units per block.  A block that holds
// part of an item leaves (maximum, sum, unnormalised output) in the workspace
// and the last of the item's blocks to arrive merges them in block order, so
// equal calls give equal bits.
//
// Measured (bf16 rows, heads of 128, of the measured 6.55 TB/s):
//   32 requests of up to 3,080 positions, 5 rows, 32 / 32 heads:  97 us, 5.3 TB/s (0.80); fp32 rows with an empty L2 115, bf16 109
//   64 requests of up to 4,096, 1 row, 32 / 8 heads:              69 us, 5.0 TB/s (0.76)
//   2 requests of 131,071, 1 row, 32 / 8 heads:                   97 us, 5.5 TB/s (0.84)
//   4 requests of up to 509 fp32 rows over up to 4,096, 32 / 8:  440 us (bf16 rows on the tensor tiles 119)
//   8 requests of up to 100, 1 fp32 row, 4 heads of 64:          8.2 us: latency
// The copies alone, without products, run the third in 81 us; conversions,
// softmax and products take issue slots beside them.  On the way (first case / second / third): codes converted for both products 179 /
// 121 / 178, scores from bytes 127 / 88 / 134, two slices a step 115 /
// 82 / 113, queries in shared memory instead of
// registers and one V buffer 97 / 71 / 101 (three blocks a multiprocessor).
// Four blocks of 128 registers spill: 118 / 87 / 113.
#include "kv8_attn.cuh"

#include <cuda_fp16.h>

#include <cmath>

namespace specdec {

namespace {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kSlice = 16;                            // positions of a slice
constexpr int kStep = 2;                              // slices a warp takes at a time: one page, or two of 16 positions
constexpr int kUnit = kSlice * kStep * kDecWarps;     // positions of a unit
constexpr int dec_ctas(int nt) { return nt == 1 ? 3 : 2; }  // blocks per SM: registers
constexpr int kChunkRows = 64;                        // rows of a kv head from which the tensor tiles are faster, given
constexpr int kChunkUnits = 24;                       // this many of this kernel's units for each of its blocks, or
constexpr float kChunkItems = 1.5f;                   // this many of its items
constexpr int kMergeAhead = 8;                        // partial results read at once
// Steps (of 32 positions) after which a warp's running sums are added to far sums in shared memory and begin anew.  One
// weight far above a long tail would swallow what follows it, since a lane adds single weights to its sum, and the tensor
// cores cut an output off at its last bit with every product.  Sixteen steps leave 64 additions and, for fp32 rows, 64
// products in a run.  64 requests of 100,000 positions, one of them 14 to 22 nats above the others, heads of 128: the
// log-sum-exp is off by 5e-6 (1.3e-4 in one run and with weights in steps of 2^-24 of the largest), outputs of fp32 rows by
// 3.3e-6 of the largest value (1.9e-4), with equal weights by 1.7e-7 (7.2e-6); verify rows as below, but fp32, take 115 us
// (109).  The outputs of bf16 rows stay in one run: up to 2^-24 of them for each 16 positions of a warp's quarter of its
// block's share, less than half a last bit of theirs below a million positions.
constexpr int kRunSteps = 16;
template <typename XT, int D, int NT>
struct DecGeom {
  static constexpr int kRows = 8 * NT;
  static constexpr int kSliceBytes = kSlice * D;            // K or V codes of a slice
  static constexpr int kHalf = kStep * kSliceBytes;         // K or V codes of a step; a multiple of 128: places within a
                                                            // row are XORed into addresses
  static constexpr int kTail = 8 * kStep;                   // per slice: the key and the value scale
  static constexpr int kRing = kDecWarps * 3 * kHalf;       // per warp two K buffers and one V buffer
  static constexpr int kTails = kDecWarps * 2 * kTail;
  static constexpr int kQuery = 3 * NT * 32 * (D / 4);      // the rows' three bytes as the products take them
  static constexpr bool kWide = sizeof(XT) == 4;            // fp32 rows: outputs have far sums too
  static constexpr int kFarRow = kWide ? 1 + D / 16 : 1;    // per eight rows and thread: (sums, maxima) of two columns, outputs
  static constexpr int kFar = NT * kFarRow * kDecThreads * 16;
  static constexpr int kFixed = kRing + kTails + kQuery + kFar;
  static constexpr int kPart = kRows * D + 2 * kRows;       // floats of a partial result
  static_assert(8 * D * 4 == kHalf, "a warp's output of eight rows fits the V buffer that it has just read");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t shared_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8 x 16-byte matrices, one row address per lane: lane l gets bytes 4 (l % 4) .. of row l / 4 of each.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix2(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
  r[2] = r[3] = 0;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// d = a b, and d += a b
__device__ __forceinline__ void mma16832_first(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, "
      "%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma16832(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 matrix of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }

// Place of a 16-byte chunk of a slice row in shared memory.  K rows are read
// eight at a time at one chunk: the chunks of rows that start in the same bank
// are spread.  V rows are read 8 lanes along a row and 4 rows (2t) at once.
template <int D>
__device__ __forceinline__ int k_place(int row, int chunk) {
  if constexpr (D == 128) return row * D + 16 * (chunk ^ (row & 7));
  if constexpr (D == 64) return row * D + 16 * (chunk ^ ((row >> 1) & 3));
  if constexpr (D == 32) return row * D + 16 * (chunk ^ ((row >> 2) & 1));
  return row * D + 16 * chunk;
}
template <int D>
__device__ __forceinline__ int v_place(int row, int chunk) {
  if constexpr (D == 128) return row * D + 16 * (chunk ^ (row & 6));
  const int r = (row & 8) | ((row & 7) >> 1) | ((row & 1) << 2);
  if constexpr (D == 64) return r * D + 16 * (chunk ^ (r & 2));
  return r * D + 16 * chunk;
}

// The request that a run of units belongs to.
struct DecReq {
  int b, q0, q, len;
  int nr, nt, t0;  // row tiles, units of an item, first unit's index along the cache
};

template <int ROWS>
__device__ __forceinline__ void dec_shape(const AttendArgs &a, DecReq &r) {
  r.nr = (r.q * a.g.G + ROWS - 1) / ROWS;
  const int lo = a.window > 0 ? max(0, r.len - r.q - a.window + 1) : 0;
  r.t0 = lo / kUnit;
  r.nt = max(1, (r.len + kUnit - 1) / kUnit - r.t0);
}
template <int ROWS>
__device__ __forceinline__ DecReq dec_req(const AttendArgs &a, const DecBatch &s, int b) {
  DecReq r;
  r.b = uniform(b);
  r.q0 = uniform(s.q0[b]);
  r.q = uniform(s.q[b]);
  r.len = uniform(s.len[b]);
  dec_shape<ROWS>(a, r);
  return r;
}

// Walks consecutive units: request, kv head, row tile, unit of the item.
template <int ROWS>
struct Cursor {
  DecReq q;
  int h, tile, unit;
  __device__ __forceinline__ void seek(const AttendArgs &a, const DecBatch &s, long long u) {
    q = dec_req<ROWS>(a, s, request_of(s.pre, a.b.B, u));
    const long long in = u - s.pre[q.b];
    const int item = static_cast<int>(quotient(in, q.nt));
    unit = uniform(static_cast<int>(in - static_cast<long long>(item) * q.nt));
    h = uniform(item / q.nr);
    tile = uniform(item - h * q.nr);
  }
  // the next item (the caller counts units)
  __device__ __forceinline__ void next_item(const AttendArgs &a, const DecBatch &s) {
    unit = 0;
    if (++tile < q.nr) return;
    tile = 0;
    if (++h < a.g.Hkv) return;
    h = 0;
    int b = q.b + 1;
    while (b < a.b.B && s.pre[b + 1] == s.pre[b]) ++b;
    b = uniform(b);
    if (b < a.b.B) q = dec_req<ROWS>(a, s, b);
  }
};

// Byte offset of word s of plane p, column tile n of this lane's queries, and a lane's words of a plane.
template <int KW>
__device__ __forceinline__ uint32_t query_place(int p, int n, int lane, int s, int nt) {
  constexpr int V = KW < 4 ? KW : 4;  // words a lane reads at once
  return ((p * nt + n) * 32 * KW + (s / V) * 32 * V + lane * V + s % V) * 4;
}
template <int KW>
__device__ __forceinline__ void query_words(uint32_t (&w)[(KW + 1) / 2 * 2], uint32_t addr) {
  if constexpr (KW >= 4) {
#pragma unroll
    for (int s = 0; s < KW; s += 4) {
      const uint4 v = lds128(addr + 128 * s);
      w[s] = v.x; w[s + 1] = v.y; w[s + 2] = v.z; w[s + 3] = v.w;
    }
  } else if constexpr (KW == 2) {
    const uint2 v = lds64(addr);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = lds32(addr);
    w[1] = 0;
  }
}

// Place of four adjacent outputs in a warp's merge area, spread over the banks.
template <int D>
__device__ __forceinline__ int merge_place(int r, int d4) {
  const int t = (r >> 1) & 3;
  if constexpr (D == 128) return r * (D / 4) + (d4 ^ ((t & 1) | ((t & 2) << 1)));
  if constexpr (D == 64) return r * (D / 4) + (d4 ^ (2 * t));
  return r * (D / 4) + d4;
}

template <typename XT, int D, int NT>
__global__ void __launch_bounds__(kDecThreads, dec_ctas(NT)) kv8_decode_kernel(const __grid_constant__ AttendArgs a) {
  using Geo = DecGeom<XT, D, NT>;
  constexpr int ROWS = Geo::kRows;
  constexpr int KS = D / 16;       // products of 16 dims per score tile, and 16-dim tiles of the output
  constexpr int KW = D / 16;       // words of codes a lane reads of a K row
  constexpr int KM = (KW + 1) / 2; // products of 32 dims per score tile
  constexpr bool F32 = Geo::kWide;  // weights as two f16 each: 22 bits
  constexpr int NP = F32 ? 2 : 1;
  extern __shared__ __align__(128) unsigned char dec_smem[];
  unsigned char *ring = dec_smem;
  DecBatch bt;
  bt.pre = reinterpret_cast<long long *>(dec_smem + Geo::kFixed);
  bt.q0 = reinterpret_cast<int *>(bt.pre + a.b.B + 1);
  bt.q = bt.q0 + a.b.B;
  bt.len = bt.q + a.b.B;
  __shared__ long long red[kDecWarps];
  __shared__ float s_m[kDecWarps][ROWS], s_l[kDecWarps][ROWS];
  __shared__ int s_last;
  // what decides on branches is made uniform over the warp by a shuffle or a vote, so that the products inside
  // them need no re-convergence
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = a.g.G, Hkv = a.g.Hkv;

  request_prefix(a.b.B, bt.pre, red, [&](int b) {
    const Kv8Req r = kv8_req(a.b, a.g.P, b);
    DecReq q{b, bt.q0[b] = r.q0, bt.q[b] = r.q, bt.len[b] = r.len, 0, 0, 0};
    dec_shape<ROWS>(a, q);
    return static_cast<long long>(q.nr) * q.nt * Hkv;
  });
  const long long total = bt.pre[a.b.B];
  const long long share = quotient(total + gridDim.x - 1, gridDim.x);
  const long long u0 = min(total, share * blockIdx.x), u1 = min(total, u0 + share);
  if (u0 >= u1) return;
  const int n_units = uniform(static_cast<int>(u1 - u0));

  // ---- this warp's buffers: K of a step and of the next, V of a step ------
  const uint32_t my_k = shared_addr(ring) + warp * 3 * Geo::kHalf, my_v = my_k + 2 * Geo::kHalf;
  const uint32_t my_tails = shared_addr(ring) + Geo::kRing + warp * 2 * Geo::kTail;
  const uint32_t queries = shared_addr(ring) + Geo::kRing + Geo::kTails;
  float4 *far = reinterpret_cast<float4 *>(ring + Geo::kRing + Geo::kTails + Geo::kQuery) + threadIdx.x;
  constexpr int kCopies = (kSlice * D / 16 + 31) / 32;  // 16-byte copies of a lane for a slice's K, and its V
  // copy c of a lane goes 512 c bytes on: 4 rows at D = 128, where the chunk order of every other copy is turned, and
  // 8 rows at D = 64, where it stays
  const uint32_t k_to = k_place<D>(lane / (D / 16), lane % (D / 16));
  const uint32_t v_to = v_place<D>(lane / (D / 16), lane % (D / 16));
  constexpr uint32_t kTurn = D == 128 ? 64 : 0;
  Cursor<ROWS> load;
  load.seek(a, bt, u0);
  int to_load = n_units;                                     // units not yet asked for
  int l_left = load.q.nt - load.unit;                        // units of the load cursor's item from here on
  int l_pos = (load.q.t0 + load.unit) * kUnit + warp * kStep * kSlice;  // this warp's part of that unit
  const int32_t *l_table = a.b.table + static_cast<long long>(load.q.b) * a.b.cols;
  const uint32_t page_bytes = static_cast<uint32_t>(D) << a.p_shift, page_blocks = 1u << (a.p_shift - a.t_shift);
  int page[2];  // pages of the part's first and last slice (one page unless it is 16 positions long)
  auto read_pages = [&]() {
    page[0] = l_pos < load.q.len ? l_table[l_pos >> a.p_shift] : -1;
    page[1] = l_pos + kSlice < load.q.len ? (a.p_shift == 4 ? l_table[(l_pos >> 4) + 1] : page[0]) : -1;
  };
  read_pages();
  uint32_t there = 0;                    // two bits a step: whether its slices' pages are there, the newest step lowest
  uint32_t v_row0 = 0, v_row1 = 0, v_in = 0, v_in1 = 0;  // where the V of the newest step lies
  auto copy = [&](const int8_t *base, uint32_t to, uint32_t row, uint32_t at) {
    const int8_t *src = base + (static_cast<unsigned long long>(row) * page_bytes + (at * D + 16 * lane));
    if (kSlice * D / 16 % 32 == 0 || lane < kSlice * D / 16) {
#pragma unroll
      for (int c = 0; c < kCopies; ++c) cp_async16((to ^ (c & 1 ? kTurn : 0)) + 512 * c, src + 512 * c);
    }
  };
  auto issue_k = [&](uint32_t par) {  // K and the scales of the next step, into buffer par
    there <<= kStep;
    if (to_load > 0) {
      // (page, kv head) rows and blocks fit 32 bits: the pool is checked against it
      v_in = l_pos & ((1u << a.p_shift) - 1);
      v_row0 = static_cast<uint32_t>(page[0]) * Hkv + load.h;
      v_row1 = static_cast<uint32_t>(page[1]) * Hkv + load.h;
      const bool ok0 = __any_sync(0xffffffffu, static_cast<uint32_t>(page[0]) < static_cast<uint32_t>(a.c.n_pages));
      const bool ok1 = __any_sync(0xffffffffu, static_cast<uint32_t>(page[1]) < static_cast<uint32_t>(a.c.n_pages));
      v_in1 = a.p_shift == 4 ? 0 : v_in + kSlice;  // the second slice's place in its page
      there |= (ok0 ? 1 : 0) | (ok1 ? 2 : 0);
      const uint32_t to = my_k + par * Geo::kHalf + k_to;
      if (ok0) copy(a.c.k, to, v_row0, v_in);
      if (ok1) copy(a.c.k, to + Geo::kSliceBytes, v_row1, v_in1);
      // lanes 0 .. 3: the slices' key and value scales
      const uint32_t block = (lane < 2 ? v_row0 : v_row1) * page_blocks + ((lane < 2 ? v_in : v_in1) >> a.t_shift);
      if (lane < 4 && (lane < 2 ? ok0 : ok1))
        cp_async4(my_tails + par * Geo::kTail + 4 * lane, ((lane & 1) ? a.c.vs : a.c.ks) + block);
      l_pos += kUnit;
      if (--l_left == 0) {
        load.next_item(a, bt);
        l_left = load.q.nt;
        l_pos = load.q.t0 * kUnit + warp * kStep * kSlice;
        l_table = a.b.table + static_cast<long long>(load.q.b) * a.b.cols;
      }
      if (--to_load > 0) read_pages();
    }
    cp_commit();
  };
  auto issue_v = [&]() {  // V of the step whose K was asked for last
    if (there & 1) copy(a.c.v, my_v + v_to, v_row0, v_in);
    if (there & 2) copy(a.c.v, my_v + v_to + Geo::kSliceBytes, v_row1, v_in1);
    cp_commit();
  };
  issue_k(0);
  issue_v();
  uint32_t par = 0;  // K buffer of the step at hand

  Cursor<ROWS> cur;
  cur.seek(a, bt, u0);
  float o[NT][KS][4], m[NT][2], l[NT][2], cs[NT][2];
  int lim[NT][2];   // last visible position of this lane's two columns (-1: none)
  // the item's row tile: its first row and rows; first and last position at which some row is cut off; this warp's
  // next position; positions at which every row sees a whole step
  int row0 = 0, n_rows = 0, min_lim = 0, max_lim = 0, p0 = 0, whole_lo = 0, whole_hi = 0;
  int run = 0, runs = 0;  // steps of the present run, runs in the far sums
  // The far sums brought to the present maximum, plus the present run.
  auto add_far = [&](int n, float4 &sums) {
    float4 f = far[n * Geo::kFarRow * kDecThreads];
    const float al[2] = {exp2_fast(f.z - m[n][0]), exp2_fast(f.w - m[n][1])};
    sums = make_float4(fmaf(f.x, al[0], l[n][0]), fmaf(f.y, al[1], l[n][1]), m[n][0], m[n][1]);
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        f = far[(n * Geo::kFarRow + 1 + s) * kDecThreads];
        o[n][s][0] = fmaf(f.x, al[0], o[n][s][0]);
        o[n][s][1] = fmaf(f.y, al[1], o[n][s][1]);
        o[n][s][2] = fmaf(f.z, al[0], o[n][s][2]);
        o[n][s][3] = fmaf(f.w, al[1], o[n][s][3]);
      }
    }
  };
  auto end_run = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float4 sums = make_float4(l[n][0], l[n][1], m[n][0], m[n][1]);
      if (runs > 0) add_far(n, sums);
      far[n * Geo::kFarRow * kDecThreads] = sums;
      l[n][0] = l[n][1] = 0.f;
      if constexpr (F32) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          far[(n * Geo::kFarRow + 1 + s) * kDecThreads] = make_float4(o[n][s][0], o[n][s][1], o[n][s][2], o[n][s][3]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][s][j] = 0.f;
        }
      }
    }
    ++runs;
    run = 0;
  };
  Quad<XT> raw[NT][KW];
  auto begin_item = [&]() {  // asks for the item's query rows
    const DecReq &q = cur.q;
    row0 = cur.tile * ROWS;
    n_rows = min(ROWS, q.q * G - row0);
    min_lim = q.len - q.q + row_at(a, row0).i;
    max_lim = q.len - q.q + row_at(a, row0 + n_rows - 1).i;
    p0 = (q.t0 + cur.unit) * kUnit + warp * kStep * kSlice;
    whole_lo = a.window > 0 ? max_lim - a.window + 1 : 0;
    whole_hi = min_lim - kStep * kSlice + 1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const bool live = 8 * n + g < n_rows;
      const RowAt at_row = row_at(a, r);
      const long long at = live ? (q.q0 + at_row.i) * a.q_row + (cur.h * G + at_row.h) * a.q_head : 0;
      const XT *src = static_cast<const XT *>(a.q) + at + 4 * t;
      auto load = [&](bool vec) {
#pragma unroll
        for (int s = 0; s < KW; ++s) raw[n][s].load(src + 16 * s, vec, live);
      };
      if (a.q_vec) load(true);
      else load(false);
    }
  };
  // The item's queries, scaled by a power of two to at most 1..2, as whole numbers v = x 2^(21 - e) rounded, where
  // 2^e <= the row's largest value < 2^(e + 1) (rows below 2^-100 count as 2^-100): 22 bits of that value.  The digits of
  // v in base 256, -128 .. 127 each, are the bytes of v + 0x808080 less 128: three products of bytes give q . k exactly.
  // Every warp finds the rows' largest values; the four convert a quarter of the words each, for all.
  auto put_queries = [&]() {
    const DecReq &q = cur.q;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float big = 0.f, bad = 0.f;  // bad: 0, or a NaN where the row has a value that is not finite
#pragma unroll
      for (int s = 0; s < KW; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          big = fmaxf(big, fabsf(raw[n][s].get(j)));
          bad = fmaf(raw[n][s].get(j), 0.f, bad);
        }
#pragma unroll
      for (int i = 1; i <= 2; i <<= 1) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, i));
        bad += __shfl_xor_sync(0xffffffffu, bad, i);
      }
      const int e = min(max(static_cast<int>(__float_as_uint(big) >> 23) - 127, -100), 127);
      const float down = __uint_as_float((127 + 21 - e) << 23), up = __uint_as_float((127 + e - 21) << 23) + bad;
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        if (s % kDecWarps != warp) continue;
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<uint32_t>(__float2int_rn(raw[n][s].get(j) * down)) + 0x808080u;
        const uint32_t a01 = __byte_perm(v[0], v[1], 0x5140), a23 = __byte_perm(v[2], v[3], 0x5140);  // bytes 0, 1
        const uint32_t b01 = __byte_perm(v[0], v[1], 0x0062), b23 = __byte_perm(v[2], v[3], 0x0062);  // byte 2
        const uint32_t w[3] = {__byte_perm(a01, a23, 0x5410), __byte_perm(a01, a23, 0x7632), __byte_perm(b01, b23, 0x5410)};
#pragma unroll
        for (int p = 0; p < 3; ++p)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(queries + query_place<KW>(p, n, lane, s, NT)), "r"(w[p] ^ 0x80808080u)
                       : "memory");
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // columns 2t + j of this tile: their row's scale sits in lane 4 (2t + j)
        cs[n][j] = __shfl_sync(0xffffffffu, up, 4 * (2 * t + j)) * (a.scale * kLog2e);
        const int rr = 8 * n + 2 * t + j;
        lim[n][j] = rr < n_rows ? q.len - q.q + row_at(a, row0 + rr).i : -1;
        m[n][j] = kNone;
        l[n][j] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][s][j] = 0.f;
    }
  };
  begin_item();
  put_queries();
  __syncthreads();
  const uint32_t k_row = lane & 15, k_half = lane >> 4;  // ldmatrix row and 16-byte chunk of this lane
  const uint32_t v_at = v_place<D>(2 * t, (KS * g) >> 4) + ((KS * g) & 15);
  for (int n_left = n_units; n_left > 0; --n_left) {
    const DecReq &q = cur.q;
    // ---- one step: kStep slices ------------------------------------------------
    const uint32_t here = there;  // this step's slices
    issue_k(par ^ 1);
    cp_wait<2>();  // this step's K and scales
    __syncwarp();
    const uint32_t slot = my_k + par * Geo::kHalf;
    const uint4 tail = lds128(my_tails + par * Geo::kTail);
    float ksc[kStep] = {__uint_as_float(tail.x), __uint_as_float(tail.z)};
    float vsc[kStep] = {__uint_as_float(tail.y), __uint_as_float(tail.w)};
    const bool whole = __all_sync(0xffffffffu, p0 >= whole_lo && p0 <= whole_hi && (here & 3) == 3);
    bool any = true;
    if (!whole) {  // scales of 0 for a slice that is not there or that no row sees
      any = false;
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int p = p0 + i * kSlice;
        const bool seen = (here >> i & 1) && p <= max_lim && (a.window <= 0 || p + kSlice - 1 > min_lim - a.window);
        ksc[i] = seen ? ksc[i] : 0.f;
        vsc[i] = seen ? vsc[i] : 0.f;
        any |= seen;
      }
    }
    if (__any_sync(0xffffffffu, any)) {
      // scores: the slices' 16 positions x the rows, exact whole numbers
      float sc[kStep][NT][4];
      uint32_t kw[kStep][KM][4];
#pragma unroll
      for (int i = 0; i < kStep; ++i)
#pragma unroll
        for (int s = 0; s < KM; ++s) {
          const uint32_t at = slot + i * Geo::kSliceBytes + k_place<D>(k_row, D == 16 ? 0 : 2 * s + k_half);
          if constexpr (D == 16) ldmatrix2(kw[i][s], at);
          else ldmatrix4(kw[i][s], at);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        int hi[kStep][4], lo[kStep][4];
        auto product = [&](int (&d)[kStep][4], int p, bool first) {
          uint32_t w[KM * 2];
          query_words<KW>(w, queries + query_place<KW>(p, n, lane, 0, NT));
#pragma unroll
          for (int s = 0; s < KM; ++s)
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
              if (first && s == 0) mma16832_first(d[i], kw[i][s], w[2 * s], w[2 * s + 1]);
              else mma16832(d[i], kw[i][s], w[2 * s], w[2 * s + 1]);
            }
        };
        product(hi, 2, true);
        product(lo, 0, true);
#pragma unroll
        for (int i = 0; i < kStep; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) hi[i][j] <<= 8;
        product(hi, 1, false);
#pragma unroll
        for (int i = 0; i < kStep; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sc[i][n][j] = fmaf(static_cast<float>(hi[i][j]), 256.f, static_cast<float>(lo[i][j]));
      }
      // softmax: this lane has positions g, g + 8 of each slice for columns 2t, 2t + 1.  Weights are held relative to
      // the largest p x sv: the value scale's exponent joins the maximum
      float x[kStep][NT][4], fev[kStep];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        fev[i] = static_cast<float>(max(static_cast<int>(__float_as_uint(vsc[i]) >> 23 & 0xff) - 127, kScaleFloor));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[i][n][j] = fmaf(sc[i][n][j], cs[n][j & 1] * ksc[i], -m[n][j & 1]);
            if (!whole) {
              const int p = p0 + i * kSlice + g + 8 * (j >> 1), last = lim[n][j & 1];
              if (p > last || (a.window > 0 && p <= last - a.window) || !(here >> i & 1)) x[i][n][j] = -INFINITY;
            }
          }
          grow |= fmaxf(fmaxf(x[i][n][0], x[i][n][1]), fmaxf(x[i][n][2], x[i][n][3])) > kLazy + kRoom - fev[i];
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
              const float f = cs[n][j] * ksc[i];
#pragma unroll
              for (int r = 0; r < 4; r += 2)
                if (x[i][n][j + r] != -INFINITY) top = fmaxf(top, sc[i][n][j + r] * f + fev[i]);
            }
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
            const float nm = fmaxf(m[n][j], top - kRoom);
            const float al = exp2_fast(m[n][j] - nm);
            m[n][j] = nm;
            l[n][j] *= al;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              o[n][s][j] *= al;
              o[n][s][j + 2] *= al;
            }
#pragma unroll
            for (int i = 0; i < kStep; ++i)
#pragma unroll
              for (int r = 0; r < 4; r += 2)
                if (x[i][n][j + r] != -INFINITY) x[i][n][j + r] = fmaf(sc[i][n][j + r], cs[n][j] * ksc[i], -nm);
          }
      }
      cp_wait<1>();  // this step's V
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        uint32_t pf[NP][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = exp2_fast(x[i][n][j]);
            l[n][j & 1] += p;
            // a scale that is not finite reaches only the rows that see its slice
            w[j] = whole || x[i][n][j] != -INFINITY ? p * vsc[i] : 0.f;
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t hi = pack_f16(w[2 * r], w[2 * r + 1]);
            pf[0][n][r] = transpose8x8(hi);
            if constexpr (F32) {
              const float2 h = unpack_f16(hi);
              pf[NP - 1][n][r] = transpose8x8(pack_f16((w[2 * r] - h.x) * kLowUp, (w[2 * r + 1] - h.y) * kLowUp));
            }
          }
        }
        // output: this lane's dims KS g .. + KS and D / 2 + KS g .. of positions 2t, 2t + 1, 2t + 8, 2t + 9
        constexpr int VB = KS < 4 ? KS : 4;  // dims a word carries
        uint32_t vw[2][4][(KS + 3) / 4];     // [half of the dims][position]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // position 2t + (r & 1) + 8 (r >> 1); D = 64 and below keep odd positions 4 rows on
            const uint32_t step = (r & 1) * (D == 128 ? D : 4 * D) + (r >> 1) * 8 * D;
            const uint32_t at = (my_v + v_at + i * Geo::kSliceBytes + step) ^ (h && D >= 64 ? D / 2 : 0);
            if constexpr (KS == 8) {
              const uint2 v = lds64(at);
              vw[h][r][0] = v.x;
              vw[h][r][1] = v.y;
            } else if constexpr (KS == 4) {
              vw[h][r][0] = lds32(at);
            } else if constexpr (KS == 2) {
              vw[h][r][0] = lds16(at + h * (D / 2));
            } else {
              vw[h][r][0] = lds8(at + h * (D / 2));
            }
          }
#pragma unroll
        for (int c = 0; c < (KS + 3) / 4; ++c) {
          uint32_t w[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) w[h][r] = vw[h][r][c] ^ 0x80808080u;
#pragma unroll
          for (int half = 0; half < (VB + 1) / 2; ++half) {
            // pairs of positions (2t, 2t + 1) and (2t + 8, 2t + 9) of dims 2 half, 2 half + 1
            uint32_t y[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 2; ++r) y[h][r] = __byte_perm(w[h][2 * r], w[h][2 * r + 1], half ? 0x7362 : 0x5140);
#pragma unroll
            for (int j = 0; j < (VB < 2 ? 1 : 2); ++j) {
              uint32_t f[4];
              const uint32_t sel = j ? 0x4342 : 0x4140;
              f[0] = f16_codes(__byte_perm(y[0][0], 0x64646464u, sel));
              f[1] = f16_codes(__byte_perm(y[1][0], 0x64646464u, sel));
              f[2] = f16_codes(__byte_perm(y[0][1], 0x64646464u, sel));
              f[3] = f16_codes(__byte_perm(y[1][1], 0x64646464u, sel));
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16816(o[n][4 * c + 2 * half + j], f, pf[0][n][0], pf[0][n][1]);
              if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = scale_f16(f[i], 1.f / kLowUp);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(o[n][4 * c + 2 * half + j], f, pf[NP - 1][n][0], pf[NP - 1][n][1]);
              }
            }
          }
        }
      }
    }
    __syncwarp();
    ++cur.unit;
    p0 += kUnit;
    par ^= 1;
    const bool last_of_item = cur.unit == q.nt || n_left == 1;
    if (!last_of_item) {
      cp_wait<1>();  // a step that no row saw has not waited for its V
      issue_v();
      if (++run == kRunSteps) end_run();
    }

    // ---- end of the item, or of this block's share of it --------------------
    if (last_of_item) {
      const long long i0 = u0 + (n_units - n_left) + 1 - cur.unit, i1 = i0 + q.nt;
      const DecReq q = cur.q;
      const int hk = cur.h, row0_now = row0, n_rows_now = n_rows;
      cur.next_item(a, bt);
      if (n_left > 1) begin_item();
      const bool all = i0 >= u0 && i1 <= u1;
      const int c0 = all ? 0 : static_cast<int>(quotient(i0, share)), c1 = all ? 0 : static_cast<int>(quotient(i1 - 1, share));
      float *part = a.part + (2 * static_cast<long long>(blockIdx.x) + (i0 >= u0 ? 1 : 0)) * Geo::kPart;
      // a warp takes rows warp, warp + 4, ...; its lanes four dims each
      constexpr int kLanes = D / 4 < 32 ? D / 4 : 32, kRowsAtOnce = kDecThreads / kLanes;
      const int r_first = threadIdx.x / kLanes, d4 = threadIdx.x % kLanes;
      auto store = [&](int r, float4 v, float lsum, float top) {
        const float inv = lsum == 0.f ? 0.f : __fdividef(1.f, lsum);  // 0: the row saw nothing
        const RowAt at_row = row_at(a, row0_now + r);
        const int i = q.q0 + at_row.i, h = hk * G + at_row.h;
        XT *dst = static_cast<XT *>(a.out) + i * a.o_row + h * a.o_head + 4 * d4;
        store4(dst, a.o_vec, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        if (a.lse && d4 == 0) a.lse[static_cast<long long>(i) * a.g.H + h] = lsum == 0.f ? -INFINITY : logf(lsum) + top * kLn2;
      };
      cp_wait<1>();  // the outputs take the place of the step's V
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NT; ++n) {  // eight rows at a time
        if (runs > 0) {
          float4 sums;
          add_far(n, sums);
          l[n][0] = sums.x;
          l[n][1] = sums.y;
        }
        float *mine = reinterpret_cast<float *>(ring + (warp * 3 + 2) * Geo::kHalf);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = l[n][j];
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
          const int r = 2 * t + j;
          if (g == 0) {
            s_m[warp][8 * n + r] = m[n][j];
            s_l[warp][8 * n + r] = sum;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d = h * (D / 2) + KS * g;
            if constexpr (KS >= 4) {
#pragma unroll
              for (int s = 0; s < KS; s += 4)
                *reinterpret_cast<float4 *>(mine + 4 * merge_place<D>(r, (d + s) / 4)) =
                    make_float4(o[n][s][j + 2 * h], o[n][s + 1][j + 2 * h], o[n][s + 2][j + 2 * h], o[n][s + 3][j + 2 * h]);
            } else {
#pragma unroll
              for (int s = 0; s < KS; ++s) mine[r * D + d + s] = o[n][s][j + 2 * h];
            }
          }
        }
        __syncthreads();
        for (int r8 = r_first; r8 < min(8, n_rows_now - 8 * n); r8 += kRowsAtOnce) {
          const int r = 8 * n + r8;
          float sm[kDecWarps], top = kNone;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            sm[w] = s_m[w][r];
            top = fmaxf(top, sm[w]);
          }
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          float lsum = 0.f;
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            const float f = exp2_fast(sm[w] - top);
            const float4 y = reinterpret_cast<const float4 *>(ring + (w * 3 + 2) * Geo::kHalf)[merge_place<D>(r8, d4)];
            lsum += s_l[w][r] * f;
            v.x += y.x * f; v.y += y.y * f; v.z += y.z * f; v.w += y.w * f;
          }
          if (all) {
            store(r, v, lsum, top);
          } else {
            *reinterpret_cast<float4 *>(part + r * D + 4 * d4) = v;
            if (d4 == 0) {
              part[ROWS * D + r] = top;
              part[ROWS * D + ROWS + r] = lsum;
            }
          }
        }
        if (NT > 1 && n + 1 < NT) __syncthreads();
      }
      if (!all) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicAdd(a.ticket + c0, 1) == c1 - c0;
        __syncthreads();
        if (s_last) {
          __threadfence();
          for (int r = r_first; r < n_rows_now; r += kRowsAtOnce) {
            float top = kNone, lsum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = c0; c <= c1; c += kMergeAhead) {
              float pm[kMergeAhead], pl[kMergeAhead];
              float4 pv[kMergeAhead];
              const float was = top;
#pragma unroll
              for (int k = 0; k < kMergeAhead; ++k) {
                const bool in = c + k <= c1;
                const float *p = a.part + (2ll * (in ? c + k : c0) + (!in || c + k == c0)) * Geo::kPart;
                pm[k] = __ldcg(p + ROWS * D + r);
                pl[k] = __ldcg(p + ROWS * D + ROWS + r);
                pv[k] = __ldcg(reinterpret_cast<const float4 *>(p) + r * (D / 4) + d4);
                if (!in) pm[k] = kNone * 2;  // weight 0
              }
#pragma unroll
              for (int k = 0; k < kMergeAhead; ++k) top = fmaxf(top, pm[k]);
              const float al = exp2_fast(was - top);
              lsum *= al;
              v.x *= al; v.y *= al; v.z *= al; v.w *= al;
#pragma unroll
              for (int k = 0; k < kMergeAhead; ++k) {
                const float f = exp2_fast(pm[k] - top);
                lsum += pl[k] * f;
                v.x += pv[k].x * f; v.y += pv[k].y * f; v.z += pv[k].z * f; v.w += pv[k].w * f;
              }
            }
            store(r, v, lsum, top);
          }
          if (threadIdx.x == 0) a.ticket[c0] = 0;
        }
      }
      run = runs = 0;
      if (n_left > 1) put_queries();
      __syncthreads();
      issue_v();
    }
  }
}

template <typename XT, int D, int NT>
constexpr int dec_smem_bytes(int B) {
  return DecGeom<XT, D, NT>::kFixed + (B + 1) * static_cast<int>(sizeof(long long)) + 3 * B * static_cast<int>(sizeof(int));
}

template <typename XT, int D, int NT>
void dec_launch(const specdec_kv8 *h, const AttendArgs &a, cudaStream_t st) {
  // at most one item per row and kv head, at least one unit per block
  const long long units = static_cast<long long>(a.b.T) * h->g.Hkv * ((static_cast<long long>(a.b.cols) * h->g.P + kUnit - 1) / kUnit);
  const int grid = static_cast<int>(std::min(units, static_cast<long long>(dec_ctas(NT)) * h->num_sms));
  op_launch("specdec_kv8_attend", kv8_decode_kernel<XT, D, NT>, dim3(grid), kDecThreads, dec_smem_bytes<XT, D, NT>(a.b.B),
            st, 1, a);
}

template <typename XT, int NT>
void dec_launch_dim(const specdec_kv8 *h, const AttendArgs &a, cudaStream_t st) {
  switch (h->g.D) {
    case 16: return dec_launch<XT, 16, NT>(h, a, st);
    case 32: return dec_launch<XT, 32, NT>(h, a, st);
    case 64: return dec_launch<XT, 64, NT>(h, a, st);
    default: return dec_launch<XT, 128, NT>(h, a, st);
  }
}

template <typename XT, int NT>
void dec_attrs(int max_batch) {
  auto set = [](auto kernel, int bytes) {
    op_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute");
  };
  set(kv8_decode_kernel<XT, 16, NT>, dec_smem_bytes<XT, 16, NT>(max_batch));
  set(kv8_decode_kernel<XT, 32, NT>, dec_smem_bytes<XT, 32, NT>(max_batch));
  set(kv8_decode_kernel<XT, 64, NT>, dec_smem_bytes<XT, 64, NT>(max_batch));
  set(kv8_decode_kernel<XT, 128, NT>, dec_smem_bytes<XT, 128, NT>(max_batch));
}

int log2i(int v) {
  int n = 0;
  while (v > 1 << n) ++n;
  return n;
}
// Whether every row and head starts at a boundary of four elements.
bool rows_aligned(const void *p, int64_t row, int64_t head, int dtype) {
  const uintptr_t size = dtype == SPECDEC_F32 ? 16 : 8;
  return reinterpret_cast<uintptr_t>(p) % size == 0 && row % 4 == 0 && head % 4 == 0;
}

}  // namespace

void kv8_attn_create(specdec_kv8 *h) {
  dec_attrs<float, 1>(kKv8MaxBatch);
  dec_attrs<float, 2>(kKv8MaxBatch);
  dec_attrs<__nv_bfloat16, 1>(kKv8MaxBatch);
  dec_attrs<__nv_bfloat16, 2>(kKv8MaxBatch);
  const size_t blocks = static_cast<size_t>(dec_ctas(1)) * h->num_sms;
  const size_t part = std::max(blocks * 2 * (16 * h->g.D + 32) * sizeof(float), kv8_chunk_part_bytes(h));
  kv8_chunk_create(h);
  op_cuda(cudaMalloc(&h->part, part), "cudaMalloc");
  const cudaError_t e = cudaMalloc(&h->ticket, (blocks + 1) * sizeof(int));
  if (e != cudaSuccess) {
    kv8_attn_destroy(h);
    op_cuda(e, "cudaMalloc");
  }
  h->err_word = h->ticket + blocks;
  cudaError_t z = cudaMemset(h->ticket, 0, (blocks + 1) * sizeof(int));
  if (z == cudaSuccess) z = cudaStreamSynchronize(nullptr);  // the first call may be on a stream that does not wait for it
  if (z != cudaSuccess) {
    kv8_attn_destroy(h);
    op_cuda(z, "cudaMemset");
  }
}

void kv8_attn_destroy(specdec_kv8 *h) {
  if (h->part) cudaFree(h->part);
  if (h->ticket) cudaFree(h->ticket);
  h->part = nullptr;
  h->ticket = nullptr;
}

}  // namespace specdec

using namespace specdec;

extern "C" int specdec_kv8_attend(specdec_kv8 *h, const specdec_kv8_layer *layer, const specdec_kv8_batch *batch,
                                  const void *q, int64_t q_row_stride, int64_t q_head_stride, int dtype, int n_tokens,
                                  void *out, int64_t out_row_stride, int64_t out_head_stride, float *lse, int max_q,
                                  float scale, int window, void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    const Kv8Layer c = kv8_layer(h, layer);
    const Kv8Batch b = kv8_batch(h, batch, n_tokens);
    op_check(dtype == SPECDEC_F32 || dtype == SPECDEC_BF16, "rows must be SPECDEC_F32 or SPECDEC_BF16");
    op_check(max_q >= 0 && window >= 0, "max_q and window must not be negative");
    op_check(std::isfinite(scale), "scale must be finite");
    if (b.B == 0 || b.T == 0) return;
    op_check(q && out, "null row buffer");
    // a window that no request can be longer than cuts nothing off, and positions less such a window pass 32 bits
    if (window >= static_cast<long long>(b.cols) * h->g.P) window = 0;
    DeviceScope scope(h->device);
    const AttendArgs a{h->g, c,   b,     q,      q_row_stride, q_head_stride, out, out_row_stride, out_head_stride,
                       lse,  scale, window, h->part, h->ticket, log2i(h->g.P), log2i(h->g.t),
                       (h->g.G & (h->g.G - 1)) == 0 ? log2i(h->g.G) : -1,
                       rows_aligned(q, q_row_stride, q_head_stride, dtype),
                       rows_aligned(out, out_row_stride, out_head_stride, dtype),
                       aligned16(q) && q_row_stride % 8 == 0 && q_head_stride % 8 == 0,
                       aligned16(out) && out_row_stride % 8 == 0 && out_head_stride % 8 == 0, h->err_word};
    const auto st = static_cast<cudaStream_t>(stream);
    // Many rows per kv head: every cached value meets all of them and the products bound the call, so they go to the
    // 128-row tensor tiles, where there is enough of it to pay for those tiles' longer start and merges: units as the
    // tables have room for, or items (row tiles x kv heads).  Measured in us, this kernel / the tensor tiles (heads of 128):
    //   units a block  14: 4 x 16 rows over 4,096, 32 / 8 heads 48 / 55       22: 32 x 8 over 3,080, 16 / 2 heads 62 / 61
    //                  28: 4 x 32 over 4,096, 32 / 8 heads    74 / 57         87: 32 x 16 over 3,080, 32 / 8    192 / 164
    //   items a block 0.9: 4 x 64 over themselves, 16 / 2     13 / 20        1.7: 4 x 64, 32 / 8 heads           19 / 20
    //                 1.7: 16 x 16 over 500, 32 / 8 heads     42 / 28        3.5: 4 x 128, 32 / 8 heads          32 / 22
    //   48 rows of a kv head: 32 x 48 over 3,080, 32 / 32 heads 521 / 536, 32 x 12, 32 / 8 heads 149 / 164
    // The host does not know the lengths, so tables that are far wider than the requests are long send small prompts to the
    // tensor tiles too (4 x 64 rows over themselves, 16 / 2 heads: 20 us instead of 13).
    const long long items = (static_cast<long long>(b.T) * h->g.G + 15) / 16 * h->g.Hkv;
    const long long units = items * ((static_cast<long long>(b.cols) * h->g.P + kUnit - 1) / kUnit);
    const long long blocks = static_cast<long long>(dec_ctas(2)) * h->num_sms;
    if (dtype == SPECDEC_BF16 && h->g.D >= 64 && b.B <= kChunkMaxBatch && static_cast<long long>(max_q) * h->g.G >= kChunkRows &&
        (units >= kChunkUnits * blocks || items >= kChunkItems * blocks)) {
      kv8_chunk_launch(h, a, st);
      return;
    }
    // rows of one kv head: one column tile of 8 where they fit, else two (64 requests of up to 4,096, 4 rows a kv head: 69 us
    // with one tile, 94 with two)
    const bool one = static_cast<long long>(max_q) * h->g.G <= 8;
    if (dtype == SPECDEC_F32)
      one ? dec_launch_dim<float, 1>(h, a, st) : dec_launch_dim<float, 2>(h, a, st);
    else
      one ? dec_launch_dim<__nv_bfloat16, 1>(h, a, st) : dec_launch_dim<__nv_bfloat16, 2>(h, a, st);
  });
}

extern "C" int specdec_kv8_check(specdec_kv8 *h, void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    DeviceScope scope(h->device);
    const auto st = static_cast<cudaStream_t>(stream);
    int bits = 0;
    op_cuda(cudaMemcpyAsync(&bits, h->err_word, sizeof(int), cudaMemcpyDeviceToHost, st), "specdec_kv8_check");
    op_cuda(cudaStreamSynchronize(st), "specdec_kv8_check");
    if (!bits) return;
    // the block that gave up has not arrived at its split items: their tickets go back to 0 with the error word behind them
    op_cuda(cudaMemsetAsync(h->ticket, 0, (h->err_word - h->ticket + 1) * sizeof(int), st), "specdec_kv8_check");
    op_fail(SPECDEC_ERR_CUDA, "a wait inside specdec_kv8_attend did not end within its limit");
  });
}
