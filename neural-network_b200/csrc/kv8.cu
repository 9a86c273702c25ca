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
// requests.
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

constexpr int kPlanThreads = 256;

struct PlanReq {
  long long q;
  int take, give;
  bool bad;
};
__device__ __forceinline__ PlanReq plan_req(const PlanArgs &a, int b) {
  const long long held = a.held[b], keep = a.keep[b], q = a.q_len[b];
  const long long cap = static_cast<long long>(a.cols) * a.P;
  PlanReq r{0, 0, 0, held < 0 || keep < 0 || keep > held || q < 0 || held > cap || keep + q > cap};
  if (!r.bad) {
    const int have = static_cast<int>((held + a.P - 1) / a.P), need = static_cast<int>((keep + q + a.P - 1) / a.P);
    r.q = q;
    r.take = max(0, need - have);
    r.give = max(0, have - need);
  }
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const PlanArgs a) {
  extern __shared__ long long plan_smem[];
  long long *cu = plan_smem;       // [B + 1] first row of a request
  long long *mv = cu + a.B + 1;    // [B + 1] pages taken (low 32 bits) and given back (high) before it
  __shared__ long long red[kPlanThreads / 32];
  int bad = 0;
  request_prefix(a.B, cu, red, [&](int b) {
    const PlanReq r = plan_req(a, b);
    bad |= r.bad;
    return r.q;
  });
  request_prefix(a.B, mv, red, [&](int b) {
    const PlanReq r = plan_req(a, b);
    return static_cast<long long>(r.take) | static_cast<long long>(r.give) << 32;
  });
  bad = __syncthreads_or(bad);
  const long long head = a.ring_state[0], count = a.ring_state[1];
  const long long takes = mv[a.B] & 0xffffffffll, gives = mv[a.B] >> 32;
  const bool ring_ok = head >= 0 && head < a.ring_cap && count >= 0 && count <= a.ring_cap;
  const int status = ((!ring_ok || takes > count) ? 1 : 0) | (bad ? 2 : 0) | (cu[a.B] > a.T ? 4 : 0) |
                     ((ring_ok && count - takes + gives > a.ring_cap) ? 2 : 0);
  const bool fine = status == 0;
  const long long tid = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  if (tid == 0) {
    *a.status = status;
    a.ring_out[0] = fine ? static_cast<int>((head + takes) % a.ring_cap) : static_cast<int>(head);
    a.ring_out[1] = fine ? static_cast<int>(count - takes + gives) : static_cast<int>(count);
  }
  for (long long b = tid; b <= a.B; b += stride) {
    a.cu_q[b] = fine ? static_cast<int>(cu[b]) : 0;
    if (b < a.B) a.kv_len[b] = fine ? a.keep[b] + a.q_len[b] : a.held[b];
  }
  auto pages = [&](int n) { return (static_cast<long long>(n) + a.P - 1) / a.P; };
  if (fine) {
    auto low = [&](int b) { return mv[b] & 0xffffffffll; };
    auto high = [&](int b) { return mv[b] >> 32; };
    auto find = [&](long long u, auto &&at) {  // the last request with at(b) <= u
      int lo = 0, hi = a.B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at(mid) <= u) lo = mid;
        else hi = mid - 1;
      }
      return lo;
    };
    for (long long i = tid; i < takes; i += stride) {
      const int b = find(i, low);
      a.table[static_cast<long long>(b) * a.cols + pages(a.held[b]) + (i - low(b))] = a.ring[(head + i) % a.ring_cap];
    }
    for (long long i = tid; i < gives; i += stride) {
      const int b = find(i, high);
      const long long need = pages(a.keep[b] + a.q_len[b]);
      a.ring[(head + count + i) % a.ring_cap] = a.table[static_cast<long long>(b) * a.cols + need + (i - high(b))];
    }
  }
  for (long long t = tid; t < a.T; t += stride) {
    int req = -1, pos = -1;
    long long slot = -1;
    if (fine && t < cu[a.B]) {
      req = request_of(cu, a.B, t);
      pos = a.keep[req] + static_cast<int>(t - cu[req]);
      const long long col = pos / a.P, have = pages(a.held[req]);
      // a page taken in this call is read from the ring: its table entry is being written
      const long long page = col < have ? a.table[static_cast<long long>(req) * a.cols + col]
                                        : a.ring[(head + (mv[req] & 0xffffffffll) + col - have) % a.ring_cap];
      slot = page * a.P + pos % a.P;
    }
    a.tok_req[t] = req;
    a.tok_pos[t] = pos;
    a.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------
// Cache write.  One unit = the new rows of one scale block, one kv head, K or
// V: a = max |x| over the finite new values, scale' = max(scale if the block
// has older rows, a x (1 / 127)); older rows are brought to scale', new rows
// become rint(x x (1 / scale')).  A scale below the smallest normal number is
// 0 (its codes are 0), so 1 / scale' is finite.
constexpr float kInv127 = 1.f / 127.f;

__device__ __forceinline__ int quant_code(float x, float inv) {
  const float c = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
  return isnan(x) ? 0 : static_cast<int>(c);
}

struct AppendArgs {
  Kv8Geom g;
  Kv8Layer c;
  Kv8Batch b;
  const void *x[2];           // K and V rows
  long long row_stride[2], head_stride[2];  // elements
};

constexpr int kAppendThreads = 128;

template <typename XT>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const AppendArgs a) {
  extern __shared__ int append_smem[];
  int *pre = append_smem;  // [B + 1] blocks touched before a request
  __shared__ int red[kAppendThreads / 32];
  __shared__ float redf[kAppendThreads / 32];
  const Kv8Geom &g = a.g;
  request_prefix(a.b.B, pre, red, [&](int b) {
    const Kv8Req r = kv8_req(a.b, g.P, b);
    return (r.q > 0 && r.len >= r.q) ? (r.len - 1) / g.t - (r.len - r.q) / g.t + 1 : 0;
  });
  const long long units = static_cast<long long>(pre[a.b.B]) * g.Hkv * 2;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int kv = static_cast<int>(u & 1), h = static_cast<int>((u >> 1) % g.Hkv);
    const int blk = static_cast<int>((u >> 1) / g.Hkv);
    const int b = request_of(pre, a.b.B, blk);
    const Kv8Req r = kv8_req(a.b, g.P, b);
    const int start = r.len - r.q;
    const int p0 = (start / g.t + blk - pre[b]) * g.t;  // the block's first position
    const int lo = max(p0, start), hi = min(p0 + g.t, r.len);
    const int page = a.b.table[static_cast<long long>(b) * a.b.cols + p0 / g.P];
    if (page < 0 || page >= a.c.n_pages) continue;
    const long long row0 = (static_cast<long long>(page) * g.Hkv + h) * g.P + p0 % g.P;
    int8_t *code = (kv ? a.c.v : a.c.k) + row0 * g.D;
    float *sc = (kv ? a.c.vs : a.c.ks) + (static_cast<long long>(page) * g.Hkv + h) * (g.P / g.t) + p0 % g.P / g.t;
    const XT *x = static_cast<const XT *>(a.x[kv]) + (r.q0 + lo - start) * a.row_stride[kv] + h * a.head_stride[kv];
    const int n = (hi - lo) * g.D, n_old = (lo - p0) * g.D;
    float m = 0.f;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const float v = fabsf(to_f32(x[i / g.D * a.row_stride[kv] + i % g.D]));
      if (v < INFINITY) m = fmaxf(m, v);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) redf[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kAppendThreads / 32; ++w) m = fmaxf(m, redf[w]);
    const float old = n_old ? *sc : 0.f;
    float s = fmaxf(old, __fmul_rn(m, kInv127));
    if (s < 1.17549435e-38f) s = 0.f;
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    const float factor = s > old ? __fdiv_rn(old, s) : 1.f;
    __syncthreads();  // every thread has read the scale and the partial maxima
    if (threadIdx.x == 0) *sc = s;
    if (factor != 1.f)
      for (int i = threadIdx.x; i < n_old; i += blockDim.x)
        code[i] = static_cast<int8_t>(rintf(__fmul_rn(static_cast<float>(code[i]), factor)));
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const float v = to_f32(x[i / g.D * a.row_stride[kv] + i % g.D]);
      code[n_old + i] = s > 0.f ? static_cast<int8_t>(quant_code(v, inv)) : 0;
    }
  }
}

// Cache read: the values code * scale of given rows, [n][Hkv][D].
struct GatherArgs {
  Kv8Geom g;
  Kv8Layer c;
  const int64_t *rows;
  int n;
  void *out[2];
};

template <typename XT>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const GatherArgs a) {
  const Kv8Geom &g = a.g;
  const long long total = static_cast<long long>(a.n) * g.Hkv * g.D;
  const long long all = static_cast<long long>(a.c.n_pages) * g.P;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int d = static_cast<int>(i % g.D), h = static_cast<int>(i / g.D % g.Hkv);
    const int64_t row = a.rows[i / g.D / g.Hkv];
    for (int kv = 0; kv < 2; ++kv) {
      if (!a.out[kv]) continue;
      float v = 0.f;
      if (row >= 0 && row < all) {
        const long long ph = row / g.P * g.Hkv + h;
        const int off = static_cast<int>(row % g.P);
        v = static_cast<float>((kv ? a.c.v : a.c.k)[(ph * g.P + off) * g.D + d]) *
            (kv ? a.c.vs : a.c.ks)[ph * (g.P / g.t) + off / g.t];
      }
      static_cast<XT *>(a.out[kv])[i] = from_f32<XT>(v);
    }
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
                                 2 * (kKv8MaxBatch + 1) * static_cast<int>(sizeof(long long))),
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
    const int work = std::max(b.T, b.B);
    const int grid = std::max(1, std::min(h->num_sms, (work + 4 * kPlanThreads - 1) / (4 * kPlanThreads)));
    op_launch("specdec_kv8_plan", kv8_plan_kernel, dim3(grid), kPlanThreads, 2 * (b.B + 1) * sizeof(long long),
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
    const AppendArgs a{h->g, c, b, {k, v}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride}};
    const long long units = (static_cast<long long>(b.T) / h->g.t + 2ll * b.B) * h->g.Hkv * 2;
    const int grid = static_cast<int>(std::min(units, 16ll * h->num_sms));
    const size_t smem = (b.B + 1) * sizeof(int);
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == SPECDEC_F32)
      op_launch("specdec_kv8_append", kv8_append_kernel<float>, dim3(grid), kAppendThreads, smem, st, 1, a);
    else
      op_launch("specdec_kv8_append", kv8_append_kernel<__nv_bfloat16>, dim3(grid), kAppendThreads, smem, st, 1, a);
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
    const GatherArgs a{h->g, c, rows, n, {out_k, out_v}};
    const long long total = static_cast<long long>(n) * h->g.Hkv * h->g.D;
    const int grid = static_cast<int>(std::min((total + 255) / 256, 16ll * h->num_sms));
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == SPECDEC_F32)
      op_launch("specdec_kv8_gather", kv8_gather_kernel<float>, dim3(grid), 256, 0, st, 1, a);
    else
      op_launch("specdec_kv8_gather", kv8_gather_kernel<__nv_bfloat16>, dim3(grid), 256, 0, st, 1, a);
  });
}

}  // extern "C"
