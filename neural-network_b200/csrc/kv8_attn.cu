// Attention over the 8-bit paged cache (specdec_kv8_attend).
#include "kv8_attn.cuh"

#include <cmath>

namespace specdec {

namespace {

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
};

// One warp per (row, head): scores and values one position at a time with a
// running maximum.  Right for every shape; nothing is reused between rows.
template <typename XT>
__global__ void __launch_bounds__(128) kv8_attend_simple_kernel(const AttendArgs a) {
  const Kv8Geom &g = a.g;
  const int lane = threadIdx.x & 31;
  const int per = (g.D + 31) / 32;
  for (long long w = blockIdx.x * 4ll + (threadIdx.x >> 5); w < static_cast<long long>(a.b.T) * g.H; w += gridDim.x * 4ll) {
    const int row = static_cast<int>(w / g.H), h = static_cast<int>(w % g.H), hk = h / g.G;
    int lo = 0, hi = a.b.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.b.cu_q[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    const Kv8Req r = kv8_req(a.b, g.P, lo);
    if (row < r.q0 || row >= r.q0 + r.q) continue;
    const int pos = r.len - r.q + row - r.q0;
    const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    float q[4], o[4], m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      o[i] = 0.f;
      q[i] = (i < per && d < g.D) ? to_f32(static_cast<const XT *>(a.q)[row * a.q_row + h * a.q_head + d]) : 0.f;
    }
    for (int p = first; p <= pos; ++p) {
      const int page = a.b.table[static_cast<long long>(lo) * a.b.cols + p / g.P];
      if (page < 0 || page >= a.c.n_pages) continue;
      const long long ph = static_cast<long long>(page) * g.Hkv + hk;
      const long long at = (ph * g.P + p % g.P) * g.D;
      const long long sat = ph * (g.P / g.t) + p % g.P / g.t;
      float dot = 0.f;
      for (int i = 0; i < per; ++i)
        if (lane + 32 * i < g.D) dot += q[i] * static_cast<float>(a.c.k[at + lane + 32 * i]);
      const float s = warp_sum(dot) * a.c.ks[sat] * a.scale;
      const float nm = fmaxf(m, s);
      const float al = expf(m - nm), e = expf(s - nm);
      m = nm;
      l = l * al + e;
      const float ev = e * a.c.vs[sat];
      for (int i = 0; i < per; ++i)
        if (lane + 32 * i < g.D) o[i] = o[i] * al + ev * static_cast<float>(a.c.v[at + lane + 32 * i]);
    }
    for (int i = 0; i < per; ++i)
      if (lane + 32 * i < g.D)
        static_cast<XT *>(a.out)[row * a.o_row + h * a.o_head + lane + 32 * i] = from_f32<XT>(l > 0.f ? o[i] / l : 0.f);
    if (a.lse && lane == 0) a.lse[w] = l > 0.f ? m + logf(l) : -INFINITY;
  }
}

}  // namespace

void kv8_attn_create(specdec_kv8 *) {}
void kv8_attn_destroy(specdec_kv8 *) {}

}  // namespace specdec

using namespace specdec;

extern "C" int specdec_kv8_attend(specdec_kv8 *h, const specdec_kv8_layer *layer, const specdec_kv8_batch *batch,
                                  const void *q, int64_t q_row_stride, int64_t q_head_stride, int dtype, int n_tokens,
                                  void *out, int64_t out_row_stride, int64_t out_head_stride, float *lse, int max_q,
                                  float scale, int window, void *stream) {
  if (!h) return SPECDEC_ERR_INVALID;
  return op_guard(h->err, [&] {
    const Kv8Layer c = kv8_layer(layer);
    const Kv8Batch b = kv8_batch(h, batch, n_tokens);
    op_check(dtype == SPECDEC_F32 || dtype == SPECDEC_BF16, "rows must be SPECDEC_F32 or SPECDEC_BF16");
    op_check(max_q >= 0 && window >= 0, "max_q and window must not be negative");
    op_check(std::isfinite(scale), "scale must be finite");
    if (b.B == 0 || b.T == 0) return;
    op_check(q && out, "null row buffer");
    DeviceScope scope(h->device);
    const AttendArgs a{h->g, c, b, q, q_row_stride, q_head_stride, out, out_row_stride, out_head_stride, lse, scale, window};
    const long long warps = static_cast<long long>(b.T) * h->g.H;
    const int grid = static_cast<int>(std::min((warps + 3) / 4, 16ll * h->num_sms));
    const auto st = static_cast<cudaStream_t>(stream);
    if (dtype == SPECDEC_F32)
      op_launch("specdec_kv8_attend", kv8_attend_simple_kernel<float>, dim3(grid), 128, 0, st, 1, a);
    else
      op_launch("specdec_kv8_attend", kv8_attend_simple_kernel<__nv_bfloat16>, dim3(grid), 128, 0, st, 1, a);
  });
}
