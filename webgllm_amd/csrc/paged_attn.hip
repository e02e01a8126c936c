// Attention over the paged cache: decode (one row a sequence) and prompts
// (rows of many sequences), both under an optional sliding window with the
// first entries kept visible.
#include "common.h"
#include "dot.h"
#include "paged_dev.h"

namespace wg {
namespace {

__device__ inline uint16_t half_of(float v) {
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}

struct RowArgs {
  const float *q;
  const int32_t *row_start;
  uint16_t *out;
  float *scores, *stats;  // of decode with weights: [sequences][H][ld_scores], [sequences][H][2]
  int ldq, ldo, M, H, KV, window, sinks;
  int64_t ld_scores;
};

// A wave a (row, query head), 64 of the entries that it sees at a time, a lane
// an entry: its score, then the running maximum and sum over the wave, then
// HD / 64 dims a lane of the weighted values.
template <int HD>
__global__ __launch_bounds__(64) void paged_row_kernel(const Paged c, const RowArgs a) {
  __shared__ float qs[HD];
  const int m = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  int b = m, back = 1;
  if (a.row_start) {
    b = find_seq(a.row_start, c.seqs, m);
    if (b < 0) return;
    back = a.row_start[b + 1] - m;
  }
  const int i = paged_len(c, b) - back, kvd = a.KV * HD;
  const Span sp = i < 0 ? Span{0, 0, 0} : paged_span(i, i, a.window, a.sinks);
  const int32_t *pages = c.table + (int64_t)b * c.ld_table;
  const int64_t head = (int64_t)(h / (a.H / a.KV)) * HD;
  for (int d = lane; d < HD; d += 64) qs[d] = a.q[(int64_t)m * a.ldq + (int64_t)h * HD + d];
  __syncthreads();
  float mx = -INFINITY, sum = 0.0f, o[HD / 64] = {};
  for (int t0 = 0; t0 < sp.count; t0 += 64) {
    const int t = t0 + lane;
    const int row = t < sp.count ? paged_row(c, pages, span_entry(sp, t)) : -1;
    float s = -INFINITY;
    if (row >= 0) {
      const _Float16 *k = reinterpret_cast<const _Float16 *>(c.k) + (int64_t)row * kvd + head;
      s = 0.0f;
      for (int d = 0; d < HD; d++) s = __builtin_fmaf(qs[d], (float)k[d], s);
    }
    if (a.scores && t < sp.count)
      a.scores[((int64_t)b * a.H + h) * a.ld_scores + t] = s;
    const float m2 = fmaxf(mx, wave_max(s)), mu = m2 == -INFINITY ? 0.0f : m2;
    const float w = __expf(s - mu), corr = __expf(mx - mu);
    sum = sum * corr + wave_sum(w);
    mx = m2;
#pragma unroll
    for (int e = 0; e < HD / 64; e++) o[e] *= corr;
    for (int u = 0; u < 64; u++) {
      const int r = __shfl(row, u, 64);
      const float wu = __shfl(w, u, 64);
      if (r < 0) continue;
      const _Float16 *v = reinterpret_cast<const _Float16 *>(c.v) + (int64_t)r * kvd + head;
#pragma unroll
      for (int e = 0; e < HD / 64; e++) o[e] = __builtin_fmaf(wu, (float)v[lane + 64 * e], o[e]);
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int e = 0; e < HD / 64; e++)
    a.out[(int64_t)m * a.ldo + (int64_t)h * HD + lane + 64 * e] = half_of(o[e] * inv);
  if (a.stats && lane == 0) {
    float *st = a.stats + ((int64_t)b * a.H + h) * 2;
    st[0] = mx == -INFINITY ? 0.0f : mx;
    st[1] = inv;
  }
}

// weights[b][entry] += its attention weight, summed over the heads in order.
__global__ __launch_bounds__(256) void paged_weights_kernel(const Paged c, const RowArgs a,
                                                            float *weights, int ldw) {
  const int b = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
  const int n = paged_len(c, b);
  if (n == 0) return;
  const Span sp = paged_span(n - 1, n - 1, a.window, a.sinks);
  if (t >= sp.count) return;
  float w = 0.0f;
  for (int h = 0; h < a.H; h++) {
    const int64_t bh = (int64_t)b * a.H + h;
    w += __expf(a.scores[bh * a.ld_scores + t] - a.stats[bh * 2]) * a.stats[bh * 2 + 1];
  }
  weights[(int64_t)b * ldw + span_entry(sp, t)] += w;
}

int check_attn(const float *q, int64_t M, int ldq, const wg_attn_shape *sh, const wg_paged_cache *c,
               int window, int sinks, const uint16_t *out, int ldo, int max_group,
               const char *who) {
  WG_REQUIRE(q && sh && out, "%s: null argument", who);
  const int H = sh->heads, KV = sh->kv_heads, hd = sh->head_dim;
  WG_REQUIRE(KV > 0 && H > 0 && H % KV == 0 && H / KV <= max_group && H <= 65535,
             "%s: %d query heads over %d KV heads", who, H, KV);
  WG_REQUIRE(hd == 64 || hd == 128, "%s: head_dim %d (64 or 128)", who, hd);
  const int rc = check_paged(c, (int64_t)KV * hd, true, who);
  if (rc) return rc;
  WG_REQUIRE(M >= 1, "%s: %lld rows", who, (long long)M);
  WG_REQUIRE(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", who, window, sinks);
  WG_REQUIRE(ldq >= (int64_t)H * hd && ldo >= (int64_t)H * hd, "%s: strides too small", who);
  WG_REQUIRE(((uintptr_t)q & 15) == 0 && ldq % 4 == 0,
             "%s: queries must be 16-byte aligned with a stride of 4k floats", who);
  WG_REQUIRE(!overlaps(q, ((size_t)(M - 1) * ldq + (size_t)H * hd) * 4, out,
                       ((size_t)(M - 1) * ldo + (size_t)H * hd) * 2),
             "%s: out overlaps q", who);
  return WG_OK;
}

int64_t score_stride(const wg_paged_cache *c) { return ((int64_t)c->max_entries + 63) / 64 * 64; }

}  // namespace
}  // namespace wg

using namespace wg;

extern "C" {

size_t wg_paged_decode_scratch_bytes(const wg_paged_cache *c, const wg_attn_shape *sh,
                                     int32_t with_weights) {
  if (!c || !sh || c->sequences < 1 || sh->heads < 1 || c->max_entries < 1) return 0;
  const int64_t rows = (int64_t)c->sequences * sh->heads;
  return with_weights ? (size_t)(((rows * 2 + 3) & ~3ll) + rows * score_stride(c)) * 4 : 0;
}

int wg_paged_attn_decode(const float *q, int32_t ldq, const wg_attn_shape *sh,
                         const wg_paged_cache *cache, int32_t window, int32_t sinks,
                         float *weights, int32_t ld_weights, uint16_t *out, int32_t ldo,
                         void *scratch, size_t scratch_bytes, void *stream) {
  int rc = check_attn(q, cache ? cache->sequences : 0, ldq, sh, cache, window, sinks, out, ldo, 64,
                      "wg_paged_attn_decode");
  if (rc) return rc;
  const size_t need = wg_paged_decode_scratch_bytes(cache, sh, weights != nullptr);
  WG_REQUIRE(scratch_bytes >= need && (!need || (scratch && ((uintptr_t)scratch & 15) == 0)),
             "wg_paged_attn_decode: scratch of %zu bytes, needs %zu (16-byte aligned)",
             scratch_bytes, need);
  WG_REQUIRE(!weights || ld_weights >= cache->max_entries,
             "wg_paged_attn_decode: weights of %d entries a sequence of up to %d", ld_weights,
             cache->max_entries);
  RowArgs a = {q, nullptr, out, nullptr, nullptr, ldq, ldo, cache->sequences, sh->heads,
               sh->kv_heads, window, sinks, score_stride(cache)};
  if (weights) {
    a.stats = (float *)scratch;
    a.scores = a.stats + (((int64_t)cache->sequences * sh->heads * 2 + 3) & ~3ll);
  }
  const Paged c = as_paged(cache);
  auto kernel = sh->head_dim == 64 ? paged_row_kernel<64> : paged_row_kernel<128>;
  kernel<<<dim3(a.M, a.H), 64, 0, as_stream(stream)>>>(c, a);
  rc = launched("wg_paged_attn_decode");
  if (rc || !weights) return rc;
  paged_weights_kernel<<<dim3((cache->max_entries + 255) / 256, a.M), 256, 0, as_stream(stream)>>>(
      c, a, weights, ld_weights);
  return launched("wg_paged_attn_decode");
}

size_t wg_paged_prefill_scratch_bytes(const wg_paged_cache *, const wg_attn_shape *, int32_t) {
  return 0;
}

int wg_paged_attn_prefill(const float *q, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                          const wg_paged_cache *cache, const int32_t *row_start, int32_t window,
                          int32_t sinks, uint16_t *out, int32_t ldo, void *scratch,
                          size_t scratch_bytes, void *stream) {
  int rc = check_attn(q, M, ldq, sh, cache, window, sinks, out, ldo, 32, "wg_paged_attn_prefill");
  if (rc) return rc;
  WG_REQUIRE(row_start, "wg_paged_attn_prefill: null row_start");
  const RowArgs a = {q, row_start, out, nullptr, nullptr, ldq, ldo, M, sh->heads, sh->kv_heads,
                     window, sinks, 0};
  auto kernel = sh->head_dim == 64 ? paged_row_kernel<64> : paged_row_kernel<128>;
  kernel<<<dim3(a.M, a.H), 64, 0, as_stream(stream)>>>(as_paged(cache), a);
  return launched("wg_paged_attn_prefill");
}

}  // extern "C"
