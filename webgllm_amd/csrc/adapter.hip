// Low-rank adapters of many requests beside a shared projection: y += s B (A x),
// each sequence's rows by its own adapter.
#include "common.h"
#include "paged_dev.h"

namespace wg {
namespace {

constexpr int PARTS = 4, MAX_RANK = 256;

struct AdapterArgs {
  const uint16_t *x, *a, *b;
  const int32_t *rank, *slot, *row_start;
  const float *scale, *row_scale;
  float *y, *t;  // t [M][parts][max_rank]: A x
  int M, ldx, ldy, slots, max_rank, K, N, parts, segments;
  int edge[PARTS];  // one past each part's last output
};

// Row m's adapter (-1: none) and its rank.
__device__ inline int adapter_of(const AdapterArgs &a, int m, int *rank) {
  int s = m, r0, r1, at;
  if (a.row_start) {
    s = find_segment(
        a.segments, m,
        [&](int i, bool whole, int *first, int *end, int *more) {
          *first = a.row_start[i];
          if (whole) {
            *end = a.row_start[i + 1];
            *more = a.slot[i];
          }
        },
        [](int first, int) { return first; }, &r0, &r1, &at);
    if (s < 0 || m >= r1) return -1;
  } else {
    at = a.slot[s];
  }
  if ((uint32_t)at >= (uint32_t)a.slots) return -1;
  *rank = min(max(a.rank[at], 0), a.max_rank);
  return *rank > 0 ? at : -1;
}

// A wave a row and factor row.
__global__ __launch_bounds__(64) void adapter_down_kernel(const AdapterArgs a) {
  const int m = blockIdx.x, part = blockIdx.z, r = blockIdx.y, lane = threadIdx.x;
  int rank;
  const int at = adapter_of(a, m, &rank);
  if (at < 0 || r >= rank) return;
  const uint16_t *w = a.a + (((int64_t)at * a.parts + part) * a.max_rank + r) * a.K;
  const uint16_t *x = a.x + (int64_t)m * a.ldx;
  float sum = 0.0f;
  for (int k = lane; k < a.K; k += 64) sum += half_to_float(w[k]) * half_to_float(x[k]);
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) a.t[((int64_t)m * a.parts + part) * a.max_rank + r] = sum;
}

// A thread a row and output.
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterArgs a) {
  const int m = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  int rank;
  const int at = adapter_of(a, m, &rank);
  if (at < 0 || n >= a.N) return;
  int part = 0;
  for (int p = 0; p + 1 < a.parts; p++) part += n >= a.edge[p];
  const uint16_t *w = a.b + ((int64_t)at * a.N + n) * a.max_rank;
  const float *t = a.t + ((int64_t)m * a.parts + part) * a.max_rank;
  float sum = 0.0f;
  for (int r = 0; r < rank; r++) sum += t[r] * half_to_float(w[r]);
  const float f = a.scale[at] * (a.row_scale ? a.row_scale[m] : 1.0f);
  a.y[(int64_t)m * a.ldy + n] += f * sum;
}

int check_adapters(const wg_adapters *ad, const char *who) {
  WG_REQUIRE(ad && ad->a && ad->b && ad->rank && ad->scale, "%s: null argument", who);
  WG_REQUIRE(ad->slots >= 1, "%s: %d adapters", who, ad->slots);
  WG_REQUIRE(ad->max_rank >= 8 && ad->max_rank <= MAX_RANK && ad->max_rank % 8 == 0,
             "%s: ranks up to %d (a multiple of 8 up to %d)", who, ad->max_rank, MAX_RANK);
  WG_REQUIRE(ad->K >= 8 && ad->K % 8 == 0, "%s: K %d (a multiple of 8)", who, ad->K);
  WG_REQUIRE(ad->parts >= 1 && ad->parts <= PARTS, "%s: %d parts (1 to %d)", who, ad->parts, PARTS);
  int64_t sum = 0;
  for (int p = 0; p < ad->parts; p++) {
    WG_REQUIRE(ad->cols[p] >= 4 && ad->cols[p] % 4 == 0, "%s: a part of %d outputs (a multiple of 4)",
               who, ad->cols[p]);
    sum += ad->cols[p];
  }
  WG_REQUIRE(sum == ad->N, "%s: parts of %lld outputs of %d", who, (long long)sum, ad->N);
  WG_REQUIRE((((uintptr_t)ad->a | (uintptr_t)ad->b) & 15) == 0,
             "%s: factors must be 16-byte aligned", who);
  return WG_OK;
}

}  // namespace
}  // namespace wg

using namespace wg;

extern "C" {

size_t wg_adapter_scratch_bytes(const wg_adapters *ad, int32_t M) {
  if (!ad || M < 1 || ad->parts < 1 || ad->parts > PARTS || ad->max_rank < 1) return 0;
  return (size_t)M * ad->parts * ad->max_rank * 4;
}

int wg_adapter_add(const uint16_t *x, int32_t M, int32_t ldx, const wg_adapters *ad,
                   const int32_t *slot, const int32_t *row_start, int32_t segments,
                   const float *row_scale, float *y, int32_t ldy, void *scratch,
                   size_t scratch_bytes, void *stream) {
  const int rc = check_adapters(ad, "wg_adapter_add");
  if (rc) return rc;
  WG_REQUIRE(x && slot && y, "wg_adapter_add: null argument");
  WG_REQUIRE(M >= 1 && segments >= 1 && segments <= 65535 && (row_start || M == segments),
             "wg_adapter_add: %d rows of %d sequences", M, segments);
  WG_REQUIRE(ldx >= ad->K && ldy >= ad->N, "wg_adapter_add: strides too small");
  WG_REQUIRE(((uintptr_t)x & 15) == 0 && ldx % 8 == 0,
             "wg_adapter_add: inputs must be 16-byte aligned with a stride of 8k halves");
  WG_REQUIRE(!overlaps(x, ((size_t)(M - 1) * ldx + ad->K) * 2, y,
                       ((size_t)(M - 1) * ldy + ad->N) * 4),
             "wg_adapter_add: y overlaps x");
  const size_t need = wg_adapter_scratch_bytes(ad, M);
  WG_REQUIRE(scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0,
             "wg_adapter_add: scratch of %zu bytes, needs %zu (16-byte aligned)", scratch_bytes,
             need);
  AdapterArgs a = {x, ad->a, ad->b, ad->rank, slot, row_start, ad->scale, row_scale, y,
                   (float *)scratch, M, ldx, ldy, ad->slots, ad->max_rank, ad->K, ad->N, ad->parts,
                   segments, {}};
  for (int p = 0, e = 0; p < ad->parts; p++) a.edge[p] = e += ad->cols[p];
  hipStream_t s = as_stream(stream);
  adapter_down_kernel<<<dim3(M, ad->max_rank, ad->parts), 64, 0, s>>>(a);
  adapter_up_kernel<<<dim3((ad->N + 255) / 256, M), 256, 0, s>>>(a);
  return launched("wg_adapter_add");
}

}  // extern "C"
