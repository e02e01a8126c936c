// Low-rank adapters of many requests beside a shared projection: y += s B (A x),
// each sequence's rows by its own adapter. Two launches, t = A x and y += s B t:
// a row a sequence on the vector units, where only the factors' bytes count;
// rows of several tokens on MFMA, where the rows of y do.
#include "common.h"
#include "dot.h"
#include "paged_dev.h"

namespace wg {
namespace {

constexpr int PARTS = 4, MAX_RANK = 256;

struct AdapterArgs {
  const uint16_t *x, *a, *b;
  const int32_t *rank, *slot, *row_start;
  const float *scale, *row_scale;
  float *y, *t;  // t [splits][M][parts][max_rank]: shares of A x
  int M, ldx, ldy, slots, max_rank, K, N, parts, segments, splits, wide, vec;
  int edge[PARTS];  // one past each part's last output
  int tile[PARTS];  // one past each part's last tile of `wide` outputs
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f4v __attribute__((ext_vector_type(4)));

// Slot `at`'s rank, 0 where it is none.
__device__ inline int rank_of(const AdapterArgs &a, int at) {
  return (uint32_t)at < (uint32_t)a.slots ? min(max(a.rank[at], 0), a.max_rank) : 0;
}

// The part and the outputs n0 .. n1 - 1 of tile i.
__device__ inline int tile_part(const AdapterArgs &a, int i, int *n0, int *n1) {
  int p = 0, t0 = 0, e0 = 0;
#pragma unroll
  for (int q = 0; q + 1 < PARTS; q++)
    if (q + 1 < a.parts && i >= a.tile[q]) p = q + 1, t0 = a.tile[q], e0 = a.edge[q];
  *n0 = e0 + (i - t0) * a.wide;
  int end = a.edge[0];
#pragma unroll
  for (int q = 1; q < PARTS; q++)
    if (q == p) end = a.edge[q];
  *n1 = min(*n0 + a.wide, end);
  return p;
}

// ------------------------------------------------------------ a row a sequence
//
// A wave takes RPW rows of the first factor, 512 of their inputs at a time as
// whole kilobytes, against the same piece of x: halves' products in pairs, sums
// in f32 (v_dot2_f32_f16).
template <int RPW>
__global__ __launch_bounds__(256) void adapter_token_down_kernel(const AdapterArgs a) {
  constexpr int U = 4;
  const int m = blockIdx.x, part = blockIdx.z, lane = threadIdx.x & 63;
  const int r0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * RPW;
  const int at = a.slot[m], rank = rank_of(a, at);
  if (r0 >= rank) return;
  const uint16_t *x = a.x + (int64_t)m * a.ldx;
  const uint16_t *w = a.a + (((int64_t)at * a.parts + part) * a.max_rank + r0) * a.K;
  float sum[RPW] = {};
  for (int k0 = lane * 8; k0 - lane * 8 < a.K; k0 += U * 512) {
    uint4 xv[U], wv[U][RPW];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int k = k0 + u * 512;
      xv[u] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < RPW; r++) wv[u][r] = make_uint4(0, 0, 0, 0);
      if (k >= a.K) continue;
      xv[u] = *reinterpret_cast<const uint4 *>(x + k);
#pragma unroll
      for (int r = 0; r < RPW; r++)  // (a row past the rank: the last one again)
        wv[u][r] = *reinterpret_cast<const uint4 *>(w + (int64_t)min(r, rank - 1 - r0) * a.K + k);
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int r = 0; r < RPW; r++) {
        sum[r] = dot2(wv[u][r].x, xv[u].x, sum[r]);
        sum[r] = dot2(wv[u][r].y, xv[u].y, sum[r]);
        sum[r] = dot2(wv[u][r].z, xv[u].z, sum[r]);
        sum[r] = dot2(wv[u][r].w, xv[u].w, sum[r]);
      }
  }
  float *t = a.t + ((int64_t)m * a.parts + part) * a.max_rank + r0;
#pragma unroll
  for (int r = 0; r < RPW; r++) {
    const float v = wave_sum_u(sum[r]);
    if (lane == 0 && r0 + r < rank) t[r] = v;
  }
}

// A thread an output of a row: its factor row in 16-byte pieces, against t, which
// is the same for the workgroup.
__global__ __launch_bounds__(256) void adapter_token_up_kernel(const AdapterArgs a) {
  const int m = blockIdx.y;
  int n0, n1;
  const int part = tile_part(a, blockIdx.x, &n0, &n1), n = n0 + threadIdx.x;
  const int at = a.slot[m], rank = rank_of(a, at);
  if (rank == 0 || n >= n1) return;
  const uint16_t *w = a.b + ((int64_t)at * a.N + n) * a.max_rank;
  const float *t = a.t + ((int64_t)m * a.parts + part) * a.max_rank;
  float *yp = a.y + (int64_t)m * a.ldy + n;
  const float y = *yp;
  float sum = 0.0f;
  constexpr int U = 8;
  int r0 = 0;
  for (; r0 < rank; r0 += 8 * U) {
    half8 v[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (r0 + 8 * u < rank) v[u] = *reinterpret_cast<const half8 *>(w + r0 + 8 * u);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int r = r0 + 8 * u + e;
        if (r < rank) sum = __builtin_fmaf(t[r], (float)v[u][e], sum);
      }
  }
  *yp = __builtin_fmaf(a.scale[at] * (a.row_scale ? a.row_scale[m] : 1.0f), sum, y);
}

// -------------------------------------------------------- rows of several tokens
//
// Blocks of 16 MT rows of one sequence. Blocks of sequence b are numbered from
// row_start[b] / (16 MT) + b on, which leaves each at least as many as it needs.
struct Block {
  int at, rank, m0, m1;  // its slot, and rows m0 .. m1 - 1 (none where m0 >= m1)
};
template <int MT>
__device__ inline Block block_of(const AdapterArgs &a, int blk) {
  constexpr int R = 16 * MT;
  auto block0 = [&](int first, int b) { return min(max(first, 0), a.M) / R + b; };
  Block k = {0, 0, 0, 0};
  int r0, r1, at;
  const int b = find_segment(
      a.segments, blk,
      [&](int i, bool whole, int *first, int *end, int *more) {
        *first = a.row_start[i];
        if (whole) {
          *end = a.row_start[i + 1];
          *more = a.slot[i];
        }
      },
      block0, &r0, &r1, &at);
  if (b < 0) return k;
  k.m0 = max(r0, 0) + (blk - block0(r0, b)) * R;
  k.m1 = min(min(r1, a.M), k.m0 + R);
  if (k.m0 >= k.m1) return k;
  k.at = at;
  k.rank = rank_of(a, at);
  return k;
}

// t = A x on v_mfma_f32_16x16x32_f16: A operand 16 factor rows, B operand 16 rows
// of x, both 16 bytes a lane straight from memory; a lane then holds 4
// neighbouring ranks of a row. The inputs are split over the workgroup's 4 waves,
// whose sums meet in LDS in order, and over `splits` workgroups.
template <int MT>
__global__ __launch_bounds__(256) void adapter_rows_down_kernel(const AdapterArgs a) {
  constexpr int RT = 4, U = MT == 1 ? 4 : 2;
  __shared__ f4v part_sum[3][MT * RT][64];
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block k = block_of<MT>(a, blockIdx.x);
  const int chunks = (a.max_rank + 63) >> 6, part = blockIdx.y / chunks;
  const int rc = blockIdx.y % chunks * 64;
  if (rc >= k.rank) return;
  const int tiles = min((k.rank - rc + 15) >> 4, RT);
  const int steps = (a.K + 31) >> 5, shares = a.splits * 4, share = blockIdx.z * 4 + wave;
  const int s0 = (int)((int64_t)steps * share / shares);
  const int s1 = (int)((int64_t)steps * (share + 1) / shares);
  const uint16_t *xp[MT], *wp[RT];
#pragma unroll
  for (int i = 0; i < MT; i++)
    xp[i] = a.x + (int64_t)min(k.m0 + 16 * i + n16, k.m1 - 1) * a.ldx + 8 * c4;
#pragma unroll
  for (int i = 0; i < RT; i++)
    wp[i] = a.a + (((int64_t)k.at * a.parts + part) * a.max_rank + min(rc + 16 * i + n16, k.rank - 1)) * a.K +
            8 * c4;
  f4v acc[MT][RT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < RT; j++) acc[i][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  half8 xv[2][U][MT], wv[2][U][RT];
  auto load = [&](int s, half8 (&x)[U][MT], half8 (&w)[U][RT]) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = (s + u) * 32;
      const bool in = s + u < s1 && at + 8 * c4 < a.K;
#pragma unroll
      for (int i = 0; i < MT; i++) {
        x[u][i] = half8{};
        if (in) x[u][i] = *reinterpret_cast<const half8 *>(xp[i] + at);
      }
#pragma unroll
      for (int j = 0; j < RT; j++) {
        w[u][j] = half8{};
        if (in && j < tiles) w[u][j] = *reinterpret_cast<const half8 *>(wp[j] + at);
      }
    }
  };
  auto multiply = [&](half8 (&x)[U][MT], half8 (&w)[U][RT]) {
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < RT; j++)
        if (j < tiles)
#pragma unroll
          for (int i = 0; i < MT; i++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[u][j], x[u][i], acc[i][j], 0, 0, 0);
  };
  load(s0, xv[0], wv[0]);
  for (int s = s0; s < s1; s += 2 * U) {
    load(s + U, xv[1], wv[1]);
    multiply(xv[0], wv[0]);
    load(s + 2 * U, xv[0], wv[0]);
    multiply(xv[1], wv[1]);
  }
  if (wave > 0)
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < RT; j++)
        if (j < tiles) part_sum[wave - 1][i * RT + j][lane] = acc[i][j];
  __syncthreads();
  if (wave > 0) return;
  float *t = a.t + (int64_t)blockIdx.z * a.M * a.parts * a.max_rank;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < RT; j++) {
      const int m = k.m0 + 16 * i + n16, r = rc + 16 * j + 4 * c4;
      if (j >= tiles || m >= k.m1 || r >= k.rank) continue;
      f4v v = acc[i][j];
#pragma unroll
      for (int w = 0; w < 3; w++) v += part_sum[w][i * RT + j][lane];
      *reinterpret_cast<f4v *>(t + ((int64_t)m * a.parts + part) * a.max_rank + r) = v;
    }
}

// y += f B t on the same instruction: A operand 16 outputs' factor rows, B operand
// 16 rows of t, each scaled by a power of two to the top of the halves and split
// into hi = half(t) and lo = half(t - hi) (22 bits of its largest value); a lane
// then holds 4 neighbouring outputs of a row. t's shares are added up in order
// once a workgroup; its `wide` outputs stream by, 32 a wave and step.
template <int MT>
__global__ __launch_bounds__(256) void adapter_rows_up_kernel(const AdapterArgs a) {
  constexpr int R = 16 * MT, NT = 2, TPR = 256 / R;  // threads that prepare a row of t
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float factor[R];
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block k = block_of<MT>(a, blockIdx.x);
  if (k.rank == 0) return;
  int n0, n1;
  const int part = tile_part(a, blockIdx.y, &n0, &n1);
  const int steps = (k.rank + 31) >> 5, stride = steps * 128 + 16;  // bytes of a row of t
  {
    const int row = threadIdx.x / TPR, sub = threadIdx.x % TPR, m = k.m0 + row;
    unsigned char *to = smem + row * stride;
    const float *t = a.t + ((int64_t)min(m, k.m1 - 1) * a.parts + part) * a.max_rank;
    const int64_t share = (int64_t)a.M * a.parts * a.max_rank;
    float big = 0.0f;
    for (int p = sub; p < steps * 8; p += TPR) {  // 4 ranks each
      f4v v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (m < k.m1 && 4 * p < k.rank) {
        for (int s = 0; s < a.splits; s++) v += *reinterpret_cast<const f4v *>(t + s * share + 4 * p);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (4 * p + e >= k.rank) v[e] = 0.0f;
          big = fmaxf(big, fabsf(v[e]));
        }
      }
      *reinterpret_cast<f4v *>(to + p * 16) = v;
    }
    // (the row's threads are neighbours)
#pragma unroll
    for (int o = 1; o < TPR; o *= 2) big = fmaxf(big, __shfl_xor(big, o, 64));
    // 2^e with big 2^e in [2^13, 2^14); an exponent that float32 holds both ways
    const int log = big > 0.0f && big < INFINITY ? ilogbf(big) : 13;
    const int e2 = min(max(13 - log, -114), 100);
    const float up = ldexpf(1.0f, e2);
    if (sub == 0)
      factor[row] = ldexpf(1.0f, -e2) * a.scale[k.at] *
                    (a.row_scale && m < k.m1 ? a.row_scale[m] : 1.0f);
    for (int p = sub; p < steps * 8; p += TPR) {
      const f4v v = *reinterpret_cast<const f4v *>(to + p * 16) * up;
      half8 h;  // 4 hi, 4 lo
#pragma unroll
      for (int e = 0; e < 4; e++) {
        h[e] = (_Float16)v[e];
        h[4 + e] = (_Float16)(v[e] - (float)h[e]);
      }
      *reinterpret_cast<half8 *>(to + p * 16) = h;
    }
  }
  __syncthreads();
  float f[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) f[i] = factor[16 * i + n16];
  for (int n = n0 + wave * 16 * NT; n < n1; n += 64 * NT) {
    f4v y[MT][NT], acc[MT][NT];
    auto place = [&](int i, int j) {
      return a.y + (int64_t)(k.m0 + 16 * i + n16) * a.ldy + n + 16 * j + 4 * c4;
    };
    auto mine = [&](int i, int j) { return k.m0 + 16 * i + n16 < k.m1 && n + 16 * j + 4 * c4 < n1; };
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) {
        acc[i][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        if (!mine(i, j)) continue;
        const float *p = place(i, j);
        if (a.vec) y[i][j] = *reinterpret_cast<const f4v *>(p);
        else y[i][j] = f4v{p[0], p[1], p[2], p[3]};
      }
    const uint16_t *wp[NT];
#pragma unroll
    for (int j = 0; j < NT; j++)
      wp[j] = a.b + ((int64_t)k.at * a.N + min(n + 16 * j + n16, n1 - 1)) * a.max_rank + 8 * c4;
    for (int s = 0; s < steps; s++) {
      const int left = k.rank - 32 * s - 8 * c4;  // of this lane's 8 ranks
      half8 w[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        w[j] = half8{};
        if (left > 0) w[j] = *reinterpret_cast<const half8 *>(wp[j] + 32 * s);
        if (left < 8)
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (e >= left) w[j][e] = (_Float16)0.0f;
      }
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const unsigned char *tp = smem + (16 * i + n16) * stride + s * 128 + c4 * 32;
        const half8 p0 = *reinterpret_cast<const half8 *>(tp);
        const half8 p1 = *reinterpret_cast<const half8 *>(tp + 16);
        const half8 hi = __builtin_shufflevector(p0, p1, 0, 1, 2, 3, 8, 9, 10, 11);
        const half8 lo = __builtin_shufflevector(p0, p1, 4, 5, 6, 7, 12, 13, 14, 15);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], hi, acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], lo, acc[i][j], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) {
        if (!mine(i, j)) continue;
        f4v v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = __builtin_fmaf(f[i], acc[i][j][e], y[i][j][e]);
        float *p = place(i, j);
        if (a.vec) {
          *reinterpret_cast<f4v *>(p) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) p[e] = v[e];
        }
      }
  }
}

// Rows a block takes (16 mt) and workgroups that share a block's inputs.
struct RowsPlan {
  int mt, splits;
  int64_t blocks;
};
RowsPlan rows_plan(const wg_adapters *ad, int64_t M, int64_t segments) {
  RowsPlan p;
  p.mt = M >= 32 * segments ? 4 : 1;
  p.blocks = (M - 1) / (16 * p.mt) + segments;
  const int64_t busy = ((M + 16 * p.mt - 1) / (16 * p.mt) + segments / 2) * ad->parts;
  const int64_t fill = 512 / busy, most = ad->K / 512;  // (a wave: 4 steps at least)
  const int64_t s = fill < most ? fill : most;
  p.splits = s < 1 ? 1 : s > 8 ? 8 : (int)s;
  return p;
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
  if (!ad || M < 1 || ad->parts < 1 || ad->parts > PARTS || ad->max_rank < 1 || ad->K < 1) return 0;
  // (the most shares that any number of sequences gives these rows)
  const int splits = rows_plan(ad, M, 1).splits;
  return (size_t)M * ad->parts * ad->max_rank * 4 * splits;
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
                   segments, 1, 256, ((uintptr_t)y & 15) == 0 && ldy % 4 == 0, {}, {}};
  hipStream_t s = as_stream(stream);
  auto tiles = [&](int wide) {
    a.wide = wide;
    int e = 0, t = 0;
    for (int p = 0; p < ad->parts; p++) {
      a.edge[p] = e += ad->cols[p];
      a.tile[p] = t += (ad->cols[p] + wide - 1) / wide;
    }
    return (unsigned)t;
  };
  if (!row_start) {
    if ((int64_t)M * ad->parts * ad->max_rank <= 2048)
      adapter_token_down_kernel<1><<<dim3(M, (ad->max_rank + 3) / 4, ad->parts), 256, 0, s>>>(a);
    else
      adapter_token_down_kernel<4><<<dim3(M, (ad->max_rank + 15) / 16, ad->parts), 256, 0, s>>>(a);
    const unsigned n = tiles(256);
    adapter_token_up_kernel<<<dim3(n, M), 256, 0, s>>>(a);
    return launched("wg_adapter_add");
  }
  const RowsPlan p = rows_plan(ad, M, segments);
  WG_REQUIRE(p.blocks <= 0x7fffffff, "wg_adapter_add: %d rows of %d sequences", M, segments);
  a.splits = p.splits;
  const dim3 down((unsigned)p.blocks, ad->parts * ((ad->max_rank + 63) / 64), p.splits);
  const int64_t busy = p.blocks * ((ad->N + 1023) / 1024);
  const unsigned n = tiles(busy >= 512 ? 1024 : busy >= 256 ? 512 : 256);
  WG_REQUIRE(n <= 65535, "wg_adapter_add: %d outputs", ad->N);
  const int lds = 16 * p.mt * ((ad->max_rank + 31) / 32 * 128 + 16);
  auto up = p.mt == 4 ? adapter_rows_up_kernel<4> : adapter_rows_up_kernel<1>;
  if (lds > 64 * 1024 - 1024) {
    const int rl = raise_lds((const void *)up, lds);
    if (rl) return rl;
  }
  if (p.mt == 4) adapter_rows_down_kernel<4><<<down, 256, 0, s>>>(a);
  else adapter_rows_down_kernel<1><<<down, 256, 0, s>>>(a);
  up<<<dim3((unsigned)p.blocks, n), 256, lds, s>>>(a);
  return launched("wg_adapter_add");
}

}  // extern "C"
