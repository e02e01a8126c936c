// Low-rank adapters of many requests beside a shared projection: y += s B (A x),
// each sequence's rows by its own adapter. Two launches, t = A x and y += s B t
// (every workgroup of the second needs all of a row's t): a row a sequence on the
// vector units, where only the factors' bytes count; rows of several tokens on MFMA,
// where the rows of y do.
#include <type_traits>

#include "common.h"
#include "dot.h"
#include "lds_load.h"
#include "paged_dev.h"

namespace wg {
namespace {

constexpr int PARTS = 4, MAX_RANK = 256;
constexpr int ONE_RANK = 16;  // ranks up to which one launch takes both factors of a token

struct AdapterArgs {
  const uint16_t *x, *a, *b;
  const int32_t *rank, *slot, *row_start;
  const float *scale, *row_scale;
  float *y, *t;  // t [splits][M][parts][max_rank]: shares of A x
  int M, ldx, ldy, slots, max_rank, K, N, parts, segments, splits, wide;
  int edge[PARTS];  // one past each part's last output
  int tile[PARTS];  // one past each part's last tile of `wide` outputs
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

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
// A wave takes RPW rows of the first factor, 512 U of their inputs at a time as
// whole kilobytes, against the same piece of x: halves' products in pairs, sums
// in f32 (v_dot2_f32_f16). Bound by HBM behind the chain slot, rank, factor: 64
// tokens of 40 adapters of ranks 8 to 64, 4096 inputs to three parts of 6144 outputs
// (42 MB in both launches) take 8.0 us here and 7.9 below, 2.6 TB/s (137 us by a
// thread an output); 24 of rank 16, 2048 inputs to 16,384 outputs (19 MB) 3.3 and 5.1.
constexpr int U = 8;
// 16 bytes of a row of K halves from its k-th on; zeros behind its end (of both
// operands: what lies there could be an infinity, and 0 times that is NaN).
__device__ inline __amdgpu_buffer_rsrc_t row_of(const uint16_t *row, int K) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)row, (short)0, (int)(2u * K), 0x00020000);
}
__device__ inline uint4 load_row(__amdgpu_buffer_rsrc_t row, int k) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(row, (int)(2u * k), 0, 0));
}
__device__ inline void load_x(const AdapterArgs &a, const uint16_t *x, int k0, uint4 (&xv)[U]) {
  const auto row = row_of(x, a.K);
#pragma unroll
  for (int u = 0; u < U; u++) xv[u] = load_row(row, k0 + u * 512 + (threadIdx.x & 63) * 8);
}
// Factor rows r0 .. r0 + RPW - 1 (w: the part's first) times x, whose first inputs
// xv holds: the wave's sums to t.
template <int RPW>
__device__ inline void token_down(const AdapterArgs &a, const uint16_t *x, uint4 (&xv)[U],
                                  const uint16_t *w, int r0, int rank, float *t) {
  const int lane = threadIdx.x & 63;
  __amdgpu_buffer_rsrc_t row[RPW];
#pragma unroll
  for (int r = 0; r < RPW; r++)  // (or the last)
    row[r] = row_of(w + (int64_t)min(r0 + r, rank - 1) * a.K, a.K);
  float sum[RPW] = {};
  for (int k0 = 0; k0 < a.K; k0 += U * 512) {
    uint4 wv[U][RPW];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int r = 0; r < RPW; r++) wv[u][r] = load_row(row[r], k0 + u * 512 + lane * 8);
    __builtin_amdgcn_sched_barrier(0);  // (the compiler would load where it multiplies)
    if (a.K > U * 512) load_x(a, x, k0, xv);
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
#pragma unroll
  for (int r = 0; r < RPW; r++) {
    const float v = wave_sum_u(sum[r]);
    if (lane == 0 && r0 + r < rank) t[r0 + r] = v;
  }
}
template <int RPW>
__global__ __launch_bounds__(256) void adapter_token_down_kernel(const AdapterArgs a) {
  const int m = blockIdx.x, part = blockIdx.z;
  const int r0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * RPW;
  const uint16_t *x = a.x + (int64_t)m * a.ldx;
  uint4 xv[U];
  load_x(a, x, 0, xv);  // (while the adapter is looked up)
  const int at = a.slot[m], rank = rank_of(a, at);
  if (r0 >= rank) return;
  token_down<RPW>(a, x, xv, a.a + ((int64_t)at * a.parts + part) * a.max_rank * a.K, r0, rank,
                  a.t + ((int64_t)m * a.parts + part) * a.max_rank);
}

// The sum over each P neighbouring lanes, on all of them (P up to 32).
template <int P>
__device__ inline float lanes_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x),
                                                              decltype(ctrl)::value, 0xf, 0xf, false));
  };
  if constexpr (P > 1) v += dpp(v, std::integral_constant<int, 0xb1>{});   // quad_perm [1, 0, 3, 2]
  if constexpr (P > 2) v += dpp(v, std::integral_constant<int, 0x4e>{});   // quad_perm [2, 3, 0, 1]
  if constexpr (P > 4) v += dpp(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (P > 8) v += dpp(v, std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (P > 16) v += xor16(v);
  return v;
}

// P lanes take a factor row of the second, 8 ranks each, so that a wave's load is
// of whole rows; lane p of them adds up P rows with the others and keeps the p-th,
// so that 64 neighbouring outputs end on the wave's 64 lanes. BOTH: the workgroup
// makes t itself, every one its own, which saves a launch where there are few.
template <int P, bool BOTH>
__global__ __launch_bounds__(256) void adapter_token_up_kernel(const AdapterArgs a) {
  constexpr int NB = P >= 8 ? 1 : 8 / P, UP = P < 8 ? P : 8;  // 64 outputs NB times; loads in flight
  __shared__ float own_t[BOTH ? ONE_RANK : 1];
  const int m = blockIdx.y, lane = threadIdx.x & 63, p = lane % P;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint16_t *x = a.x + (int64_t)m * a.ldx;
  uint4 xv[U];
  if constexpr (BOTH) load_x(a, x, 0, xv);  // (while the adapter is looked up)
  int n0, n1;
  const int part = tile_part(a, blockIdx.x, &n0, &n1);
  const int at = a.slot[m], rank = rank_of(a, at);
  if (rank == 0) return;
  n0 += wave * 64 * NB;
  // (behind the rank what lies last under it again, not a row's lines that count nothing:
  // 64 tokens of rank 16 in slots of 256, 2048 inputs to 16,384 outputs, 37 us, 109)
  const uint16_t *w = a.b + (int64_t)at * a.N * a.max_rank + min(8 * p, (rank - 1) & ~7);
  float y[NB], mine[NB];
  half8 v[NB][UP];
  float *yp = a.y + (int64_t)m * a.ldy;
  auto load = [&](int j0) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < UP; j++)
        v[b][j] = *reinterpret_cast<const half8 *>(
            w + (int64_t)min(n0 + 64 * b + (lane - p) + j0 + j, n1 - 1) * a.max_rank);
  };
#pragma unroll
  for (int b = 0; b < NB; b++) y[b] = yp[min(n0 + 64 * b + lane, n1 - 1)];
  const float *tp = a.t + ((int64_t)m * a.parts + part) * a.max_rank;
  if constexpr (BOTH) {
    load(0);
    for (int r0 = 2 * wave; r0 < rank; r0 += 8)
      token_down<2>(a, x, xv, a.a + ((int64_t)at * a.parts + part) * a.max_rank * a.K, r0, rank,
                    own_t);
    __syncthreads();
    tp = own_t;
  }
  if (n0 >= n1) return;
  // this lane's 8 ranks of t; nothing behind the rank, there and in the factor
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; e++) t[e] = 8 * p + e < rank ? tp[8 * p + e] : 0.0f;
  u4v keep;
#pragma unroll
  for (int i = 0; i < 4; i++)
    keep[i] = (uint32_t)((1ull << min(max((rank - 8 * p - 2 * i) * 16, 0), 32)) - 1);
  const float f = a.scale[at] * (a.row_scale ? a.row_scale[m] : 1.0f);
#pragma unroll
  for (int j0 = 0; j0 < P; j0 += UP) {
    if (!BOTH || j0) load(j0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < UP; j++) {
        const half8 h = __builtin_bit_cast(half8, __builtin_bit_cast(u4v, v[b][j]) & keep);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) s = __builtin_fmaf(t[e], (float)h[e], s);
        s = lanes_sum<P>(s);
        mine[b] = j0 + j == 0 || j0 + j == p ? s : mine[b];
      }
  }
#pragma unroll
  for (int b = 0; b < NB; b++)
    if (n0 + 64 * b + lane < n1) yp[n0 + 64 * b + lane] = __builtin_fmaf(f, mine[b], y[b]);
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
  const int at_blk = blk - block0(r0, b);
  if (at_blk < 0) return k;  // (starts that do not ascend)
  k.m0 = max(r0, 0) + at_blk * R;
  k.m1 = min(min(r1, a.M), k.m0 + R);
  if (k.m0 >= k.m1) return k;
  k.at = at;
  k.rank = rank_of(a, at);
  return k;
}

// t = A x on v_mfma_f32_16x16x32_f16, A operand 16 factor rows, B operand 16 rows
// of x; a lane then holds 4 neighbouring ranks of a row. A workgroup takes 4 tiles
// of 16 factor rows, of whichever parts, and 128 inputs at a time: 256 bytes of
// each row by direct-to-LDS loads, a step's two steps ahead, of which each of its
// 4 waves multiplies 32 (loads into registers as the operands lie would take 64
// bytes of 16 rows each, and half the time again). The waves' sums meet in LDS in
// order. 5 prompts of 131 to 900 rows, ranks up to 64, 4096 inputs to three parts:
// 13.8 us, latency (x and the factors are 23 MB); 2048 rows of rank 32 10.6. `splits`
// workgroups share the inputs: those of one share are 8 / splits
// XCDs', so that x and A come into few L2s.
constexpr int KB = 128;  // inputs a step
template <int MT>
constexpr int DOWN_LDS = 3 * 16 * (MT + 4) * KB * 2;
template <int MT, int RT>
__device__ inline void rows_down(const AdapterArgs &a, const Block &k, int split, int tile0,
                                 unsigned char *smem) {
  constexpr int ROWB = KB * 2, LPW = MT + RT, TILE = 16 * LPW * ROWB;
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (k.rank + 15) >> 4;
  // each load takes 4 rows, this lane's rl of a tile, 16-byte piece p at p ^ rl
  const int rl = 4 * wave + c4, col = (n16 ^ rl) * 8;
  const uint16_t *from[LPW];
  int part[RT], r0[RT];
#pragma unroll
  for (int i = 0; i < MT; i++) from[i] = a.x + (int64_t)min(k.m0 + 16 * i + rl, k.m1 - 1) * a.ldx;
#pragma unroll
  for (int j = 0; j < RT; j++) {
    part[j] = (tile0 + j) / per;
    r0[j] = (tile0 + j) % per * 16;
    from[MT + j] =
        a.a + (((int64_t)k.at * a.parts + part[j]) * a.max_rank + min(r0[j] + rl, k.rank - 1)) * a.K;
  }
  const int steps = (a.K + KB - 1) / KB;
  const int s0 = (int)((int64_t)steps * split / a.splits);
  const int s1 = (int)((int64_t)steps * (split + 1) / a.splits);
  const uint32_t lds = (uint32_t)(uintptr_t)smem + 4 * wave * ROWB;
  auto issue = [&](int s) {
    const int at = min(s * KB + col, a.K - 8);  // (behind K: what the row holds, cleared below)
#pragma unroll
    for (int i = 0; i < LPW; i++)
      dma16(from[i] + at, __builtin_amdgcn_readfirstlane(lds + (s - s0) % 3 * TILE + 16 * i * ROWB));
  };
  f4v acc[MT][RT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < RT; j++) acc[i][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  if (s0 < s1) issue(s0);
  if (s0 + 1 < s1) issue(s0 + 1);
  for (int s = s0; s < s1; s++) {
    // this step's loads have landed, and every wave is done with the one before
    if (s + 1 < s1) wait_vm<LPW>();
    else wait_vm<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    barrier();
    if (s + 2 < s1) issue(s + 2);
    const unsigned char *tile =
        smem + (s - s0) % 3 * TILE + n16 * ROWB + (((4 * wave + c4) ^ n16) * 16);
    half8 x[MT], w[RT];
#pragma unroll
    for (int i = 0; i < MT; i++) x[i] = *reinterpret_cast<const half8 *>(tile + 16 * i * ROWB);
#pragma unroll
    for (int j = 0; j < RT; j++) w[j] = *reinterpret_cast<const half8 *>(tile + 16 * (MT + j) * ROWB);
    if (s * KB + 32 * wave + 32 > a.K) {
      const bool in = s * KB + 32 * wave + 8 * c4 < a.K;
#pragma unroll
      for (int i = 0; i < MT; i++) x[i] = in ? x[i] : half8{};
#pragma unroll
      for (int j = 0; j < RT; j++) w[j] = in ? w[j] : half8{};  // (an infinity times 0 is NaN)
    }
#pragma unroll
    for (int j = 0; j < RT; j++)
#pragma unroll
      for (int i = 0; i < MT; i++)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], x[i], acc[i][j], 0, 0, 0);
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  barrier();
  f4v *sums = reinterpret_cast<f4v *>(smem);  // [3][MT * RT][64], over the tiles
  if (wave > 0)
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < RT; j++) sums[((wave - 1) * MT * RT + i * RT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (wave > 0) return;
  float *t = a.t + (int64_t)split * a.M * a.parts * a.max_rank;
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < RT; j++) {
      const int m = k.m0 + 16 * i + n16, r = r0[j] + 4 * c4;
      if (m >= k.m1 || r >= k.rank) continue;
      f4v v = acc[i][j];
#pragma unroll
      for (int w = 0; w < 3; w++) v += sums[(w * MT * RT + i * RT + j) * 64 + lane];
      *reinterpret_cast<f4v *>(t + ((int64_t)m * a.parts + part[j]) * a.max_rank + r) = v;
    }
}
template <int MT>
__global__ __launch_bounds__(256) void adapter_rows_down_kernel(const AdapterArgs a) {
  extern __shared__ __align__(1024) unsigned char tiles_lds[];  // DOWN_LDS<MT>
  const int split = blockIdx.x % a.splits, tile0 = blockIdx.y * 4;
  const Block k = block_of<MT>(a, blockIdx.x / a.splits);
  const int tiles = ((k.rank + 15) >> 4) * a.parts - tile0;
  if (tiles >= 4) rows_down<MT, 4>(a, k, split, tile0, tiles_lds);
  else if (tiles == 3) rows_down<MT, 3>(a, k, split, tile0, tiles_lds);
  else if (tiles == 2) rows_down<MT, 2>(a, k, split, tile0, tiles_lds);
  else if (tiles == 1) rows_down<MT, 1>(a, k, split, tile0, tiles_lds);
}

// y += f B t on the same instruction: A operand 16 outputs' factor rows, B operand
// 16 rows of t, each scaled by a power of two to the top of the halves and split
// into hi = half(t) and lo = half(t - hi) (22 bits of its largest value). t's
// shares are added up in order once a workgroup; its `wide` outputs stream by, 32
// a wave and step, the next step's y under this one's products. A lane's sums are
// 4 neighbouring outputs of a row; through LDS 8 lanes take a row's 32, so that
// memory sees whole lines. Bound by HBM, y read and written: 2048 rows of 28,672
// outputs (470 MB) take 95 us, 4.9 TB/s (adding to as much in place: 5.9 to 7.3); 5
// prompts of 131 to 900 rows of 6144 outputs (107 MB) 24 to 26 us by box, 4.3 TB/s. Two waves a
// SIMD are asked for (blocks of 64 rows fit in 256 registers with the rare path's
// values spilled; in more, one wave, those prompts take 38.7 us for both launches, 35.3).
template <int MT, bool VEC>
__global__ __launch_bounds__(256, MT == 4 ? 2 : 4) void adapter_rows_up_kernel(const AdapterArgs a) {
  constexpr int R = 16 * MT, NT = 2, W = 16 * NT, TPR = 256 / R;  // threads that prepare a row of t
  constexpr int NY = R / 8, LS = W + 4;  // y loads a wave and step; a row of sums in LDS
  extern __shared__ __align__(16) unsigned char smem[];  // [4 waves][R][LS] floats, then t
  __shared__ float factor[R];
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = a.tile[a.parts - 1];
  const Block k = block_of<MT>(a, blockIdx.x / tiles);
  if (k.rank == 0) return;
  int n0, n1;
  const int part = tile_part(a, blockIdx.x % tiles, &n0, &n1);
  // this lane's y: rows 8 i + lane / 8, outputs 4 (lane % 8) .. + 3 of a step
  const int yr = lane >> 3, yc = (lane & 7) * 4;
  // (loads without a condition: behind the last row or output it is the last again)
  auto load = [&](int n, f4v (&y)[NY]) {
#pragma unroll
    for (int i = 0; i < NY; i++) {
      const float *p = a.y + (int64_t)min(k.m0 + 8 * i + yr, k.m1 - 1) * a.ldy + min(n + yc, n1 - 4);
      if (VEC) y[i] = *reinterpret_cast<const f4v *>(p);
      else y[i] = f4v{p[0], p[1], p[2], p[3]};
    }
  };
  // the factor rows of outputs n + 16 j + n16, ranks 32 s + 8 c4 .. + 7; of two s
  auto load_w1 = [&](int n, int j, int s) {
    const uint16_t *p = a.b + ((int64_t)k.at * a.N + min(n + 16 * j + n16, n1 - 1)) * a.max_rank;
    return *reinterpret_cast<const half8 *>(p + min(32 * s + 8 * c4, a.max_rank - 8));
  };
  constexpr int WS = 2;
  auto load_w = [&](int n, int s0, half8 (&w)[WS][NT]) {
#pragma unroll
    for (int s = 0; s < WS; s++)
#pragma unroll
      for (int j = 0; j < NT; j++) w[s][j] = load_w1(n, j, s0 + s);
  };
  f4v y[NY], next[NY];
  half8 w[WS][NT], w_next[WS][NT];
  load_w(n0 + wave * W, 0, w);
  load(n0 + wave * W, y);
  const int steps = (k.rank + 31) >> 5, stride = steps * 128 + 16;  // bytes of a row of t
  unsigned char *ts = smem + 4 * R * LS * 4;
  {
    const int row = threadIdx.x / TPR, sub = threadIdx.x % TPR, m = k.m0 + row;
    unsigned char *to = ts + row * stride;
    const float *t = a.t + ((int64_t)min(m, k.m1 - 1) * a.parts + part) * a.max_rank;
    const int64_t share = (int64_t)a.M * a.parts * a.max_rank;
    float big = 0.0f;
    for (int p = sub; p < steps * 8; p += TPR) {  // 4 ranks each
      f4v v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (m < k.m1 && 4 * p < k.rank) {
        for (int s0 = 0; s0 < a.splits; s0 += 4) {  // (4 in flight)
          f4v u[4];
#pragma unroll
          for (int s = 0; s < 4; s++)
            u[s] = *reinterpret_cast<const f4v *>(t + min(s0 + s, a.splits - 1) * share + 4 * p);
#pragma unroll
          for (int s = 0; s < 4; s++) v = s0 + s < a.splits ? v + u[s] : v;
        }
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
    if (__builtin_expect(big == INFINITY, 0)) {  // (the whole row's threads)
      big = 0.0f;
      for (int p = sub; p < steps * 8; p += TPR) {
        const f4v v = *reinterpret_cast<const f4v *>(to + p * 16);
#pragma unroll
        for (int e = 0; e < 4; e++) big = fmaxf(big, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
      }
#pragma unroll
      for (int o = 1; o < TPR; o *= 2) big = fmaxf(big, __shfl_xor(big, o, 64));
    }
    // 2^e with big 2^e in [2^13, 2^14), of what is finite; an exponent that float32
    // holds both ways
    const int log = big > 0.0f ? ilogbf(big) : 13;
    const int e2 = min(max(13 - log, -114), 100);
    const float up = ldexpf(1.0f, e2);
    if (sub == 0)
      factor[row] = ldexpf(1.0f, -e2) * (a.scale[k.at] *
                                         (a.row_scale && m < k.m1 ? a.row_scale[m] : 1.0f));
    for (int p = sub; p < steps * 8; p += TPR) {
      const f4v v = *reinterpret_cast<const f4v *>(to + p * 16) * up;
      half8 h;  // 4 hi, 4 lo
#pragma unroll
      for (int e = 0; e < 4; e++) {
        h[e] = (_Float16)v[e];
        // (at most 4; a finite number too behind what is not finite)
        h[4 + e] = (_Float16)__builtin_amdgcn_fmed3f(v[e] - (float)h[e], -4.0f, 4.0f);
      }
      *reinterpret_cast<half8 *>(to + p * 16) = h;
    }
  }
  __syncthreads();
  float *sums = reinterpret_cast<float *>(smem) + wave * R * LS;
  u4v last;  // of this lane's 8 ranks in the last step, those that there are
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int bits = min(max((k.rank - 32 * (steps - 1) - 8 * c4 - 2 * i) * 16, 0), 32);
    last[i] = (uint32_t)((1ull << bits) - 1);
  }
  const bool all = k.m1 - k.m0 == R;
  auto take_next = [&]() {
#pragma unroll
    for (int s = 0; s < WS; s++)
#pragma unroll
      for (int j = 0; j < NT; j++) w[s][j] = w_next[s][j];
  };
  auto clear = [&](f4v (&acc)[MT][NT]) {
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int i = 0; i < MT; i++) acc[i][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  };
  auto cut = [&](half8 (&w)[NT]) {  // (behind the rank: not 0 times what is there)
#pragma unroll
    for (int j = 0; j < NT; j++) w[j] = __builtin_bit_cast(half8, __builtin_bit_cast(u4v, w[j]) & last);
  };
  auto load_t = [&](int i, int s, half8 (&t)[2]) {  // hi and lo
    const unsigned char *tp = ts + (16 * i + n16) * stride + s * 128 + c4 * 32;
    const half8 p0 = *reinterpret_cast<const half8 *>(tp);
    const half8 p1 = *reinterpret_cast<const half8 *>(tp + 16);
    t[0] = __builtin_shufflevector(p0, p1, 0, 1, 2, 3, 8, 9, 10, 11);
    t[1] = __builtin_shufflevector(p0, p1, 4, 5, 6, 7, 12, 13, 14, 15);
  };
  // f B t of outputs n .. to y
  auto add = [&](int n, f4v (&acc)[MT][NT], f4v (&y)[NY]) {
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++)
        *reinterpret_cast<f4v *>(sums + (16 * i + n16) * LS + 16 * j + 4 * c4) = acc[i][j];
    __builtin_amdgcn_wave_barrier();  // (the wave's own: in order in LDS)
#pragma unroll
    for (int i = 0; i < NY; i++) {
      const f4v v = *reinterpret_cast<const f4v *>(sums + (8 * i + yr) * LS + yc);
      const float f = factor[8 * i + yr];
#pragma unroll
      for (int e = 0; e < 4; e++) y[i][e] = __builtin_fmaf(f, v[e], y[i][e]);
    }
    auto store = [&](int i) {
      float *p = a.y + (int64_t)(k.m0 + 8 * i + yr) * a.ldy + n + yc;
      if (VEC) {
        *reinterpret_cast<f4v *>(p) = y[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = y[i][e];
      }
    };
    if (all && n + W <= n1) {
#pragma unroll
      for (int i = 0; i < NY; i++) store(i);
    } else {
#pragma unroll
      for (int i = 0; i < NY; i++)
        if (k.m0 + 8 * i + yr < k.m1 && n + yc < n1) store(i);
    }
    __builtin_amdgcn_wave_barrier();
  };
  // The products of outputs n .. again, where a factor among them is not finite:
  // times lo, of any sign or 0, that would be another value than times hi, so there
  // it is left out.
  auto multiply_odd = [&](int n, f4v (&acc)[MT][NT]) {
    clear(acc);
    half8 u[NT];
#pragma unroll 1
    for (int s = 0; s < steps; s++) {
#pragma unroll
      for (int j = 0; j < NT; j++) u[j] = load_w1(n, j, s);
      if (s == steps - 1) cut(u);
#pragma unroll
      for (int part = 0; part < 2; part++) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
          half8 t[2];
          load_t(i, s, t);
#pragma unroll
          for (int j = 0; j < NT; j++)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u[j], t[part], acc[i][j], 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int e = 0; e < 8; e++)
            u[j][e] = __builtin_fabsf16(u[j][e]) < (_Float16)INFINITY ? u[j][e] : (_Float16)0.0f;
      }
    }
  };
  // (LONG: more ranks than two steps hold, loaded two steps ahead)
  auto stream = [&](auto long_ranks) {
    constexpr bool LONG = decltype(long_ranks)::value;
    for (int n = n0 + wave * W; n < n1; n += 4 * W) {
      if constexpr (!LONG) load_w(n + 4 * W, 0, w_next);
      load(n + 4 * W, next);
      __builtin_amdgcn_sched_barrier(0);
      f4v acc[MT][NT];
      clear(acc);
      // 0 times the factors: NaN where one is not finite. (Ranks of 128, 8 prompts of 33
      // rows to 28,672 outputs: 39.3 us by products with a tile of zeros, 39.8 by
      // v_dot2, 39.1 without; ranks up to 64, 5 prompts: 36.4, 34.3, 34.4.)
      f4v zero = {0.0f, 0.0f, 0.0f, 0.0f};
      auto multiply = [&](int s, half8 (&w)[NT]) {
        if (s == steps - 1) cut(w);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          if constexpr (LONG) {
            zero = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], half8{}, zero, 0, 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) zero[0] = dot2(__builtin_bit_cast(u4v, w[j])[e], 0u, zero[0]);
          }
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
          half8 t[2];
          load_t(i, s, t);
#pragma unroll
          for (int j = 0; j < NT; j++) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], t[0], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], t[1], acc[i][j], 0, 0, 0);
          }
        }
      };
      if constexpr (LONG) {
        for (int s = 0; s < steps; s += WS) {
          const bool more = s + WS < steps;
          load_w(more ? n : n + 4 * W, more ? s + WS : 0, w_next);
          __builtin_amdgcn_sched_barrier(0);
          multiply(s, w[0]);
          if (s + 1 < steps) multiply(s + 1, w[1]);
          take_next();
        }
      } else {
        multiply(0, w[0]);
        if (steps > 1) multiply(1, w[1]);
      }
      float odd = zero[0];
      if constexpr (LONG) odd = zero[0] + zero[1] + zero[2] + zero[3];
      if (__builtin_expect(__any(odd != odd), 0)) multiply_odd(n, acc);
      add(n, acc, y);
#pragma unroll
      for (int i = 0; i < NY; i++) y[i] = next[i];
      if constexpr (!LONG) take_next();
    }
  };
  if (steps > WS) stream(std::true_type{});
  else stream(std::false_type{});
}

// Rows a block takes (16 times these), and workgroups that share a block's inputs:
// up to two a compute unit (5 prompts of 2272 rows, 4096 inputs, ranks up to 64: A x
// 13.8 us in 2 shares, 16.7 in one), but each is a share of t that every workgroup of
// the second launch adds up (8 prompts of 33 rows to 6144 outputs, both launches: ranks
// of 128 28.7 us in 2 shares, 42.9 in 16; of 64 20.1 in 4, 28.3 in 16; of 16 14.2 in 8,
// 15.0 in 16). Blocks of 64 rows, one workgroup a compute unit, read the first factor
// half as often, where that has several times 64 rows, of which some slots may use few
// (both launches, blocks of 64 and of 32, three parts of 6144 outputs: 16 prompts of 34
// rows, ranks of 128 32, 42; 8 of 64, of 256 41, 49; 8 of 128, of 128 35.5, 42; 4000
// rows, of 128 86, 92, of 64 61, 66, of 32 57, 53; 5 of up to 900, of 11 to 64 36.1,
// 35.3). And they write y from 32 rows a sequence on (8 of 33 rows to 28,672 outputs,
// ranks of 128: 39.3 us, in blocks of 16 56.9; of 16 23.2, 22.8).
struct RowsPlan {
  int down, up, splits;
  int64_t down_blocks, up_blocks;
};
int64_t down_tiles(const wg_adapters *ad) {  // of 64 rows of the first factor
  return (ad->parts * ((ad->max_rank + 15) / 16) + 3) / 4;
}
int most_splits(const wg_adapters *ad) {
  int n = 8;
  while (n > 1 && (n * 2 * KB > ad->K || n * ad->max_rank > 256)) n /= 2;
  return n;
}
RowsPlan rows_plan(const wg_adapters *ad, int64_t M, int64_t segments) {
  RowsPlan p;
  const int64_t tiles = down_tiles(ad);
  p.down = M > 32 * segments && tiles >= 4 ? 4 : M >= 16 * segments ? 2 : 1;
  p.up = M >= 32 * segments ? 4 : 1;
  p.down_blocks = (M - 1) / (16 * p.down) + segments;
  p.up_blocks = (M - 1) / (16 * p.up) + segments;
  const int64_t busy = (M + 16 * p.down - 1) / (16 * p.down) * tiles;
  p.splits = most_splits(ad);
  while (p.splits > 1 && p.splits * busy > (p.down == 4 ? 250 : 500)) p.splits /= 2;
  return p;
}

void launch_token_up(int p, dim3 grid, hipStream_t s, const AdapterArgs &a) {
  auto up = p == 1    ? adapter_token_up_kernel<1, false>
            : p == 2  ? adapter_token_up_kernel<2, false>
            : p == 4  ? adapter_token_up_kernel<4, false>
            : p == 8  ? adapter_token_up_kernel<8, false>
            : p == 16 ? adapter_token_up_kernel<16, false>
                      : adapter_token_up_kernel<32, false>;
  up<<<grid, 256, 0, s>>>(a);
}

int check_adapters(const wg_adapters *ad, const char *who) {
  WG_REQUIRE(ad && ad->a && ad->b && ad->rank && ad->scale, "%s: null argument", who);
  WG_REQUIRE(ad->slots >= 1, "%s: %d adapters", who, ad->slots);
  WG_REQUIRE(ad->max_rank >= 8 && ad->max_rank <= MAX_RANK && ad->max_rank % 8 == 0,
             "%s: ranks up to %d (a multiple of 8 up to %d)", who, ad->max_rank, MAX_RANK);
  WG_REQUIRE(ad->K >= 8 && ad->K % 8 == 0 && ad->K <= 1 << 30 && ad->N <= 1 << 30,
             "%s: K %d (a multiple of 8), N %d (both up to 2^30)", who, ad->K, ad->N);
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
  if (!ad || M < 1 || ad->parts < 1 || ad->parts > PARTS || ad->max_rank < 1 ||
      ad->max_rank > MAX_RANK || ad->K < 1)
    return 0;
  // enough for fewer rows too, and any number of sequences: where there are several
  // shares, they times the blocks' tiles are up to 500 (of 64 rows 250)
  const int64_t shared = 16000 / down_tiles(ad), all = (int64_t)M * most_splits(ad);
  const int64_t rows = all < shared ? all : shared;
  return (size_t)(rows > M ? rows : M) * ad->parts * ad->max_rank * 4;
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
                   segments, 1, 256, {}, {}};
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
    const int p = ad->max_rank <= 8 ? 1 : 1 << (32 - __builtin_clz(ad->max_rank / 8 - 1));
    const unsigned n = tiles(256 * (p >= 8 ? 1 : 8 / p));
    // One launch where few workgroups make t again (us in a graph, one launch and two,
    // of 1 to 32 tokens: ranks of 8, 4096 inputs, 6144 outputs 3.9 to 4.0, 5.4 to 5.5;
    // of 16, 4.4 to 4.8 up to 16 tokens, 5.2 to 5.4, for 32 7.0, 5.7; 2048 inputs, 16,384
    // outputs 4.4 to 4.6 up to 8, 5.2 to 5.3, for 32 11.1, 6.1), and 4 us less of the
    // host's.
    const int64_t groups = (int64_t)M * n;
    if (ad->max_rank <= ONE_RANK && groups <= 256 && groups * ad->max_rank * ad->K <= 6500000) {
      auto both = p == 1 ? adapter_token_up_kernel<1, true> : adapter_token_up_kernel<2, true>;
      both<<<dim3(n, M), 256, 0, s>>>(a);
    } else {
      if ((int64_t)M * ad->parts * ad->max_rank <= 2048)
        adapter_token_down_kernel<1><<<dim3(M, (ad->max_rank + 3) / 4, ad->parts), 256, 0, s>>>(a);
      else
        adapter_token_down_kernel<2><<<dim3(M, (ad->max_rank + 7) / 8, ad->parts), 256, 0, s>>>(a);
      launch_token_up(p, dim3(n, M), s, a);
    }
    return launched("wg_adapter_add");
  }
  const RowsPlan p = rows_plan(ad, M, segments);
  WG_REQUIRE(p.down_blocks * p.splits <= MAX_GROUPS - 7 && p.up_blocks <= MAX_GROUPS,
             "wg_adapter_add: %d rows of %d sequences", M, segments);
  a.splits = p.splits;
  const dim3 down(((unsigned)p.down_blocks * p.splits + 7) / 8 * 8,  // (a block's tiles: on one XCD)
                  (ad->parts * ((ad->max_rank + 15) / 16) + 3) / 4);
  const int64_t wide = (p.up_blocks * ad->N / 512 + 127) / 128 * 128;
  const unsigned n = tiles(wide < 128 ? 128 : wide > ad->N ? (ad->N + 127) / 128 * 128 : (int)wide);
  WG_REQUIRE(p.up_blocks * n <= MAX_GROUPS, "wg_adapter_add: %d rows of %d outputs", M, ad->N);
  const int lds = 16 * p.up * (4 * 36 * 4 + (ad->max_rank + 31) / 32 * 128 + 16);
  const bool vec = ((uintptr_t)y & 15) == 0 && ldy % 4 == 0;
  auto up = p.up == 4 ? (vec ? adapter_rows_up_kernel<4, true> : adapter_rows_up_kernel<4, false>)
                      : (vec ? adapter_rows_up_kernel<1, true> : adapter_rows_up_kernel<1, false>);
  if (lds > 63 * 1024) {
    const int rl = raise_lds((const void *)up, lds);
    if (rl) return rl;
  }
  const int down_lds = p.down == 4 ? DOWN_LDS<4> : p.down == 2 ? DOWN_LDS<2> : DOWN_LDS<1>;
  auto down_kernel = p.down == 4 ? adapter_rows_down_kernel<4> : p.down == 2 ? adapter_rows_down_kernel<2> : adapter_rows_down_kernel<1>;
  if (down_lds > 64 * 1024) {
    const int rl = raise_lds((const void *)down_kernel, down_lds);
    if (rl) return rl;
  }
  down_kernel<<<down, 256, down_lds, s>>>(a);
  up<<<(unsigned)p.up_blocks * n, 256, lds, s>>>(a);
  return launched("wg_adapter_add");
}

}  // extern "C"
