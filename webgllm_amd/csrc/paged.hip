// The paged cache (wg_paged_cache): head preparation of many sequences' rows
// into its pages, and eviction by accumulated attention weight.
#include "attn_core.h"
#include "common.h"
#include "dot.h"
#include "paged_dev.h"

namespace wg {

int check_paged(const wg_paged_cache *c, int64_t kvd, bool lens, const char *who) {
  WG_REQUIRE(c && c->k && c->v && c->table && (!lens || c->lens), "%s: null cache argument", who);
  WG_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "%s: pages must be 16-byte aligned",
             who);
  WG_REQUIRE(c->page_size >= 1 && (c->page_size & (c->page_size - 1)) == 0,
             "%s: pages of %d entries (a power of two)", who, c->page_size);
  WG_REQUIRE(c->pages >= 1 && (int64_t)c->pages * c->page_size <= 0x7fffffff,
             "%s: %d pages of %d entries (fewer than 2^31 entries)", who, c->pages, c->page_size);
  WG_REQUIRE(c->sequences >= 1 && c->sequences <= 65535, "%s: %d sequences", who, c->sequences);
  WG_REQUIRE(c->ld_table >= 1 && c->max_entries >= 1 && c->max_entries <= 1 << 30 &&
                 c->max_entries <= (int64_t)c->ld_table * c->page_size,
             "%s: %d entries a sequence over %d pages of %d", who, c->max_entries, c->ld_table,
             c->page_size);
  const size_t bytes = (size_t)c->pages * c->page_size * kvd * 2;
  WG_REQUIRE(!overlaps(c->k, bytes, c->v, bytes), "%s: key and value pages overlap", who);
  return WG_OK;
}

Paged as_paged(const wg_paged_cache *c) {
  return {c->k, c->v, c->table, c->lens, c->pages, __builtin_ctz((unsigned)c->page_size),
          c->ld_table, c->sequences, c->max_entries};
}

namespace {

constexpr int MAX_HD = 256;

__device__ inline uint16_t to_h(float v) {
  v = fminf(fmaxf(v, -65504.0f), 65504.0f);
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}

struct PrepArgs {
  const float *qkv, *q_norm, *k_norm, *rope;
  const int32_t *pos, *row_start;
  float *q_out;
  int ldq, ldqo, M, H, KV, hd, use_norm, rot, rope_rows;
  float eps;
  RopeAxes axes;  // (where the kernel is one of several axes)
  int ld_pos;
};

// The pool row (-1: none) and position (of the first axis) of row m; false where
// the row is no sequence's (it is then left as it was).
template <bool AXES>
__device__ inline bool row_place(const Paged &c, const PrepArgs &a, int m, int *row, int *pos) {
  int b = m, i;
  if (a.row_start) {
    int r0, r1, n;
    b = find_last(c, a.row_start, m, [](int first, int) { return first; }, &r0, &r1, &n);
    if (b < 0 || m >= r1) return false;
    i = n - (r1 - m);
  } else {
    i = paged_len(c, b) - 1;
  }
  *row = i >= 0 ? paged_row(c, c.table + (int64_t)b * c.ld_table, i) : -1;
  if constexpr (AXES) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (e >= a.axes.axes) break;
      const int p = a.pos[(int64_t)m * a.ld_pos + e];
      if (e == 0) *pos = p;
      if (p < 0 || 1024 + (p >> 10) >= a.rope_rows) *row = -1;
    }
    return true;
  }
  *pos = a.pos ? a.pos[m] : i;
  if (*pos < 0 || 1024 + (*pos >> 10) >= a.rope_rows) *row = -1;
  return true;
}
// Row m's cos and sin of frequency f under several axes.
__device__ inline void axes_angle(const PrepArgs &a, int m, int f, float *cs, float *sn) {
  int p = a.pos[(int64_t)m * a.ld_pos + rope_axis(a.axes, f)];
  if (p < 0 || 1024 + (p >> 10) >= a.rope_rows) p = 0;  // (a row that is not stored)
  const float *lo = a.rope + (int64_t)(p & 1023) * a.hd + f;
  const float *hi = a.rope + (int64_t)(1024 + (p >> 10)) * a.hd + f;
  rope_angle(lo[0], lo[a.hd / 2], hi[0], hi[a.hd / 2], cs, sn);
}

// A wave a head of any size and rotation: wg_head_prep's arithmetic
// (head_norm_inv, rope_rotate in their fixed order), so its bits.
template <bool AXES>
__global__ __launch_bounds__(64) void paged_prep_kernel(const Paged c, const PrepArgs a) {
  const int slot = blockIdx.y, m = blockIdx.x, lane = threadIdx.x;
  const int hd = a.hd, P = a.rot / 2, kvd = a.KV * hd;
  const float *x = a.qkv + (int64_t)m * a.ldq + (int64_t)slot * hd;
  const bool is_q = slot < a.H, is_v = slot >= a.H + a.KV;
  const float *nw = is_q ? a.q_norm : a.k_norm;
  float xv[4], wv[4], xp[4], wp[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int t = lane + 64 * i;
    xv[i] = xp[i] = 0.0f;
    wv[i] = wp[i] = 1.0f;
    if (t < hd) {
      xv[i] = x[t];
      if (!is_v && a.use_norm) wv[i] = nw[t];
      if (!is_v && t < 2 * P) {
        const int tp = t < P ? t + P : t - P;  // the rotation partner
        xp[i] = x[tp];
        if (a.use_norm) wp[i] = nw[tp];
      }
    }
  }
  int row, pos;
  if (!row_place<AXES>(c, a, m, &row, &pos)) return;
  if (row < 0) {
    if (is_q)
      for (int t = lane; t < hd; t += 64) a.q_out[(int64_t)m * a.ldqo + (int64_t)slot * hd + t] = 0.0f;
    return;
  }
  if (is_v) {
    uint16_t *vo = c.v + (int64_t)row * kvd + (int64_t)(slot - a.H - a.KV) * hd;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (lane + 64 * i < hd) vo[lane + 64 * i] = to_h(xv[i]);
    return;
  }
  float inv = 1.0f;
  if (a.use_norm) {
    // lane q < 4 walks dims 32 t + 8 q + e (held by lane (32 t + 8 q + e) % 64, element t / 2)
    const int q = lane & 3;
    float part = 0.0f;
    for (int t = 0; 32 * t < hd; t++) {
      float xs = xv[0];
#pragma unroll
      for (int i = 1; i < 4; i++)
        if (i == (t >> 1)) xs = xv[i];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float y = __shfl(xs, (32 * t + 8 * q + e) & 63, 64);
        part = __builtin_fmaf(y, y, part);
      }
    }
    const float total = (__shfl(part, 0, 64) + __shfl(part, 1, 64)) +
                        (__shfl(part, 2, 64) + __shfl(part, 3, 64));
    inv = head_norm_inv(total, hd, a.eps);
  }
  const float *r_lo = a.rope + (int64_t)(pos & 1023) * hd;
  const float *r_hi = a.rope + (int64_t)(1024 + (pos >> 10)) * hd;
  const float scale = is_q ? 1.0f / sqrtf((float)hd) : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int t = lane + 64 * i;
    if (t >= hd) break;
    const float v = xv[i] * (a.use_norm ? inv * wv[i] : 1.0f);
    float r = v;
    if (t < 2 * P) {
      const bool first = t < P;
      const int f = first ? t : t - P;
      const float p = xp[i] * (a.use_norm ? inv * wp[i] : 1.0f);
      if constexpr (AXES) {
        float cs, sn;
        axes_angle(a, m, f, &cs, &sn);
        r = rope_turn(v, p, first, cs, sn);
      } else {
        r = rope_rotate(v, p, first, r_lo[f], r_lo[hd / 2 + f], r_hi[f], r_hi[hd / 2 + f]);
      }
    }
    if (is_q) a.q_out[(int64_t)m * a.ldqo + (int64_t)slot * hd + t] = r * scale;
    else c.k[(int64_t)row * kvd + (int64_t)(slot - a.H) * hd + t] = to_h(r);
  }
}

// The same bits with 16 dims a thread in 16-byte pieces (8 and their rotation
// partners), a workgroup a row: heads of 64 and 128, all rotated, everything
// aligned. The row's loads wait for nothing; only the rope table and the stores
// wait for its place. Bound by HBM: 3997 rows of 48 heads of 64 with norms (86 MB
// moved) take 18.4 us, 4.7 TB/s, by the kernel above 76; 64 rows 4.2 us, latency.
// Under several axes a frequency's table rows are its own, so the row's cosines
// and sines are made once, a thread each, and lie in LDS for all heads.
template <int HD, bool AXES>
__global__ __launch_bounds__(1024) void paged_prep_rows_kernel(const Paged c, const PrepArgs a) {
  constexpr int TPH = HD / 16;  // threads a head (4 or 8)
  const int m = blockIdx.x, slots = a.H + 2 * a.KV, kvd = a.KV * HD;
  int row = -1, pos = 0;
  bool ours = false, placed = false;
  __shared__ float turn[AXES ? 2 : 1][AXES ? HD / 2 : 1];  // cos, sin
  // (whole waves together: a head's lanes exchange, and the search takes them all)
  for (int t = threadIdx.x; t - (int)(threadIdx.x & 63) < slots * TPH; t += blockDim.x) {
    const int ch = t % TPH, slot = min(t / TPH, slots - 1);
    const bool in = t < slots * TPH, is_q = slot < a.H, is_v = slot >= a.H + a.KV;
    // [0]: dims 8 ch .., [1]: their partners
    float x[2][8], w[2][8];
    const float *from = a.qkv + (int64_t)m * a.ldq + (int64_t)slot * HD + 8 * ch;
    const float *nw = (is_q ? a.q_norm : a.k_norm) + 8 * ch;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float4 v = *reinterpret_cast<const float4 *>(from + p * (HD / 2) + 4 * u);
        float4 n = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (a.use_norm && !is_v) n = *reinterpret_cast<const float4 *>(nw + p * (HD / 2) + 4 * u);
        x[p][4 * u] = v.x, x[p][4 * u + 1] = v.y, x[p][4 * u + 2] = v.z, x[p][4 * u + 3] = v.w;
        w[p][4 * u] = n.x, w[p][4 * u + 1] = n.y, w[p][4 * u + 2] = n.z, w[p][4 * u + 3] = n.w;
      }
    if (!placed) {
      if constexpr (AXES)  // (before the row's place, so that neither waits for the other)
        for (int f = threadIdx.x; f < HD / 2; f += blockDim.x) axes_angle(a, m, f, &turn[0][f], &turn[1][f]);
      ours = row_place<AXES>(c, a, m, &row, &pos);
      placed = true;
      if constexpr (AXES) __syncthreads();  // (every wave comes by here once)
    }
    if (!ours) return;
    float inv = 1.0f;
    if (a.use_norm) {  // the sum of squares in head_norm_inv's order
      const int lane = threadIdx.x & 63, head0 = lane - ch;
      float part = 0.0f;
      if constexpr (HD == 64) {
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
          for (int e = 0; e < 8; e++) part = __builtin_fmaf(x[p][e], x[p][e], part);
      } else {
        // t = 0, 2 on threads ch < 4, t = 1, 3 on threads ch + 4
#pragma unroll
        for (int q = 0; q < 4; q++) {
          if (q) part = __shfl(part, head0 + (ch ^ 4), 64);
#pragma unroll
          for (int e = 0; e < 8; e++) part = __builtin_fmaf(x[q >> 1][e], x[q >> 1][e], part);
        }
      }
      constexpr int END = HD == 64 ? 0 : 4;  // the chains that began at t = 0 ended there
      const float total = (__shfl(part, head0 + END, 64) + __shfl(part, head0 + END + 1, 64)) +
                          (__shfl(part, head0 + END + 2, 64) + __shfl(part, head0 + END + 3, 64));
      inv = head_norm_inv(total, HD, a.eps);
    }
    if (!in || (row < 0 && !is_q)) continue;
    float r[2][8];
    if (row < 0) {
#pragma unroll
      for (int e = 0; e < 8; e++) r[0][e] = r[1][e] = 0.0f;
    } else if (is_v) {
#pragma unroll
      for (int e = 0; e < 8; e++) r[0][e] = x[0][e], r[1][e] = x[1][e];
    } else if constexpr (AXES) {
      const float scale = is_q ? 1.0f / sqrtf((float)HD) : 1.0f;
#pragma unroll
      for (int d = 0; d < 8; d++) {
        const float cs = turn[0][8 * ch + d], sn = turn[1][8 * ch + d];
        const float y0 = x[0][d] * (a.use_norm ? inv * w[0][d] : 1.0f);
        const float y1 = x[1][d] * (a.use_norm ? inv * w[1][d] : 1.0f);
        r[0][d] = rope_turn(y0, y1, true, cs, sn);
        r[1][d] = rope_turn(y1, y0, false, cs, sn);
        if (is_q) {
          r[0][d] *= scale;
          r[1][d] *= scale;
        }
      }
    } else {
      const float *r_lo = a.rope + (int64_t)(pos & 1023) * HD + 8 * ch;
      const float *r_hi = a.rope + (int64_t)(1024 + (pos >> 10)) * HD + 8 * ch;
      const float scale = is_q ? 1.0f / sqrtf((float)HD) : 1.0f;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float4 c1 = *reinterpret_cast<const float4 *>(r_lo + 4 * u);
        const float4 s1 = *reinterpret_cast<const float4 *>(r_lo + HD / 2 + 4 * u);
        const float4 c2 = *reinterpret_cast<const float4 *>(r_hi + 4 * u);
        const float4 s2 = *reinterpret_cast<const float4 *>(r_hi + HD / 2 + 4 * u);
        const float fc1[4] = {c1.x, c1.y, c1.z, c1.w}, fs1[4] = {s1.x, s1.y, s1.z, s1.w};
        const float fc2[4] = {c2.x, c2.y, c2.z, c2.w}, fs2[4] = {s2.x, s2.y, s2.z, s2.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int d = 4 * u + e;
          const float y0 = x[0][d] * (a.use_norm ? inv * w[0][d] : 1.0f);
          const float y1 = x[1][d] * (a.use_norm ? inv * w[1][d] : 1.0f);
          r[0][d] = rope_rotate(y0, y1, true, fc1[e], fs1[e], fc2[e], fs2[e]);
          r[1][d] = rope_rotate(y1, y0, false, fc1[e], fs1[e], fc2[e], fs2[e]);
          if (is_q) {
            r[0][d] *= scale;
            r[1][d] *= scale;
          }
        }
      }
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
      if (is_q) {
        float *o = a.q_out + (int64_t)m * a.ldqo + (int64_t)slot * HD + 8 * ch + p * (HD / 2);
        *reinterpret_cast<float4 *>(o) = make_float4(r[p][0], r[p][1], r[p][2], r[p][3]);
        *reinterpret_cast<float4 *>(o + 4) = make_float4(r[p][4], r[p][5], r[p][6], r[p][7]);
      } else {
        uint16_t *o = (is_v ? c.v : c.k) + (int64_t)row * kvd +
                      (int64_t)(slot - a.H - (is_v ? a.KV : 0)) * HD + 8 * ch + p * (HD / 2);
        *reinterpret_cast<uint4 *>(o) =
            make_uint4(to_h(r[p][0]) | (uint32_t)to_h(r[p][1]) << 16,
                       to_h(r[p][2]) | (uint32_t)to_h(r[p][3]) << 16,
                       to_h(r[p][4]) | (uint32_t)to_h(r[p][5]) << 16,
                       to_h(r[p][6]) | (uint32_t)to_h(r[p][7]) << 16);
      }
    }
  }
}

// ------------------------------------------------------------------ eviction

// A weight as a number that sorts like it: larger weights larger, -0 as 0,
// NaN as -infinity.
__device__ inline uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
  const float *weights;
  int32_t *to_lens, *kept;
  float *to_weights;
  int ldw, ld_kept, ld_tow, keep, sinks, recent;
};

constexpr int SEL = 1024;  // threads that select
constexpr int KEYS1 = 16;  // entries a thread holds where one workgroup selects
constexpr int KEYS2 = 8;   // the same of a chunk
constexpr int CHUNK_ENTRIES = SEL * KEYS2;

// What stays is found by the kept weights' least: its sorting key digit by digit
// (11, 11 and 10 bits), counts of the digits in LDS. The entries are held in
// registers, a wave 64 K neighbouring ones, so that ranks in order are counts of
// ballots. The choice is bound by the chain of counts and scans: 577 entries 6.8
// us, 16 sequences of up to 6000 9.9. The copies are bound by HBM (107 MB moved
// for those 16: 25 us, 4.3 TB/s).
constexpr int DIGITS = 2048;
__device__ inline int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ inline uint32_t digit_of(uint32_t key, int pass) {
  return pass == 2 ? key & 1023 : (key >> digit_shift(pass)) & 2047;
}

// The sum of sums[0 .. wave - 1] (SEL / 64 of them, in LDS), on every lane.
__device__ inline uint32_t waves_before(const uint32_t *sums, int wave) {
  const int lane = threadIdx.x & 63;
  const uint32_t run = wave_scan(lane < SEL / 64 ? sums[lane] : 0);
  return wave ? __builtin_amdgcn_readlane(run, wave - 1) : 0;
}

// Inclusive sums over the workgroup's threads; sums[SEL / 64] in LDS.
__device__ inline uint32_t block_scan(uint32_t v, uint32_t *sums) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  v = wave_scan(v);
  __syncthreads();  // (sums is free)
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  return v + waves_before(sums, wave);
}

// The digit in which the need-th largest lies (need >= 1, of at least as many),
// h[0] and h[1] the counts of digits 2047 - 2 t and 2046 - 2 t on thread t, and
// how many lie above it.
__device__ inline void find_digit(const uint32_t (&h)[2], uint32_t need, uint32_t *sums,
                                  uint32_t *found, uint32_t *digit, uint32_t *above) {
  const uint32_t run = block_scan(h[0] + h[1], sums), over = run - h[0] - h[1];
  if (over < need && run >= need) {
    const bool second = over + h[0] < need;
    found[0] = DIGITS - 1 - 2 * threadIdx.x - (second ? 1 : 0);
    found[1] = over + (second ? h[0] : 0);
  }
  __syncthreads();
  *digit = found[0];
  *above = found[1];
}

// The ranks of this thread's K entries (wave w holds from + 64 K w .., entry
// from + 64 (K w + k) + lane) behind `before` kept ones and `equal` equal ones:
// always kept ones, those of a larger key, and the first `need` of an equal one.
template <int K>
__device__ inline void keep_in_order(const EvictArgs &a, int b, int from, int count, int hi,
                                     bool any, uint32_t least, uint32_t need, uint32_t before,
                                     uint32_t equal, const float (&x)[K],
                                     const uint32_t (&key)[K], int per, uint32_t *sums) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int32_t *kept = a.kept + (int64_t)b * a.ld_kept;
  float *tow = a.to_weights ? a.to_weights + (int64_t)b * a.ld_tow : nullptr;
  uint64_t gb[K], eb[K];
  uint32_t gt = 0, eq = 0;
#pragma unroll
  for (int k = 0; k < K; k++) {
    gb[k] = eb[k] = 0;
    if (k >= per) continue;  // (uniform)
    const int i = from + (wave * per + k) * 64 + lane;
    const bool in = i < count, must = in && (i < a.sinks || i >= hi);
    gb[k] = __ballot(must || (in && any && key[k] > least));
    eb[k] = __ballot(in && !must && any && key[k] == least);
    gt += __popcll(gb[k]);
    eq += __popcll(eb[k]);
  }
  // the waves before this one
  __syncthreads();
  if (lane == 0) {
    sums[wave] = gt;
    sums[SEL / 64 + wave] = eq;
  }
  __syncthreads();
  before += waves_before(sums, wave);
  equal += waves_before(sums + SEL / 64, wave);
  const uint64_t mine = 1ull << lane, below = mine - 1;
#pragma unroll
  for (int k = 0; k < K; k++) {
    if (k >= per) continue;
    const uint32_t e = equal + __popcll(eb[k] & below);
    if ((gb[k] & mine) || ((eb[k] & mine) && e < need)) {
      const int64_t to = before + __popcll(gb[k] & below) + min(e, need);
      kept[to] = from + (wave * per + k) * 64 + lane;
      if (tow) tow[to] = x[k];
    }
    before += __popcll(gb[k]);
    equal += __popcll(eb[k]);
  }
}

// The rest of a sequence's kept row; its new length.
__device__ inline void finish_kept(const EvictArgs &a, int b, int n) {
  const int m = min(n, a.keep);
  for (int i = m + threadIdx.x; i < a.keep; i += SEL) {
    a.kept[(int64_t)b * a.ld_kept + i] = -1;
    if (a.to_weights) a.to_weights[(int64_t)b * a.ld_tow + i] = 0.0f;
  }
  if (threadIdx.x == 0) a.to_lens[b] = m;
}

// One workgroup a sequence, for up to SEL * KEYS1 entries.
__global__ __launch_bounds__(SEL) void evict_select_kernel(const Paged c, const EvictArgs a) {
  __shared__ uint32_t hist[DIGITS], sums[2 * SEL / 64], found[2];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = paged_len(c, b), hi = n - a.recent;  // the middle is [sinks, hi)
  const float *w = a.weights + (int64_t)b * a.ldw;
  const int per = (n + SEL - 1) / SEL;  // entries a thread holds
  float x[KEYS1];
  uint32_t key[KEYS1];
#pragma unroll
  for (int k = 0; k < KEYS1; k++) {
    const int i = (wave * per + k) * 64 + lane;
    x[k] = k < per && i < n ? w[i] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < KEYS1; k++)
    if (k < per) key[k] = weight_key(x[k]);
  __syncthreads();  // (to_lens may be lens)
  finish_kept(a, b, n);
  uint32_t need = n > a.keep ? a.keep - a.sinks - a.recent : 0, least = 0;
  const bool any = need > 0;
  if (any) {
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
      hist[tid] = hist[tid + SEL] = 0;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < KEYS1; k++) {
        if (k >= per) continue;  // (uniform)
        const int i = (wave * per + k) * 64 + lane;
        if (i >= a.sinks && i < hi && (pass == 0 || key[k] >> digit_shift(pass - 1) == least))
          atomicAdd(&hist[digit_of(key[k], pass)], 1u);
      }
      __syncthreads();
      const uint32_t h[2] = {hist[DIGITS - 1 - 2 * tid], hist[DIGITS - 2 - 2 * tid]};
      uint32_t digit, above;
      find_digit(h, need, sums, found, &digit, &above);
      least = least << (pass == 2 ? 10 : 11) | digit;
      need -= above;
    }
  }
  // (all of a shorter sequence: its middle is empty)
  keep_in_order<KEYS1>(a, b, 0, n, n > a.keep ? hi : 0, any, least, need, 0, 0, x, key, per, sums);
}

// Longer sequences in chunks of CHUNK_ENTRIES, a workgroup each and a launch a
// digit: pass p counts its chunk's digits into counts[b][chunk][p] and adds up
// those that all chunks of the sequence counted in pass p - 1, which gives the
// digit; the last launch has the whole key, the kept ones of the chunks before
// its own, and writes.
struct EvictScratch {
  uint32_t *counts;  // [sequences][chunks][3][DIGITS]
  uint32_t *above;   // [sequences][chunks][2]: entries of a larger digit, passes 0 and 1
  uint32_t *state;   // [sequences][2][2]: the key so far, what is still needed of it
  int32_t *lens;     // [sequences]: the lengths as the first launch read them
  int chunks;
};
template <int PASS>
__global__ __launch_bounds__(SEL) void evict_chunk_kernel(const Paged c, const EvictArgs a,
                                                          const EvictScratch sc) {
  __shared__ uint32_t hist[DIGITS], sums[2 * SEL / 64], found[2];
  const int b = blockIdx.y, chunk = blockIdx.x, from = chunk * CHUNK_ENTRIES;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (to_lens, which the last launch writes, may be lens)
  const int n = PASS == 0 ? paged_len(c, b) : sc.lens[b], hi = n - a.recent;
  if (PASS == 0 && chunk == 0 && tid == 0) sc.lens[b] = n;
  const bool any = n > a.keep && a.keep > a.sinks + a.recent;
  if (from >= n && chunk > 0) return;
  if (PASS < 3 && !any) return;
  const float *w = a.weights + (int64_t)b * a.ldw;
  float x[KEYS2];
  uint32_t key[KEYS2];
#pragma unroll
  for (int k = 0; k < KEYS2; k++) {
    const int i = from + (wave * KEYS2 + k) * 64 + lane;
    x[k] = i < n ? w[i] : 0.0f;
  }
  uint32_t *mine = sc.counts + ((int64_t)b * sc.chunks + chunk) * 3 * DIGITS;
  uint32_t least = 0, need = any ? a.keep - a.sinks - a.recent : 0;
  uint32_t before = 0, equal = 0;  // kept and equal ones of the chunks before this one
  if (PASS > 0 && any) {
    const int p = PASS - 1, live = (n + CHUNK_ENTRIES - 1) / CHUNK_ENTRIES;
    if (p > 0) {
      least = sc.state[(b * 2 + p - 1) * 2];
      need = sc.state[(b * 2 + p - 1) * 2 + 1];
    }
    // thread t: digits 2047 - 2 t and 2046 - 2 t of all chunks, and of those before
    uint32_t h[2] = {0, 0}, hb[2] = {0, 0}, own[2] = {0, 0};
    const uint32_t *row = sc.counts + ((int64_t)b * sc.chunks * 3 + p) * DIGITS + DIGITS - 2 - 2 * tid;
#pragma unroll 8
    for (int q = 0; q < live; q++) {
      const uint2 v = *reinterpret_cast<const uint2 *>(row + (int64_t)q * 3 * DIGITS);
      h[0] += v.y, h[1] += v.x;
      if (q < chunk) hb[0] += v.y, hb[1] += v.x;
      if (q == chunk) own[0] = v.y, own[1] = v.x;
    }
    uint32_t digit, above;
    find_digit(h, need, sums, found, &digit, &above);
    least = least << (p == 2 ? 10 : 11) | digit;
    need -= above;
    const uint32_t d0 = DIGITS - 1 - 2 * tid, d1 = d0 - 1;
    if (PASS < 3) {
      const uint32_t got = block_scan((d0 > digit ? own[0] : 0) + (d1 > digit ? own[1] : 0), sums);
      if (tid == SEL - 1) sc.above[((int64_t)b * sc.chunks + chunk) * 2 + p] = got;
      if (chunk == 0 && tid == 0) {
        sc.state[(b * 2 + p) * 2] = least;
        sc.state[(b * 2 + p) * 2 + 1] = need;
      }
    } else {
      uint32_t g = (d0 > digit ? hb[0] : 0) + (d1 > digit ? hb[1] : 0);
      for (int q = tid; q < chunk; q += SEL)
        g += sc.above[((int64_t)b * sc.chunks + q) * 2] +
             sc.above[((int64_t)b * sc.chunks + q) * 2 + 1];
      const uint32_t e = (d0 == digit ? hb[0] : 0) + (d1 == digit ? hb[1] : 0);
      const uint32_t gs = block_scan(g, sums);
      if (tid == SEL - 1) found[0] = gs;
      const uint32_t es = block_scan(e, sums);
      if (tid == SEL - 1) found[1] = es;
      __syncthreads();
      before = found[0];
      equal = found[1];
    }
  }
#pragma unroll
  for (int k = 0; k < KEYS2; k++) key[k] = weight_key(x[k]);
  if constexpr (PASS < 3) {
    hist[tid] = hist[tid + SEL] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS2; k++) {
      const int i = from + (wave * KEYS2 + k) * 64 + lane;
      if (i >= a.sinks && i < hi && (PASS == 0 || key[k] >> digit_shift(PASS - 1) == least))
        atomicAdd(&hist[digit_of(key[k], PASS)], 1u);
    }
    __syncthreads();
    *reinterpret_cast<uint2 *>(mine + PASS * DIGITS + 2 * tid) = make_uint2(hist[2 * tid], hist[2 * tid + 1]);
  } else {
    if (chunk == 0) finish_kept(a, b, n);
    const int mid = n > a.keep ? hi : 0;  // (all of a shorter sequence is kept)
    // the always kept ones before this chunk, and the equal ones that stay
    before += n > a.keep ? min(from, a.sinks) + max(0, from - hi) : from;
    keep_in_order<KEYS2>(a, b, from, n, mid, any, least, need, before, equal, x, key,
                         KEYS2, sums);
  }
}

// The kept entries' copies: a workgroup for `group` neighbouring ones, 8 pieces
// of 16 bytes a thread in flight. An entry without a page becomes zeros: its new
// place is among the new length's entries, so what it held before (another
// sequence's, say) would be seen.
__global__ __launch_bounds__(256) void evict_copy_kernel(const Paged c, const Paged to,
                                                         const int32_t *to_lens,
                                                         const int32_t *kept, int ld_kept,
                                                         int pieces, int group) {
  __shared__ int src[64], dst[64];
  const int b = blockIdx.y, i0 = blockIdx.x * group;
  const int n = min(group, min(to_lens[b], to.max_entries) - i0);
  if (n <= 0) return;
  if ((int)threadIdx.x < n) {
    const int i = i0 + threadIdx.x;
    const int s = paged_row(c, c.table + (int64_t)b * c.ld_table, kept[(int64_t)b * ld_kept + i]);
    src[threadIdx.x] = s;
    dst[threadIdx.x] = paged_row(to, to.table + (int64_t)b * to.ld_table, i);
  }
  __syncthreads();
  const int all = n * 2 * pieces;
  for (int p0 = threadIdx.x; p0 < all; p0 += 256 * 8) {
    uint4 x[8];
    uint4 *at[8];
    bool ok[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int p = min(p0 + 256 * e, all - 1), i = p / (2 * pieces), q = p - i * 2 * pieces;
      const bool v = q >= pieces;
      const int64_t r = v ? q - pieces : q;
      const int s = src[i], d = dst[i];
      ok[e] = p0 + 256 * e < all && d >= 0;
      at[e] = reinterpret_cast<uint4 *>(v ? to.v : to.k) + (int64_t)d * pieces + r;
      x[e] = make_uint4(0u, 0u, 0u, 0u);
      if (ok[e] && s >= 0)
        x[e] = reinterpret_cast<const uint4 *>(v ? c.v : c.k)[(int64_t)s * pieces + r];
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (ok[e]) *at[e] = x[e];
  }
}

// Chunks of a sequence, 0 where one workgroup takes it all, as long as its
// registers hold the entries: that is faster up to there (one sequence of 2000
// entries 12 us against 20 in chunks, of 16,000 20 against 24; 16 of 16,000 28
// against 34). Two sequences of up to 131,000 entries take 29 us in the four
// launches (about 3 us of each are its start and end) and 13 in the copies.
int evict_chunks(const wg_paged_cache *c) {
  return c->max_entries <= SEL * KEYS1 ? 0
                                       : (c->max_entries + CHUNK_ENTRIES - 1) / CHUNK_ENTRIES;
}

// Both head preparations; axes NULL: one position a row.
int head_prep(const char *who, const float *qkv, int32_t M, int32_t ldq, const wg_attn_shape *sh,
              const float *q_norm, const float *k_norm, const float *rope, int32_t rope_rows,
              const int32_t *pos, int32_t ld_pos, const wg_rope_axes *axes,
              const wg_paged_cache *cache, const int32_t *row_start, float *q_out, int32_t ldqo,
              void *stream) {
  WG_REQUIRE(qkv && sh && rope && q_out, "%s: null argument", who);
  WG_REQUIRE(sh->kv_heads > 0 && sh->heads > 0 && sh->heads % sh->kv_heads == 0,
             "%s: %d query heads over %d KV heads", who, sh->heads, sh->kv_heads);
  const int hd = sh->head_dim;
  WG_REQUIRE(hd >= 8 && hd <= MAX_HD && hd % 8 == 0,
             "%s: head_dim %d (a multiple of 8 up to %d)", who, hd, MAX_HD);
  const int64_t slots = (int64_t)sh->heads + 2 * (int64_t)sh->kv_heads;
  WG_REQUIRE(slots <= 65535, "%s: %lld heads a row", who, (long long)slots);
  int rc = check_paged(cache, (int64_t)sh->kv_heads * hd, true, who);
  if (rc) return rc;
  WG_REQUIRE(M >= 1 && (row_start || M == cache->sequences),
             "%s: %d rows for %d sequences", who, M, cache->sequences);
  WG_REQUIRE(sh->rotated_dims >= 0 && sh->rotated_dims <= hd && sh->rotated_dims % 2 == 0,
             "%s: rotated dims %d", who, sh->rotated_dims);
  WG_REQUIRE(!sh->use_norm || (q_norm && k_norm), "%s: norm weights missing", who);
  WG_REQUIRE(rope_rows > 1024, "%s: a rope table of %d rows", who, rope_rows);
  WG_REQUIRE(ldq >= slots * hd && ldqo >= (int64_t)sh->heads * hd, "%s: strides too small", who);
  WG_REQUIRE(!overlaps(qkv, ((size_t)(M - 1) * ldq + slots * hd) * 4, q_out,
                       ((size_t)(M - 1) * ldqo + (size_t)sh->heads * hd) * 4),
             "%s: q_out overlaps qkv", who);
  RopeAxes ra = {};
  if (axes) {
    WG_REQUIRE(axes->axes >= 1 && axes->axes <= 4 && ld_pos >= axes->axes,
               "%s: %d axes (1 to 4) of %d positions a row", who, axes->axes, ld_pos);
    int64_t sum = 0;
    ra.axes = axes->axes;
    ra.interleaved = axes->interleaved != 0;
    for (int e = 0; e < axes->axes; e++) {
      const int n = ra.n[e] = axes->sections[e];
      WG_REQUIRE(n >= 0, "%s: a section of %d frequencies", who, n);
      sum += n;
    }
    WG_REQUIRE(sum == sh->rotated_dims / 2, "%s: sections of %lld frequencies for %d rotated dims", who,
               (long long)sum, sh->rotated_dims);
  }
  const PrepArgs a = {qkv, q_norm, k_norm, rope, pos, row_start, q_out, ldq, ldqo, M, sh->heads,
                      sh->kv_heads, hd, sh->use_norm, sh->rotated_dims, rope_rows, sh->eps, ra,
                      ld_pos};
  const uintptr_t ptrs = (uintptr_t)qkv | (uintptr_t)q_norm | (uintptr_t)k_norm |
                         (uintptr_t)rope | (uintptr_t)q_out;
  if ((hd == 64 || hd == 128) && sh->rotated_dims == hd && (ptrs & 15) == 0 && ldq % 4 == 0 &&
      ldqo % 4 == 0) {
    // Half the threads, twice each, where there are more rows' than run at once: up to
    // twice as many, or under several axes, whose angles each workgroup makes first. Us
    // with all and with half of them, heads normalised: of 32 query and 8 KV heads of
    // 128, 1400 rows 16.5, 14.5, 2142 21.7, 19.7, 8000 73.8, 74.3 (under 3 axes 19.1,
    // 14.9; 25.3, 21.5; 79.1, 78.3); of 64, 3997 rows 20.1, 19.1, 8000 without norms 36.0,
    // 36.9 (axes 22.7, 20.4; 44.3, 40.8); 14 and 2 of 64, 8000 rows 16.6, 17.7.
    int64_t threads = (slots * (hd / 16) + 63) / 64 * 64;
    if (threads >= 192 && M * threads > 2048 * 256 && (axes || M * threads <= 2048 * 512))
      threads = (threads / 2 + 63) / 64 * 64;
    auto kernel = axes ? (hd == 64 ? paged_prep_rows_kernel<64, true>
                                   : paged_prep_rows_kernel<128, true>)
                       : (hd == 64 ? paged_prep_rows_kernel<64, false>
                                   : paged_prep_rows_kernel<128, false>);
    kernel<<<M, threads < 1024 ? (unsigned)threads : 1024, 0, as_stream(stream)>>>(
        as_paged(cache), a);
  } else {
    auto kernel = axes ? paged_prep_kernel<true> : paged_prep_kernel<false>;
    kernel<<<dim3(M, (unsigned)slots), 64, 0, as_stream(stream)>>>(as_paged(cache), a);
  }
  return launched(who);
}

}  // namespace
}  // namespace wg

using namespace wg;

extern "C" {

int wg_paged_head_prep(const float *qkv, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                       const float *q_norm, const float *k_norm, const float *rope,
                       int32_t rope_rows, const int32_t *pos, const wg_paged_cache *cache,
                       const int32_t *row_start, float *q_out, int32_t ldqo, void *stream) {
  return head_prep("wg_paged_head_prep", qkv, M, ldq, sh, q_norm, k_norm, rope, rope_rows, pos, 1,
                   nullptr, cache, row_start, q_out, ldqo, stream);
}

int wg_paged_head_prep_axes(const float *qkv, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                            const float *q_norm, const float *k_norm, const float *rope,
                            int32_t rope_rows, const int32_t *pos, int32_t ld_pos,
                            const wg_rope_axes *axes, const wg_paged_cache *cache,
                            const int32_t *row_start, float *q_out, int32_t ldqo, void *stream) {
  WG_REQUIRE(axes && pos, "wg_paged_head_prep_axes: null argument");
  return head_prep("wg_paged_head_prep_axes", qkv, M, ldq, sh, q_norm, k_norm, rope, rope_rows,
                   pos, ld_pos, axes, cache, row_start, q_out, ldqo, stream);
}

size_t wg_paged_evict_scratch_bytes(const wg_paged_cache *c) {
  if (!c || c->sequences < 1 || c->max_entries < 1) return 0;
  const size_t chunks = evict_chunks(c);
  return chunks ? c->sequences * (chunks * (3 * DIGITS + 2) + 5) * 4 : 0;
}

int wg_paged_evict(const wg_paged_cache *cache, int32_t kv_dim, const float *weights,
                   int32_t ld_weights, int32_t keep, int32_t sinks, int32_t recent,
                   const wg_paged_cache *to, int32_t *to_lens, float *to_weights,
                   int32_t ld_to_weights, int32_t *kept, int32_t ld_kept, void *scratch,
                   size_t scratch_bytes, void *stream) {
  WG_REQUIRE(weights && to_lens && kept, "wg_paged_evict: null argument");
  WG_REQUIRE(kv_dim >= 8 && kv_dim % 8 == 0, "wg_paged_evict: %d values an entry (a multiple of 8)",
             kv_dim);
  int rc = check_paged(cache, kv_dim, true, "wg_paged_evict");
  if (!rc) rc = check_paged(to, kv_dim, false, "wg_paged_evict (to)");
  if (rc) return rc;
  const int n = cache->sequences;
  WG_REQUIRE(to->sequences == n, "wg_paged_evict: %d sequences to %d", n, to->sequences);
  WG_REQUIRE(keep >= 1 && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep,
             "wg_paged_evict: %d sinks and %d recent entries of %d kept", sinks, recent, keep);
  const int most = keep < cache->max_entries ? keep : cache->max_entries;
  WG_REQUIRE(to->max_entries >= most, "wg_paged_evict: room for %d entries of %d kept",
             to->max_entries, most);
  WG_REQUIRE(ld_weights >= cache->max_entries && ld_kept >= keep &&
                 (!to_weights || ld_to_weights >= keep),
             "wg_paged_evict: strides too small");
  WG_REQUIRE(!to_weights || !overlaps(weights, ((size_t)(n - 1) * ld_weights + cache->max_entries) * 4,
                                      to_weights, ((size_t)(n - 1) * ld_to_weights + keep) * 4),
             "wg_paged_evict: to_weights overlaps weights");
  const EvictArgs a = {weights, to_lens, kept, to_weights, ld_weights, ld_kept, ld_to_weights,
                       keep, sinks, recent};
  const size_t need = wg_paged_evict_scratch_bytes(cache);
  WG_REQUIRE(scratch_bytes >= need && (!need || (scratch && ((uintptr_t)scratch & 15) == 0)),
             "wg_paged_evict: scratch of %zu bytes, needs %zu (16-byte aligned)", scratch_bytes,
             need);
  const Paged c = as_paged(cache);
  hipStream_t s = as_stream(stream);
  if (const int chunks = evict_chunks(cache)) {
    uint32_t *m = (uint32_t *)scratch;
    const size_t counts = (size_t)n * chunks * 3 * DIGITS;
    uint32_t *above = m + counts, *state = above + (size_t)n * chunks * 2;
    const EvictScratch sc = {m, above, state, (int32_t *)state + (size_t)n * 4, chunks};
    evict_chunk_kernel<0><<<dim3(chunks, n), SEL, 0, s>>>(c, a, sc);
    evict_chunk_kernel<1><<<dim3(chunks, n), SEL, 0, s>>>(c, a, sc);
    evict_chunk_kernel<2><<<dim3(chunks, n), SEL, 0, s>>>(c, a, sc);
    evict_chunk_kernel<3><<<dim3(chunks, n), SEL, 0, s>>>(c, a, sc);
  } else {
    evict_select_kernel<<<n, SEL, 0, s>>>(c, a);
  }
  rc = launched("wg_paged_evict");
  if (rc) return rc;
  const int pieces = kv_dim / 8, fit = 2048 / (2 * pieces);  // (8 pieces a thread)
  const int group = fit < 1 ? 1 : fit > 64 ? 64 : fit;
  evict_copy_kernel<<<dim3((most + group - 1) / group, n), 256, 0, s>>>(
      c, as_paged(to), to_lens, kept, ld_kept, pieces, group);
  return launched("wg_paged_evict");
}

}  // extern "C"
