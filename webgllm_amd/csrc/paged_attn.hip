// Attention over the paged cache: decode (one row a sequence) and prompts
// (rows of many sequences), both under an optional sliding window with the
// first entries kept visible.
#include "common.h"
#include "dot.h"
#include "lds_load.h"
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
  int ldq, ldo, M, H, KV, window, sinks;
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
}

// ---------------------------------------------------------------- decode
//
// Flash decoding over all sequences at once. A unit is (sequence, KV head,
// group of up to 16 of its query heads); what it sees is cut into tiles of 32
// entries, and the tiles of all units, one after another, into even runs of
// `workers` workgroups: however ragged the lengths, every compute unit streams
// the same number of bytes, and the lengths stay on the device. A workgroup's
// waves take the tiles of its run in turn, each with its own running maximum,
// sum and weighted values, which meet in LDS where a unit ends. A unit inside
// one run is finished there; the others leave a part per run, and
// paged_join_kernel adds them up in order.
constexpr int TK = 32;           // entries a tile
constexpr int DW = 4;            // waves a workgroup
constexpr int MAX_WORKERS = 512; // two workgroups a compute unit
constexpr int QC = 16;           // query heads a unit

struct DecodeArgs {
  const float *q;
  uint16_t *out;
  float *parts;  // [workers][2][group][HD + 4]: values, then maximum and sum
  int *joins;    // [workers][4]: unit's sequence (-1: none), unit, first run, last run
  float *stats;  // [sequences][H][2]: maximum (log2) and 1 / sum; or NULL
  float *scores; // [sequences][H][ld_scores], log2; or NULL
  int64_t ld_scores;
  int ldq, ldo, H, KV, window, sinks;
};

// Entries that sequence b's newest row sees.
__device__ inline Span decode_span(const Paged &c, int b, int window, int sinks) {
  const int n = paged_len(c, b);
  return n > 0 ? paged_span(n - 1, n - 1, window, sinks) : Span{0, 0, 0};
}
__device__ inline int64_t wave_scan(int64_t v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

// The runs: `workers` of them over `total` tiles, run w from start(w) on.
struct Runs {
  int64_t total;
  int workers;
  __device__ int64_t start(int w) const { return w * total / workers; }
  __device__ int of(int64_t tile) const { return (int)(((tile + 1) * workers - 1) / total); }
};

// Sums the sequences' tiles (64 lanes over the sequences, each a stretch of
// them) and finds the sequence that holds tile `at(runs)`; *first its first tile.
template <typename At>
__device__ inline Runs find_run(const Paged &c, const DecodeArgs &a, int units, int grid, At at,
                                int *seq, int64_t *first) {
  const int lane = threadIdx.x & 63, per = (c.seqs + 63) >> 6;
  int64_t mine = 0;
  int full = 0;
  for (int i = 0; i < per; i++) {
    const int b = lane * per + i;
    if (b >= c.seqs) break;
    const int t = (decode_span(c, b, a.window, a.sinks).count + TK - 1) / TK;
    mine += t;
    full += t > 0;
  }
  const int64_t sum = wave_scan(mine);
  Runs r;
  r.total = __shfl(sum, 63, 64) * units;
  int live = full;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) live += __shfl_xor(live, d, 64);
  // as many runs as give every wave a tile, and at least one a unit
  const int64_t want = max((r.total + DW - 1) / DW, (int64_t)live * units);
  r.workers = (int)min((int64_t)grid, want);
  *seq = -1;
  if (r.total == 0) return r;
  const int64_t t = at(r) / units;  // a unit's tiles follow one another: sequence by division
  // the lane whose stretch holds tile t of the sequences' tiles
  const uint64_t past = __ballot(sum > t);
  const int l = __ffsll((unsigned long long)past) - 1;
  int64_t base = l > 0 ? __shfl(sum, l - 1, 64) : 0;
  for (int b0 = l * per; b0 < (l + 1) * per; b0 += 64) {
    const int b = b0 + lane;
    int tiles = 0;
    if (b < c.seqs && b < (l + 1) * per)
      tiles = (decode_span(c, b, a.window, a.sinks).count + TK - 1) / TK;
    const int64_t run = base + wave_scan(tiles);
    const uint64_t over = __ballot(run > t);
    if (over) {
      const int f = __ffsll((unsigned long long)over) - 1;
      *seq = b0 + f;
      *first = (f > 0 ? __shfl(run, f - 1, 64) : base) * units;
      return r;
    }
    base = __shfl(run, 63, 64);
  }
  return r;
}

template <int HD>
__host__ __device__ constexpr int decode_lds(int group) {
  return DW * 2 * TK * HD * 2 + DW * group * (HD + 4) * 4;
}

// Scores as S^T = K Q^T on v_mfma_f32_16x16x32_f16: A = 16 entries' keys
// straight from memory (each lane's 8 dims are 16 bytes of a row), B = the
// queries, each scaled by a power of two to the top of the halves and split
// into hi = half(q) and lo = half(q - hi), so that scores keep 22 bits of any
// finite query. A lane then holds 8 entries of one query, and its weights,
// split alike, are the B operand of O^T = V^T P^T as they stand: entry
// 16 (e / 4) + 4 (lane / 16) + e % 4 is k-index 8 (lane / 16) + e, and the
// value tile's transposing LDS loads read the same entries.
// Entries of no page, or past the last, read the tile's first entry that has
// one and weigh nothing: bits that the row does not see never enter.
template <int HD>
__global__ __launch_bounds__(DW * 64, 2) void paged_decode_kernel(const Paged c,
                                                                 const DecodeArgs a) {
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  typedef short short4v __attribute__((ext_vector_type(4)));
  typedef float f4v __attribute__((ext_vector_type(4)));
  constexpr int KP = HD / 8, ROWB = HD * 2, TILE = TK * ROWB, RPI = 64 / KP, NI = TK / RPI;
  constexpr int QS = HD / 32, DT = HD / 16, MS = HD + 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.H / a.KV, QG = (G + QC - 1) / QC, units = a.KV * QG, kvd = a.KV * HD;
  const int GS = min(G, QC);  // a part's query heads
  // rows r of a value tile keep 16-byte piece p at p ^ swz(r): the 16 rows that
  // a transposing load takes 32 bytes of lie two to a bank
  auto swz = [](int r) { return KP == 16 ? r & 15 : ((r >> 1) & 3) << 1; };
  unsigned char *vt = smem + wave * 2 * TILE;
  const uint32_t vlds = (uint32_t)(uintptr_t)vt;
  float *mrg = reinterpret_cast<float *>(smem + DW * 2 * TILE);

  const int w = blockIdx.x;
  int b;
  int64_t first;
  const Runs runs = find_run(
      c, a, units, gridDim.x, [&](const Runs &r) { return w < r.workers ? r.start(w) : 0; }, &b,
      &first);
  // rows that see nothing
  for (int z = w; z < c.seqs; z += gridDim.x)
    if (decode_span(c, z, a.window, a.sinks).count == 0) {
      for (int d = threadIdx.x; d < a.H * HD; d += DW * 64) a.out[(int64_t)z * a.ldo + d] = 0;
      if (a.stats)
        for (int h = threadIdx.x; h < a.H; h += DW * 64)
          a.stats[((int64_t)z * a.H + h) * 2] = a.stats[((int64_t)z * a.H + h) * 2 + 1] = 0.0f;
    }
  if (w >= runs.workers || b < 0) {
    if (threadIdx.x == 0) a.joins[4 * w] = -1;
    return;
  }
  const int64_t from = runs.start(w), upto = runs.start(w + 1);
  int64_t at = from;
  Span sp = decode_span(c, b, a.window, a.sinks);
  int tiles = (sp.count + TK - 1) / TK;
  int u = (int)((at - first) / tiles);
  while (true) {
    // unit u of sequence b: its tiles t0 .. t1 - 1 are this run's
    const int64_t unit0 = first + (int64_t)u * tiles;
    const int t0 = (int)(at - unit0), t1 = (int)min((int64_t)tiles, upto - unit0);
    const int kh = u / QG, qg = u % QG, GQ = min(QC, G - qg * QC);
    const int32_t *pages = c.table + (int64_t)b * c.ld_table;
    const bool mine = n16 < GQ;
    const int head = kh * G + qg * QC + n16;
    // this lane's entry of a tile: its pool row, or -1
    auto row_of = [&](int t) {
      const int i = t * TK + (lane & 31);
      return t < t1 && i < sp.count ? paged_row(c, pages, span_entry(sp, i)) : -1;
    };
    int t = t0 + wave;
    int row = row_of(t), row_next = row_of(t + DW);
    float4 qraw[QS][2];
    {
      const float *qp = a.q + (int64_t)b * a.ldq + (int64_t)(mine ? head : 0) * HD + 8 * c4;
#pragma unroll
      for (int s = 0; s < QS; s++) {
        qraw[s][0] = *reinterpret_cast<const float4 *>(qp + 32 * s);
        qraw[s][1] = *reinterpret_cast<const float4 *>(qp + 32 * s + 4);
      }
    }
    uint32_t seen, seen_next = 0;
    half8 kc[2][QS], kn[2][QS];
    auto issue = [&](int r, int buf, half8 (&k)[2][QS]) -> uint32_t {
      const uint32_t live = (uint32_t)__ballot(r >= 0);
      if (live == 0) return 0;
      const int some = __builtin_amdgcn_readlane(r, __builtin_ctz(live));
      r = r < 0 ? some : r;
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        const int kr = __shfl(r, 16 * kt + n16, 64);
        const uint16_t *kp = c.k + (int64_t)kr * kvd + kh * HD + 8 * c4;
#pragma unroll
        for (int s = 0; s < QS; s++) k[kt][s] = *reinterpret_cast<const half8 *>(kp + 32 * s);
      }
#pragma unroll
      for (int ii = 0; ii < NI; ii++) {
        const int vr = ii * RPI + lane / KP;
        const int pr = __shfl(r, vr, 64);
        dma16(c.v + (int64_t)pr * kvd + kh * HD + ((lane % KP) ^ swz(vr)) * 8,
              vlds + buf * TILE + ii * 1024);
      }
      return live;
    };
    seen = issue(row, 0, kc);
    row = row_next;
    row_next = row_of(t + 2 * DW);
    // the queries as B operands: dims 32 s + 8 c4 .. + 7
    half8 qhi[QS], qlo[QS];
    float scale;
    {
      float v[QS][8], big = 0.0f;
#pragma unroll
      for (int s = 0; s < QS; s++) {
        const float4 x = qraw[s][0], y = qraw[s][1];
        const float e8[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; e++) {
          v[s][e] = mine ? e8[e] : 0.0f;
          big = fmaxf(big, fabsf(v[s][e]));
        }
      }
      big = fmaxf(big, xor16(big));
      big = fmaxf(big, xor32(big));
      // 2^k with big 2^k in [2^13, 2^14); an exponent that float32 holds both ways
      const int e = big > 0.0f && big < INFINITY ? ilogbf(big) : 13;
      const int k = min(max(13 - e, -114), 100);
      const float up = ldexpf(1.0f, k);
      scale = ldexpf(1.44269504088896340736f, -k);
#pragma unroll
      for (int s = 0; s < QS; s++)
#pragma unroll
        for (int e8 = 0; e8 < 8; e8++) {
          const float x = v[s][e8] * up;
          const _Float16 hi = (_Float16)x;
          qhi[s][e8] = hi;
          qlo[s][e8] = (_Float16)(x - (float)hi);
        }
    }
    float m_run = -INFINITY, l_run = 0.0f;
    f4v o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    for (int buf = 0; t < t1; t += DW, buf ^= 1) {
      // this tile's loads have landed; the other buffer's reads are done
      wait_vm<0>();
      __builtin_amdgcn_s_waitcnt(0xc07f);
      asm volatile("" ::: "memory");
      seen_next = t + DW < t1 ? issue(row, buf ^ 1, kn) : 0;
      row = row_next;
      row_next = row_of(t + 3 * DW);
      if (seen) {
        float sc[2][4], tmax = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
          f4v st = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int s = 0; s < QS; s++) {
            st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kt][s], qhi[s], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kt][s], qlo[s], st, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const bool vis = (seen >> (16 * kt + 4 * c4 + i)) & 1;
            sc[kt][i] = vis ? st[i] * scale : -INFINITY;
            tmax = fmaxf(tmax, sc[kt][i]);
          }
        }
        if (a.scores && mine) {
          float *sp_ = a.scores + ((int64_t)b * a.H + head) * a.ld_scores + t * TK + 4 * c4;
          *reinterpret_cast<f4v *>(sp_) = f4v{sc[0][0], sc[0][1], sc[0][2], sc[0][3]};
          *reinterpret_cast<f4v *>(sp_ + 16) = f4v{sc[1][0], sc[1][1], sc[1][2], sc[1][3]};
        }
        tmax = fmaxf(tmax, xor16(tmax));
        tmax = fmaxf(tmax, xor32(tmax));
        const float m_new = fmaxf(m_run, tmax), mu = m_new == -INFINITY ? 0.0f : m_new;
        if (__ballot(m_new != m_run)) {
          const float corr = __builtin_amdgcn_exp2f(m_run - mu);
          l_run *= corr;
#pragma unroll
          for (int dt = 0; dt < DT; dt++) o[dt] *= corr;
          m_run = m_new;
        }
        half8 phi, plo;
        float psum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float p = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - mu);
          psum += p;
          const _Float16 hi = (_Float16)p;
          phi[e] = hi;
          plo[e] = (_Float16)(p - (float)hi);
        }
        psum += xor16(psum);
        psum += xor32(psum);
        l_run += psum;
        const unsigned char *vb = vt + buf * TILE;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          half8 va;
#pragma unroll
          for (int hh = 0; hh < 2; hh++) {
            const int r = 16 * hh + 4 * c4 + (n16 >> 2), col = 16 * dt + 4 * (n16 & 3);
            const unsigned char *p = vb + r * ROWB + (((col >> 3) ^ swz(r)) * 16) + (col & 7) * 2;
            const half4 h4 = __builtin_bit_cast(
                half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) short4v *)(uint32_t)(uintptr_t)p));
#pragma unroll
            for (int e = 0; e < 4; e++) va[4 * hh + e] = h4[e];
          }
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, phi, o[dt], 0, 0, 0);
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, plo, o[dt], 0, 0, 0);
        }
      } else if (a.scores && mine) {  // no entry of the tile has a page
        float *sp_ = a.scores + ((int64_t)b * a.H + head) * a.ld_scores + t * TK + 4 * c4;
        const f4v none = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        *reinterpret_cast<f4v *>(sp_) = none;
        *reinterpret_cast<f4v *>(sp_ + 16) = none;
      }
      seen = seen_next;
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int s = 0; s < QS; s++) kc[kt][s] = kn[kt][s];
    }
    wait_vm<0>();
    // the waves' sums meet: lane (query, c4) holds dims 16 dt + 4 c4 .. + 3
    if (mine) {
      float *mw = mrg + (wave * GS + n16) * MS;
#pragma unroll
      for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f4v *>(mw + 16 * dt + 4 * c4) = o[dt];
      if (c4 == 0) {
        mw[HD] = m_run;
        mw[HD + 1] = l_run;
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    for (int i = threadIdx.x; i < GQ * (HD / 4); i += DW * 64) {
      const int g = i / (HD / 4), d = i % (HD / 4) * 4;
      const float *mw = mrg + g * MS;
      float mx = -INFINITY, l = 0.0f;
#pragma unroll
      for (int v = 0; v < DW; v++) mx = fmaxf(mx, mw[v * GS * MS + HD]);
      const float mu = mx == -INFINITY ? 0.0f : mx;
      f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int v = 0; v < DW; v++) {
        const float *p = mw + v * GS * MS;
        const float e = __builtin_amdgcn_exp2f(p[HD] - mu);
        l += p[HD + 1] * e;
        x += *reinterpret_cast<const f4v *>(p + d) * e;
      }
      const int h = kh * G + qg * QC + g;
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t *op = a.out + (int64_t)b * a.ldo + (int64_t)h * HD + d;
#pragma unroll
        for (int e = 0; e < 4; e++) op[e] = half_of(x[e] * inv);
        if (a.stats && d == 0) {
          a.stats[((int64_t)b * a.H + h) * 2] = mu;
          a.stats[((int64_t)b * a.H + h) * 2 + 1] = inv;
        }
      } else {
        float *pp = a.parts + ((int64_t)(2 * w + (at != from)) * GS + g) * MS;
        *reinterpret_cast<f4v *>(pp + d) = x;
        if (d == 0) {
          pp[HD] = mx;
          pp[HD + 1] = l;
        }
      }
    }
    // The run that first takes up a unit begun before it joins its parts.
    if (threadIdx.x == 0 && at == from) {
      const int lead = runs.of(unit0);
      const bool joins = t0 > 0 && lead + 1 == w;
      a.joins[4 * w] = joins ? b : -1;
      a.joins[4 * w + 1] = u;
      // (the sign: whether the unit began with its first run or inside it)
      a.joins[4 * w + 2] = runs.start(lead) == unit0 ? lead : -1 - lead;
      a.joins[4 * w + 3] = runs.of(unit0 + tiles - 1);
    }
    at = unit0 + t1;
    if (at >= upto) break;
    if (++u == units) {
      first += (int64_t)units * tiles;
      u = 0;
      do {
        if (++b >= c.seqs) return;
        sp = decode_span(c, b, a.window, a.sinks);
        tiles = (sp.count + TK - 1) / TK;
      } while (tiles == 0);
    }
    __syncthreads();  // the sums' place is free again
  }
}

// The parts of a unit that several runs took, in the runs' order: threads over
// its values (4 each), as many stretches of the parts side by side as fit.
template <int HD>
__global__ __launch_bounds__(1024) void paged_join_kernel(const Paged c, const DecodeArgs a) {
  typedef float f4v __attribute__((ext_vector_type(4)));
  constexpr int MS = HD + 4;
  __shared__ f4v xs[1024];
  __shared__ float ms[1024], ls[1024];
  const int w = blockIdx.x, b = a.joins[4 * w];
  if (b < 0) return;
  const int u = a.joins[4 * w + 1], lead = a.joins[4 * w + 2], last = a.joins[4 * w + 3];
  const int w0 = lead < 0 ? -1 - lead : lead, n = last - w0 + 1;
  const int G = a.H / a.KV, QG = (G + QC - 1) / QC, GS = min(G, QC);
  const int kh = u / QG, qg = u % QG, GQ = min(QC, G - qg * QC);
  const int cols = GQ * (HD / 4), sets = 1024 / cols;
  const int i = threadIdx.x % cols, set = threadIdx.x / cols;
  const int g = i / (HD / 4), d = i % (HD / 4) * 4;
  float mx = -INFINITY, l = 0.0f;
  f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
  if (set < sets) {
    const int per = (n + sets - 1) / sets;
#pragma unroll 4
    for (int p = set * per; p < min(n, set * per + per); p++) {
      // a run's first part, or its second where the unit began inside the run
      const float *pp =
          a.parts + ((int64_t)(2 * (w0 + p) + (p == 0 && lead < 0)) * GS + g) * MS;
      const float m2 = pp[HD], l2 = pp[HD + 1];
      const f4v y = *reinterpret_cast<const f4v *>(pp + d);
      const float top = fmaxf(mx, m2), mu = top == -INFINITY ? 0.0f : top;
      const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2 - mu);
      x = x * e1 + y * e2;
      l = l * e1 + l2 * e2;
      mx = top;
    }
  }
  xs[threadIdx.x] = x;
  ms[threadIdx.x] = mx;
  ls[threadIdx.x] = l;
  __syncthreads();
  if (set != 0) return;
  for (int s = 1; s < sets; s++) {
    const int j = s * cols + i;
    const float m2 = ms[j], top = fmaxf(mx, m2), mu = top == -INFINITY ? 0.0f : top;
    const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2 - mu);
    x = x * e1 + xs[j] * e2;
    l = l * e1 + ls[j] * e2;
    mx = top;
  }
  const int h = kh * G + qg * QC + g;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t *op = a.out + (int64_t)b * a.ldo + (int64_t)h * HD + d;
#pragma unroll
  for (int e = 0; e < 4; e++) op[e] = half_of(x[e] * inv);
  if (a.stats && d == 0) {
    a.stats[((int64_t)b * a.H + h) * 2] = mx == -INFINITY ? 0.0f : mx;
    a.stats[((int64_t)b * a.H + h) * 2 + 1] = inv;
  }
}

// weights[b][entry] += its attention weight, summed over the heads in order.
__global__ __launch_bounds__(256) void paged_weights_kernel(const Paged c, const DecodeArgs a,
                                                            float *weights, int ldw) {
  const int b = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
  const Span sp = decode_span(c, b, a.window, a.sinks);
  if (t >= sp.count) return;
  float w = 0.0f;
  for (int h = 0; h < a.H; h++) {
    const int64_t bh = (int64_t)b * a.H + h;
    w += __builtin_amdgcn_exp2f(a.scores[bh * a.ld_scores + t] - a.stats[bh * 2]) *
         a.stats[bh * 2 + 1];
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

// The decode scratch: parts, joins, then (with weights) stats and scores.
struct DecodeScratch {
  size_t parts, joins, stats, scores, end;  // byte offsets
  int64_t ld_scores;
};
DecodeScratch decode_scratch(const wg_paged_cache *c, const wg_attn_shape *sh, bool weights) {
  const int G = sh->heads / sh->kv_heads;
  DecodeScratch d;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  d.parts = 0;
  d.joins = up((size_t)MAX_WORKERS * 2 * (G < QC ? G : QC) * (sh->head_dim + 4) * 4);
  d.stats = d.joins + up(MAX_WORKERS * 16);
  const size_t rows = (size_t)c->sequences * sh->heads;
  d.scores = d.stats + (weights ? up(rows * 8) : 0);
  d.ld_scores = ((int64_t)c->max_entries + TK - 1) / TK * TK;
  d.end = d.scores + (weights ? rows * d.ld_scores * 4 : 0);
  return d;
}

template <int HD>
int launch_decode(const Paged &c, const DecodeArgs &a, int grid, hipStream_t s) {
  const int G = a.H / a.KV, lds = decode_lds<HD>(G < QC ? G : QC);
  const int rc = raise_lds((const void *)paged_decode_kernel<HD>, lds);
  if (rc) return rc;
  paged_decode_kernel<HD><<<grid, DW * 64, lds, s>>>(c, a);
  if (grid > 1) paged_join_kernel<HD><<<grid, 1024, 0, s>>>(c, a);
  return launched("wg_paged_attn_decode");
}

}  // namespace
}  // namespace wg

using namespace wg;

extern "C" {

size_t wg_paged_decode_scratch_bytes(const wg_paged_cache *c, const wg_attn_shape *sh,
                                     int32_t with_weights) {
  if (!c || !sh || c->sequences < 1 || sh->heads < 1 || sh->kv_heads < 1 || sh->head_dim < 1 ||
      c->max_entries < 1)
    return 0;
  return decode_scratch(c, sh, with_weights != 0).end;
}

int wg_paged_attn_decode(const float *q, int32_t ldq, const wg_attn_shape *sh,
                         const wg_paged_cache *cache, int32_t window, int32_t sinks,
                         float *weights, int32_t ld_weights, uint16_t *out, int32_t ldo,
                         void *scratch, size_t scratch_bytes, void *stream) {
  int rc = check_attn(q, cache ? cache->sequences : 0, ldq, sh, cache, window, sinks, out, ldo, 64,
                      "wg_paged_attn_decode");
  if (rc) return rc;
  const DecodeScratch d = decode_scratch(cache, sh, weights != nullptr);
  WG_REQUIRE(scratch && scratch_bytes >= d.end && ((uintptr_t)scratch & 15) == 0,
             "wg_paged_attn_decode: scratch of %zu bytes, needs %zu (16-byte aligned)",
             scratch_bytes, d.end);
  WG_REQUIRE(!weights || ld_weights >= cache->max_entries,
             "wg_paged_attn_decode: weights of %d entries a sequence of up to %d", ld_weights,
             cache->max_entries);
  unsigned char *m = (unsigned char *)scratch;
  const DecodeArgs a = {q, out, (float *)(m + d.parts), (int *)(m + d.joins),
                        weights ? (float *)(m + d.stats) : nullptr,
                        weights ? (float *)(m + d.scores) : nullptr, d.ld_scores, ldq, ldo,
                        sh->heads, sh->kv_heads, window, sinks};
  const Paged c = as_paged(cache);
  hipStream_t s = as_stream(stream);
  // as many runs as the longest sequences could use
  const int64_t most = window > 0 ? (int64_t)window + sinks : cache->max_entries;
  const int64_t entries = most < cache->max_entries ? most : cache->max_entries;
  const int64_t units = (int64_t)cache->sequences * sh->kv_heads *
                        ((sh->heads / sh->kv_heads + QC - 1) / QC);
  const int64_t tiles = (entries + TK - 1) / TK, per = (tiles + DW - 1) / DW;
  const int grid = units * per < MAX_WORKERS ? (int)(units * per) : MAX_WORKERS;
  rc = sh->head_dim == 64 ? launch_decode<64>(c, a, grid, s) : launch_decode<128>(c, a, grid, s);
  if (rc || !weights) return rc;
  paged_weights_kernel<<<dim3((unsigned)((entries + 255) / 256), cache->sequences), 256, 0, s>>>(
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
  const RowArgs a = {q, row_start, out, ldq, ldo, M, sh->heads, sh->kv_heads, window, sinks};
  auto kernel = sh->head_dim == 64 ? paged_row_kernel<64> : paged_row_kernel<128>;
  kernel<<<dim3(a.M, a.H), 64, 0, as_stream(stream)>>>(as_paged(cache), a);
  return launched("wg_paged_attn_prefill");
}

}  // extern "C"
