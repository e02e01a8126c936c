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
// Flash decoding over all sequences at once. A workgroup's 4 waves stand side
// by side on `wide` KV heads (as many of 4, 2 or 1 as divide the KV heads) and,
// where those are fewer than the waves, on neighbouring tiles of 32 entries: a
// step is 4 / wide tiles of `wide` heads, which lie together in an entry's row
// (one head of 128 alone is 256 bytes of every 2 KB; reading 131,072 entries
// of 8 such heads, K and V, 4 heads together reach 6.1 to 6.3 TB/s on this
// card, one at a time 5.3 to 5.9).
// A unit is (sequence, those heads, a group of up to 16 query heads of each);
// the steps of all units, one after another, are cut into even runs of
// `workers` workgroups: however ragged the lengths, every compute unit streams
// the same number of bytes, and the lengths stay on the device. Each wave has
// its own running maximum, sum and weighted values; waves of one head add
// theirs up in LDS where a unit ends. A unit inside one run is finished there;
// the others leave a part per run, and paged_join_kernel adds them up in order.
constexpr int TK = 32;           // entries a tile
constexpr int DW = 4;            // waves a workgroup
constexpr int MAX_WORKERS = 512; // two workgroups a compute unit
constexpr int QC = 16;           // query heads a KV head and unit
constexpr int MIN_STEPS = 2;     // steps of a run, where there are so many

struct DecodeArgs {
  const float *q;
  uint16_t *out;
  float *parts;  // [workers][2][wide][group][HD + 4]: values, then maximum and sum
  int *joins;    // [units][4]: first run (-1: finished there), its part, last run
  float *stats;  // [sequences][H][2]: maximum (log2) and 1 / sum; or NULL
  float *scores; // [sequences][H][ld_scores], log2; or NULL
  int64_t ld_scores;
  int ldq, ldo, H, KV, window, sinks, wide;
};

// 4 output halves at dim `at` of row b; 8 bytes at once where they are aligned.
typedef float f4x __attribute__((ext_vector_type(4)));
__device__ inline void store_half4(const DecodeArgs &a, int b, int64_t at, f4x x) {
  uint16_t *op = a.out + (int64_t)b * a.ldo + at;
  if (((uintptr_t)op & 7) == 0) {
    *reinterpret_cast<uint2 *>(op) = make_uint2(half_of(x[0]) | (uint32_t)half_of(x[1]) << 16,
                                                half_of(x[2]) | (uint32_t)half_of(x[3]) << 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) op[e] = half_of(x[e]);
  }
}

// Entries that sequence b's newest row sees.
__device__ inline Span decode_span(const Paged &c, int b, int window, int sinks) {
  const int n = paged_len(c, b);
  return n > 0 ? paged_span(n - 1, n - 1, window, sinks) : Span{0, 0, 0};
}
// Steps of `entries` entries.
__device__ inline int span_steps(const Span &s, int entries) {
  return (int)((uint32_t)(s.count + entries - 1) / (uint32_t)entries);
}
// Inclusive sums over the wave, by DPP: shifts within rows of 16 lanes, then a
// row's and the lower half's sum into what follows.
__device__ inline uint32_t wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
__device__ inline uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// The runs: `workers` of them over all steps (fewer than 2^31), the first
// `longer` of `each` + 1 steps, the others of `each`.
struct Runs {
  uint32_t workers, each, longer;
  __device__ uint32_t start(uint32_t w) const { return w * each + min(w, longer); }
  __device__ uint32_t of(uint32_t step) const {
    const uint32_t edge = longer * (each + 1);
    return step < edge ? step / (each + 1) : longer + (step - edge) / each;
  }
};

// Sums the sequences' steps (each lane a stretch of them) and finds the
// sequence that holds run w's first step; *first is that sequence's first.
__device__ inline Runs find_run(const Paged &c, const DecodeArgs &a, uint32_t units, int entries,
                                uint32_t grid, uint32_t w, int *seq, uint32_t *first) {
  const int lane = threadIdx.x & 63, per = (c.seqs + 63) >> 6;
  uint32_t mine = 0, live = 0;
  for (int i = 0; i < per; i++) {
    const int b = lane * per + i;
    const uint32_t t =
        b < c.seqs ? span_steps(decode_span(c, b, a.window, a.sinks), entries) : 0;
    mine += t;
    live += t > 0;
  }
  const uint32_t sum = wave_scan(mine);
  const uint32_t total = uniform(__shfl(sum, 63, 64)) * units;
  const uint32_t all = uniform(__shfl(wave_scan(live), 63, 64)) * units;
  // runs of MIN_STEPS at least, but one a unit at least
  Runs r;
  r.workers = min(grid, max((total + MIN_STEPS - 1) / MIN_STEPS, all));
  *seq = -1;
  *first = 0;
  if (w >= r.workers) return r;
  r.each = total / r.workers;
  r.longer = total - r.each * r.workers;
  // a sequence's units follow one another: its steps are those of t = step / units
  const uint32_t t = r.start(w) / units;
  const int l = __ffsll((unsigned long long)__ballot(sum > t)) - 1;
  uint32_t base = l > 0 ? uniform(__shfl(sum, l - 1, 64)) : 0;
  if (per == 1) {
    *seq = l;
    *first = base * units;
    return r;
  }
  for (int b0 = l * per; b0 < (l + 1) * per; b0 += 64) {
    const int b = b0 + lane;
    const bool in = b < c.seqs && b < (l + 1) * per;
    const uint32_t run =
        base + wave_scan(in ? span_steps(decode_span(c, b, a.window, a.sinks), entries) : 0);
    const uint64_t over = __ballot(run > t);
    if (over) {
      const int f = __ffsll((unsigned long long)over) - 1;
      *seq = b0 + f;
      *first = (f > 0 ? uniform(__shfl(run, f - 1, 64)) : base) * units;
      return r;
    }
    base = uniform(__shfl(run, 63, 64));
  }
  return r;
}

// A wave's place in its workgroup's run: step t of steps t0 .. t1 - 1 of the
// unit of its KV head kh and query group qg of sequence b; `left` steps from
// the unit's first to the run's end.
struct Slot {
  int b, kh, qg, t, t0, t1, steps;
  Span sp;
  uint32_t left;
  bool ok;
  __device__ bool last() const { return t + 1 >= t1; }
};
__device__ inline void next_slot(Slot &s, const Paged &c, const DecodeArgs &a, int QG, int hw,
                                 int entries) {
  if (!s.last()) {
    s.t++;
    return;
  }
  s.ok = s.ok && s.left > (uint32_t)s.steps;
  if (!s.ok) return;
  s.left -= s.steps;
  if (++s.qg == QG) {
    s.qg = 0;
    s.kh += a.wide;
  }
  if (s.kh >= a.KV) {
    s.kh = hw;
    do {
      if (++s.b >= c.seqs) {
        s.ok = false;
        return;
      }
      s.sp = decode_span(c, s.b, a.window, a.sinks);
      s.steps = span_steps(s.sp, entries);
    } while (s.steps == 0);
  }
  s.t0 = s.t = 0;
  s.t1 = (int)min((uint32_t)s.steps, s.left);
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
// A wave's tiles are loaded one ahead and their pages looked up two ahead,
// across the ends of units.
template <int HD>
__global__ __launch_bounds__(DW * 64, 2) void paged_decode_kernel(const Paged c,
                                                                 const DecodeArgs a) {
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  typedef short short4v __attribute__((ext_vector_type(4)));
  typedef float f4v __attribute__((ext_vector_type(4)));
  constexpr int KP = HD / 8, ROWB = HD * 2, TILE = TK * ROWB, RPI = 64 / KP, NI = TK / RPI;
  constexpr int QS = HD / 32, DT = HD / 16, MS = HD + 4;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, n16 = lane & 15, c4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wide = a.wide, hw = wave & (wide - 1);
  const int EW = wide == 4 ? 1 : wide == 2 ? 2 : 4, ew = wide == 4 ? 0 : wide == 2 ? wave >> 1 : wave;
  const int entries = EW * TK;  // of a step
  const int G = a.H / a.KV, QG = (G + QC - 1) / QC, units = a.KV / wide * QG, kvd = a.KV * HD;
  const int GS = min(G, QC);  // a part's query heads of a KV head
  // rows r of a value tile keep 16-byte piece p at p ^ swz(r): the 16 rows that
  // a transposing load takes 32 bytes of lie two to a bank
  auto swz = [](int r) { return KP == 16 ? r & 15 : ((r >> 1) & 3) << 1; };
  unsigned char *vt = smem + wave * 2 * TILE;
  const uint32_t vlds = (uint32_t)(uintptr_t)vt;
  float *mrg = reinterpret_cast<float *>(smem + DW * 2 * TILE);

  const uint32_t w = blockIdx.x;
  int b0;
  uint32_t first;
  const Runs runs = find_run(c, a, units, entries, gridDim.x, w, &b0, &first);
  // rows that see nothing
  for (int z = w; z < c.seqs; z += gridDim.x)
    if (decode_span(c, z, a.window, a.sinks).count == 0) {
      for (int d = threadIdx.x; d < a.H * HD; d += DW * 64) a.out[(int64_t)z * a.ldo + d] = 0;
      for (int u = threadIdx.x; u < units; u += DW * 64) a.joins[4 * ((int64_t)z * units + u)] = -1;
    }
  Slot cur;
  cur.b = b0;
  cur.sp = b0 < 0 ? Span{0, 0, 0} : decode_span(c, b0, a.window, a.sinks);
  cur.steps = span_steps(cur.sp, entries);
  if (cur.steps == 0) return;  // no run for this workgroup
  const uint32_t upto = runs.start(w + 1);
  {
    const uint32_t from = runs.start(w);
    const int u = (int)((from - first) / cur.steps);
    const uint32_t unit0 = first + (uint32_t)u * cur.steps;
    cur.kh = u / QG * wide + hw;
    cur.qg = u % QG;
    cur.t = cur.t0 = (int)(from - unit0);
    cur.left = upto - unit0;
    cur.t1 = (int)min((uint32_t)cur.steps, cur.left);
    cur.ok = true;
  }
  int unit_no = 0;  // the run's units so far
  // this lane's entry of a tile: its page (-1: none), looked up two tiles
  // ahead, and its pool row, made when the tile's loads are issued
  auto page_of = [&](const Slot &s) {
    const int i = (s.t * EW + ew) * TK + (lane & 31);
    return s.ok && i < s.sp.count
               ? c.table[(int64_t)s.b * c.ld_table + (span_entry(s.sp, i) >> c.shift)]
               : -1;
  };
  auto row_in = [&](const Slot &s, int page) {
    const int i = span_entry(s.sp, (s.t * EW + ew) * TK + (lane & 31));
    return (uint32_t)page < (uint32_t)c.pages ? (page << c.shift) + (i & ((1 << c.shift) - 1))
                                              : -1;
  };
  auto head_of = [&](const Slot &s) { return s.kh * G + s.qg * QC; };  // its first query head
  auto heads_in = [&](const Slot &s) { return min(QC, G - s.qg * QC); };
  float4 qraw[QS][2];
  auto load_q = [&](const Slot &s) {
    const float *qp =
        a.q + (int64_t)s.b * a.ldq + (int64_t)(n16 < heads_in(s) ? head_of(s) + n16 : 0) * HD + 8 * c4;
#pragma unroll
    for (int i = 0; i < QS; i++) {
      qraw[i][0] = *reinterpret_cast<const float4 *>(qp + 32 * i);
      qraw[i][1] = *reinterpret_cast<const float4 *>(qp + 32 * i + 4);
    }
  };
  half8 kc[2][QS], kn[2][QS];
  auto issue = [&](const Slot &s, int page, int buf, half8 (&k)[2][QS]) -> uint32_t {
    int r = row_in(s, page);
    const uint32_t live = (uint32_t)__ballot(r >= 0);
    if (live == 0) return 0;
    const int some = __builtin_amdgcn_readlane(r, __builtin_ctz(live));
    r = r < 0 ? some : r;
    const int kh = s.kh;
    int ln = lane;  // (opaque: these addresses are made anew, not kept in registers)
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
      const int kr = __shfl(r, 16 * kt + n16, 64);
      const uint16_t *kp = c.k + (int64_t)kr * kvd + kh * HD + 8 * c4;
#pragma unroll
      for (int i = 0; i < QS; i++) k[kt][i] = *reinterpret_cast<const half8 *>(kp + 32 * i);
    }
#pragma unroll
    for (int ii = 0; ii < NI; ii++) {
      const int vr = ii * RPI + ln / KP;
      const int pr = __shfl(r, vr, 64);
      dma16(c.v + (int64_t)pr * kvd + kh * HD + ((ln % KP) ^ swz(vr)) * 8,
            __builtin_amdgcn_readfirstlane(vlds + buf * TILE + ii * 1024));
    }
    return live;
  };
  // the queries as B operands: dims 32 i + 8 c4 .. + 7
  half8 qhi[QS], qlo[QS];
  float scale;
  auto split_q = [&](const Slot &s) {
    const bool mine = n16 < heads_in(s);
    float v[QS][8], big = 0.0f;
#pragma unroll
    for (int i = 0; i < QS; i++) {
      const float4 x = qraw[i][0], y = qraw[i][1];
      const float e8[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; e++) {
        v[i][e] = mine ? e8[e] : 0.0f;
        big = fmaxf(big, fabsf(v[i][e]));
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
    for (int i = 0; i < QS; i++)
#pragma unroll
      for (int e8 = 0; e8 < 8; e8++) {
        const float x = v[i][e8] * up;
        const _Float16 hi = (_Float16)x;
        qhi[i][e8] = hi;
        qlo[i][e8] = (_Float16)(x - (float)hi);
      }
  };
  Slot nxt = cur;
  next_slot(nxt, c, a, QG, hw, entries);
  const int page = page_of(cur);
  int page_nxt = page_of(nxt);
  load_q(cur);
  uint32_t seen = issue(cur, page, 0, kc);
  split_q(cur);
  float m_run = -INFINITY, l_run = 0.0f;
  f4v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) o[dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  for (int buf = 0;; buf ^= 1) {
    Slot far = nxt;
    next_slot(far, c, a, QG, hw, entries);
    // this tile's loads have landed; the other buffer's reads are done
    wait_vm<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
    const uint32_t seen_nxt = issue(nxt, page_nxt, buf ^ 1, kn);
    const int page_far = page_of(far);
    const bool last = cur.last();
    float *scores = nullptr;
    if (a.scores && n16 < heads_in(cur))
      scores = a.scores + ((int64_t)cur.b * a.H + head_of(cur) + n16) * a.ld_scores +
               (cur.t * EW + ew) * TK + 4 * c4;
    if (seen) {
      float sc[2][4], tmax = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; kt++) {
        f4v st = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < QS; i++) {
          st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kt][i], qhi[i], st, 0, 0, 0);
          st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[kt][i], qlo[i], st, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const bool vis = (seen >> (16 * kt + 4 * c4 + i)) & 1;
          sc[kt][i] = vis ? st[i] * scale : -INFINITY;
          tmax = fmaxf(tmax, sc[kt][i]);
        }
      }
      if (scores) {
        *reinterpret_cast<f4v *>(scores) = f4v{sc[0][0], sc[0][1], sc[0][2], sc[0][3]};
        *reinterpret_cast<f4v *>(scores + 16) = f4v{sc[1][0], sc[1][1], sc[1][2], sc[1][3]};
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
      // dims 16 dt + 4 (n16 % 4) .. + 3 of row 16 hh + 4 c4 + n16 / 4: piece 2 dt
      // or the next, dt 32 bytes on before the swizzle, so one xor
      const int vr = 4 * c4 + (n16 >> 2);
      uint32_t va0 = vlds + buf * TILE + vr * ROWB + ((((n16 >> 1) & 1) ^ swz(vr)) * 16) +
                     (n16 & 1) * 8;
      asm volatile("" : "+v"(va0));
#pragma unroll
      for (int dt = 0; dt < DT; dt++) {
        half8 va;
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {  // (swz(r + 16) == swz(r))
          const half4 h4 = __builtin_bit_cast(
              half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                         (__attribute__((address_space(3))) short4v *)((va0 ^ (dt * 32)) +
                                                                       hh * 16 * ROWB)));
#pragma unroll
          for (int e = 0; e < 4; e++) va[4 * hh + e] = h4[e];
        }
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, phi, o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, plo, o[dt], 0, 0, 0);
      }
    } else if (scores) {  // no entry of the tile has a page
      const f4v none = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      *reinterpret_cast<f4v *>(scores) = none;
      *reinterpret_cast<f4v *>(scores + 16) = none;
    }
    if (last) {
      // the sums go through LDS, where those of one KV head's waves meet: lane
      // (query, c4) holds dims 16 dt + 4 c4 .. + 3
      const int GQ = heads_in(cur);
      if (n16 < GQ) {
        float *mw = mrg + (wave * GS + n16) * MS;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f4v *>(mw + 16 * dt + 4 * c4) = o[dt];
        if (c4 == 0) {
          mw[HD] = m_run;
          mw[HD + 1] = l_run;
        }
      }
      if (nxt.ok) load_q(nxt);  // (in flight while the sums meet)
      __builtin_amdgcn_s_waitcnt(0xc07f);
      if (EW > 1) barrier();
      else asm volatile("" ::: "memory");
      const bool whole = cur.t0 == 0 && cur.t1 == cur.steps;
      // each wave's share of its head's values, 4 a lane
      for (int i = ew * 64 + lane; i < GQ * (HD / 4); i += EW * 64) {
        const int g = i / (HD / 4), d = i % (HD / 4) * 4;
        const float *mw = mrg + (hw * GS + g) * MS;
        float mx = -INFINITY, l = 0.0f;
        for (int v = 0; v < EW; v++) mx = fmaxf(mx, mw[v * wide * GS * MS + HD]);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int v = 0; v < EW; v++) {
          const float *p = mw + v * wide * GS * MS;
          const float e = __builtin_amdgcn_exp2f(p[HD] - mu);
          l += p[HD + 1] * e;
          x += *reinterpret_cast<const f4v *>(p + d) * e;
        }
        const int h = head_of(cur) + g;
        if (whole) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          store_half4(a, cur.b, (int64_t)h * HD + d, x * inv);
          if (a.stats && d == 0) {
            float *st = a.stats + ((int64_t)cur.b * a.H + h) * 2;
            st[0] = mu;
            st[1] = inv;
          }
        } else {
          float *pp = a.parts + (((int64_t)(2 * w + (unit_no > 0)) * wide + hw) * GS + g) * MS;
          *reinterpret_cast<f4v *>(pp + d) = x;
          if (d == 0) {
            pp[HD] = mx;
            pp[HD + 1] = l;
          }
        }
      }
      // the run that begins a unit tells the join where its parts are
      if (threadIdx.x == 0 && cur.t0 == 0) {
        const int u = (wide == 4 ? cur.kh >> 2 : wide == 2 ? cur.kh >> 1 : cur.kh) * QG + cur.qg;
        int *jn = a.joins + 4 * ((int64_t)cur.b * units + u);
        jn[0] = whole ? -1 : (int)w;
        jn[1] = unit_no > 0;
        jn[2] = (int)runs.of(upto - cur.left + cur.steps - 1);
      }
      if (!nxt.ok) break;
      unit_no++;
      split_q(nxt);
      m_run = -INFINITY;
      l_run = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; dt++) o[dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
      __builtin_amdgcn_s_waitcnt(0xc07f);
      if (EW > 1) barrier();  // the sums' place is free again
      else asm volatile("" ::: "memory");
    }
    cur = nxt;
    nxt = far;
    page_nxt = page_far;
    seen = seen_nxt;
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
      for (int i = 0; i < QS; i++) kc[kt][i] = kn[kt][i];
  }
}

// The parts of a unit that several runs took, in the runs' order: a workgroup
// a query head (or several, in turn) and 4 COLS of its values, threads over
// those, 4 each, and over stretches of the parts.
constexpr int JT = 256;
template <int HD, int COLS>
__device__ inline void join_head(const DecodeArgs &a, int b, int u, int w0, int second, int n,
                                 int hw, int g, int QG, int GS) {
  typedef float f4v __attribute__((ext_vector_type(4)));
  constexpr int MS = HD + 4, SETS = JT / COLS;
  __shared__ f4v xs[JT];
  __shared__ float ms[JT], ls[JT];
  const int i = threadIdx.x % COLS, set = threadIdx.x / COLS, per = (n + SETS - 1) / SETS;
  const int d = (blockIdx.z * COLS + i) * 4;
  float mx = -INFINITY, l = 0.0f;
  f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
  const int end = min(n, set * per + per);
  for (int p0 = set * per; p0 < end; p0 += 4) {  // 4 parts' loads together
    float m2[4], l2[4];
    f4v y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int p = min(p0 + e, end - 1);
      // a run's first part, or its second where the unit began inside the run
      const float *pp =
          a.parts +
          (((int64_t)(2 * (w0 + p) + (p == 0 ? second : 0)) * a.wide + hw) * GS + g) * MS;
      m2[e] = pp[HD];
      l2[e] = pp[HD + 1];
      y[e] = *reinterpret_cast<const f4v *>(pp + d);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float top = fmaxf(mx, m2[e]), mu = top == -INFINITY ? 0.0f : top;
      const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2[e] - mu);
      if (p0 + e < end) {  // (not 0 times a part that is not finite)
        x = x * e1 + y[e] * e2;
        l = l * e1 + l2[e] * e2;
        mx = top;
      }
    }
  }
  xs[threadIdx.x] = x;
  ms[threadIdx.x] = mx;
  ls[threadIdx.x] = l;
  __syncthreads();
  if (set == 0) {
#pragma unroll
    for (int s = 1; s < SETS; s++) {
      const int j = s * COLS + i;
      const float m2 = ms[j], top = fmaxf(mx, m2), mu = top == -INFINITY ? 0.0f : top;
      const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2 - mu);
      x = x * e1 + xs[j] * e2;
      l = l * e1 + ls[j] * e2;
      mx = top;
    }
    const int h = (u / QG * a.wide + hw) * (a.H / a.KV) + u % QG * QC + g;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store_half4(a, b, (int64_t)h * HD + d, x * inv);
    if (a.stats && d == 0) {
      a.stats[((int64_t)b * a.H + h) * 2] = mx == -INFINITY ? 0.0f : mx;
      a.stats[((int64_t)b * a.H + h) * 2 + 1] = inv;
    }
  }
}
template <int HD, int COLS>
__global__ __launch_bounds__(JT) void paged_join_kernel(const DecodeArgs a, int units) {
  const int *jn = a.joins + 4 * (int64_t)blockIdx.x;
  const int w0 = jn[0], second = jn[1], last = jn[2];
  if (w0 < 0) return;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int G = a.H / a.KV, QG = (G + QC - 1) / QC, GQ = min(QC, G - u % QG * QC);
  for (int i = blockIdx.y; i < a.wide * GQ; i += gridDim.y) {
    join_head<HD, COLS>(a, b, u, w0, second, last - w0 + 1, i / GQ, i % GQ, QG, min(G, QC));
    __syncthreads();
  }
}

// weights[b][entry] += its attention weight, summed over the heads in order:
// 4 entries a lane, 8 heads' scores in flight.
__global__ __launch_bounds__(64) void paged_weights_kernel(const Paged c, const DecodeArgs a,
                                                           float *weights, int ldw) {
  typedef float f4v __attribute__((ext_vector_type(4)));
  const int b = blockIdx.y, t = (blockIdx.x * 64 + threadIdx.x) * 4;
  const Span sp = decode_span(c, b, a.window, a.sinks);
  if (t >= sp.count) return;
  const float *sc = a.scores + (int64_t)b * a.H * a.ld_scores + t;
  const float *st = a.stats + (int64_t)b * a.H * 2;
  float old[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    old[e] = t + e < sp.count ? weights[(int64_t)b * ldw + span_entry(sp, t + e)] : 0.0f;
  f4v w = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int h0 = 0; h0 < a.H; h0 += 8) {
    f4v s[8];
    float m[8], inv[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int h = min(h0 + e, a.H - 1);
      s[e] = *reinterpret_cast<const f4v *>(sc + (int64_t)h * a.ld_scores);
      m[e] = st[2 * h];
      inv[e] = h0 + e < a.H ? st[2 * h + 1] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (h0 + e < a.H)
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] += __builtin_amdgcn_exp2f(s[e][i] - m[e]) * inv[e];
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (t + e < sp.count) weights[(int64_t)b * ldw + span_entry(sp, t + e)] = old[e] + w[e];
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

// KV heads side by side in a workgroup, and units of a sequence.
int decode_wide(int kv_heads) { return kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1; }
int decode_units(const wg_attn_shape *sh) {
  return sh->kv_heads / decode_wide(sh->kv_heads) * ((sh->heads / sh->kv_heads + QC - 1) / QC);
}

// The decode scratch: parts, joins, then (with weights) stats and scores.
struct DecodeScratch {
  size_t parts, joins, stats, scores, end;  // byte offsets
  int64_t ld_scores;
};
DecodeScratch decode_scratch(const wg_paged_cache *c, const wg_attn_shape *sh, bool weights) {
  const int G = sh->heads / sh->kv_heads, wide = decode_wide(sh->kv_heads);
  DecodeScratch d;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  d.parts = 0;
  d.joins = up((size_t)MAX_WORKERS * 2 * wide * (G < QC ? G : QC) * (sh->head_dim + 4) * 4);
  const size_t rows = (size_t)c->sequences * sh->heads;
  d.stats = d.joins + up((size_t)c->sequences * decode_units(sh) * 16);
  d.scores = d.stats + (weights ? up(rows * 8) : 0);
  d.ld_scores = ((int64_t)c->max_entries + DW * TK - 1) / (DW * TK) * (DW * TK);
  d.end = d.scores + (weights ? rows * d.ld_scores * 4 : 0);
  return d;
}

template <int HD>
int launch_decode(const Paged &c, const DecodeArgs &a, const wg_attn_shape *sh, int grid,
                  hipStream_t s) {
  const int G = a.H / a.KV, lds = decode_lds<HD>(G < QC ? G : QC);
  const int rc = raise_lds((const void *)paged_decode_kernel<HD>, lds);
  if (rc) return rc;
  paged_decode_kernel<HD><<<grid, DW * 64, lds, s>>>(c, a);
  if (grid > 1) {
    // a workgroup a unit and query head while those are no more than 4096
    // (most units of many sequences have no parts), and each a quarter or half
    // of the values where they leave compute units idle
    const int units = decode_units(sh), heads = a.wide * (G < QC ? G : QC);
    const int64_t all = (int64_t)c.seqs * units;
    const int y = all * heads <= 4096 ? heads : all >= 4096 ? 1 : (int)(4096 / all);
    if (all * heads <= 256)
      paged_join_kernel<HD, 8><<<dim3((unsigned)all, y, HD / 32), JT, 0, s>>>(a, units);
    else
      paged_join_kernel<HD, HD / 4><<<dim3((unsigned)all, y), JT, 0, s>>>(a, units);
  }
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
                        sh->heads, sh->kv_heads, window, sinks, decode_wide(sh->kv_heads)};
  const Paged c = as_paged(cache);
  hipStream_t s = as_stream(stream);
  // as many runs as the longest sequences could use
  const int64_t most = window > 0 ? (int64_t)window + sinks : cache->max_entries;
  const int64_t entries = most < cache->max_entries ? most : cache->max_entries;
  const int64_t units = (int64_t)cache->sequences * decode_units(sh);
  const int64_t steps = (entries * a.wide + DW * TK - 1) / (DW * TK);
  WG_REQUIRE(units * steps <= 0x7fffffff,
             "wg_paged_attn_decode: %d sequences of %lld entries over %d KV heads (fewer than "
             "2^31 steps)", cache->sequences, (long long)entries, sh->kv_heads);
  const int64_t runs = units * ((steps + MIN_STEPS - 1) / MIN_STEPS);
  const int grid = runs < MAX_WORKERS ? (int)runs : MAX_WORKERS;
  rc = sh->head_dim == 64 ? launch_decode<64>(c, a, sh, grid, s)
                          : launch_decode<128>(c, a, sh, grid, s);
  if (rc || !weights) return rc;
  paged_weights_kernel<<<dim3((unsigned)((entries + 255) / 256), cache->sequences), 64, 0, s>>>(
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
