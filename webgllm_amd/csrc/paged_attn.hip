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

// 4 output halves; 8 bytes at once where they are aligned.
typedef float f4x __attribute__((ext_vector_type(4)));
__device__ inline void store_half4(uint16_t *op, f4x x) {
  if (((uintptr_t)op & 7) == 0) {
    *reinterpret_cast<uint2 *>(op) = make_uint2(half_of(x[0]) | (uint32_t)half_of(x[1]) << 16,
                                                half_of(x[2]) | (uint32_t)half_of(x[3]) << 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) op[e] = half_of(x[e]);
  }
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
// Bound by HBM: 131,000 entries of 8 heads of 128 (537 MB) take 98 us, 5.4 TB/s
// (a pass that only reads as much reaches 6.0), and the join 6; 64 sequences of up
// to 1028 such entries (177 MB) 41 + 6 us, with a new table row, query and part
// every few tiles; 24 of up to 6000 entries of 8 heads of 64 (112 MB), their
// weights summed, 28.5 + 4.7 and 4.8 for the sums. 45 entries: 5.5 us, latency.
constexpr int TK = 32;           // entries a tile
constexpr int DW = 4;            // waves a workgroup
constexpr int MAX_WORKERS = 512; // two a compute unit (768 and 1024: 3 to 4 us more parts)
constexpr int QC = 16;           // query heads a KV head and unit
constexpr int MIN_STEPS = 2;     // steps of a run, where there are so many (1, 4: the same)

// Weights are 2^(score - base), score in log2 units, and a sum of them and of
// weighted values belongs to its base. A score more than BASE_MAX over it moves
// it to BASE_TOP under that score. So the largest weight seen lies between 2^12
// and 2^15 (a half ends at 65504), and what the halves' smallest steps round
// away of a small one is 2^-37 of it at most: the sum over a long cache behind
// one strong entry (131072 of them: 2^-20) is not lost, as it would be with
// weights of 1 and less (2^-8). And the sums are rescaled a few times a row,
// not with each new largest score.
constexpr float BASE_TOP = 12.0f, BASE_MAX = 15.0f;
__device__ inline float base_under(float top) {
  const float b = top - BASE_TOP;
  return top - b > BASE_MAX ? top : b;  // (past 2^26 a float32's steps are 8 and more)
}

struct DecodeArgs {
  const float *q;
  uint16_t *out;
  float *parts;  // [workers][2][wide][group][HD + 4]: values, then maximum and sum
  int *joins;    // [units][4]: first run (-1: finished there, -2: in `whole`), its part, last run,
                 // whether a prefix goes before
  float *stats;  // [sequences][H][2]: maximum (log2) and 1 / sum; or NULL
  float *scores; // [sequences][H][ld_scores], log2; or NULL
  int64_t ld_scores;
  int ldq, ldo, H, KV, window, sinks, wide;
  // behind a shared prefix: each sequence's first entry that is not its group's
  // (or 0), and [sequences][H][HD + 4] for the parts of units inside one run
  const int32_t *first;
  float *whole;
};

// Where a decode run finds a sequence's span: from its length and the window; or,
// behind a shared prefix (the entries that are not its group's), from that first
// entry in memory, or from a table of spans that the workgroup made in LDS. UNITS: as
// WINDOW, but a workgroup's run is one unit, whatever its length.
enum { WINDOW, FIRST, TABLE, UNITS };
struct Spans {
  const int2 *table;  // first entry, count
};
// Entries that sequence b's newest row sees (behind a shared prefix: of its own).
template <int MODE>
__device__ inline Span decode_span(const Paged &c, int b, const DecodeArgs &a, const Spans &sp) {
  if constexpr (MODE == TABLE) {
    const int2 s = sp.table[b];
    return Span{0, s.x, s.y};
  }
  const int n = paged_len(c, b);
  if constexpr (MODE == FIRST) {
    const int f = a.first[b];
    return Span{0, f, n - f};
  }
  return n > 0 ? paged_span(n - 1, n - 1, a.window, a.sinks) : Span{0, 0, 0};
}
// Steps of `entries` entries.
__device__ inline int span_steps(const Span &s, int entries) {
  return (int)((uint32_t)(s.count + entries - 1) / (uint32_t)entries);
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
template <int MODE>
__device__ inline Runs find_run(const Paged &c, const DecodeArgs &a, const Spans &spans,
                                uint32_t units, int entries, uint32_t grid, uint32_t w, int *seq,
                                uint32_t *first) {
  const int lane = threadIdx.x & 63, per = (c.seqs + 63) >> 6;
  uint32_t mine = 0, live = 0;
  for (int i = 0; i < per; i++) {
    const int b = lane * per + i;
    const uint32_t t =
        b < c.seqs ? span_steps(decode_span<MODE>(c, b, a, spans), entries) : 0;
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
        base + wave_scan(in ? span_steps(decode_span<MODE>(c, b, a, spans), entries) : 0);
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
template <int MODE>
__device__ inline void next_slot(Slot &s, const Paged &c, const DecodeArgs &a, const Spans &spans,
                                 int QG, int hw, int entries) {
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
      s.sp = decode_span<MODE>(c, s.b, a, spans);
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
template <int HD, int MODE>
__device__ __forceinline__ void decode_run(const Paged &c, const DecodeArgs &a, const Spans &spans,
                                           uint32_t w, uint32_t grid, unsigned char *smem) {
  constexpr bool BEHIND = MODE == FIRST || MODE == TABLE;
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  typedef short short4v __attribute__((ext_vector_type(4)));
  typedef float f4v __attribute__((ext_vector_type(4)));
  constexpr int KP = HD / 8, ROWB = HD * 2, TILE = TK * ROWB, RPI = 64 / KP, NI = TK / RPI;
  constexpr int QS = HD / 32, DT = HD / 16, MS = HD + 4;
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

  int b0 = w / units;
  uint32_t first = 0;
  Runs runs = {};
  if constexpr (MODE != UNITS)
    runs = find_run<MODE>(c, a, spans, units, entries, grid, w, &b0, &first);
  // rows that see nothing
  for (int z = w; z < c.seqs; z += grid)
    if (decode_span<MODE>(c, z, a, spans).count == 0) {
      for (int d = threadIdx.x; d < a.H * HD; d += DW * 64) a.out[(int64_t)z * a.ldo + d] = 0;
      for (int u = threadIdx.x; MODE != UNITS && u < units; u += DW * 64)
        a.joins[4 * ((int64_t)z * units + u)] = -1;
    }
  Slot cur;
  cur.b = b0;
  cur.sp = b0 < 0 ? Span{0, 0, 0} : decode_span<MODE>(c, b0, a, spans);
  cur.steps = span_steps(cur.sp, entries);
  if (cur.steps == 0) return;  // no run for this workgroup
  const uint32_t upto = MODE == UNITS ? cur.steps : runs.start(w + 1);
  if constexpr (MODE == UNITS) {
    const int u = (int)(w % units);
    cur.kh = u / QG * wide + hw;
    cur.qg = u % QG;
    cur.t = cur.t0 = 0;
    cur.left = cur.t1 = cur.steps;
    cur.ok = true;
  } else {
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
  next_slot<MODE>(nxt, c, a, spans, QG, hw, entries);
  const int page = page_of(cur);
  int page_nxt = page_of(nxt);
  load_q(cur);
  uint32_t seen = issue(cur, page, 0, kc);
  split_q(cur);
  float base = -INFINITY, l_run = 0.0f;
  f4v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++) o[dt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  for (int buf = 0;; buf ^= 1) {
    Slot far = nxt;
    next_slot<MODE>(far, c, a, spans, QG, hw, entries);
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
      if (__ballot(tmax - base > BASE_MAX)) {
        const float to = fmaxf(base, base_under(tmax));
        const float corr = __builtin_amdgcn_exp2f(base - (to == -INFINITY ? 0.0f : to));
        l_run *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] *= corr;
        base = to;
      }
      const float mu = base == -INFINITY ? 0.0f : base;  // (nothing visible yet: weights 0)
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
          mw[HD] = base;
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
        if (whole && !(BEHIND && cur.sp.gap)) {
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          store_half4(a.out + (int64_t)cur.b * a.ldo + (int64_t)h * HD + d, x * inv);
          if (a.stats && d == 0) {
            float *st = a.stats + ((int64_t)cur.b * a.H + h) * 2;
            st[0] = mu;
            st[1] = inv;
          }
        } else {
          float *pp = a.parts + (((int64_t)(2 * w + (unit_no > 0)) * wide + hw) * GS + g) * MS;
          if (BEHIND && whole) pp = a.whole + ((int64_t)cur.b * a.H + h) * MS;
          *reinterpret_cast<f4v *>(pp + d) = x;
          if (d == 0) {
            pp[HD] = mx;
            pp[HD + 1] = l;
          }
        }
      }
      // the run that begins a unit tells the join where its parts are
      if (MODE != UNITS && threadIdx.x == 0 && cur.t0 == 0) {
        const int u = (wide == 4 ? cur.kh >> 2 : wide == 2 ? cur.kh >> 1 : cur.kh) * QG + cur.qg;
        int *jn = a.joins + 4 * ((int64_t)cur.b * units + u);
        jn[0] = !whole ? (int)w : BEHIND && cur.sp.gap ? -2 : -1;
        jn[1] = unit_no > 0;
        jn[2] = (int)runs.of(upto - cur.left + cur.steps - 1);
        if (BEHIND) jn[3] = cur.sp.gap > 0;
      }
      if (!nxt.ok) break;
      unit_no++;
      split_q(nxt);
      base = -INFINITY;
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

template <int HD>
__global__ __launch_bounds__(DW * 64, 2) void paged_decode_kernel(const Paged c,
                                                                 const DecodeArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  decode_run<HD, WINDOW>(c, a, Spans{}, blockIdx.x, gridDim.x, smem);
}

// The same of sequences so short that a workgroup takes each unit: no parts, no join,
// and no sum over the lengths before (3 sequences of up to 104 entries, 14 heads of 64:
// 6.2 us, latency).
template <int HD>
__global__ __launch_bounds__(DW * 64, 2) void paged_decode_units_kernel(const Paged c,
                                                                       const DecodeArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  decode_run<HD, UNITS>(c, a, Spans{}, blockIdx.x, gridDim.x, smem);
}

// Parts p0 .. end - 1 of a query head added in order to x, l and mx, 4 values of
// theirs from d on, U parts' loads together.
template <int HD, int U, typename Part>
__device__ inline void add_parts(int p0, int end, int d, Part part, f4x &x, float &l, float &mx) {
  for (; p0 < end; p0 += U) {
    float m2[U], l2[U];
    f4x y[U];
#pragma unroll
    for (int e = 0; e < U; e++) {
      const float *pp = part(min(p0 + e, end - 1));
      m2[e] = pp[HD];
      l2[e] = pp[HD + 1];
      y[e] = *reinterpret_cast<const f4x *>(pp + d);
    }
#pragma unroll
    for (int e = 0; e < U; e++) {
      const float top = fmaxf(mx, m2[e]), mu = top == -INFINITY ? 0.0f : top;
      const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2[e] - mu);
      if (p0 + e < end) {  // (not 0 times a part that is not finite)
        x = x * e1 + y[e] * e2;
        l = l * e1 + l2[e] * e2;
        mx = top;
      }
    }
  }
}

// The parts of one query head, in order: NT threads (a workgroup, or a wave) over
// 4 COLS of its values, 4 each, and over stretches of the n parts, which meet in
// LDS. part(p) is part
// p's values, maximum and sum. On the first COLS threads x is the head's values
// from d on, mx its maximum (log2) and inv 1 / its sum.
constexpr int JT = 256;
template <int HD, int COLS, int NT = JT, typename Part>
__device__ inline void join_parts(int n, int d, Part part, f4x *x_out, float *mx_out,
                                  float *inv_out) {
  constexpr int SETS = NT / COLS;
  const int i = threadIdx.x % COLS, set = threadIdx.x % NT / COLS, per = (n + SETS - 1) / SETS;
  float mx = -INFINITY, l = 0.0f;
  f4x x = {0.0f, 0.0f, 0.0f, 0.0f};
  add_parts<HD, 4>(set * per, min(n, set * per + per), d, part, x, l, mx);
  // one sum into another: both sides of an exchange take the same two, so every
  // lane of a column ends with the same bits
  auto add = [&](float m2, float l2, f4x y) {
    const float top = fmaxf(mx, m2), mu = top == -INFINITY ? 0.0f : top;
    const float e1 = __builtin_amdgcn_exp2f(mx - mu), e2 = __builtin_amdgcn_exp2f(m2 - mu);
    x = x * e1 + y * e2;
    l = l * e1 + l2 * e2;
    mx = top;
  };
#pragma unroll
  for (int o = COLS; o < 64; o *= 2) {  // the wave's stretches
    const float m2 = __shfl_xor(mx, o, 64), l2 = __shfl_xor(l, o, 64);
    f4x y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = __shfl_xor(x[e], o, 64);
    add(m2, l2, y);
  }
  if constexpr (NT > 64) {
    __shared__ f4x xs[NT / 64 * COLS];
    __shared__ float ms[NT / 64 * COLS], ls[NT / 64 * COLS];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < COLS) {
      xs[wave * COLS + i] = x;
      ms[wave * COLS + i] = mx;
      ls[wave * COLS + i] = l;
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int v = 1; v < NT / 64; v++) add(ms[v * COLS + i], ls[v * COLS + i], xs[v * COLS + i]);
    }
    __syncthreads();
  }
  *x_out = x;
  *mx_out = mx == -INFINITY ? 0.0f : mx;
  *inv_out = l == 0.0f ? 0.0f : 1.0f / l;
}
// A workgroup a unit and query head (or several, in turn) that several runs
// took, and 4 COLS of its values.
template <int HD, int COLS>
__global__ __launch_bounds__(JT) void paged_join_kernel(const DecodeArgs a, int units) {
  constexpr int MS = HD + 4;
  const int *jn = a.joins + 4 * (int64_t)blockIdx.x;
  const int w0 = jn[0], second = jn[1], last = jn[2];
  if (w0 < 0) return;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int G = a.H / a.KV, QG = (G + QC - 1) / QC, GS = min(G, QC), GQ = min(QC, G - u % QG * QC);
  const int d = (blockIdx.z * COLS + threadIdx.x % COLS) * 4;
  for (int i = blockIdx.y; i < a.wide * GQ; i += gridDim.y) {
    const int hw = i / GQ, g = i % GQ, h = (u / QG * a.wide + hw) * G + u % QG * QC + g;
    f4x x;
    float mx, inv;
    // a run's first part, or its second where the unit began inside the run
    join_parts<HD, COLS>(
        last - w0 + 1, d,
        [&](int p) {
          return a.parts +
                 (((int64_t)(2 * (w0 + p) + (p == 0 ? second : 0)) * a.wide + hw) * GS + g) * MS;
        },
        &x, &mx, &inv);
    if (threadIdx.x < COLS) {
      store_half4(a.out + (int64_t)b * a.ldo + (int64_t)h * HD + d, x * inv);
      if (a.stats && d == 0) {
        a.stats[((int64_t)b * a.H + h) * 2] = mx;
        a.stats[((int64_t)b * a.H + h) * 2 + 1] = inv;
      }
    }
  }
}

// weights[b][entry] += its attention weight, summed over the heads in order: 4
// entries a lane, the heads in WW stretches, a wave each with 8 heads' scores in
// flight, whose sums meet in LDS in order.
constexpr int WW = 4;
__global__ __launch_bounds__(WW * 64) void paged_weights_kernel(const Paged c, const DecodeArgs a,
                                                                float *weights, int ldw) {
  __shared__ f4x part[WW - 1][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y, t = (blockIdx.x * 64 + lane) * 4;
  const Span sp = decode_span<WINDOW>(c, b, a, Spans{});
  if ((int)blockIdx.x * 256 >= sp.count) return;
  const float *sc = a.scores + (int64_t)b * a.H * a.ld_scores + t;
  const float *st = a.stats + (int64_t)b * a.H * 2;
  const int per = (a.H + WW - 1) / WW, h1 = min(a.H, (wave + 1) * per);
  float old[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    old[e] = wave == 0 && t + e < sp.count ? weights[(int64_t)b * ldw + span_entry(sp, t + e)] : 0.0f;
  f4x w = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int h0 = wave * per; h0 < h1; h0 += 8) {
    f4x s[8];
    float m[8], inv[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int h = min(h0 + e, h1 - 1);
      s[e] = f4x{0.0f, 0.0f, 0.0f, 0.0f};
      if (t < sp.count) s[e] = *reinterpret_cast<const f4x *>(sc + (int64_t)h * a.ld_scores);
      m[e] = st[2 * h];
      inv[e] = st[2 * h + 1];
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (h0 + e < h1)
#pragma unroll
        for (int i = 0; i < 4; i++)  // (no page: -inf, and nothing, of a sum that is not finite too)
          w[i] += s[e][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[e][i] - m[e]) * inv[e];
  }
  if (wave > 0) part[wave - 1][lane] = w;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int v = 0; v < WW - 1; v++) w += part[v][lane];
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (t + e < sp.count) weights[(int64_t)b * ldw + span_entry(sp, t + e)] = old[e] + w[e];
}

// ---------------------------------------------------------------- prompts
//
// A workgroup takes R rows of one sequence (QW waves of 32 queries: rows x the
// KV head's query heads) and one KV head, and walks what those rows see
// together, the first entries and then the window's, KEYS at a time:
//  - scores as S^T = K Q^T on v_mfma_f32_32x32x16_f16: A = 32 keys of the tile,
//    B = the wave's queries, each scaled by a power of two to the top of the
//    halves and split into hi = half(q) and lo = half(q - hi): scores keep 22
//    bits of any finite query. Lane i holds 16 keys of query i % 32 (keys
//    8 (j / 4) + 4 (i / 32) + j % 4 of the tile), so the softmax runs in the
//    lane, plus one exchange between the half-waves;
//  - weighted values as O^T = V^T P^T: B = the lane's own weights, split alike
//    (the upper 11 bits by a mask, then half(the rest): 21 bits; split by a
//    rounding and what it leaves, 253 us where the mask takes 247), A = the values
//    of those keys by transposing LDS loads. One half a weight (11 bits) would
//    take 199 us (2048 rows of 32 heads of 128 under a window of 4096) and leave
//    an error of the size of the half output's own rounding.
// Tiles come by direct-to-LDS loads one step ahead, their pages looked up two
// ahead. KW groups of QW waves take the steps in turn where queries alone leave
// compute units idle, their sums merged in LDS, and beyond that `splits`
// workgroups share a block's steps, as many as its own length is worth, and leave
// parts for paged_part_join_kernel (and their number, beside the first).
// Entries of no page, or past the last, read the step's first entry that has
// one and weigh nothing. What a row does not see is a bit mask over the step, in
// the steps at the ends of what the rows see alone. A wave's softmax goes before
// another's products on the same SIMD (s_setprio), so that the matrix cores have
// both waves' products to fill up with (with one half a weight 193 us instead of
// 205; products first: 205).
// Bound by the matrix cores and the vector units in turn, which overlap little:
// 2048 rows of 32 heads of 128 under a window of 4096 take 237 to 252 us by card
// (58 and 48 % of the cycles), 1.1 PFLOP/s with the products of the low halves,
// 0.55 to 0.58 without; a large matrix product reaches 1.3. Tried against it and
// slower (with one half a weight, 222 us then): 8 waves whose halves take products
// and softmax in turn between barriers (262 us), the next step's products under
// this step's softmax in one wave a SIMD (307). 7 prompts of 33 to 1500 rows of 14
// heads of 64 behind up to 900 entries take 33 us, some 4 of each workgroup's time
// before its first tile is there; 5 rows behind 6000 entries 9.5 us and 3 in the
// join.
struct PromptArgs {
  const float *q;
  const int32_t *row_start;
  uint16_t *out;
  float *parts;  // [M][H][splits][HD + 4] where splits > 1
  int ldq, ldo, M, H, KV, window, sinks, R, blocks, splits;
  const int32_t *group_start, *shared;  // a shared prefix's groups and their entries
  int groups;
};
// What of its rows' entries a prompt kernel takes: all; the ones that a group of
// sequences shares (for all the group's rows at once); the ones behind those.
enum { ALL, PREFIX, OWN };

// Entries that sequences s0 .. s1 - 1 share: one sequence alone nothing, where decode
// runs cut its entries evenly with the others'; of prompt blocks (rows) there are as
// many shares of a prefix as of its own entries or more (32 sequences of 4 rows, two
// of them alone in their group behind 8000 entries: 86 us instead of 111).
__device__ inline int group_entries(const Paged &c, int s0, int s1, int shared, bool rows) {
  return min(s1, c.seqs) - max(s0, 0) < (rows ? 1 : 2) ? 0 : min(max(shared, 0), c.max_entries);
}
// The first entry of a sequence of len entries and so many rows that is not its
// group's: 0 where the shared ones do not end before its rows.
__device__ inline int own_first(int shared, int len, int rows) {
  return len - max(rows, 1) >= shared ? shared : 0;
}

// How many shares so many entries are worth. Each costs a part of every query,
// written and read, which few rows (of one wave of queries) feel less, and the
// launch that joins them some 3 us: 5 rows behind 3000 entries take 12 us in 7
// shares, 28 in one; 256 rows (heads of 64) behind 3000 entries 31 us in 4
// shares, 43 in one, behind 1000 entries 19.1 us in 2, 20.5 in one.
__host__ __device__ inline int64_t shares_of(int64_t entries, int qw, bool joined = false) {
  if (joined) return entries < 256 ? 1 : entries / 128;  // (behind a prefix there is a join anyway)
  const int64_t n = entries / (qw == 1 ? 256 : 512);
  return n < (qw == 1 ? 3 : 5) ? 1 : n;
}

// Whether BYTES in LDS hold a half that is not finite: 0 times it is not 0.
template <int BYTES>
__device__ inline bool any_not_finite(const unsigned char *tile) {
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  half2v sum[4] = {};
#pragma unroll 4
  for (int i = 0; i < BYTES / 1024; i++) {
    const uint4 x = *reinterpret_cast<const uint4 *>(tile + i * 1024 + (threadIdx.x & 63) * 16);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
      sum[e] = __builtin_elementwise_fma(__builtin_bit_cast(half2v, w[e]), half2v{}, sum[e]);
  }
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) any |= __builtin_bit_cast(uint32_t, sum[e]);
  return __ballot(any != 0) != 0;
}
// 0x8000 in each half of x that is not finite, else 0.
__device__ inline uint32_t not_finite(uint32_t x) {
  return ((x & 0x7c007c00) + 0x04000400) & 0x80008000;
}

// (block: of R rows and a KV head, the last rows first; share: of its entries)
template <int HD, int QW, int KW, int KT, int PART>
__device__ __forceinline__ void prompt_block(const Paged &c, const PromptArgs &a, uint32_t block,
                                             uint32_t share_no, unsigned char *smem) {
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef _Float16 half4 __attribute__((ext_vector_type(4)));
  typedef short short4v __attribute__((ext_vector_type(4)));
  typedef float f4v __attribute__((ext_vector_type(4)));
  typedef float float16v __attribute__((ext_vector_type(16)));
  constexpr int KEYS = 32 * KT;  // a step's
  constexpr int KP = HD / 8, ROWB = HD * 2, TILE = KEYS * ROWB, RPI = 64 / KP, NI = KEYS / RPI;
  constexpr int KS = HD / 16, DT = HD / 32;
  constexpr int LPW = NI / QW;  // loads (1 KB) of keys a wave issues a step, and of values
  static_assert(LPW * QW == NI, "loads split evenly");
  constexpr int MERGE = 64 * (16 * DT + 2) * 4;  // bytes a merged wave leaves
  static_assert((KW - 1) * QW * MERGE <= KW * 4 * TILE, "merge area");
  // smem: [KW][2 buffers][K tile, V tile]
  auto swz = [](int r) { return KP == 16 ? (r & 15) : ((r >> 1) & 7); };
  // V rows: 4 rows' 4 neighbouring pieces, which a transposing load takes at
  // once, land on 16 distinct bank groups
  auto swzv = [](int r) {
    return (KP == 16 ? (r & 3) << 2 : (r & 2) << 1) | ((r >> 2) & 3);
  };
  // the last rows, which see the most, first
  const int kh = block % a.KV;
  int blk = a.blocks - 1 - block / a.KV;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = wave % QW, kg = wave / QW;
  const int hh = lane >> 5, c32 = lane & 31, n16 = lane & 15;
  const int G = a.H / a.KV, kvd = a.KV * HD;
  // Blocks of R rows: those of sequence b are numbered from row_start[b] / R + b
  // on, which leaves each at least as many as it needs, so that a workgroup finds
  // its sequence without a sum over the ones before.
  auto block0 = [&](int first, int b) { return min(max(first, 0), a.M) / a.R + b; };
  int r0, r1, len, b;
  float own_entries = 0.0f;  // (PREFIX) behind the prefixes, of all sequences, about
  if constexpr (PART == PREFIX) {  // b: the group's first sequence that sees the prefix
    auto row0 = [&](int g) {
      const int s = min(max(a.group_start[g], 0), c.seqs);
      return a.row_start ? a.row_start[s] : s;
    };
    const int g = find_segment(
        a.groups, blk,
        [&](int at, bool whole, int *first, int *end, int *shared) {
          *first = row0(at);
          if (whole) {
            *end = row0(at + 1);
            *shared = group_entries(c, a.group_start[at], a.group_start[at + 1], a.shared[at],
                                    a.row_start != nullptr);
          }
        },
        block0, &r0, &r1, &len);
    if (g < 0 || len == 0) return;
    const int s1 = min(a.group_start[g + 1], c.seqs);
    b = -1;  // (an empty one's table row may name no pages)
    int seen = 0;
    float entries = 0.0f;  // of their own, of `seen` sequences (up to 256 or so)
    for (int s = max(a.group_start[g], 0); s < s1 && (b < 0 || seen < 192); s += 64) {
      const int i = s + lane, n = i < s1 ? paged_len(c, i) : 0;
      const bool in =
          i < s1 && own_first(len, n, a.row_start ? a.row_start[i + 1] - a.row_start[i] : 1) > 0;
      const uint64_t sees = __ballot(in);
      if (sees && b < 0) b = s + __ffsll((unsigned long long)sees) - 1;
      entries += in ? (float)(n - len) : 0.0f;
      seen += __popcll(sees);
    }
    if (b < 0) return;
    own_entries = wave_sum_u(entries) / seen * c.seqs;
    blk -= block0(r0, g);
  } else {
    b = find_last(c, a.row_start, blk, block0, &r0, &r1, &len);
    if (b < 0) return;
    blk -= block0(r0, b);
  }
  const int m_end = min(r1, a.M), m0 = max(r0, 0) + blk * a.R;
  if (m0 >= m_end || blk < 0) return;  // (under 0: starts that do not ascend)
  const int m_last = min(m0 + a.R, m_end) - 1;
  // row m's entry (where the group shares it: behind what it sees, all of it)
  auto entry = [&](int m) { return PART == PREFIX ? len - 1 : len - r1 + m; };
  const int32_t *pages = c.table + (int64_t)b * c.ld_table;
  int own = 0;
  if constexpr (PART == OWN) {
    int s0, s1, shared;
    const int g = find_segment(
        a.groups, b,
        [&](int at, bool whole, int *first, int *end, int *more) {
          *first = a.group_start[at];
          if (whole) {
            *end = a.group_start[at + 1];
            *more = group_entries(c, *first, *end, a.shared[at], true);
          }
        },
        [](int first, int) { return first; }, &s0, &s1, &shared);
    if (g >= 0 && b < s1) own = own_first(shared, len, r1 - r0);
  }
  const Span sp = entry(m_last) < 0 ? Span{0, 0, 0}
                  : PART == OWN
                      ? Span{0, own, entry(m_last) + 1 - own}
                      : paged_span(max(entry(m0), 0), entry(m_last), a.window, a.sinks);
  // this lane's query (slot qs): row qm, entry qe
  const int qs = wq * 32 + c32;
  const int qm = m0 + qs / G;
  const bool qvalid = qs < G * a.R && qm <= m_last;
  const int qe = entry(qm);
  // the wave's first and last row's entries
  const bool w_any = m0 + wq * 32 / G <= m_last && wq * 32 < G * a.R;
  const int w_first = entry(m0 + wq * 32 / G);
  const int w_last = entry(min(m0 + min(wq * 32 + 31, G * a.R - 1) / G, m_last));
  // the span's indexes that the query sees: under q_end, and from q_first on or sinks
  const int q_end = qe < 0 ? 0 : (qe < sp.sinks ? qe : qe - sp.gap) + 1;
  const int q_first = a.window > 0 && qe >= a.window ? max(qe - a.window + 1 - sp.gap, 0) : 0;
  const uint32_t all = (sp.count + KEYS - 1) / KEYS;  // the block's steps; this workgroup's:
  // (all < 2^25 and at most 64 splits: 32 bits hold it)
  uint32_t splits = min((uint32_t)a.splits, (uint32_t)shares_of((int64_t)all * KEYS, QW, PART != ALL));
  // Half of a prefix's shares, one workgroup a compute unit beside one that takes own
  // entries, where those last (us at 3.9 TB/s) half as long as it would (1.6 a step),
  // or shares are short
  if (PART == PREFIX && splits > 1) {
    const float halves = 8.0f + 1.6f * (float)all / (float)(splits / 2 * KW);
    const float others = 6.0f + own_entries * (float)(a.KV * HD * 4) * (1.0f / 3.9e6f);
    if (all * KEYS < 512 * splits || 2.0f * others > halves) splits /= 2;
  }
  if (share_no >= splits) return;
  const int s0 = splits == 1 ? 0 : (int)(all * share_no / splits);
  const int s1 = splits == 1 ? all : (int)(all * (share_no + 1) / splits);
  unsigned char *tiles = smem + kg * 4 * TILE;
  const uint32_t sbase = (uint32_t)(uintptr_t)smem + kg * 4 * TILE;
  auto page_of = [&](int s) {
    const int t = s * KEYS + (lane & (KEYS - 1));
    return s < s1 && t < sp.count ? pages[span_entry(sp, t) >> c.shift] : -1;
  };
  const int kr0 = wq * RPI + lane / KP;
  const int kcol = kh * HD + ((lane % KP) ^ swz(kr0)) * 8;
  const int vcol = kh * HD + ((lane % KP) ^ swzv(kr0)) * 8;
  // step s's loads into buffer buf: the mask of its entries that have a page
  auto issue = [&](int s, int page, int buf) -> uint64_t {
    const int i = span_entry(sp, s * KEYS + (lane & (KEYS - 1)));
    int r = (uint32_t)page < (uint32_t)c.pages ? (page << c.shift) + (i & ((1 << c.shift) - 1))
                                               : -1;
    uint64_t live = __ballot(r >= 0);
    if constexpr (KEYS == 32) live &= 0xffffffffu;
    if (live == 0) return 0;
    const int some = __builtin_amdgcn_readlane(r, __builtin_ctzll(live));
    r = r < 0 ? some : r;
    // each of the wave's loads takes RPI rows, this lane's kr0 past a multiple
    // of the group's; the swizzles are bit selections, so of those rows apart
    int pr[LPW];
#pragma unroll
    for (int l = 0; l < LPW; l++) pr[l] = __shfl(r, kr0 + l * QW * RPI, 64);
#pragma unroll
    for (int l = 0; l < LPW; l++)
      dma16(c.k + (int64_t)pr[l] * kvd + (kcol ^ swz(l * QW * RPI) * 8),
            __builtin_amdgcn_readfirstlane(sbase + buf * 2 * TILE + (l * QW + wq) * 1024));
#pragma unroll
    for (int l = 0; l < LPW; l++)
      dma16(c.v + (int64_t)pr[l] * kvd + (vcol ^ swzv(l * QW * RPI) * 8),
            __builtin_amdgcn_readfirstlane(sbase + buf * 2 * TILE + TILE + (l * QW + wq) * 1024));
    return live;
  };
  const int iters = (s1 - s0 + KW - 1) / KW;  // of every group
  uint64_t live = 0, live_nxt = 0;
  const int page0 = page_of(s0 + kg);
  int page = page_of(s0 + kg + KW);
  if (s0 + kg < s1) live = issue(s0 + kg, page0, 0);
  half8 qb_hi[KS], qb_lo[KS];
  float scale;  // of a query's raw scores, to log2
  {
    const float *qp =
        a.q + (int64_t)(qvalid ? qm : m0) * a.ldq + (int64_t)(kh * G + qs % G) * HD + 8 * hh;
    float v[KS][8], big = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const float4 x = *reinterpret_cast<const float4 *>(qp + 16 * ks);
      const float4 y = *reinterpret_cast<const float4 *>(qp + 16 * ks + 4);
      const float e8[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int t = 0; t < 8; t++) {
        v[ks][t] = qvalid ? e8[t] : 0.0f;
        big = fmaxf(big, fabsf(v[ks][t]));
      }
    }
    big = fmaxf(big, xor32(big));
    // 2^k with big 2^k in [2^13, 2^14); an exponent that float32 holds both ways
    const int e = big > 0.0f && big < INFINITY ? ilogbf(big) : 13;
    const int k = min(max(13 - e, -114), 100);
    const float up = ldexpf(1.0f, k);
    scale = ldexpf(1.44269504088896340736f, -k);
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int t = 0; t < 8; t++) {
        const float x = v[ks][t] * up;
        const _Float16 hi = (_Float16)x;
        qb_hi[ks][t] = hi;
        qb_lo[ks][t] = (_Float16)(x - (float)hi);
      }
  }
  float base = -INFINITY, l_run = 0.0f;
  float16v o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int j = 0; j < 16; j++) o[dt][j] = 0.0f;
  // The value tile at `at`, step s's, without what is not finite: first every wave
  // marks its queries' sums, a key at a time, then the group's waves clear it.
  auto mend_tile = [&](int s, int at) {
    unsigned char *v = tiles + at;
    for (int key = 0; key < (s < s1 ? KEYS : 0); key++) {
      const bool sees = ((live >> key) & 1) &&
                        paged_sees(qe, span_entry(sp, s * KEYS + key), a.window, a.sinks);
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) {  // dims 32 dt + 8 j + 4 hh .. + 3
          const uint2 x = *reinterpret_cast<const uint2 *>(
              v + key * ROWB + (((4 * dt + j) ^ swzv(key)) * 16) + 8 * hh);
          const uint32_t n[2] = {sees ? not_finite(x.x) : 0, sees ? not_finite(x.y) : 0};
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (n[e >> 1] & (e & 1 ? 0x80000000 : 0x8000)) o[dt][4 * j + e] = __builtin_nanf("");
        }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    if constexpr (QW > 1) barrier();
    else asm volatile("" ::: "memory");
    for (int i = wq; i < TILE / 1024; i += QW) {
      uint4 *x = reinterpret_cast<uint4 *>(v + i * 1024 + lane * 16);
      x->x &= ~((not_finite(x->x) >> 15) * 0xffff);
      x->y &= ~((not_finite(x->y) >> 15) * 0xffff);
      x->z &= ~((not_finite(x->z) >> 15) * 0xffff);
      x->w &= ~((not_finite(x->w) >> 15) * 0xffff);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    if constexpr (QW > 1) barrier();
    else asm volatile("" ::: "memory");
  };
  const int vrow0 = 4 * hh + (n16 >> 2);  // + 32 kt + 16 sl + 8 t: a transposing load's row
  for (int it = 0; it < iters; it++, live = live_nxt) {
    const int s = s0 + it * KW + kg, t0 = s * KEYS;
    // this step's loads have landed, and every wave of the group is done
    // with the other buffer
    wait_vm<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);
    if constexpr (QW > 1) barrier();
    else asm volatile("" ::: "memory");
    live_nxt = s + KW < s1 ? issue(s + KW, page, (it + 1) & 1) : 0;
    page = page_of(s + 2 * KW);
    // An entry that a query does not see has a weight of 0, but 0 times a value
    // that is not finite is NaN. Where not all of the block's rows see all of the
    // workgroup's steps, such values make NaN of the sums of the queries that see
    // them here, and are 0 in the tile from then on. (5 rows behind 6000 entries
    // take 12.6 us with it, 12.1 without; large chunks the same.)
    if constexpr (PART != PREFIX) {
      const int ta = (s - kg) * KEYS, tb = min(min(ta + KW * KEYS, s1 * KEYS), sp.count) - 1;
      const int lo = span_entry(sp, ta), hi = span_entry(sp, tb);
      if (hi > entry(m0) || (a.window > 0 && hi >= a.sinks && lo <= entry(m_last) - a.window)) {
        bool bad = false;  // in any group's tile: the same for all waves, which meet below
#pragma unroll
        for (int g = 0; g < (QW > 1 ? KW : 1); g++)  // (a group without a step: what LDS held)
          if ((QW == 1 ? s : s - kg + g) < s1)
            bad |= any_not_finite<TILE>((QW > 1 ? smem + g * 4 * TILE : tiles) + (it & 1) * 2 * TILE +
                                      TILE);
        if (__builtin_expect(bad, 0)) mend_tile(s, (it & 1) * 2 * TILE + TILE);
      }
    }
    if (s >= s1 || live == 0 || !w_any) continue;  // wave-uniform
    const int j_lo = span_entry(sp, t0), j_hi = span_entry(sp, min(t0 + KEYS, sp.count) - 1);
    if (j_lo > w_last ||
        (a.window > 0 && j_lo >= a.sinks && j_hi <= w_first - a.window))
      continue;  // none of the wave's rows sees any of it
    const unsigned char *kt0 = tiles + (it & 1) * 2 * TILE, *vt0 = kt0 + TILE;
    float16v st[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int j = 0; j < 16; j++) st[kt][j] = 0.0f;
    half8 ka[2][KT];
    auto kread = [&](int ks) {
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        const int r = 32 * kt + c32;
        ka[ks & 1][kt] = *reinterpret_cast<const half8 *>(kt0 + r * ROWB +
                                                          (((2 * ks + hh) ^ swz(r)) * 16));
      }
    };
    __builtin_amdgcn_s_setprio(0);  // (products give way to the other wave's softmax)
    kread(0);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      if (ks + 1 < KS) kread(ks + 1);  // under this slice's products
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kt = 0; kt < KT; kt++)
        st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[ks & 1][kt], qb_hi[ks], st[kt], 0, 0, 0);
#pragma unroll
      for (int kt = 0; kt < KT; kt++)
        st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka[ks & 1][kt], qb_lo[ks], st[kt], 0, 0, 0);
    }
    __builtin_amdgcn_s_setprio(1);
    const bool full = KEYS == 32 ? live == 0xffffffffu : live == ~0ull;
    if (!full || j_hi > w_first ||
        (a.window > 0 && j_hi >= a.sinks && j_lo <= w_last - a.window)) {  // wave-uniform
      asm volatile("" ::: "memory");  // (stays a branch, not selects for every score)
      auto below = [&](int t) {  // the step's entries under index t, a bit each
        const int n = t - t0;
        return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
      };
      const uint64_t vis =
          (live & below(q_end) & (~below(q_first) | below(a.sinks))) >> (4 * hh);
#pragma unroll
      for (int kt = 0; kt < KT; kt++) {
        const int v = (int)(uint32_t)(vis >> (32 * kt));
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const int all = v << (31 - (8 * (j >> 2) + (j & 3))) >> 31;  // the bit, over the word
          st[kt][j] = __int_as_float((__float_as_int(st[kt][j]) & all) | (0xff800000 & ~all));
        }
      }
    }
    float tmax = st[0][0];
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int j = 0; j < 16; j++) tmax = fmaxf(tmax, st[kt][j]);
    tmax = fmaxf(tmax, xor32(tmax));
    tmax *= scale;
    if (__ballot(tmax - base > BASE_MAX)) {
      const float to = fmaxf(base, base_under(tmax));
      const float corr = __builtin_amdgcn_exp2f(base - (to == -INFINITY ? 0.0f : to));
      l_run *= corr;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[dt][j] *= corr;
      base = to;
    }
    const float mu = base == -INFINITY ? 0.0f : base;  // (nothing visible yet: weights 0)
    float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int j = 0; j < 16; j++) {
        st[kt][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][j], scale, -mu));
        ps[j & 3] += st[kt][j];
      }
    float psum = (ps[0] + ps[1]) + (ps[2] + ps[3]);
    psum += xor32(psum);
    l_run += psum;
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
      for (int sl = 0; sl < 2; sl++) {
        half8 phi, plo;
#pragma unroll
        for (int t = 0; t < 8; t++) {
          const float p = st[kt][8 * sl + t];
          const float hi = __int_as_float(__float_as_int(p) & 0xffffe000);  // (a half's bits)
          phi[t] = (_Float16)hi;
          plo[t] = (_Float16)(p - hi);
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
          half8 va;
#pragma unroll
          for (int t2 = 0; t2 < 2; t2++) {
            // source lane n16 of each 16: row vrow0, dims 32 dt + 16 (their
            // half of 32) + 4 (n16 % 4) .. + 3; it receives dim 32 dt + c32
            // of 4 rows
            const int r = 32 * kt + 16 * sl + 8 * t2 + vrow0;
            const int col = 32 * dt + (lane & 16) + 4 * (n16 & 3);
            const unsigned char *at = vt0 + r * ROWB + (((col >> 3) ^ swzv(r)) * 16) + (col & 7) * 2;
            const half4 h4 = __builtin_bit_cast(
                half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) short4v *)(uint32_t)(uintptr_t)at));
#pragma unroll
            for (int e = 0; e < 4; e++) va[4 * t2 + e] = h4[e];
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, phi, o[dt], 0, 0, 0);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, plo, o[dt], 0, 0, 0);
        }
      }
  }
  wait_vm<0>();
  if constexpr (KW > 1) {  // the groups' sums meet in LDS, over the tiles
    const int groups = min(KW, s1 - s0);  // that had steps (uniform)
    auto part = [&](int g) {
      return reinterpret_cast<float *>(smem) + ((g - 1) * QW + wq) * (MERGE / 4);
    };
    if (groups > 1) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      barrier();
      if (kg > 0 && kg < groups) {
        float *w = part(kg);
        w[lane] = base;
        w[64 + lane] = l_run;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            *reinterpret_cast<f4v *>(w + 128 + ((4 * dt + j) * 64 + lane) * 4) =
                f4v{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);
      barrier();
    }
    if (kg > 0) return;
    for (int g = 1; g < groups; g++) {
      const float *w = part(g);
      const float m2 = w[lane], mx = fmaxf(base, m2);
      const float mu = mx == -INFINITY ? 0.0f : mx;
      const float a1 = __builtin_amdgcn_exp2f(base - mu), a2 = __builtin_amdgcn_exp2f(m2 - mu);
      l_run = l_run * a1 + w[64 + lane] * a2;
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const f4v v = *reinterpret_cast<const f4v *>(w + 128 + ((4 * dt + j) * 64 + lane) * 4);
#pragma unroll
          for (int e = 0; e < 4; e++) o[dt][4 * j + e] = o[dt][4 * j + e] * a1 + v[e] * a2;
        }
      base = mx;
    }
  }
  if (!qvalid) return;
  const int h = kh * G + qs % G;
  if (PART != ALL || a.splits > 1) {
    float *pp = a.parts + (((int64_t)qm * a.H + h) * a.splits + share_no) * (HD + 4);
    if (hh == 0 && share_no == 0) {
      pp[HD + 2] = __int_as_float((int)splits);
      if (PART == OWN) pp[HD + 3] = __int_as_float(own);
    }
    if (splits > 1 || PART == PREFIX || own) {
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          *reinterpret_cast<f4v *>(pp + 32 * dt + 8 * j + 4 * hh) =
              f4v{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
      if (hh == 0) {
        pp[HD] = base;
        pp[HD + 1] = l_run;
      }
      return;
    }
  }
  const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int j = 0; j < 4; j++)
      store_half4(a.out + (int64_t)qm * a.ldo + (int64_t)h * HD + 32 * dt + 8 * j + 4 * hh,
                  f4x{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]} * inv);
}

template <int HD, int QW, int KW, int KT>
__global__ __launch_bounds__(QW * KW * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_prompt_kernel(const Paged c, const PromptArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  prompt_block<HD, QW, KW, KT, ALL>(c, a, blockIdx.x, blockIdx.y, smem);
}

// The parts of a row's query heads, where there are any: a workgroup each, or
// (many rows, of few parts) HD / 4 threads each.
template <int HD, bool MANY>
__global__ __launch_bounds__(JT) void paged_part_join_kernel(const PromptArgs a, int seqs) {
  constexpr int COLS = HD / 4, MS = HD + 4, PER = MANY ? JT / COLS : 1;
  const int64_t i = (int64_t)blockIdx.x * PER + (MANY ? threadIdx.x / COLS : 0);
  if (i >= (int64_t)a.M * a.H) return;
  const int m = (int)(i / a.H), h = (int)(i - (int64_t)m * a.H), d = threadIdx.x % COLS * 4;
  const float *pp = a.parts + i * a.splits * MS;
  const int n = min(__float_as_int(pp[HD + 2]), a.splits);
  if (m < a.row_start[0] || m >= a.row_start[seqs]) return;  // (of no sequence: nothing there)
  if (n <= 1) return;                                        // (one share: written already)
  f4x x = {0.0f, 0.0f, 0.0f, 0.0f};
  float mx = -INFINITY, inv, l = 0.0f;
  auto part = [&](int p) { return pp + p * MS; };
  if constexpr (MANY) {
    add_parts<HD, 4>(0, n, d, part, x, l, mx);
    inv = l == 0.0f ? 0.0f : 1.0f / l;
  } else {
    join_parts<HD, COLS>(n, d, part, &x, &mx, &inv);
    if (threadIdx.x >= COLS) return;
  }
  store_half4(a.out + (int64_t)m * a.ldo + (int64_t)h * HD + d, x * inv);
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

// Workgroups for sequences of up to `entries` seen entries.
int decode_grid(const char *who, const wg_paged_cache *c, const wg_attn_shape *sh, int64_t entries,
                int *grid) {
  const int64_t units = (int64_t)c->sequences * decode_units(sh);
  const int64_t steps = (entries * decode_wide(sh->kv_heads) + DW * TK - 1) / (DW * TK);
  WG_REQUIRE(units * steps <= 0x7fffffff,
             "%s: %d sequences of %lld entries over %d KV heads (fewer than 2^31 steps)", who,
             c->sequences, (long long)entries, sh->kv_heads);
  WG_REQUIRE(units <= MAX_GROUPS, "%s: %d sequences of %d KV heads", who, c->sequences, sh->kv_heads);
  const int64_t runs = units * ((steps + MIN_STEPS - 1) / MIN_STEPS);
  *grid = runs < MAX_WORKERS ? (int)runs : MAX_WORKERS;
  return WG_OK;
}

template <int HD>
int launch_units(const Paged &c, const DecodeArgs &a, unsigned grid, hipStream_t s) {
  const int G = a.H / a.KV, lds = decode_lds<HD>(G < QC ? G : QC);
  if (lds > 64 * 1024) {
    const int rc = raise_lds((const void *)paged_decode_units_kernel<HD>, lds);
    if (rc) return rc;
  }
  paged_decode_units_kernel<HD><<<grid, DW * 64, lds, s>>>(c, a);
  return launched("wg_paged_attn_shared");
}

template <int HD>
int launch_decode(const char *who, const Paged &c, const DecodeArgs &a, const wg_attn_shape *sh,
                  int grid, hipStream_t s) {
  const int G = a.H / a.KV, lds = decode_lds<HD>(G < QC ? G : QC);
  if (lds > 64 * 1024) {  // (half a microsecond of the host's)
    const int rc = raise_lds((const void *)paged_decode_kernel<HD>, lds);
    if (rc) return rc;
  }
  paged_decode_kernel<HD><<<grid, DW * 64, lds, s>>>(c, a);
  if (grid > 1) {
    // a workgroup a unit and query head while those are no more than 4096
    // (most units of many sequences have no parts), and each a quarter or half
    // of the values where they leave compute units idle (131,000 entries: 103.7
    // us instead of 108.9, 8000: 15.0 instead of 17.6)
    const int units = decode_units(sh), heads = a.wide * (G < QC ? G : QC);
    const int64_t all = (int64_t)c.seqs * units;
    const int y = all * heads <= 4096 ? heads : all >= 4096 ? 1 : (int)(4096 / all);
    if (all * heads <= 256)
      paged_join_kernel<HD, 8><<<dim3((unsigned)all, y, HD / 32), JT, 0, s>>>(a, units);
    else
      paged_join_kernel<HD, HD / 4><<<dim3((unsigned)all, y), JT, 0, s>>>(a, units);
  }
  return launched(who);
}

// The prompt kernel's shape for M rows: waves of queries and of keys, and how
// many workgroups share a block's entries.
struct PromptPlan {
  int qw, kw, R;
  int64_t blocks;  // of R rows, at most
  int splits;
};
PromptPlan prompt_plan(const wg_paged_cache *c, const wg_attn_shape *sh, int64_t M) {
  const int G = sh->heads / sh->kv_heads;
  // blocks over all KV heads, for so many waves of queries: about (each sequence's
  // last is half full)
  auto groups = [&](int qw) {
    const int R = qw * 32 / G;
    return sh->kv_heads * ((M + R - 1) / R + c->sequences / 2);
  };
  // Few blocks: groups of waves on the keys. One sequence's rows of 32 query and 8
  // KV heads behind (fresh, 3000, 16000) entries, in us, of shapes (waves of queries
  // x groups of keys):
  //   heads of 64, 128 rows (64 blocks of 2): 1x4 7.0, 23, 64, 2x2 7.4, 25, 55;
  //     512 rows: 1x4 10.6, 46, 197, 2x2 11.8, 46, 168; 1024: 25, 90, 384, 20, 77, 320;
  //     2000 rows: 2x2 52, 160, 637, 4x1 54, 153, 599; 2500 (1250 blocks): 75, 216,
  //     824, 72, 247, 903; 3500: 134, 327, 1173, 124, 312, 1146
  //   heads of 128, 128 rows: 1x4 9.6, 30, 103, 2x2 10.2, 37, 86; 256 (128 blocks):
  //     11, 45, 184, 13, 47, 153; 512: 22, 88, 367, 19, 76, 288;
  //     1024 rows: 2x2 36, 134, 555, 4x1 41, 131, 496; 1536 (768 blocks): 56, 227,
  //     949, 66, 206, 807; 2000: 85, 279, 1108, 87, 257, 981
  // The lines stand between what fresh and what deep rows want: behind 16,000
  // entries the shape of more queries wins well before them.
  PromptPlan p;
  const int64_t two = groups(2);
  if (two < (sh->head_dim == 64 ? 64 : 128)) p.qw = 1, p.kw = 4;
  else if (two < (sh->head_dim == 64 ? 1200 : 768)) p.qw = 2, p.kw = 2;
  else p.qw = 4, p.kw = 1;
  p.R = p.qw * 32 / G;
  p.blocks = (M - 1) / p.R + c->sequences;  // (block0's last, at most, and one)
  // shares that fill the workgroups which run at once (LDS holds one or two a
  // compute unit)
  const int64_t fill = (sh->head_dim == 128 && p.qw == 1 ? 256 : 512) / groups(p.qw);
  const int64_t most = shares_of(c->max_entries, p.qw);
  const int64_t s = fill < most ? fill : most;
  p.splits = s < 1 ? 1 : s > 64 ? 64 : (int)s;
  return p;
}

template <int HD, int QW, int KW, int KT>
constexpr int PROMPT_LDS = KW * 4 * 32 * KT * HD * 2;

template <int HD, int QW, int KW, int KT>
int launch_prompt(const char *who, const Paged &c, const PromptArgs &a, hipStream_t s) {
  constexpr int LDS = PROMPT_LDS<HD, QW, KW, KT>;
  if (LDS > 64 * 1024) {
    const int rc = raise_lds((const void *)paged_prompt_kernel<HD, QW, KW, KT>, LDS);
    if (rc) return rc;
  }
  paged_prompt_kernel<HD, QW, KW, KT>
      <<<dim3((unsigned)a.blocks * a.KV, a.splits), QW * KW * 64, LDS, s>>>(c, a);
  if (a.splits > 1) {
    // a workgroup a head while those are few (5 rows of 32 heads behind 6000
    // entries: 12.1 us instead of 16.2 by HD / 4 threads; 96 rows: 29.3, 27.6)
    const int64_t heads = (int64_t)a.M * a.H, per = JT / (HD / 4);
    if (heads <= 2048)
      paged_part_join_kernel<HD, false><<<(unsigned)heads, JT, 0, s>>>(a, c.seqs);
    else
      paged_part_join_kernel<HD, true><<<(unsigned)((heads + per - 1) / per), JT, 0, s>>>(a, c.seqs);
  }
  return launched(who);
}

// -------------------------------------------------------- a shared prefix
//
// Softmax over a union of entries from the parts' running maxima m, sums l and
// weighted values o: with mu = max m, (sum o 2^(m - mu)) / (sum l 2^(m - mu)). What
// a group of sequences shares is read once for all its rows (prompt blocks over the
// group's queries), what each has of its own by the decode kernel's runs (one row a
// sequence) or prompt blocks, and a row's parts are joined in order, the prefix's
// first.
// The prefix is bound by the matrix cores where a group has many rows: 32 sequences
// of 32 query and 8 KV heads of 128 behind 100,000 entries (425 MB, 105 GFLOP with
// the low halves' products) take 133 us; two workgroups a compute unit run 64 queries
// by 64 entries in 2.1 us, 1.0 PFLOP/s (a large matrix product reaches 1.2), one
// alone in 1.6. Else by what a workgroup does besides, 8 us: the group and its
// first rows 1.3, its span 1.3, queries 3, merge and write 2. 64 sequences of up to
// 2000 entries behind 6000 (160 MB) take 47 us, 45 of 32 heads of 64 in five groups
// (55 MB) 27, 16 of 4 to 9 rows behind 8000 54; and the join 4 to 7. (The decode
// kernel over all entries, us a call in a graph, shared and not: 64 sequences behind
// 4096 entries 31, 99; behind 16,384 62, 315; 8 behind 4096 20, 29.)

// Sequence b's first own entry, its group among the starts by halves.
__device__ inline int first_of(const Paged &c, int b, const int32_t *group_start,
                               const int32_t *shared, int groups) {
  int lo = 0, hi = groups;  // the last group that begins at b or before it: lo - 1
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (group_start[mid] <= b) lo = mid + 1;
    else hi = mid;
  }
  if (lo == 0 || b >= group_start[lo]) return 0;
  return own_first(group_entries(c, group_start[lo - 1], group_start[lo], shared[lo - 1], false),
                   paged_len(c, b), 1);
}
// The sequences' first own entries into memory, where they are more than a table
// in LDS takes.
__global__ __launch_bounds__(256) void paged_first_kernel(const Paged c, const int32_t *group_start,
                                                          const int32_t *shared, int groups,
                                                          int32_t *first) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < c.seqs) first[b] = first_of(c, b, group_start, shared, groups);
}
constexpr int SPANS = 512;  // sequences of a table

// Both at once: the first `owns` workgroups take the sequences' own entries (the
// decode kernel's runs, or prompt blocks), the others the groups' prefixes, so that
// memory and the matrix cores work beside each other (64 sequences behind 6000
// entries 53 us, 67 by a launch each; rows of several tokens behind 8000 72, 78).
// Runs are as many as there are compute units, which leaves each a place for a
// prefix's workgroup (384 and 512 runs were no faster, nor were the prefixes first)
// where LDS holds two: heads of 64; of 128 with up to 5 query heads a KV head, or 6 and
// 7 and some 460 and 200 sequences. With more, the prefixes wait for runs to end (64
// sequences of up to 1000 entries behind 6000, 8 KV heads of 128, us a call in a graph,
// shared and not: 32 query heads 43, 148; 48 53, 151; 64 76, 195; 128 107, 203).
template <int HD, int QW, int KW, int KT, bool DECODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_shared_kernel(const Paged c, const PromptArgs pre, const PromptArgs own,
                         const DecodeArgs a, uint32_t owns, uint32_t table) {
  extern __shared__ __align__(1024) unsigned char smem[];
  if (blockIdx.x >= owns) {
    const uint32_t i = blockIdx.x - owns, blocks = (uint32_t)pre.blocks * pre.KV;
    prompt_block<HD, QW, KW, KT, PREFIX>(c, pre, i % blocks, i / blocks, smem);
  } else if constexpr (DECODE) {
    if (table == 0) {
      decode_run<HD, FIRST>(c, a, Spans{}, blockIdx.x, owns, smem);
      return;
    }
    // the groups where the tiles come later, the spans behind
    int32_t *starts = reinterpret_cast<int32_t *>(smem), *shared = starts + SPANS + 1;
    int2 *spans = reinterpret_cast<int2 *>(smem + table);
    for (int g = threadIdx.x; g <= pre.groups; g += 256) {
      starts[g] = pre.group_start[g];
      if (g < pre.groups) shared[g] = pre.shared[g];
    }
    __syncthreads();
    for (int b = threadIdx.x; b < c.seqs; b += 256) {
      const int f = first_of(c, b, starts, shared, pre.groups);
      spans[b] = make_int2(f, paged_len(c, b) - f);
    }
    __syncthreads();
    decode_run<HD, TABLE>(c, a, Spans{spans}, blockIdx.x, owns, smem);
  } else {
    const uint32_t blocks = (uint32_t)own.blocks * own.KV;
    prompt_block<HD, QW, KW, KT, OWN>(c, own, blockIdx.x % blocks, blockIdx.x / blocks, smem);
  }
}

// A workgroup (or, MANY, a wave) a row and query head: the prefix's parts, then its
// own.
template <int HD, bool DECODE, bool MANY>
__global__ __launch_bounds__(JT) void paged_shared_join_kernel(const PromptArgs pre,
                                                               const PromptArgs own,
                                                               const DecodeArgs a, int seqs) {
  constexpr int MS = HD + 4, COLS = HD / 4;
  const int64_t i = MANY ? (int64_t)blockIdx.x * (JT / 64) +
                               __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                         : blockIdx.x;
  if (MANY && i >= (int64_t)pre.M * pre.H) return;
  const int m = (int)(i / pre.H), h = (int)(i - (int64_t)m * pre.H);
  const int d = threadIdx.x % COLS * 4;
  const float *p1 = pre.parts + i * pre.splits * MS, *p2;
  int n1 = __float_as_int(p1[HD + 2]), n2, w0 = 0, second = 0, hw = 0, g = 0, GS = 0;
  bool behind;
  if constexpr (DECODE) {
    const int G = a.H / a.KV, QG = (G + QC - 1) / QC, units = a.KV / a.wide * QG;
    const int kh = h / G, qg = h % G / QC;
    const int4 jn = *reinterpret_cast<const int4 *>(
        a.joins + 4 * ((int64_t)m * units + kh / a.wide * QG + qg));
    w0 = jn.x, second = jn.y;
    if (w0 == -1) return;
    behind = jn.w > 0;
    n2 = w0 == -2 ? 1 : jn.z - w0 + 1;
    p2 = w0 == -2 ? a.whole + i * MS : a.parts;
    hw = kh % a.wide, g = h % G % QC, GS = min(G, QC);
  } else {
    if (m < own.row_start[0] || m >= own.row_start[seqs]) return;  // (of no sequence)
    p2 = own.parts + i * own.splits * MS;
    n2 = min(__float_as_int(p2[HD + 2]), own.splits);
    behind = __float_as_int(p2[HD + 3]) > 0;
    if (!behind && n2 <= 1) return;  // (written already)
  }
  n1 = behind ? min(max(n1, 0), pre.splits) : 0;
  f4x x;
  float mx, inv;
  join_parts<HD, COLS, MANY ? 64 : JT>(
      n1 + n2, d,
      [&](int p) {
        if (p < n1) return p1 + p * MS;
        p -= n1;
        if (!DECODE || w0 == -2) return p2 + p * MS;
        return p2 + (((int64_t)(2 * (w0 + p) + (p == 0 ? second : 0)) * a.wide + hw) * GS + g) * MS;
      },
      &x, &mx, &inv);
  if (threadIdx.x % (MANY ? 64 : JT) >= COLS) return;
  store_half4((DECODE ? a.out : own.out) + (int64_t)m * pre.ldo + (int64_t)h * HD + d, x * inv);
}

// The shapes of both kinds of blocks (waves of queries; all of one call alike) and
// how many workgroups share a block's entries.
struct SharedPlan {
  int qw, R;
  int64_t pre_blocks, own_blocks;  // of R rows, at most
  int pre_splits, own_splits;
};
SharedPlan shared_plan(const wg_paged_cache *c, const wg_attn_shape *sh, int64_t M, int groups) {
  const int G = sh->heads / sh->kv_heads;
  SharedPlan p;
  p.qw = sh->head_dim == 64 && M * G <= 32 * (int64_t)groups ? 1 : 2;
  p.R = p.qw * 32 / G;
  p.pre_blocks = (M - 1) / p.R + groups;
  p.own_blocks = (M - 1) / p.R + c->sequences;
  const int64_t most = shares_of(c->max_entries, p.qw, true);
  auto splits = [&](int64_t segments) {
    const int64_t fill = 512 / (sh->kv_heads * ((M + p.R - 1) / p.R + segments / 2));
    const int64_t s = fill < most ? fill : most;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
  };
  p.pre_splits = splits(groups);
  p.own_splits = splits(c->sequences);
  return p;
}

// Whether rows of several tokens run as a prompt that shares nothing: where a
// sequence's queries fill a block of 64 by themselves, its keys and values are read
// once for them anyway, and a short prefix is not worth the join. Us a call, shared
// and as prompts, of 8 sequences of R rows behind P entries (32 query and 8 KV heads
// of 128): P 1000, R 2 to 32: 19, 15; 20, 24; 22, 19; 30, 21; 39, 31; P 8000: 26, 50;
// 32, 59; 45, 53; 59, 90; 96, 96; 64 rows: 170, 213; of 32 sequences in 4 groups,
// P 1000: 27, 29; 30, 30; 48, 31; 63, 41; P 8000: 78, 139; 108, 119; 124, 181; 237,
// 224; 455, 426. (Rows are counted on the device alone, so this goes by the average: 63
// sequences of a row beside one of 500 rows behind 6000 entries 194, 325; beside one of
// 1000, which runs all as prompts, 456, as two calls 56 and 222.)
bool as_prompt(const wg_paged_cache *c, const wg_attn_shape *sh, int64_t M) {
  return M * (sh->heads / sh->kv_heads) > 64 * (int64_t)c->sequences || c->max_entries < 2048;
}

// Whether a row a sequence runs by a workgroup a unit, without parts and a join: where
// the longest unit is no more than 7 steps, or 5 of 128 dims. Us a call in a graph, so
// and as below, of 3 and 200 sequences, by steps: 32 query and 8 KV heads of 128: 3 10.2,
// 14.2 and 13, 22; 4 11.5, 14.1 and 16, 23; 6 15, 14 and 22, 23; 14 and 2 of 64: 2 6.0,
// 8.8 and 6.5, 10.3; 4 8.2, 10.4 and 8.7, 16; 7 11.2, 11.5 and 12, 16; 13 17, 11 and 18,
// 16; 32 and 8 of 64: 3 6.9, 11.1 and 8.6, 15; 6 9.9, 11.1 and 13.5, 18.
bool by_units(const wg_paged_cache *c, const wg_attn_shape *sh) {
  const int64_t entries = DW * TK / decode_wide(sh->kv_heads);  // of a step
  return c->max_entries <= entries * (sh->head_dim == 64 ? 7 : 5);
}
// Whether a row a sequence runs as wg_paged_attn_decode, which reads a prefix once a
// sequence: where all that the sequences may hold is so few bytes that a launch and
// its join take longest. Us a call in a graph, shared and not, of so many MB: 32 query
// and 8 KV heads of 128: 7 MB 15.1, 14.2; 25 15.8, 14.5; 27 15.4, 16.0; 38 19.4, 15.6;
// 44 18.1, 18.5; 55 19.8, 18.6; 78 19.2, 21.6; 14 and 2 of 64: 1 MB 12.9, 11.6; 22
// 15.7, 14.0; 36 15.6, 15.7; 55 16.7, 18.4; 32 and 8 of 64: 9 MB 12.8, 11.6; 29 15.1,
// 12.6; 39 14.0, 15.4; 55 15.9, 16.0; 75 16.4, 18.5.
bool as_decode(const wg_paged_cache *c, const wg_attn_shape *sh) {
  return (double)c->sequences * c->max_entries * sh->kv_heads * sh->head_dim * 4 <= 32 << 20;
}

// Scratch of a call of M rows: each sequence's first own entry, the prefix's
// parts, then the decode kernel's scratch and whole parts, or the parts of the
// rows' own entries.
struct SharedScratch {
  size_t first, prefix, own, whole, end;
};
SharedScratch shared_scratch(const wg_paged_cache *c, const wg_attn_shape *sh, int64_t M,
                             const SharedPlan &p, bool decode) {
  SharedScratch d;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  const size_t part = (size_t)M * sh->heads * (sh->head_dim + 4) * 4;
  d.first = 0;
  d.prefix = up((size_t)c->sequences * 4);
  d.own = d.prefix + up(part * p.pre_splits);
  d.whole = d.own + (decode ? up(decode_scratch(c, sh, false).end) : up(part * p.own_splits));
  d.end = d.whole + (decode ? up(part) : 0);
  return d;
}

template <int HD, int QW, int KW, int KT, bool DECODE>
int launch_shared(const Paged &c, const PromptArgs &pre, const PromptArgs &own, const DecodeArgs &a,
                  int grid, hipStream_t s) {
  const int G = pre.H / pre.KV;
  int lds = PROMPT_LDS<HD, QW, KW, KT>, table = 0;
  if (DECODE) {
    int own_lds = decode_lds<HD>(G < QC ? G : QC);
    if (c.seqs <= SPANS) {
      table = own_lds;
      own_lds += c.seqs * 8;
    } else {
      paged_first_kernel<<<(c.seqs + 255) / 256, 256, 0, s>>>(c, pre.group_start, pre.shared,
                                                              pre.groups, (int32_t *)a.first);
    }
    if (own_lds > lds) lds = own_lds;
  }
  if (lds > 64 * 1024) {
    const int rc = raise_lds((const void *)paged_shared_kernel<HD, QW, KW, KT, DECODE>, lds);
    if (rc) return rc;
  }
  const unsigned owns = DECODE ? grid : (unsigned)own.blocks * own.KV * own.splits;
  const unsigned all = owns + (unsigned)pre.blocks * pre.KV * pre.splits;
  paged_shared_kernel<HD, QW, KW, KT, DECODE><<<all, 256, lds, s>>>(c, pre, own, a, owns, table);
  const unsigned heads = (unsigned)((int64_t)pre.M * pre.H);
  // a wave a head where those are many (us, by a workgroup each and by a wave: 6400
  // heads 12.8, 6.4; 3200: 7.8, 7.2; 2048 of few parts 5.3, 4.0; 1440: 5.3, 4.9;
  // 1024: 7.1, 7.9; 512 of many parts 6.7, 10.1)
  if (heads >= 1280)
    paged_shared_join_kernel<HD, DECODE, true><<<(heads + 3) / 4, JT, 0, s>>>(pre, own, a, c.seqs);
  else
    paged_shared_join_kernel<HD, DECODE, false><<<heads, JT, 0, s>>>(pre, own, a, c.seqs);
  return launched("wg_paged_attn_shared");
}

// wg_paged_attn_decode and wg_paged_attn_prefill, also under the name of a call that
// runs as one of them.
int attn_decode(const char *who, const float *q, int32_t ldq, const wg_attn_shape *sh,
                const wg_paged_cache *cache, int32_t window, int32_t sinks, float *weights,
                int32_t ld_weights, uint16_t *out, int32_t ldo, void *scratch,
                size_t scratch_bytes, void *stream) {
  int rc = check_attn(q, cache ? cache->sequences : 0, ldq, sh, cache, window, sinks, out, ldo, 64,
                      who);
  if (rc) return rc;
  if (window >= cache->max_entries) window = 0;  // (hides nothing)
  const DecodeScratch d = decode_scratch(cache, sh, weights != nullptr);
  WG_REQUIRE(scratch && scratch_bytes >= d.end && ((uintptr_t)scratch & 15) == 0,
             "%s: scratch of %zu bytes, needs %zu (16-byte aligned)", who, scratch_bytes, d.end);
  WG_REQUIRE(!weights || ld_weights >= cache->max_entries,
             "%s: weights of %d entries a sequence of up to %d", who, ld_weights,
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
  int grid;
  rc = decode_grid(who, cache, sh, entries, &grid);
  if (rc) return rc;
  rc = sh->head_dim == 64 ? launch_decode<64>(who, c, a, sh, grid, s)
                          : launch_decode<128>(who, c, a, sh, grid, s);
  if (rc || !weights) return rc;
  paged_weights_kernel<<<dim3((unsigned)((entries + 255) / 256), cache->sequences), WW * 64, 0,
                         s>>>(c, a, weights, ld_weights);
  return launched(who);
}

size_t prompt_scratch(const PromptPlan &p, const wg_attn_shape *sh, int64_t M) {
  return p.splits > 1 ? (size_t)M * sh->heads * p.splits * (sh->head_dim + 4) * 4 : 0;
}
int attn_prompt(const char *who, const float *q, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                const wg_paged_cache *cache, const int32_t *row_start, int32_t window,
                int32_t sinks, uint16_t *out, int32_t ldo, void *scratch, size_t scratch_bytes,
                void *stream) {
  int rc = check_attn(q, M, ldq, sh, cache, window, sinks, out, ldo, 32, who);
  if (rc) return rc;
  WG_REQUIRE(row_start, "%s: null row_start", who);
  if (window >= cache->max_entries) window = 0;  // (hides nothing)
  PromptPlan p = prompt_plan(cache, sh, M);
  const size_t need = prompt_scratch(p, sh, M);
  WG_REQUIRE(scratch_bytes >= need && (!need || (scratch && ((uintptr_t)scratch & 15) == 0)),
             "%s: scratch of %zu bytes, needs %zu (16-byte aligned)", who, scratch_bytes, need);
  // a block sees no more than its rows, a window and the sinks
  const int64_t seen = window > 0 ? (int64_t)window + sinks + p.R : cache->max_entries;
  const int64_t most = shares_of(seen, p.qw);
  if (p.splits > most) p.splits = (int)most;
  WG_REQUIRE(p.blocks * sh->kv_heads <= MAX_GROUPS, "%s: %d rows", who, M);
  const PromptArgs a = {q, row_start, out, (float *)scratch, ldq, ldo, M, sh->heads, sh->kv_heads,
                        window, sinks, p.R, (int)p.blocks, p.splits};
  const Paged c = as_paged(cache);
  hipStream_t s = as_stream(stream);
  if (sh->head_dim == 64)
    return p.qw == 1   ? launch_prompt<64, 1, 4, 1>(who, c, a, s)
           : p.qw == 4 ? launch_prompt<64, 4, 1, 2>(who, c, a, s)
                       : launch_prompt<64, 2, 2, 2>(who, c, a, s);
  return p.qw == 1   ? launch_prompt<128, 1, 4, 1>(who, c, a, s)
         : p.qw == 4 ? launch_prompt<128, 4, 1, 2>(who, c, a, s)
                     : launch_prompt<128, 2, 2, 1>(who, c, a, s);
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
  return attn_decode("wg_paged_attn_decode", q, ldq, sh, cache, window, sinks, weights, ld_weights,
                     out, ldo, scratch, scratch_bytes, stream);
}

size_t wg_paged_prefill_scratch_bytes(const wg_paged_cache *c, const wg_attn_shape *sh,
                                      int32_t M) {
  if (!c || !sh || M < 1 || c->sequences < 1 || sh->kv_heads < 1 ||
      sh->heads < sh->kv_heads || sh->heads / sh->kv_heads > 32 || c->max_entries < 1)
    return 0;
  return prompt_scratch(prompt_plan(c, sh, M), sh, M);
}

int wg_paged_attn_prefill(const float *q, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                          const wg_paged_cache *cache, const int32_t *row_start, int32_t window,
                          int32_t sinks, uint16_t *out, int32_t ldo, void *scratch,
                          size_t scratch_bytes, void *stream) {
  return attn_prompt("wg_paged_attn_prefill", q, M, ldq, sh, cache, row_start, window, sinks, out,
                     ldo, scratch, scratch_bytes, stream);
}

size_t wg_paged_shared_scratch_bytes(const wg_paged_cache *c, const wg_attn_shape *sh, int32_t M,
                                     int32_t groups) {
  if (!c || !sh || M < 1 || groups < 1 || c->sequences < 1 || sh->kv_heads < 1 ||
      sh->heads < sh->kv_heads || sh->heads / sh->kv_heads > 32 || c->max_entries < 1)
    return 0;
  const SharedPlan p = shared_plan(c, sh, M, groups);
  const size_t rows = as_prompt(c, sh, M) ? wg_paged_prefill_scratch_bytes(c, sh, M)
                                          : shared_scratch(c, sh, M, p, false).end;
  const size_t one = M != c->sequences   ? 0
                     : by_units(c, sh) || as_decode(c, sh) ? decode_scratch(c, sh, false).end
                                                           : shared_scratch(c, sh, M, p, true).end;
  return rows > one ? rows : one;
}

int wg_paged_attn_shared(const float *q, int32_t M, int32_t ldq, const wg_attn_shape *sh,
                         const wg_paged_cache *cache, const int32_t *row_start,
                         const int32_t *group_start, const int32_t *shared, int32_t groups,
                         uint16_t *out, int32_t ldo, void *scratch, size_t scratch_bytes,
                         void *stream) {
  const char *who = "wg_paged_attn_shared";
  int rc = check_attn(q, M, ldq, sh, cache, 0, 0, out, ldo, 32, who);
  if (rc) return rc;
  WG_REQUIRE(group_start && shared, "wg_paged_attn_shared: null argument");
  WG_REQUIRE(groups >= 1 && groups <= cache->sequences,
             "wg_paged_attn_shared: %d groups of %d sequences", groups, cache->sequences);
  WG_REQUIRE(row_start || M == cache->sequences, "wg_paged_attn_shared: %d rows for %d sequences",
             M, cache->sequences);
  const bool decode = !row_start;
  if (!decode && as_prompt(cache, sh, M))
    return attn_prompt(who, q, M, ldq, sh, cache, row_start, 0, 0, out, ldo, scratch,
                       scratch_bytes, stream);
  if (decode && by_units(cache, sh)) {
    // (as of caches somewhat longer, though nothing is written: scratch is asked for by
    // one rule, which wg_paged_shared_scratch_bytes states)
    const size_t need = decode_scratch(cache, sh, false).end;
    WG_REQUIRE(scratch && scratch_bytes >= need && ((uintptr_t)scratch & 15) == 0,
               "wg_paged_attn_shared: scratch of %zu bytes, needs %zu (16-byte aligned)",
               scratch_bytes, need);
    DecodeArgs a = {};
    a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo, a.H = sh->heads, a.KV = sh->kv_heads;
    a.wide = decode_wide(sh->kv_heads);
    const int64_t grid = (int64_t)cache->sequences * decode_units(sh);
    WG_REQUIRE(grid <= MAX_GROUPS, "wg_paged_attn_shared: %d rows of %d heads", M, sh->heads);
    return sh->head_dim == 64
               ? launch_units<64>(as_paged(cache), a, (unsigned)grid, as_stream(stream))
               : launch_units<128>(as_paged(cache), a, (unsigned)grid, as_stream(stream));
  }
  if (decode && as_decode(cache, sh))
    return attn_decode(who, q, ldq, sh, cache, 0, 0, nullptr, 0, out, ldo, scratch, scratch_bytes,
                       stream);
  const SharedPlan p = shared_plan(cache, sh, M, groups);
  const SharedScratch d = shared_scratch(cache, sh, M, p, decode);
  WG_REQUIRE(scratch && scratch_bytes >= d.end && ((uintptr_t)scratch & 15) == 0,
             "wg_paged_attn_shared: scratch of %zu bytes, needs %zu (16-byte aligned)",
             scratch_bytes, d.end);
  int grid = 0;
  if (decode) {
    rc = decode_grid("wg_paged_attn_shared", cache, sh, cache->max_entries, &grid);
    if (rc) return rc;
    if (grid > 256) grid = 256;
  }
  const int64_t owns = decode ? grid : p.own_blocks * p.own_splits * sh->kv_heads;
  WG_REQUIRE(owns + p.pre_blocks * p.pre_splits * sh->kv_heads <= MAX_GROUPS &&
                 ((int64_t)M * sh->heads + 3) / 4 <= MAX_GROUPS,
             "wg_paged_attn_shared: %d rows of %d heads", M, sh->heads);
  unsigned char *m = (unsigned char *)scratch;
  const Paged c = as_paged(cache);
  hipStream_t s = as_stream(stream);
  int32_t *first = (int32_t *)(m + d.first);
  const PromptArgs pre = {q, row_start, out, (float *)(m + d.prefix), ldq, ldo, M, sh->heads,
                          sh->kv_heads, 0, 0, p.R, (int)p.pre_blocks, p.pre_splits, group_start,
                          shared, groups};
  PromptArgs own = pre;
  own.parts = (float *)(m + d.own);
  own.blocks = (int)p.own_blocks, own.splits = p.own_splits;
  DecodeArgs a = {};
  if (decode) {
    const DecodeScratch ds = decode_scratch(cache, sh, false);
    unsigned char *o = m + d.own;
    a = {q, out, (float *)(o + ds.parts), (int *)(o + ds.joins), nullptr, nullptr, 0, ldq, ldo,
         sh->heads, sh->kv_heads, 0, 0, decode_wide(sh->kv_heads), first, (float *)(m + d.whole)};
  }
  if (sh->head_dim == 64) {
    if (p.qw == 1)
      return decode ? launch_shared<64, 1, 4, 1, true>(c, pre, own, a, grid, s)
                    : launch_shared<64, 1, 4, 1, false>(c, pre, own, a, grid, s);
    return decode ? launch_shared<64, 2, 2, 2, true>(c, pre, own, a, grid, s)
                  : launch_shared<64, 2, 2, 2, false>(c, pre, own, a, grid, s);
  }
  return decode ? launch_shared<128, 2, 2, 1, true>(c, pre, own, a, grid, s)
                : launch_shared<128, 2, 2, 1, false>(c, pre, own, a, grid, s);
}

}  // extern "C"
