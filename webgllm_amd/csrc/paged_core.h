// The paged cache's arithmetic, shared by its kernels and compiled by itself
// on the host for its tests: where an entry lies and which entries a row sees.
#pragma once
#include <cstdint>

#ifndef __HIP__
#define __host__
#define __device__
#endif

namespace wg {

// wg_paged_cache as the kernels take it (page_size = 1 << shift).
struct Paged {
  uint16_t *k, *v;
  const int32_t *table, *lens;
  int32_t pages, shift, ld_table, seqs, max_entries;
};

// Entries of sequence b (a length outside [0, max_entries] is cut to it, so
// no table index leaves its row).
__host__ __device__ inline int paged_len(const Paged &c, int b) {
  const int n = c.lens[b];
  return n < 0 ? 0 : n > c.max_entries ? c.max_entries : n;
}

// The pool row of entry i (in [0, max_entries)) of the sequence whose table
// row is `pages_of`, or -1 where the table names no page of the pool.
__host__ __device__ inline int paged_row(const Paged &c, const int32_t *pages_of, int i) {
  const int p = pages_of[i >> c.shift];
  return (uint32_t)p < (uint32_t)c.pages ? (p << c.shift) + (i & ((1 << c.shift) - 1)) : -1;
}

// What rows first .. last (entries of one sequence) see together: the entries
// [0, sinks) and [lo, last], counted through without the gap: index t is
// entry t for t < sinks, else t + gap.
struct Span {
  int sinks, gap, count;
};
__host__ __device__ inline Span paged_span(int first, int last, int window, int sinks) {
  const int lo = window > 0 && first - window + 1 > 0 ? first - window + 1 : 0;
  const int s = sinks < lo ? sinks : lo;
  return {s, lo - s, last + 1 - (lo - s)};
}
__host__ __device__ inline int span_entry(const Span &s, int t) {
  return t < s.sinks ? t : t + s.gap;
}
// Whether entry i's row sees entry j.
__host__ __device__ inline bool paged_sees(int i, int j, int window, int sinks) {
  return j <= i && (window <= 0 || j < sinks || j > i - window);
}

// Rotary positions of several axes (wg_rope_axes): the axis whose position turns
// frequency f. n[a] frequencies are axis a's, one axis after another; or
// interleaved: f is axis f % axes' where f < axes n[f % axes], and axis 0's behind.
struct RopeAxes {
  int axes, interleaved, n[4];
};
__host__ __device__ inline int rope_axis(const RopeAxes &r, int f) {
  if (r.interleaved) {
    const int a = r.axes == 1 ? 0 : r.axes == 2 ? f & 1 : r.axes == 3 ? f % 3 : f & 3;
    const int n = a == 0 ? r.n[0] : a == 1 ? r.n[1] : a == 2 ? r.n[2] : r.n[3];
    return f < r.axes * n ? a : 0;
  }
  const int e0 = r.n[0], e1 = e0 + r.n[1], e2 = e1 + r.n[2];
  return (f >= e0) + (f >= e1) + (f >= e2);  // (axes that there are not have no frequencies)
}

}  // namespace wg
