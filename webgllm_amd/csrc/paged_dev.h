// What the paged cache's kernels share on the device and in their checks.
#pragma once

#include "common.h"
#include "paged_core.h"

namespace wg {

// A cache descriptor's checks (0, or a status with the message set); kvd
// values an entry. `lens` is read only where the caller says so.
int check_paged(const wg_paged_cache *c, int64_t kvd, bool lens, const char *who);
Paged as_paged(const wg_paged_cache *c);

// The last of n segments whose key(first, segment) is at most x (keys ascending),
// or -1; the whole wave calls it, x uniform. load(segment, whole, &first, &end,
// &more) reads a segment's first (and, where `whole`, the others too). 64 of the
// segments are looked at a time, spread over what is left: one load up to 64
// segments, two up to 4096. The last look brings *first, *end and *more along,
// which would be a trip to memory more.
template <typename Load, typename Key>
__device__ inline int find_segment(int n, int x, Load load, Key key, int *first, int *end,
                                   int *more) {
  const int lane = threadIdx.x & 63, all = n;
  int lo = 0;
  while (true) {
    const int step = (n + 63) >> 6, at = lo + lane * step;
    const bool in = lane * step < n;
    int f = 0, e = 0, v = 0;
    if (in) load(at, step == 1, &f, &e, &v);
    const int below = __popcll(__ballot(in && key(f, at) <= x));  // (ascending: a prefix)
    if (below == 0) return -1;
    if (step == 1) {
      *first = __builtin_amdgcn_readlane(f, below - 1);
      *end = __builtin_amdgcn_readlane(e, below - 1);
      *more = __builtin_amdgcn_readlane(v, below - 1);
      return lo + below - 1;
    }
    lo += (below - 1) * step;
    n = min(step, all - lo);
  }
}
// The same over the sequences by their first rows, with the sequence's rows
// *r0 .. *r1 - 1 and its entries *len.
template <typename Key>
__device__ inline int find_last(const Paged &c, const int32_t *row_start, int x, Key key, int *r0,
                                int *r1, int *len) {
  return find_segment(
      c.seqs, x,
      [&](int at, bool whole, int *first, int *end, int *entries) {
        *first = row_start[at];
        if (whole) {
          *end = row_start[at + 1];
          *entries = paged_len(c, at);
        }
      },
      key, r0, r1, len);
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

}  // namespace wg
