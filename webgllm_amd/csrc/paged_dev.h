// What the paged cache's kernels share on the device and in their checks.
#pragma once

#include "common.h"
#include "paged_core.h"

namespace wg {

// A cache descriptor's checks (0, or a status with the message set); kvd
// values an entry. `lens` is read only where the caller says so.
int check_paged(const wg_paged_cache *c, int64_t kvd, bool lens, const char *who);
Paged as_paged(const wg_paged_cache *c);

// The sequence that row m belongs to (row_start ascending), or -1; the whole
// wave calls it, m uniform. 64 of the starts are looked at a time, spread
// over what is left: one load up to 64 sequences, two up to 4096.
__device__ inline int find_seq(const int32_t *row_start, int seqs, int m) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = seqs;  // row_start[lo] <= m if any is; the answer is in lo .. lo + n - 1
  while (true) {
    const int step = (n + 63) >> 6;
    const int at = lo + lane * step;
    const bool below = lane * step < n && row_start[at] <= m;
    const int c = __popcll(__ballot(below));  // (ascending: a prefix)
    if (c == 0) return -1;
    lo += (c - 1) * step;
    if (step == 1) break;
    n = min(step, seqs - lo);
  }
  return m < row_start[lo + 1] ? lo : -1;
}

}  // namespace wg
