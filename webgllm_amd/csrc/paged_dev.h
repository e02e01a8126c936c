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
