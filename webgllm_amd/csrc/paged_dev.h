// What the paged cache's kernels share on the device and in their checks.
#pragma once

#include "common.h"
#include "paged_core.h"

namespace wg {

// A cache descriptor's checks (0, or a status with the message set); kvd
// values an entry. `lens` is read only where the caller says so.
int check_paged(const wg_paged_cache *c, int64_t kvd, bool lens, const char *who);
Paged as_paged(const wg_paged_cache *c);

// The last sequence whose first row's key(row_start[b], b) is at most x (keys
// ascending), or -1; the whole wave calls it, x uniform. 64 of the starts are
// looked at a time, spread over what is left: one load up to 64 sequences, two
// up to 4096. The last look brings the sequence's rows *r0 .. *r1 - 1 and its
// entries *len along, which would be a trip to memory more.
template <typename Key>
__device__ inline int find_last(const Paged &c, const int32_t *row_start, int x, Key key, int *r0,
                                int *r1, int *len) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = c.seqs;
  while (true) {
    const int step = (n + 63) >> 6, at = lo + lane * step;
    const bool in = lane * step < n;
    int first = 0, end = 0, entries = 0;
    if (in) {
      first = row_start[at];
      if (step == 1) {
        end = row_start[at + 1];
        entries = paged_len(c, at);
      }
    }
    const int below = __popcll(__ballot(in && key(first, at) <= x));  // (ascending: a prefix)
    if (below == 0) return -1;
    if (step == 1) {
      *r0 = __builtin_amdgcn_readlane(first, below - 1);
      *r1 = __builtin_amdgcn_readlane(end, below - 1);
      *len = __builtin_amdgcn_readlane(entries, below - 1);
      return lo + below - 1;
    }
    lo += (below - 1) * step;
    n = min(step, c.seqs - lo);
  }
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
