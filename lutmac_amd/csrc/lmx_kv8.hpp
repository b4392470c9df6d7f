// lmx_kv8.hpp -- device-side building blocks of the 8-bit paged cache
// (include/lutmac_kv8.h): the arguments, the search for a work unit's
// sequence, and the digits of queries and weights.
#ifndef LMX_KV8_HPP
#define LMX_KV8_HPP

#include <hip/hip_runtime.h>

#include "lmx_lanes.hpp"
#include "lmx_internal.hpp"
#include "lmx_types.hpp"
#include "lutmac_kv8.h"

namespace lmx {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kPage = LMX_KV8_PAGE, kBlock = LMX_KV8_BLOCK, kPageBlocks = kPage / kBlock;

struct Kv8Args {
  int8_t *k, *v;
  float *k_scale, *v_scale;
  const int *offsets, *lengths, *pages;
  int n_pages, n_kv, n_seqs, max_pages, n_rows;
  int n_heads, group;
};

// The sequence that work unit u belongs to, where sequence s begins at unit
// floor(offsets[s] * mul / 16) + s * per (at least its units follow, and less
// than `per` more): -1 past the last.  The wave looks at 64 sequences a load.
__device__ __forceinline__ int unit_sequence(const Kv8Args &a, int u, int mul, int per, int lane, int &first) {
  int lo = 0, n = a.n_seqs;
  const auto begin = [&](int s) {
    return int((static_cast<long long>(min(max(a.offsets[s], 0), a.n_rows)) * mul) >> 4) + s * per;
  };
  while (true) {
    const int step = (n + kWave - 1) / kWave, s = lo + lane * step;
    const bool in = lane * step < n && begin(min(s, a.n_seqs - 1)) <= u;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
    if (step == 1) break;
  }
  first = begin(lo);
  return lo;
}

// One sequence's rows of the call.
struct SeqRows {
  int r0, n;         // first row, count
  int start, len;    // position of the first row (may be negative), tokens with the rows
  __device__ __forceinline__ SeqRows(const Kv8Args &a, int s) {
    r0 = min(max(a.offsets[s], 0), a.n_rows);
    n = min(max(a.offsets[s + 1], r0), a.n_rows) - r0;
    len = max(a.lengths[s], 0);
    start = len - n;
  }
};

__device__ __forceinline__ bool page_ok(const Kv8Args &a, int page) { return page >= 0 && page < a.n_pages; }

}  // namespace lmx

#endif  // LMX_KV8_HPP
