// lmx_pages.hip -- the page table of the 8-bit cache kept on the device
// (lmx_kv8_extend, lmx_kv8_trim): which sequences get their tokens, where each
// row goes, and the stack of free pages.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lmx_internal.hpp"
#include "lutmac_kv8.h"

namespace lmx {
namespace {

constexpr int kPage = LMX_KV8_PAGE, kThreads = 1024, kWaves = kThreads / kWave;

struct PagesArgs {
  int *pages, *lengths, *free_pages, *n_free;
  int n_seqs, n_pages;
  size_t max_pages;
  const int *count;   // new or dropped tokens
  int n_rows;
  int *offsets, *granted, *positions;
  long long *slots;
};

// Sums that stop at 2^32 - 1, past every limit that they are compared with: in
// any order they come out the same.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive sums over the workgroup's threads of N numbers each on top of
// base[N], which grows by all of them.
template <int N>
__device__ __forceinline__ void block_sums(uint32_t (&v)[N], uint32_t (&base)[N], uint32_t (*waves)[kWaves]) {
  const int lane = threadIdx.x & (kWave - 1), wave = int(threadIdx.x) / kWave;
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const uint32_t o = __shfl_up(v[n], d);
      if (lane >= d) v[n] = add_sat(v[n], o);
    }
    if (lane == kWave - 1) waves[n][wave] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t before = base[n], all = base[n];
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t o = waves[n][w];
      if (w < wave) before = add_sat(before, o);
      all = add_sat(all, o);
    }
    v[n] = add_sat(v[n], before);
    base[n] = all;
  }
  __syncthreads();
}

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens) { return (tokens + kPage - 1) / kPage; }

// n pages between a table row (from its entry `first` on) and the stack (from its
// place `top` down), taken from it or (PUSH) given back.  One or two by the thread
// itself, of up to kLong by 16 lanes, kAtOnce times 4 sequences at a time with their
// loads on the way together, of more by the wave (1000 sequences of 31 pages in one
// workgroup: 41 us thread by thread, 17 a wave for each, 11 so).  Returns whether what this
// thread gave back held an entry that is no page (negative).
constexpr int kAtOnce = 4, kLong = 128;
template <bool PUSH>
__device__ __forceinline__ bool move_pages(const PagesArgs &a, uint32_t n, size_t first, uint32_t top) {
  bool hole = false;
  const auto take = [&](size_t entry, uint32_t place) __attribute__((always_inline)) { return PUSH ? a.pages[entry] : a.free_pages[place]; };
  const auto give = [&](size_t entry, uint32_t place, int page) __attribute__((always_inline)) {
    a.pages[entry] = PUSH ? -1 : page;
    if (PUSH) hole |= page < 0;
    if (PUSH && place < uint32_t(a.n_pages)) a.free_pages[place] = page;   // (pages freed twice may be more than there are)
  };
  if (n <= 2)
    for (uint32_t j = 0; j < n; ++j) give(first + j, top - j, take(first + j, top - j));
  const int lane = threadIdx.x & (kWave - 1);
  for (uint64_t huge = __builtin_amdgcn_ballot_w64(n > kLong); huge; huge &= huge - 1) {
    const int src = __builtin_ctzll(huge);
    const uint32_t count = __shfl(n, src), from = __shfl(top, src);
    const size_t entry = size_t(__shfl(uint32_t(first >> 32), src)) << 32 | __shfl(uint32_t(first), src);
    for (uint32_t j = uint32_t(lane); j < count; j += 4 * kWave) {
      int page[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) page[b] = take(entry + min(j + b * kWave, count - 1), from - min(j + b * kWave, count - 1));
#pragma unroll
      for (int b = 0; b < 4; ++b) asm volatile("" ::"v"(page[b]));
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (j + b * kWave < count) give(entry + j + b * kWave, from - (j + b * kWave), page[b]);
    }
  }
  const uint32_t big = n > 2 && n <= kLong ? n : 0;
  const uint64_t many = __builtin_amdgcn_ballot_w64(big != 0);
  for (int q0 = 0; q0 < kWave; q0 += 4 * kAtOnce) {
    if (!(many >> q0 & ((uint64_t(1) << (4 * kAtOnce)) - 1))) continue;
    uint32_t count[kAtOnce], from[kAtOnce];
    size_t entry[kAtOnce];
#pragma unroll
    for (int b = 0; b < kAtOnce; ++b) {
      const int src = q0 + 4 * b + lane / 16;
      count[b] = __shfl(big, src), from[b] = __shfl(top, src);
      entry[b] = size_t(__shfl(uint32_t(first >> 32), src)) << 32 | __shfl(uint32_t(first), src);
    }
    for (uint32_t j = uint32_t(lane) % 16;; j += 32) {
      bool more = false;
      int page[2 * kAtOnce];   // (those of no use: the first entry or place, as some page moves there is one)
#pragma unroll
      for (int b = 0; b < 2 * kAtOnce; ++b) {
        const uint32_t i = j + 16 * (b % 2);
        const bool yes = i < count[b / 2];
        page[b] = take(yes ? entry[b / 2] + i : 0, yes ? from[b / 2] - i : 0);
        more |= i + 32 < count[b / 2];
      }
      // (all here before the first store: else each store's branch would wait for the store before)
#pragma unroll
      for (int b = 0; b < 2 * kAtOnce; ++b) asm volatile("" ::"v"(page[b]));
#pragma unroll
      for (int b = 0; b < 2 * kAtOnce; ++b) {
        const uint32_t i = j + 16 * (b % 2);
        if (i < count[b / 2]) give(entry[b / 2] + i, from[b / 2] - i, page[b]);
      }
      if (!__builtin_amdgcn_ballot_w64(more)) break;
    }
  }
  return hole;
}

// Row r is the token at `pos` of sequence s.
__device__ __forceinline__ void place_row(const PagesArgs &a, int r, int s, int pos) {
  a.positions[r] = pos;
  if (!a.slots) return;
  const int page = a.pages[size_t(s) * a.max_pages + pos / kPage];
  a.slots[r] = page < 0 ? -1 : (long long)page * kPage + pos % kPage;
}

// The last of n ascending numbers (the first of which is at most r) that is at
// most r.
__device__ __forceinline__ int last_at_most(const int *v, int n, int r) {
  int lo = 0;
  while (n > 1) {
    const int half = n / 2;
    const bool up = v[lo + half] <= r;
    lo = up ? lo + half : lo;
    n = up ? n - half : half;
  }
  return lo;
}

// One workgroup over all sequences, a thread each, kThreads of them at a time:
// the sums of new tokens, pages and granted tokens are all that couples them.  (64
// sequences' step 4.4 us, most of it the launch and three trips to memory; 1000 prompts' decisions 6.7.)
// ROWS: moves the pages and places the rows as well.
template <bool ROWS>
__global__ __launch_bounds__(kThreads) void extend_kernel(PagesArgs a) {
  __shared__ uint32_t waves[2][kWaves], used;
  __shared__ int begin[kThreads], start[kThreads];
  const uint32_t have = uint32_t(min(max(*a.n_free, 0), a.n_pages));
  uint32_t asked[2] = {0, 0}, rows[1] = {0};
  if (threadIdx.x == 0) used = 0, a.offsets[0] = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += kThreads) {
    const int s = s0 + int(threadIdx.x);
    const bool live = s < a.n_seqs;
    const uint32_t old = live ? uint32_t(max(a.lengths[s], 0)) : 0;
    uint32_t add = live ? uint32_t(max(a.count[s], 0)) : 0;
    if (size_t(old) + add > min(a.max_pages * kPage, size_t(0x7FFFFFFF))) add = 0;
    const uint32_t first = pages_of(old), need = add ? pages_of(old + add) - first : 0;
    uint32_t v[2] = {add, need};
    block_sums<2>(v, asked, waves);
    const bool yes = add && v[0] <= uint32_t(a.n_rows) && (need == 0 || v[1] <= have);
    const uint32_t before = rows[0];
    uint32_t g[1] = {yes ? add : 0};
    block_sums<1>(g, rows, waves);
    if (live) {
      a.granted[s] = yes ? int(add) : 0;
      a.offsets[s + 1] = int(g[0]);
      if (yes) a.lengths[s] = int(old + add);
    }
    // (a sequence that gets pages is behind none that needed some and got none)
    const uint32_t take = yes ? need : 0;
    if (take) atomicMax(&used, v[1]);
    if constexpr (ROWS) {
      move_pages<false>(a, take, size_t(s) * a.max_pages + first, have - 1 - (v[1] - need));
      begin[threadIdx.x] = int(g[0]) - (yes ? int(add) : 0);
      start[threadIdx.x] = int(old);
      __syncthreads();
      const int n = min(kThreads, a.n_seqs - s0);
      for (int r = int(before + threadIdx.x); r < int(rows[0]); r += kThreads) {
        const int i = last_at_most(begin, n, r);
        place_row(a, r, s0 + i, start[i] + r - begin[i]);
      }
    }
    __syncthreads();
  }
  __syncthreads();
  if (threadIdx.x == 0) *a.n_free = int(have - used);
}

// The new pages of a call of many rows, once it is known who gets them: up to
// kMovers workgroups, which sum anew what precedes their sequences.  (A workgroup of its
// own for each few sequences, since one CU issues too little for them all.)
constexpr int kMovers = 64;
__global__ __launch_bounds__(256) void new_pages_kernel(PagesArgs a) {
  __shared__ uint32_t sums[2][4];
  const int lane = threadIdx.x & (kWave - 1), wave = int(threadIdx.x) / kWave;
  const int share = ((a.n_seqs + int(gridDim.x) - 1) / int(gridDim.x) + kWave - 1) / kWave * kWave;
  const int begin = min(int(blockIdx.x) * share, a.n_seqs), end = min(begin + share, a.n_seqs);
  if (begin == end) return;
  struct Taken { uint32_t first, need; };
  const auto taken = [&](int s) __attribute__((always_inline)) {
    const uint32_t got = uint32_t(a.granted[s]), now = uint32_t(max(a.lengths[s], 0)), first = pages_of(now - got);
    return Taken{first, got ? pages_of(now) - first : 0};
  };
  uint32_t before = 0, all = 0;
  for (int s = int(threadIdx.x); s < a.n_seqs; s += 256) {
    const uint32_t need = taken(s).need;
    all += need;
    if (s < begin) before += need;
  }
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) all += __shfl_xor(all, d), before += __shfl_xor(before, d);
  if (lane == 0) sums[0][wave] = before, sums[1][wave] = all;
  __syncthreads();
  before = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  uint32_t top = uint32_t(*a.n_free) + sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3] - 1 - before;   // of the next sequence
  // every wave goes over the workgroup's sequences, and moves the pages of a quarter of each 64
  for (int s0 = begin; s0 < end; s0 += kWave) {
    const int s = s0 + lane;
    const Taken t = s < end ? taken(s) : Taken{0, 0};
    uint32_t upto = t.need;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const uint32_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    move_pages<false>(a, lane / 16 == wave ? t.need : 0, size_t(s) * a.max_pages + t.first, top - (upto - t.need));
    top -= __shfl(upto, kWave - 1);
  }
}

// The last sequence whose first row is at most r (the first row is 0), by a wave.
__device__ __forceinline__ int wave_search(const int *offsets, int n, int r) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave, i = lane * step;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && offsets[lo + min(i, n - 1)] <= r));
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  return lo;
}

// The rows of the call, where they are many, kEach neighbours a thread: 12 bytes
// written a row (2 million rows 11 us, 2.2 TB/s; one a thread 17).
constexpr int kEach = 4;
__global__ __launch_bounds__(256) void rows_kernel(PagesArgs a) {
  const int rows = a.offsets[a.n_seqs], first = int(blockIdx.x * 256 + (threadIdx.x & ~(kWave - 1))) * kEach;
  if (first >= rows) return;   // (the wave's)
  const int lo = wave_search(a.offsets, a.n_seqs, first), hi = wave_search(a.offsets, a.n_seqs, min(first + kWave * kEach, rows) - 1);
  const int r0 = first + int(threadIdx.x & (kWave - 1)) * kEach;
  if (r0 >= rows) return;
  int s = lo + last_at_most(a.offsets + lo, hi - lo + 1, r0), end = a.offsets[s + 1], pos = a.lengths[s] - end + r0, page = 0, known = -1;
  int at[kEach];
  long long slot[kEach];
  const int n = min(kEach, rows - r0);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (j >= n) break;
    if (r0 + j >= end) {   // the next sequence that has rows
      do end = a.offsets[++s + 1];
      while (r0 + j >= end);
      pos = a.lengths[s] - end + r0 + j;
      known = -1;
    }
    if (a.slots && pos / kPage != known) known = pos / kPage, page = a.pages[size_t(s) * a.max_pages + known];
    at[j] = pos;
    slot[j] = page < 0 ? -1 : (long long)page * kPage + pos % kPage;
    ++pos;
  }
  if (n == kEach && reinterpret_cast<size_t>(a.positions) % 16 == 0) {
    *reinterpret_cast<int4 *>(a.positions + r0) = make_int4(at[0], at[1], at[2], at[3]);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (j < n) a.positions[r0 + j] = at[j];
  }
  if (!a.slots) return;
  if (n == kEach && reinterpret_cast<size_t>(a.slots) % 16 == 0) {
    *reinterpret_cast<longlong2 *>(a.slots + r0) = make_longlong2(slot[0], slot[1]);
    *reinterpret_cast<longlong2 *>(a.slots + r0 + 2) = make_longlong2(slot[2], slot[3]);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (j < n) a.slots[r0 + j] = slot[j];
  }
}

__global__ __launch_bounds__(kThreads) void trim_kernel(PagesArgs a) {
  __shared__ uint32_t waves[1][kWaves];
  __shared__ int holes;
  const uint32_t have = uint32_t(min(max(*a.n_free, 0), a.n_pages));
  if (threadIdx.x == 0) holes = 0;
  struct Cut { uint32_t keep, kept, gone; bool live, past; };   // past: longer than the table row
  const auto cut = [&](int s) {
    Cut c{};
    c.live = s < a.n_seqs;
    if (!c.live) return c;
    const uint32_t old = uint32_t(max(a.lengths[s], 0)), drop = uint32_t(max(a.count[s], 0));
    c.past = old > a.max_pages * kPage;
    c.keep = old - min(old, drop);
    c.kept = uint32_t(min(size_t(pages_of(c.keep)), a.max_pages));
    c.gone = uint32_t(min(size_t(pages_of(old)), a.max_pages)) - c.kept;
    return c;
  };
  uint32_t all[1] = {0}, before[1] = {0};   // pages of the whole call, and up to here
  for (int s0 = 0; a.n_seqs > kThreads && s0 < a.n_seqs; s0 += kThreads) {
    uint32_t v[1] = {cut(s0 + int(threadIdx.x)).gone};
    block_sums<1>(v, all, waves);
  }
  for (int s0 = 0; s0 < a.n_seqs; s0 += kThreads) {
    const int s = s0 + int(threadIdx.x);
    const Cut c = cut(s);
    uint32_t v[1] = {c.gone};
    block_sums<1>(v, before, waves);
    if (a.n_seqs <= kThreads) all[0] = before[0];
    const bool hole = move_pages<true>(a, c.gone, size_t(s) * a.max_pages + c.kept, have + all[0] - 1 - (v[0] - c.gone));
    if (hole | c.past) atomicOr(&holes, int(hole) | 2 * int(c.past));
    if (c.live) a.lengths[s] = int(c.keep);
  }
  __syncthreads();
  const uint32_t end = min(add_sat(have, all[0]), uint32_t(a.n_pages));
  uint32_t pages[1] = {end - have};
  if (holes == 1) {   // what is no page leaves the stack again (a chunk is read before any of it is written)
    pages[0] = 0;
    for (uint32_t p0 = have; p0 < end; p0 += kThreads) {
      const uint32_t p = p0 + threadIdx.x;
      const int page = p < end ? a.free_pages[p] : -1;
      const bool ok = page >= 0;
      uint32_t v[1] = {ok};
      block_sums<1>(v, pages, waves);
      if (ok) a.free_pages[have + v[0] - 1] = page;
    }
  }
  if (threadIdx.x == 0) *a.n_free = int(have + pages[0]);
}

int launch_err(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

int check_pages(const lmx_kv8_pages *p) {
  if (!p) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (p->n_seqs > (1u << 20) || p->max_pages > (1u << 24) || p->n_pages >= (1u << 31))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu sequences of %zu pages, %zu pages: at most 2^20, 2^24 and 2^31 - 1", p->n_seqs, p->max_pages, p->n_pages);
  return LMX_OK;
}
int check_pointers(const lmx_kv8_pages *p, const int32_t *count) {
  if (!p->n_free || (p->n_seqs && (!p->lengths || !count)) || (p->n_seqs && p->max_pages && !p->pages) || (p->n_pages && !p->free_pages))
    return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if ((reinterpret_cast<size_t>(p->lengths) | reinterpret_cast<size_t>(p->n_free) | reinterpret_cast<size_t>(p->pages) |
       reinterpret_cast<size_t>(p->free_pages) | reinterpret_cast<size_t>(count)) % 4)
    return fail(LMX_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
  return LMX_OK;
}
PagesArgs pages_args(const lmx_kv8_pages *p, const int32_t *count) {
  PagesArgs a{};
  a.pages = p->pages, a.lengths = p->lengths, a.free_pages = p->free_pages, a.n_free = p->n_free;
  a.n_seqs = int(p->n_seqs), a.n_pages = int(p->n_pages), a.max_pages = p->max_pages, a.count = count;
  return a;
}

// Rows that the one workgroup places itself.
constexpr size_t kFewRows = 8192;

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_kv8_extend(const lmx_kv8_pages *pages, const int32_t *new_tokens, size_t n_rows, int32_t *offsets, int32_t *granted,
                   int32_t *positions, int64_t *slots, void *stream) {
  int r = check_pages(pages);
  if (r) return r;
  if (n_rows > (1u << 24)) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu rows: at most 2^24", n_rows);
  if (!offsets || (pages->n_seqs && !granted) || (n_rows && !positions)) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if ((reinterpret_cast<size_t>(offsets) | reinterpret_cast<size_t>(granted) | reinterpret_cast<size_t>(positions)) % 4 ||
      reinterpret_cast<size_t>(slots) % 8)
    return fail(LMX_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
  if ((r = check_pointers(pages, new_tokens))) return r;
  PagesArgs a = pages_args(pages, new_tokens);
  a.n_rows = int(n_rows);
  a.offsets = offsets, a.granted = granted, a.positions = positions, a.slots = reinterpret_cast<long long *>(slots);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n_rows <= kFewRows) {
    extend_kernel<true><<<1, kThreads, 0, st>>>(a);
    return launch_err("kv8 extend");
  }
  extend_kernel<false><<<1, kThreads, 0, st>>>(a);
  if ((r = launch_err("kv8 extend"))) return r;
  if (pages->n_seqs == 0) return LMX_OK;
  new_pages_kernel<<<unsigned(std::min<size_t>((pages->n_seqs + kWave - 1) / kWave, kMovers)), 256, 0, st>>>(a);
  if ((r = launch_err("kv8 extend pages"))) return r;
  rows_kernel<<<unsigned((n_rows + 256 * kEach - 1) / (256 * kEach)), 256, 0, st>>>(a);
  return launch_err("kv8 extend rows");
}

int lmx_kv8_trim(const lmx_kv8_pages *pages, const int32_t *drop, void *stream) {
  int r = check_pages(pages);
  if (r || pages->n_seqs == 0) return r;
  if ((r = check_pointers(pages, drop))) return r;
  trim_kernel<<<1, kThreads, 0, static_cast<hipStream_t>(stream)>>>(pages_args(pages, drop));
  return launch_err("kv8 trim");
}

}  // extern "C"
