// lmx_verify.hip -- verification of drafted tokens (include/lutmac_verify.h).
//
// Everything that decides is computed in 64 bits: a token is the first whose
// cumulative weight passes a threshold, and with weights off by 2^-24 of
// themselves a pick from a vocabulary of 10^5 would now and then be a neighbour.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lmx_internal.hpp"
#include "lmx_lanes.hpp"
#include "lmx_types.hpp"
#include "lutmac_verify.h"

namespace lmx {
namespace {

// What a part of a row holds: its largest logit, the sum of e^((l - top) / T), or,
// greedily, the place of the first of the largest.
struct Part {
  double sum;
  float top;
  int best;
};

struct VerifyArgs {
  const int *offsets, *drafts;
  const float2 *uniforms;
  const float *temperature;
  int n_seqs, n_rows, vocab;
  const void *logits;
  size_t stride;
  const float *probs;
  size_t probs_stride;
  int *accepted, *tokens;
  Part *parts;        // [n_rows][n_parts]
  double *rest;       // [n_seqs][n_parts] sums of what p has over q, where a sequence needs them
  unsigned *tickets;  // [n_seqs], zero when a pick begins
  int n_parts;
  int groups;         // workgroups of a sequence where q may be needed
};

// A part of a row is what a wave takes at a time: kPieces pieces of 16 bytes a lane.
constexpr int kPieces = 4, kPart = kPieces * kWave;   // (pieces of a part)
constexpr int kStatsThreads = 256, kThreads = 512, kWaves = kThreads / kWave;

// Sums over a wave, the same bits in every lane, and inclusive sums over its lanes
// (without LDS: a shuffle of 64 bits takes two trips through it).
template <int D = kWave / 2>
__device__ __forceinline__ double wave_sum(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t o = uint64_t(lane_xor_u32<D>(uint32_t(u >> 32), lane)) << 32 | lane_xor_u32<D>(uint32_t(u), lane);
  v += __builtin_bit_cast(double, o);
  if constexpr (D > 1) return wave_sum<D / 2>(v, lane);
  else return v;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {   // v plus that of another lane, where there is one
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CTRL, ROWS, 0xF, false));
  const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CTRL, ROWS, 0xF, false));
  return v + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v = dpp_add<0x111, 0xF>(v);   // the lane 1, 2, 4, 8 below in a row of 16
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<0x142, 0xA>(v);   // rows 0 and 2 to the next
  return dpp_add<0x143, 0xC>(v);   // the lower half to the upper
}
__device__ __forceinline__ double lane_value(double v, int from) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u)), from)), hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u >> 32)), from));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ float wave_max(float v, int lane) { return lane_max<kWave / 2>(v, lane); }
template <int D = kWave / 2>
__device__ __forceinline__ int wave_min(int v, int lane) {
  v = min(v, int(lane_xor_u32<D>(uint32_t(v), lane)));
  if constexpr (D > 1) return wave_min<D / 2>(v, lane);
  else return v;
}

// The last sequence whose first row is at most r (-1: none), by a wave.
__device__ __forceinline__ int sequence_of(const int *offsets, int n, int r, int lane) {
  int lo = 0;
  while (n > 0) {
    const int step = (n + kWave - 1) / kWave, i = lane * step;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && offsets[lo + min(i, n - 1)] <= r));
    if (c == 0) return -1;
    if (step == 1) return lo + c - 1;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  return -1;
}

// A sequence's temperature (0: greedy) and what a difference of logits is
// multiplied by to become a power of two; `least`: the difference that gives 2^-1100.
struct Heat {
  float t;
  double by, least;
};
__device__ __forceinline__ Heat heat_of(const VerifyArgs &a, int s) {
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  const double by = fmax(1.4426950408889634074 / double(t), 1e-300);
  return t > 0.0f ? Heat{t, by, -1100.0 / by} : Heat{0.0f, 0.0, 0.0};
}
// e^((l - top) / t): with y = (l - top) by, 2^k times 1 + f P(f), f = y - k within
// 1/2 and P of degree 8 the interpolation of (2^f - 1) / f at Chebyshev's points (2^f is off by 2^-44.6 at
// most).  Adding 1.5 * 2^52 leaves k in the low word.  -inf, or a part of only such
// (-inf - -inf), weighs nothing.  15 operations in 64 bits, which cost as much as in
// 32 here.
__device__ __forceinline__ double weight_of(float l, float top, const Heat &h) {
  constexpr double kRound = 6755399441055744.0;
  const double d = fmax(double(l) - double(top), h.least);
  const double n = fma(d, h.by, kRound), f = fma(d, h.by, kRound - n);
  double p = 1.0203121138901363e-07;
  p = fma(p, f, 1.325522487892511e-06);
  p = fma(p, f, 1.525268684597521e-05);
  p = fma(p, f, 1.5403455852451678e-04);
  p = fma(p, f, 1.3333558179043376e-03);
  p = fma(p, f, 9.618129159402562e-03);
  p = fma(p, f, 5.5504108664760424e-02);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return ldexp(p, int(uint32_t(__builtin_bit_cast(uint64_t, n))));
}

// A row's elements in pieces of 16 bytes, E of them from element c E on, whatever
// the row's alignment (the loads need none).  Elements past the row's end are -inf,
// which weighs nothing.
template <class T>
struct RowOf {
  static constexpr int E = 16 / int(sizeof(T));
  typedef T Values __attribute__((ext_vector_type(E)));
  typedef T Anywhere __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  const T *x;
  int vocab;
  __device__ __forceinline__ RowOf(const VerifyArgs &a, int row) : x(static_cast<const T *>(a.logits) + size_t(row) * a.stride), vocab(a.vocab) {}
  __device__ __forceinline__ Values piece(int c) const {
    const int i = c * E;
    if (i + E <= vocab) return *reinterpret_cast<const Anywhere *>(x + i);
    Values v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = i + e < vocab ? x[i + e] : T(-INFINITY);
    return v;
  }
  // A part's pieces, all on their way at once.
  __device__ __forceinline__ void part(int part, int lane, Values (&v)[kPieces]) const {
    const bool whole = (part + 1) * (kPart * E) <= vocab;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int c = part * kPart + j * kWave + lane;
      if (whole) v[j] = *reinterpret_cast<const Anywhere *>(x + c * E);
      else v[j] = piece(c);
    }
  }
};

// Sums, largest and first of the largest of each part of each row, a wave a run of
// parts, the next of them on its way while one is summed.  Bound by the vector unit:
// 24 operations an element (64 x 0..7 drafts, 151936 logits, bf16: 38 us, 2.1 TB/s).
template <class T>
__global__ __launch_bounds__(kStatsThreads) void stats_kernel(VerifyArgs a) {
  typedef typename RowOf<T>::Values Values;
  constexpr int E = RowOf<T>::E;
  const int lane = threadIdx.x & (kWave - 1);
  const size_t waves = size_t(gridDim.x) * (kStatsThreads / kWave), units = size_t(a.n_rows) * a.n_parts;
  const size_t wave = size_t(blockIdx.x) * (kStatsThreads / kWave) + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const size_t each = units / waves, more = units % waves;   // (the first `more` waves take one more)
  size_t left = each + (wave < more);
  const size_t begin = wave * each + min(wave, more);
  int row = int(begin / a.n_parts), part = int(begin % a.n_parts), known = -1, s = -1;
  if (left == 0) return;
  Values next[kPieces];
  RowOf<T>(a, row).part(part, lane, next);
  Heat h{};
  bool mine = false;   // whether the row is any sequence's
  while (true) {
    Values x[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) x[j] = next[j];
    const int this_row = row, this_part = part;
    if (++part == a.n_parts) part = 0, ++row;
    if (--left) RowOf<T>(a, row).part(part, lane, next);
    if (this_row != known) {
      known = this_row;
      s = sequence_of(a.offsets, a.n_seqs, known, lane);
      mine = s >= 0 && known < a.offsets[s + 1];
      if (mine) {
        h = heat_of(a, s);
        if (lane == 0 && known == max(a.offsets[s], 0)) a.tickets[s] = 0;
      }
    }
    if (mine) {
      float top = -INFINITY;   // (a NaN stays)
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) top = __builtin_elementwise_maximum(top, float(x[j][e]));
      const bool nan = top != top;
      top = wave_max(top, lane);
      double sum = 0.0;
      int first = 0x7FFFFFFF;
      if (h.t > 0.0f) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e) sum += weight_of(float(x[j][e]), top, h);
      } else {
#pragma unroll
        for (int j = 0; j < kPieces; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (float(x[j][e]) == top) first = min(first, (this_part * kPart + j * kWave + lane) * E + e);
        first = wave_min(first, lane);
      }
      if (nan || top == INFINITY) sum = __builtin_nan("");
      sum = wave_sum(sum, lane);
      if (lane == 0) a.parts[size_t(this_row) * a.n_parts + this_part] = Part{sum, top, first};
    }
    if (left == 0) return;
  }
}

// A row's distribution: weights over `total`.
struct Row {
  double total;   // not positive: none
  float top;
  int best;
};
// A part's weights in a row's units.
__device__ __forceinline__ double part_weight(const Part &p, float top, const Heat &h) { return p.sum * weight_of(p.top, top, h); }
// By a wave, each lane with its first part (of lane `lane`) in `first`; share: that part's weights.
__device__ __forceinline__ Row row_of(const Part *p, int n, const Part &first, const Heat &h, int lane, double &share) {
  Row r{0.0, first.top, 0x7FFFFFFF};
  for (int i = lane + kWave; i < n; i += kWave) r.top = fmaxf(r.top, p[i].top);
  r.top = wave_max(r.top, lane);
  if (h.t > 0.0f) {
    share = part_weight(first, r.top, h);
    r.total = share;
    for (int i = lane + kWave; i < n; i += kWave) r.total += part_weight(p[i], r.top, h);
    r.total = wave_sum(r.total, lane);
  } else {
    bool bad = first.sum != first.sum;
    if (first.top == r.top) r.best = first.best;
    for (int i = lane + kWave; i < n; i += kWave) {
      bad |= p[i].sum != p[i].sum;
      if (p[i].top == r.top) r.best = min(r.best, p[i].best);
    }
    r.best = wave_min(r.best, lane);
    r.total = __builtin_amdgcn_ballot_w64(bad) ? 0.0 : 1.0;
  }
  if (r.top == -INFINITY || !(r.total > 0.0)) r.total = 0.0;
  return r;
}

// The weights of a row's pieces: OVER: what p has over q, times the total, else p's,
// but for `skip`.
template <class T>
struct Piece : RowOf<T> {
  using RowOf<T>::E, RowOf<T>::vocab;
  typedef float Shares __attribute__((ext_vector_type(E)));
  typedef float AnyShares __attribute__((ext_vector_type(E), aligned(4)));
  const Row &r;
  const Heat &h;
  const float *q;
  __device__ __forceinline__ Piece(const VerifyArgs &a, int row, const Row &r, const Heat &h)
      : RowOf<T>(a, row), r(r), h(h), q(a.probs + size_t(row) * a.probs_stride) {}
  __device__ __forceinline__ Shares shares(int c) const {
    const int i = c * E;
    if (i + E <= vocab) return *reinterpret_cast<const AnyShares *>(q + i);
    Shares v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = i + e < vocab ? q[i + e] : 0.0f;
    return v;
  }
  __device__ __forceinline__ double over(T l, float share) const { return fmax(fma(double(share), -r.total, weight_of(float(l), r.top, h)), 0.0); }
  template <bool OVER>
  __device__ __forceinline__ void weights(int c, int skip, double (&w)[E]) const {
    const typename RowOf<T>::Values v = this->piece(c);
    Shares u;
    if constexpr (OVER) u = shares(c);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (OVER) w[e] = over(v[e], u[e]);
      else w[e] = c * E + e == skip ? 0.0 : weight_of(float(v[e]), r.top, h);
    }
  }
  // The sum of a part's weights, by a wave.
  template <bool OVER>
  __device__ __forceinline__ double part_sum(int part, int skip, int lane) const {
    typename RowOf<T>::Values v[kPieces];
    Shares u[kPieces];
    if constexpr (OVER) {
      const bool whole = (part + 1) * (kPart * E) <= vocab;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int c = part * kPart + j * kWave + lane;
        if (whole) u[j] = *reinterpret_cast<const AnyShares *>(q + c * E);
        else u[j] = shares(c);
      }
    }
    this->part(part, lane, v);
    double all = 0.0;
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (OVER) all += over(v[j][e], u[j][e]);
        else all += (part * kPart + j * kWave + lane) * E + e == skip ? 0.0 : weight_of(float(v[j][e]), r.top, h);
      }
    return wave_sum(all, lane);
  }
};

// The place among up to 64 parts a time, of n, where a wave's sums of weights first
// pass u times all of them: the part, and what is left of the threshold in it
// (infinite: its last token with a weight).  v0: the lane's first sum, of(i): part i's.
struct Place {
  int part;   // -1: nothing weighs anything
  double target;
};
template <class F>
__device__ __forceinline__ Place place_of(int n, double u, double v0, int lane, F of) {
  double all = wave_sum(v0, lane);
  for (int i = kWave; i < n; i += kWave) all += wave_sum(i + lane < n ? of(i + lane) : 0.0, lane);
  if (!(all > 0.0)) return {-1, 0.0};
  const double target = u * all;
  double before = 0.0;
  int behind = -1;
  for (int i = 0; i < n; i += kWave) {
    const double v = i == 0 ? v0 : i + lane < n ? of(i + lane) : 0.0, upto = before + wave_scan(v);
    const uint64_t some = __builtin_amdgcn_ballot_w64(v > 0.0), past = some & __builtin_amdgcn_ballot_w64(upto > target);
    if (past) {
      const int found = __builtin_ctzll(past);
      return {i + found, target - lane_value(upto - v, found)};
    }
    if (some) behind = i + 63 - __builtin_clzll(some);
    before = lane_value(upto, kWave - 1);
  }
  return {behind, INFINITY};   // (rounding, or a number of 1 and more)
}

// A workgroup a sequence, or, where q may be needed, some: each finds the row that
// the sequence stops at, a wave a row at a time.  The token there: parts' sums are
// known, or, of p - q, taken by the sequence's workgroups; the row's wave (of the last
// workgroup) finds the part that the threshold falls into, the workgroup the
// element in it.  What it costs is its chain of loads: offsets, then parts' sums
// and drafts, then the drafted tokens' logits, then the part found (one sequence of 128256
// 9 us; 64 of 151936, p - q summed by 640 workgroups, 23).
template <class T>
__global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a) {
  constexpr int E = RowOf<T>::E;
  static_assert(kPart <= kThreads, "a piece a thread");
  __shared__ Row rows[kWaves];
  __shared__ int stops[kWaves];
  constexpr int kNear = kWaves;
  __shared__ double scan[kWaves], near[kNear];   // (sums of one workgroup's few parts stay here)
  __shared__ Place place;
  __shared__ int at, last, joins, without;
  const int s = int(blockIdx.x), group = int(blockIdx.y), lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int begin = max(a.offsets[s], 0), end = min(a.offsets[s + 1], a.n_rows);
  const Heat h = heat_of(a, s);
  if (begin >= end) {
    if (group == 0 && threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  int row = begin, owner, token = -1;
  double share = 0.0, weight = 0.0;   // of this wave's row: the lane's part's, the drafted token's
  bool known = false;
  float2 u = {0.0f, 0.0f};
  for (;; row += kWaves) {
    const int mine = row + wave;
    if (mine < end) {
      const Part *parts = a.parts + size_t(mine) * a.n_parts;
      const Part first = lane < a.n_parts ? parts[lane] : Part{0.0, -INFINITY, 0x7FFFFFFF};
      token = a.drafts[mine];
      u = a.uniforms[mine];
      known = mine != end - 1 && token >= 0 && token < a.vocab;
      float l = -INFINITY, q = 1.0f;
      if (known) {
        l = float((static_cast<const T *>(a.logits) + size_t(mine) * a.stride)[token]);
        if (a.probs) q = a.probs[size_t(mine) * a.probs_stride + token];
      }
      const Row x = row_of(parts, a.n_parts, first, h, lane, share);
      weight = h.t > 0.0f ? weight_of(l, x.top, h) : token == x.best ? 1.0 : 0.0;
      const bool go = known && x.total > 0.0 && double(u.x) * double(q) * x.total < weight;
      if (lane == 0) rows[wave] = x, stops[wave] = !go;
    } else if (lane == 0) {
      stops[wave] = 1;
    }
    __syncthreads();
    owner = 0;
    while (owner < kWaves && !stops[owner]) ++owner;
    if (owner < kWaves) break;   // (the last row stops)
    __syncthreads();
  }
  row += owner;
  const Row r = rows[owner];
  if (group == 0) {
    for (int i = begin + int(threadIdx.x); i < end; i += kThreads)
      if (i != row) a.tokens[i] = i < row ? a.drafts[i] : -1;
    if (threadIdx.x == 0) {
      a.accepted[s] = row - begin;
      // (greedily: whatever q is, all that p has over it is there)
      if (!(r.total > 0.0) || h.t == 0.0f) a.tokens[row] = r.total > 0.0 ? r.best : -1;
    }
  }
  if (!(r.total > 0.0) || h.t == 0.0f) return;
  const bool over = row != end - 1 && a.probs;
  if (!over && group != 0) return;
  const Piece<T> x(a, row, r, h);
  const Part *parts = a.parts + size_t(row) * a.n_parts;
  if (threadIdx.x == 0) at = 0x7FFFFFFF, last = -1;
  bool from_rest = over;   // weights are those of p - q
  int skip = -1;           // the token that p is to lack
  if (over) {
    double *sums = a.rest + size_t(s) * a.n_parts;
    for (int part = group * kWaves + wave; part < a.n_parts; part += a.groups * kWaves) {
      const double sum = x.template part_sum<true>(part, -1, lane);
      if (lane != 0) continue;
      if (a.groups == 1 && part < kNear) near[part] = sum;
      else __hip_atomic_store(sums + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // (The sums go past the caches and are there before the ticket is taken; a fence
    // would write back the whole L2, 100 us in all for 64 sequences' workgroups.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (a.groups > 1) {
      if (threadIdx.x == 0)
        joins = __hip_atomic_fetch_add(a.tickets + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == unsigned(a.groups - 1);
      __syncthreads();
      if (!joins) return;
    }
    if (wave == owner) {
      const auto of = [&](int i) __attribute__((always_inline)) {
        return a.groups == 1 && i < kNear ? near[i] : __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      };
      const Place p = place_of(a.n_parts, double(u.y), lane < a.n_parts ? of(lane) : 0.0, lane, of);
      if (lane == 0) place = p;
    }
    __syncthreads();
    from_rest = place.part >= 0;   // (nothing is left: from p)
    __syncthreads();
  }
  if (!from_rest) {
    if (wave == owner) {
      // the part that lacks the drafted token: the difference keeps 42 bits, or it
      // is summed without the token
      int lacking = -1;
      double less = 0.0;
      if (!over && known) {
        lacking = token / (kPart * E);
        const double with = lacking < kWave ? lane_value(share, lacking) : part_weight(parts[lacking], r.top, h);
        less = with - weight;
        if (!(less > with * 0x1p-10)) less = x.template part_sum<false>(lacking, token, lane);
      }
      const auto of = [&](int i) __attribute__((always_inline)) { return i == lacking ? less : part_weight(parts[i], r.top, h); };
      const double v0 = lane < a.n_parts ? lane == lacking ? less : share : 0.0;
      Place p = place_of(a.n_parts, double(u.y), v0, lane, of);
      if (p.part < 0) {   // nothing is left without the token: from p
        lacking = -1;
        p = place_of(a.n_parts, double(u.y), lane < a.n_parts ? share : 0.0, lane, of);
      }
      if (lane == 0) place = p, without = lacking >= 0 ? token : -1;
    }
    __syncthreads();
    skip = without;
    if (place.part < 0) return;   // (p weighs something)
  }
  // The first piece past the threshold (or the last with a weight), then in it the
  // element: a piece a thread.
  const double target = place.target;
  const int piece = place.part * kPart + int(threadIdx.x);
  double w[E], mine = 0.0;
  if (threadIdx.x < kPart) {
    if (from_rest) x.template weights<true>(piece, -1, w);
    else x.template weights<false>(piece, skip, w);
#pragma unroll
    for (int e = 0; e < E; ++e) mine += w[e];
  }
  const double upto = wave_scan(mine);
  if (lane == kWave - 1) scan[wave] = upto;
  __syncthreads();
  double before = upto - mine;
#pragma unroll
  for (int v = 0; v < kWaves; ++v)
    if (v < wave) before += scan[v];
  // (what precedes a thread and with it is, but for rounding, what precedes the next)
  const bool past = mine > 0.0 && before + mine > target;
  if (past) atomicMin(&at, int(threadIdx.x));
  if (mine > 0.0) atomicMax(&last, int(threadIdx.x));
  __syncthreads();
  if (int(threadIdx.x) != (at < 0x7FFFFFFF ? at : last)) return;
  int found = -1;
  bool done = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    before += w[e];
    if (!done && w[e] > 0.0) found = piece * E + e;
    done = done || (past && w[e] > 0.0 && before > target);
  }
  a.tokens[row] = found;
}

int launch_err(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

int check_sizes(const lmx_drafts *d, int type) {
  if (!d) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (d->n_seqs > (1u << 20) || d->n_rows > (1u << 20) || d->vocab == 0 || d->vocab > (1u << 24))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu sequences, %zu rows of %zu: at most 2^20, 2^20 and 1..2^24", d->n_seqs, d->n_rows, d->vocab);
  return LMX_OK;
}

size_t parts_of(size_t vocab, int type) {
  const size_t part = kPart * (16 / type_bytes(type));
  return (vocab + part - 1) / part;
}

template <class T>
int launch(const VerifyArgs &a, hipStream_t st) {
  // (four waves a SIMD, each with a few parts to go through; two or eight take as long)
  const size_t units = size_t(a.n_rows) * a.n_parts, most = 256 * 16;
  if (units) stats_kernel<T><<<unsigned((std::min(units, most) + 3) / 4), kStatsThreads, 0, st>>>(a);
  const int r = launch_err("verify");
  if (r) return r;
  pick_kernel<T><<<dim3(unsigned(a.n_seqs), unsigned(a.groups)), kThreads, 0, st>>>(a);
  return launch_err("verify pick");
}

// Workgroups of a sequence for p - q: a part a wave, as long as that is four
// workgroups a CU at most (9 sequences of 16 parts: one workgroup each 16.5 us, two 14.4).
int groups_of(const VerifyArgs &a) {
  if (!a.probs || a.n_parts <= kWaves) return 1;
  return std::max(1, std::min((a.n_parts + kWaves - 1) / kWaves, 1024 / a.n_seqs));
}

struct Layout { size_t rest, tickets, all; };
Layout layout(const lmx_drafts *d, int type) {
  const size_t parts = parts_of(d->vocab, type);
  Layout l{};
  l.rest = d->n_rows * parts * sizeof(Part);
  l.tickets = l.rest + d->n_seqs * parts * sizeof(double);
  l.all = l.tickets + d->n_seqs * sizeof(unsigned);
  return l;
}

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_verify_drafts_workspace(const lmx_drafts *d, int type, size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int r = check_sizes(d, type);
  if (r) return r;
  *bytes = layout(d, type).all;
  return LMX_OK;
}

int lmx_verify_drafts(const lmx_drafts *d, int type, const void *logits, size_t stride, const float *probs, size_t probs_stride,
                      int32_t *accepted, int32_t *tokens, void *workspace, size_t workspace_bytes, void *stream) {
  size_t need = 0;
  const int r = lmx_verify_drafts_workspace(d, type, &need);
  if (r) return r;
  if (d->n_seqs == 0) return LMX_OK;
  if (!d->offsets || !accepted) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (d->n_rows && (!d->drafts || !d->uniforms || !logits || !tokens)) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  const size_t e = type_bytes(type);
  if ((reinterpret_cast<size_t>(d->offsets) | reinterpret_cast<size_t>(d->drafts) | reinterpret_cast<size_t>(d->temperature) |
       reinterpret_cast<size_t>(probs) | reinterpret_cast<size_t>(accepted) | reinterpret_cast<size_t>(tokens)) % 4 ||
      reinterpret_cast<size_t>(d->uniforms) % 8 || reinterpret_cast<size_t>(logits) % e)
    return fail(LMX_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements, uniforms to their pairs");
  if (d->n_rows && tokens == d->drafts) return fail(LMX_ERR_INVALID_ARGUMENT, "tokens and drafts are the same memory");
  if (d->n_rows > 1 && (stride < d->vocab || stride >> 40 || (probs && (probs_stride < d->vocab || probs_stride >> 40))))
    return fail(LMX_ERR_INVALID_ARGUMENT, "row strides %zu and %zu of rows of %zu", stride, probs_stride, d->vocab);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<size_t>(workspace) % 16))
    return fail(LMX_ERR_INVALID_ARGUMENT, "workspace of %zu bytes at %p: %zu bytes, 16-byte aligned, are needed", workspace_bytes,
                workspace, need);
  VerifyArgs a{};
  a.offsets = d->offsets, a.drafts = d->drafts, a.uniforms = reinterpret_cast<const float2 *>(d->uniforms);
  a.temperature = d->temperature;
  a.n_seqs = int(d->n_seqs), a.n_rows = int(d->n_rows), a.vocab = int(d->vocab);
  a.logits = logits, a.stride = stride, a.probs = probs, a.probs_stride = probs_stride;
  a.accepted = accepted, a.tokens = tokens;
  const Layout l = layout(d, type);
  char *work = static_cast<char *>(workspace);
  a.parts = reinterpret_cast<Part *>(work), a.rest = reinterpret_cast<double *>(work + l.rest);
  a.tickets = reinterpret_cast<unsigned *>(work + l.tickets);
  a.n_parts = int(parts_of(d->vocab, type));
  a.groups = groups_of(a);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch<float>(a, st);
  case LMX_F16: return launch<f16>(a, st);
  default: return launch<bf16>(a, st);
  }
}

}  // extern "C"
