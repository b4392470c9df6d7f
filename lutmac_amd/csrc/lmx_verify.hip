// lmx_verify.hip -- verification of drafted tokens (include/lutmac_verify.h).
//
// Everything that decides is computed in 64 bits: a token is the first whose
// cumulative weight passes a threshold, and with weights off by 2^-24 of
// themselves one in some hundred picks from a vocabulary of 10^5 would be a neighbour.
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
};

constexpr int kThreads = 256, kWaves = kThreads / kWave;

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

// A row's elements in pieces of 16 bytes: piece c holds elements c E - lead .. + E - 1,
// so that pieces are aligned wherever the row begins.
template <class T>
struct RowOf {
  static constexpr int E = 16 / int(sizeof(T));
  const T *x;
  int lead, vocab;
  __device__ __forceinline__ RowOf(const VerifyArgs &a, int row)
      : x(static_cast<const T *>(a.logits) + size_t(row) * a.stride), lead(int(reinterpret_cast<size_t>(x) / sizeof(T) % E)), vocab(a.vocab) {}
  typedef uint32_t Raw __attribute__((ext_vector_type(4)));
  typedef T Values __attribute__((ext_vector_type(E)));
  // (elements past the row's ends: -inf, which weighs nothing)
  __device__ __forceinline__ Raw raw(int c) const {
    const int i = c * E - lead;
    if (i >= 0 && i + E <= vocab) return *reinterpret_cast<const Raw *>(x + i);
    Values v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = T(-INFINITY);
    if (i < vocab)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= 0 && i + e < vocab) v[e] = x[i + e];
    return __builtin_bit_cast(Raw, v);
  }
  static __device__ __forceinline__ void floats(Raw r, float (&v)[E]) {
    const Values u = __builtin_bit_cast(Values, r);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = float(u[e]);
  }
  __device__ __forceinline__ void load(int c, float (&v)[E]) const { floats(raw(c), v); }
};

// Sums, largest and first of the largest of each part of each row: J pieces a
// thread.
template <class T, int J>
__global__ __launch_bounds__(kThreads) void stats_kernel(VerifyArgs a) {
  constexpr int E = RowOf<T>::E;
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int firsts[kWaves];
  const int part = int(blockIdx.y), row = int(blockIdx.x), lane = threadIdx.x & (kWave - 1), wave = int(threadIdx.x) / kWave;
  const RowOf<T> r(a, row);
  const int c0 = part * (J * kThreads) + int(threadIdx.x);
  typename RowOf<T>::Raw raw[J];
  const int i0 = part * (J * kThreads * E) - r.lead;
  if (i0 >= 0 && i0 + J * kThreads * E <= a.vocab) {   // the whole part is inside the row
    const typename RowOf<T>::Raw *from = reinterpret_cast<const typename RowOf<T>::Raw *>(r.x + i0) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < J; ++j) raw[j] = from[j * kThreads];
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) raw[j] = r.raw(c0 + j * kThreads);
  }
  const int s = sequence_of(a.offsets, a.n_seqs, row, lane);
  if (s < 0 || row >= a.offsets[s + 1]) return;
  const Heat h = heat_of(a, s);
  if (part == 0 && threadIdx.x == 0 && row == max(a.offsets[s], 0)) a.tickets[s] = 0;
  float top = -INFINITY;   // (a NaN stays)
#pragma unroll
  for (int j = 0; j < J; ++j) {
    float v[E];
    r.floats(raw[j], v);
#pragma unroll
    for (int e = 0; e < E; ++e) top = __builtin_elementwise_maximum(top, v[e]);
  }
  const bool nan = top != top;
  top = wave_max(top, lane);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
  // (from the packed values again: as floats they would take the registers of half the waves)
#pragma unroll
  for (int j = 0; j < J; ++j) asm volatile("" : "+v"(raw[j]));
  double sum = 0.0;
  int first = 0x7FFFFFFF;
  if (h.t > 0.0f) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float v[E];
      r.floats(raw[j], v);
#pragma unroll
      for (int e = 0; e < E; ++e) sum += weight_of(v[e], top, h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float v[E];
      r.floats(raw[j], v);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[e] == top) first = min(first, (c0 + j * kThreads) * E - r.lead + e);
    }
    first = wave_min(first, lane);
  }
  if (nan || top == INFINITY) sum = __builtin_nan("");
  sum = wave_sum(sum, lane);
  if (lane == 0) sums[wave] = sum, firsts[wave] = first;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += sums[w], first = min(first, firsts[w]);
  a.parts[size_t(row) * a.n_parts + part] = Part{sum, top, first};
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
  using RowOf<T>::E, RowOf<T>::lead, RowOf<T>::vocab;
  const Row &r;
  const Heat &h;
  const float *q;
  bool q_aligned;
  __device__ __forceinline__ Piece(const VerifyArgs &a, int row, const Row &r, const Heat &h)
      : RowOf<T>(a, row), r(r), h(h), q(a.probs + size_t(row) * a.probs_stride), q_aligned(lead == 0 && reinterpret_cast<size_t>(q) % 16 == 0) {}
  template <bool OVER>
  __device__ __forceinline__ void weights(int c, int skip, double (&w)[E]) const {
    float v[E], u[E];
    const int i0 = c * E - lead;
    if constexpr (OVER) {
      if (q_aligned && i0 + E <= vocab) {
        load_floats<E>(q + i0, u);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = i0 + e >= 0 && i0 + e < vocab ? q[i0 + e] : 0.0f;
      }
    }
    this->load(c, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = weight_of(v[e], r.top, h);
      if constexpr (OVER) w[e] = fmax(fma(double(u[e]), -r.total, w[e]), 0.0);
      else if (i0 + e == skip) w[e] = 0.0;
    }
  }
  template <bool OVER, int J>
  __device__ __forceinline__ void sums(int part, int skip, double (&mine)[J]) const {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      double w[E];
      weights<OVER>((part * J + j) * kThreads + int(threadIdx.x), skip, w);
      mine[j] = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) mine[j] += w[e];
    }
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

// A workgroup a sequence, or one for each part where q may be needed: each finds
// the row that the sequence stops at, four rows at a time, a wave each.  The token
// there: parts' sums are known, or, of p - q, taken by the sequence's workgroups;
// the row's wave (or the last workgroup) finds the part that the threshold falls into,
// the workgroup the element in it.  What it costs is its chain of loads: offsets,
// then parts' sums and drafts, then the drafted tokens' logits, then the part found.
template <class T, int J>
__global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a) {
  constexpr int E = RowOf<T>::E, PART = J * kThreads;   // pieces of a part
  __shared__ Row rows[kWaves];
  __shared__ int stops[kWaves];
  __shared__ double scan[J][kWaves];
  __shared__ Place place;
  __shared__ int at, last, joins;
  const int s = int(blockIdx.x), part = int(blockIdx.y), lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int begin = max(a.offsets[s], 0), end = min(a.offsets[s + 1], a.n_rows);
  const Heat h = heat_of(a, s);
  if (begin >= end) {
    if (part == 0 && threadIdx.x == 0) a.accepted[s] = 0;
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
  if (part == 0) {
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
  if (!over && part != 0) return;
  const Piece<T> x(a, row, r, h);
  const Part *parts = a.parts + size_t(row) * a.n_parts;
  double mine[J];
  // the sum of every thread's pieces over the workgroup
  const auto block_sum = [&]() __attribute__((always_inline)) {
    double all = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) all += mine[j];
    all = wave_sum(all, lane);
    if (lane == 0) scan[0][wave] = all;
    __syncthreads();
    all = scan[0][0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) all += scan[0][v];
    __syncthreads();
    return all;
  };
  bool from_rest = over;   // weights are those of p - q
  int skip = -1;           // the token that p is to lack
  if (threadIdx.x == 0) at = 0x7FFFFFFF, last = -1;
  if (over) {
    double *sums = a.rest + size_t(s) * a.n_parts;
    x.template sums<true, J>(part, -1, mine);
    const double sum = block_sum();
    if (threadIdx.x == 0) {
      __hip_atomic_store(sums + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __threadfence();
      joins = atomicAdd(a.tickets + s, 1u) == unsigned(a.n_parts - 1);
    }
    __syncthreads();
    if (!joins) return;
    __threadfence();
    if (wave == owner) {
      const auto of = [&](int i) __attribute__((always_inline)) { return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
      const Place p = place_of(a.n_parts, double(u.y), lane < a.n_parts ? of(lane) : 0.0, lane, of);
      if (lane == 0) place = p;
    }
    __syncthreads();
    if (place.part < 0) from_rest = false;   // nothing is left: from p
    __syncthreads();
  } else {
    // the part that lacks the drafted token: the difference keeps 42 bits, or it is
    // summed without the token
    __shared__ int without;
    if (wave == owner) {
      const int lacking = known ? (token + x.lead) / (PART * E) : -1;
      const double with = lane == lacking ? share : lacking >= kWave ? part_weight(parts[lacking], r.top, h) : INFINITY;
      const bool lost = lacking >= 0 && __builtin_amdgcn_ballot_w64(!(with - weight > with * 0x1p-10) && with < INFINITY) != 0;
      if (lane == 0) without = known ? token : -1, joins = lost;
    }
    __syncthreads();
    skip = without;
    if (joins) {
      x.template sums<false, J>((skip + x.lead) / (PART * E), skip, mine);
      weight = block_sum();
    }
  }
  if (!from_rest) {
    for (int again = 0; again < 2; ++again) {
      if (wave == owner) {
        const int lacking = skip >= 0 ? (skip + x.lead) / (PART * E) : -1;
        const auto less = [&](int i, double v) __attribute__((always_inline)) { return i != lacking ? v : joins && !over ? weight : v - weight; };
        const auto of = [&](int i) __attribute__((always_inline)) { return less(i, part_weight(parts[i], r.top, h)); };
        const Place p = place_of(a.n_parts, double(u.y), lane < a.n_parts ? less(lane, share) : 0.0, lane, of);
        if (lane == 0) place = p;
      }
      __syncthreads();
      if (place.part >= 0) break;
      skip = -1;   // nothing is left without the token: from p
      __syncthreads();
    }
    if (place.part < 0) return;   // (p weighs something)
  }
  // the first piece past the threshold (or the last with a weight), then in it the
  // element, by the piece's thread
  const double target = place.target;
  const int c0 = place.part * PART;
  if (from_rest) x.template sums<true, J>(place.part, -1, mine);
  else x.template sums<false, J>(place.part, skip, mine);
  double upto[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    upto[j] = wave_scan(mine[j]);
    if (lane == kWave - 1) scan[j][wave] = upto[j];
  }
  __syncthreads();
  double before = 0.0, base = 0.0;
  int past = 0x7FFFFFFF, behind = -1;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    double here = base;   // all before this wave's pieces of round j
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      if (v < wave) here += scan[j][v];
      base += scan[j][v];
    }
    if (mine[j] > 0.0) {
      behind = j * kThreads + int(threadIdx.x);
      if (past == 0x7FFFFFFF && here + upto[j] > target) past = behind, before = here + (upto[j] - mine[j]);
    }
  }
  if (past < 0x7FFFFFFF) atomicMin(&at, past);
  if (behind >= 0) atomicMax(&last, behind);
  __syncthreads();
  const int piece = at < 0x7FFFFFFF ? at : last;
  if (piece < 0 || piece % kThreads != int(threadIdx.x)) return;
  double w[E];
  if (from_rest) x.template weights<true>(c0 + piece, -1, w);
  else x.template weights<false>(c0 + piece, skip, w);
  int token_at = -1;
  bool done = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    before += w[e];
    if (!done && w[e] > 0.0) token_at = (c0 + piece) * E - x.lead + e;
    done = done || (piece == past && w[e] > 0.0 && before > target);
  }
  a.tokens[row] = token_at;
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

// Pieces of 16 bytes a thread: parts of 4 while that still makes four workgroups a
// CU, else of 2.
int pieces_of(size_t rows, size_t vocab, int type) {
  const size_t part = kThreads * 8 * (16 / type_bytes(type));
  return rows * (vocab / part) >= 1024 ? 8 : 2;
}
size_t parts_of(size_t rows, size_t vocab, int type) {
  const size_t e = 16 / type_bytes(type), part = kThreads * e * pieces_of(rows, vocab, type);
  return (vocab + e - 1 + part - 1) / part;   // (wherever in a piece a row begins)
}

template <class T, int J>
int launch(const VerifyArgs &a, hipStream_t st) {
  if (a.n_rows) stats_kernel<T, J><<<dim3(unsigned(a.n_rows), unsigned(a.n_parts)), kThreads, 0, st>>>(a);
  const int r = launch_err("verify");
  if (r) return r;
  pick_kernel<T, J><<<dim3(unsigned(a.n_seqs), a.probs ? unsigned(a.n_parts) : 1u), kThreads, 0, st>>>(a);
  return launch_err("verify pick");
}
template <class T>
int launch(const VerifyArgs &a, int pieces, hipStream_t st) {
  return pieces == 8 ? launch<T, 8>(a, st) : launch<T, 2>(a, st);
}

struct Layout { size_t rest, tickets, all; };
Layout layout(const lmx_drafts *d, int type) {
  const size_t parts = parts_of(d->n_rows, d->vocab, type);
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
  a.n_parts = int(parts_of(d->n_rows, d->vocab, type));
  const int pieces = pieces_of(d->n_rows, d->vocab, type);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch<float>(a, pieces, st);
  case LMX_F16: return launch<f16>(a, pieces, st);
  default: return launch<bf16>(a, pieces, st);
  }
}

}  // extern "C"
