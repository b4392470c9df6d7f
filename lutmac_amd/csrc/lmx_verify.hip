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
  // (elements past the row's ends: -inf, which weighs nothing)
  __device__ __forceinline__ void load(int c, float (&v)[E]) const {
    const int i = c * E - lead;
    if (i >= 0 && i + E <= vocab) {
      load_floats<E>(x + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = -INFINITY;
      if (i < vocab)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i + e >= 0 && i + e < vocab) v[e] = float(x[i + e]);
    }
  }
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
  float v[J][E];
#pragma unroll
  for (int j = 0; j < J; ++j) r.load(c0 + j * kThreads, v[j]);
  const int s = sequence_of(a.offsets, a.n_seqs, row, lane);
  if (s < 0 || row >= a.offsets[s + 1]) return;
  const Heat h = heat_of(a, s);
  if (part == 0 && threadIdx.x == 0 && row == max(a.offsets[s], 0)) a.tickets[s] = 0;
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      nan |= v[j][e] != v[j][e];
      top = fmaxf(top, v[j][e]);
    }
  top = wave_max(top, lane);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
  double sum = 0.0;
  int first = 0x7FFFFFFF;
  if (h.t > 0.0f) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) sum += weight_of(v[j][e], top, h);
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[j][e] == top) first = min(first, (c0 + j * kThreads) * E - r.lead + e);
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
__device__ __forceinline__ double part_weight(const Part &p, const Row &r, const Heat &h) { return p.sum * weight_of(p.top, r.top, h); }
// By a wave, each lane with its first part (of lane `lane`) in `first`.
__device__ __forceinline__ Row row_of(const Part *p, int n, const Part &first, const Heat &h, int lane) {
  Row r{0.0, first.top, 0x7FFFFFFF};
  for (int i = lane + kWave; i < n; i += kWave) r.top = fmaxf(r.top, p[i].top);
  r.top = wave_max(r.top, lane);
  const auto add = [&](const Part &q) {
    r.total += h.t > 0.0f || q.sum != q.sum ? q.sum * weight_of(q.top, r.top, h) : 0.0;
    if (q.top == r.top) r.best = min(r.best, q.best);
  };
  add(first);
  for (int i = lane + kWave; i < n; i += kWave) add(p[i]);
  r.total = wave_sum(r.total, lane);
  if (h.t == 0.0f) {
    r.best = wave_min(r.best, lane);
    if (r.total == 0.0) r.total = 1.0;
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

// A workgroup a sequence, or one for each part where q may be needed: each finds
// the row that the sequence stops at, four rows at a time.  The token there: parts'
// sums are known, or, of p - q, taken by the sequence's workgroups; the last of them
// finds the part that the threshold falls into, then the element in it.
template <class T, int J>
__global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a) {
  constexpr int E = RowOf<T>::E, PART = J * kThreads;   // pieces of a part
  __shared__ Row rows[kWaves];
  __shared__ int stops[kWaves];
  __shared__ double scan[J][kWaves];
  __shared__ double chosen_target;
  __shared__ int chosen, at, last, joins;
  const int s = int(blockIdx.x), part = int(blockIdx.y), lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int begin = max(a.offsets[s], 0), end = min(a.offsets[s + 1], a.n_rows);
  const Heat h = heat_of(a, s);
  if (begin >= end) {
    if (part == 0 && threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  int row = begin;
  Row r;
  for (;; row += kWaves) {
    const int mine = row + wave;
    if (mine < end) {
      // (parts and token on their way at once, then the token's logit and share)
      const Part *parts = a.parts + size_t(mine) * a.n_parts;
      const Part first = lane < a.n_parts ? parts[lane] : Part{0.0, -INFINITY, 0x7FFFFFFF};
      const int token = a.drafts[mine];
      const double u = a.uniforms[mine].x;
      const bool drafted = mine != end - 1 && token >= 0 && token < a.vocab;
      float l = 0.0f, q = 1.0f;
      if (drafted) {
        l = float((static_cast<const T *>(a.logits) + size_t(mine) * a.stride)[token]);
        if (a.probs) q = a.probs[size_t(mine) * a.probs_stride + token];
      }
      const Row x = row_of(parts, a.n_parts, first, h, lane);
      const double w = h.t > 0.0f ? weight_of(l, x.top, h) : token == x.best ? 1.0 : 0.0;
      const bool go = drafted && x.total > 0.0 && u * double(q) * x.total < w;
      if (lane == 0) rows[wave] = x, stops[wave] = !go;
    } else if (lane == 0) {
      stops[wave] = 1;
    }
    __syncthreads();
    int n = 0;
    while (n < kWaves && !stops[n]) ++n;
    if (n < kWaves) {   // (the last row stops)
      row += n;
      r = rows[n];
      break;
    }
    __syncthreads();
  }
  if (part == 0) {
    for (int i = begin + int(threadIdx.x); i < end; i += kThreads)
      if (i != row) a.tokens[i] = i < row ? a.drafts[i] : -1;
    if (threadIdx.x == 0) {
      a.accepted[s] = row - begin;
      if (!(r.total > 0.0)) a.tokens[row] = -1;
    }
  }
  if (!(r.total > 0.0)) return;
  if (h.t == 0.0f) {   // (whatever q is: all that p has over it is there)
    if (part == 0 && threadIdx.x == 0) a.tokens[row] = r.best;
    return;
  }
  const int token = a.drafts[row];
  const bool rest = row != end - 1, known = token >= 0 && token < a.vocab;
  const bool over = rest && a.probs;
  if (!over && part != 0) return;
  const Piece<T> x(a, row, r, h);
  double *sums = a.rest + size_t(s) * a.n_parts;
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
  int skip = -1;           // the token that p is to lack, its part and what is left of that
  int lacking = -1;
  double less = 0.0;
  if (over) {
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
  } else if (rest && known) {
    // (the difference keeps 42 bits, or the part is summed without the token)
    skip = token;
    lacking = (token + x.lead) / (PART * E);
    const double with = part_weight(parts[lacking], r, h);
    less = with - weight_of(float(x.x[token]), r.top, h);
    if (!(less > with * 0x1p-10)) {
      x.template sums<false, J>(lacking, skip, mine);
      less = block_sum();
    }
  }
  // Parts' sums in order, and the first that the threshold falls into: a wave, 64
  // parts at a time.
  for (int again = 0; again < 2; ++again) {
    if (wave == 0) {
      const auto sum_of = [&](int i) __attribute__((always_inline)) {
        if (i >= a.n_parts) return 0.0;
        if (from_rest) return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return i == lacking ? less : part_weight(parts[i], r, h);
      };
      const double v0 = sum_of(lane);
      double all = wave_sum(v0, lane);
      for (int i = kWave; i < a.n_parts; i += kWave) all += wave_sum(sum_of(i + lane), lane);
      int found = -1, behind = -1;
      double target = double(a.uniforms[row].y) * all, before = 0.0;
      for (int i = 0; i < a.n_parts && found < 0; i += kWave) {
        const double v = i == 0 ? v0 : sum_of(i + lane), upto = before + wave_scan(v);
        const uint64_t past = __builtin_amdgcn_ballot_w64(v > 0.0 && upto > target), some = __builtin_amdgcn_ballot_w64(v > 0.0);
        if (past) {
          found = __builtin_ctzll(past);
          target -= lane_value(upto - v, found);
          found += i;
        } else {
          if (some) behind = i + 63 - __builtin_clzll(some);
          before = lane_value(upto, kWave - 1);
        }
      }
      if (found < 0) found = behind, target = INFINITY;   // (rounding, or a number of 1 and more: the last)
      if (lane == 0) chosen = all > 0.0 ? found : -1, chosen_target = target, at = 0x7FFFFFFF, last = -1;
    }
    __syncthreads();
    if (chosen >= 0) break;
    // nothing is left: from p
    from_rest = false;
    skip = lacking = -1;
    __syncthreads();
  }
  if (chosen < 0) return;   // (p weighs something)
  // the first piece past the threshold (or the last with a weight), then in it the
  // element, by the piece's thread
  const double target = chosen_target;
  if (from_rest) x.template sums<true, J>(chosen, -1, mine);
  else x.template sums<false, J>(chosen, skip, mine);
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
  const int c = chosen * PART + piece;
  if (from_rest) x.template weights<true>(c, -1, w);
  else x.template weights<false>(c, skip, w);
  int token_at = -1;
  bool done = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    before += w[e];
    if (!done && w[e] > 0.0) token_at = c * E - x.lead + e;
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
  const size_t part = kThreads * 4 * (16 / type_bytes(type));
  return rows * (vocab / part) >= 1024 ? 4 : 2;
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
  return pieces == 4 ? launch<T, 4>(a, st) : launch<T, 2>(a, st);
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
