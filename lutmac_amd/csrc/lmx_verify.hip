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

// 2^y for y <= 0: 2^k times the series of 2^f, |f| <= 1/2, to the 10th power (the
// next term is below 2^-42).  Far below, and for NaN (-inf - -inf), 0.
__device__ __forceinline__ double exp2_neg(double y) {
  y = fmax(y, -1100.0);
  const double k = rint(y), f = y - k;
  double p = 7.054911620801123e-09;   // log(2)^n / n!
  p = fma(p, f, 1.0178086009239699e-07);
  p = fma(p, f, 1.321548679014431e-06);
  p = fma(p, f, 1.525273380405984e-05);
  p = fma(p, f, 1.5403530393381608e-04);
  p = fma(p, f, 1.3333558146428443e-03);
  p = fma(p, f, 9.618129107628477e-03);
  p = fma(p, f, 5.550410866482158e-02);
  p = fma(p, f, 2.402265069591007e-01);
  p = fma(p, f, 6.931471805599453e-01);
  p = fma(p, f, 1.0);
  return ldexp(p, int(k));
}
constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) v = fmaxf(v, __shfl_xor(v, d));
  return v;
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

// A sequence's temperature and what logits' differences are multiplied by: (0, 0)
// for a greedy one.
struct Heat {
  float t;
  double by;
};
__device__ __forceinline__ Heat heat_of(const VerifyArgs &a, int s) {
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  return t > 0.0f ? Heat{t, kLog2e / double(t)} : Heat{0.0f, 0.0};
}
__device__ __forceinline__ double weight_of(float l, float top, double by) { return exp2_neg((double(l) - double(top)) * by); }

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
  top = wave_max(top);
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
      for (int e = 0; e < E; ++e) sum += weight_of(v[j][e], top, h.by);
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[j][e] == top) first = min(first, (c0 + j * kThreads) * E - r.lead + e);
#pragma unroll
    for (int d = kWave / 2; d; d /= 2) first = min(first, __shfl_xor(first, d));
  }
  if (nan || top == INFINITY) sum = __builtin_nan("");
  sum = wave_sum(sum);
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
// By a wave.
__device__ __forceinline__ Row row_of(const VerifyArgs &a, int row, const Heat &h, int lane) {
  const Part *p = a.parts + size_t(row) * a.n_parts;
  Row r{0.0, -INFINITY, 0x7FFFFFFF};
  for (int i = lane; i < a.n_parts; i += kWave) r.top = fmaxf(r.top, p[i].top);
  r.top = wave_max(r.top);
  for (int i = lane; i < a.n_parts; i += kWave) {
    const Part q = p[i];
    r.total += h.t > 0.0f || q.sum != q.sum ? q.sum * weight_of(q.top, r.top, h.by) : 0.0;
    if (q.top == r.top) r.best = min(r.best, q.best);
  }
  r.total = wave_sum(r.total);
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) r.best = min(r.best, __shfl_xor(r.best, d));
  if (h.t == 0.0f && r.total == 0.0) r.total = 1.0;
  if (r.top == -INFINITY || !(r.total > 0.0)) r.total = 0.0;
  return r;
}

// Inclusive sums over a wave's lanes.
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const double o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// A workgroup a sequence, or one for each part where q may be needed: each finds
// the row that the sequence stops at, four rows at a time.  The token there: parts'
// sums are known, or, of p - q, taken by the sequence's workgroups; the last of them
// finds the part that the threshold falls into, then the element in it.
template <class T, int J>
__global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a) {
  constexpr int E = RowOf<T>::E;
  __shared__ Row rows[kWaves];
  __shared__ int stops[kWaves];
  __shared__ double scan[J][kWaves];
  __shared__ double chosen_sum;
  __shared__ int chosen, at, last, joins;
  const int s = int(blockIdx.x), part = int(blockIdx.y), lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int begin = max(a.offsets[s], 0), end = min(a.offsets[s + 1], a.n_rows);
  if (begin >= end) {
    if (part == 0 && threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  const Heat h = heat_of(a, s);
  int row = begin;
  Row r;
  for (;; row += kWaves) {
    const int mine = row + wave;
    if (mine < end) {
      const int token = a.drafts[mine];
      const bool drafted = mine != end - 1 && token >= 0 && token < a.vocab;
      float l = 0.0f, q = 1.0f;
      if (drafted) {
        l = float((static_cast<const T *>(a.logits) + size_t(mine) * a.stride)[token]);
        if (a.probs) q = a.probs[size_t(mine) * a.probs_stride + token];
      }
      const Row x = row_of(a, mine, h, lane);
      const double w = h.t > 0.0f ? weight_of(l, x.top, h.by) : token == x.best ? 1.0 : 0.0;
      const bool go = drafted && x.total > 0.0 && double(a.uniforms[mine].x) * double(q) * x.total < w;
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
  const int token = a.drafts[row];
  const bool rest = row != end - 1;
  const float *q = rest && a.probs ? a.probs + size_t(row) * a.probs_stride : nullptr;
  const bool q_aligned = q && reinterpret_cast<size_t>(q) % 16 == 0;
  const RowOf<T> x(a, row);
  // weights of a piece: of p, of p without the drafted token, or of what p has over q
  enum Kind { kAll, kWithout, kOver };
  const auto weights = [&](int c, Kind kind, double (&w)[E]) {
    float v[E];
    x.load(c, v);
    const int i0 = c * E - x.lead;
    float u[E];
    if (kind == kOver) {
      if (q_aligned && x.lead == 0 && i0 + E <= a.vocab) {
        load_floats<E>(q + i0, u);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = i0 + e >= 0 && i0 + e < a.vocab ? q[i0 + e] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = h.t > 0.0f ? weight_of(v[e], r.top, h.by) : i0 + e == r.best ? 1.0 : 0.0;
      if (kind == kOver) w[e] = fmax(w[e] - double(u[e]) * r.total, 0.0);
      else if (kind == kWithout && i0 + e == token) w[e] = 0.0;
    }
  };
  // the sum of a part's weights, of every thread's J pieces (mine) and over the workgroup
  const auto part_sum = [&](int part, Kind kind, double (&mine)[J]) {
    double all = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      double w[E];
      weights(part * (J * kThreads) + j * kThreads + int(threadIdx.x), kind, w);
      mine[j] = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) mine[j] += w[e];
      all += mine[j];
    }
    all = wave_sum(all);
    __syncthreads();
    if (lane == 0) scan[0][wave] = all;
    __syncthreads();
    all = scan[0][0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) all += scan[0][v];
    __syncthreads();
    return all;
  };
  double mine[J];
  Kind kind = q ? kOver : rest && token >= 0 && token < a.vocab ? kWithout : kAll;
  double *sums = a.rest + size_t(s) * a.n_parts;
  if (kind == kOver) {
    const double sum = part_sum(part, kind, mine);
    if (threadIdx.x == 0) {
      __hip_atomic_store(sums + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __threadfence();
      joins = atomicAdd(a.tickets + s, 1u) == unsigned(a.n_parts - 1);
    }
    __syncthreads();
    if (!joins) return;
    __threadfence();
  } else if (part != 0) {
    return;
  }
  // Parts' sums in order, and the first that the threshold falls into: a wave, 64
  // parts at a time.
  const int without = kind == kWithout ? (token + x.lead) / (J * kThreads * E) : -1;   // the part that lacks a token
  double less = 0.0;
  if (without >= 0) less = part_sum(without, kWithout, mine);
  const Part *parts = a.parts + size_t(row) * a.n_parts;
  for (int again = 0; again < 2; ++again) {
    if (wave == 0) {
      const auto sum_of = [&](int i) {
        if (i >= a.n_parts) return 0.0;
        if (kind == kOver) return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (i == without && kind == kWithout) return less;
        if (h.t == 0.0f) return parts[i].best == r.best && parts[i].top == r.top ? 1.0 : 0.0;
        return parts[i].sum * weight_of(parts[i].top, r.top, h.by);
      };
      double all = 0.0;
      for (int i = 0; i < a.n_parts; i += kWave) all += wave_sum(sum_of(i + lane));
      int found = -1, behind = -1;
      double target = double(a.uniforms[row].y) * all, before = 0.0;
      for (int i = 0; i < a.n_parts && found < 0; i += kWave) {
        const double v = sum_of(i + lane), upto = before + wave_scan(v, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(v > 0.0 && upto > target), some = __builtin_amdgcn_ballot_w64(v > 0.0);
        if (past) {
          found = __builtin_ctzll(past);
          target -= __shfl(upto - v, found);
          found += i;
        } else {
          if (some) behind = i + 63 - __builtin_clzll(some);
          before = __shfl(upto, kWave - 1);
        }
      }
      if (found < 0) found = behind, target = INFINITY;   // (rounding, or a number of 1 and more: the last)
      if (lane == 0) chosen = all > 0.0 ? found : -1, chosen_sum = target, at = 0x7FFFFFFF, last = -1;
    }
    __syncthreads();
    if (chosen >= 0) break;
    // nothing is left of p - q: from p
    kind = kAll;
    __syncthreads();
  }
  if (chosen < 0) return;   // (p weighs something)
  const double target = chosen_sum;
  part_sum(chosen, kind, mine);
  double upto[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    upto[j] = wave_scan(mine[j], lane);
    if (lane == kWave - 1) scan[j][wave] = upto[j];
  }
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    double base = before;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      if (v < wave) base += scan[j][v];
      before += scan[j][v];
    }
    const int c = chosen * (J * kThreads) + j * kThreads + int(threadIdx.x);
    if (mine[j] > 0.0) {
      double w[E];
      weights(c, kind, w);
      double sum = base + (upto[j] - mine[j]);
      const bool here = base + upto[j] > target;
      int end_at = -1, found = -1;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sum += w[e];
        if (w[e] > 0.0) end_at = c * E - x.lead + e;
        if (found < 0 && sum > target) found = c * E - x.lead + e;
      }
      if (here) atomicMin(&at, found >= 0 ? found : end_at);
      atomicMax(&last, end_at);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.tokens[row] = at < 0x7FFFFFFF ? at : last;
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

// Pieces of 16 bytes a thread: parts of 8 while that still makes four workgroups a
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
