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
  Part *parts;   // [n_rows][n_parts]
  int n_parts;
};

// e^y for y <= 0: 2^k times the series of e^f, |f| <= log(2) / 2, to the 11th power
// (the next term is below 2^-47).  -inf gives 0.
__device__ __forceinline__ double exp_neg(double y) {
  const double k = rint(fmax(y, -800.0) * 1.4426950408889634074);
  const double f = fma(k, -2.3190468138462996e-17, fma(k, -0.69314718055994528623, fmax(y, -800.0)));
  double p = 1.0 / 39916800.0;
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return ldexp(p, int(k));
}

__device__ __forceinline__ double lane_xor_f64(double v, int d) { return __shfl_xor(v, d); }
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = kWave / 2; d; d /= 2) v += lane_xor_f64(v, d);
  return v;
}

// The last sequence whose first row is at most r (-1: none).
__device__ __forceinline__ int sequence_of(const int *offsets, int n, int r) {
  if (n == 0 || offsets[0] > r) return -1;
  int lo = 0;
  while (n > 1) {
    const int half = n / 2;
    const bool up = offsets[lo + half] <= r;
    lo = up ? lo + half : lo;
    n = up ? n - half : half;
  }
  return lo;
}

__device__ __forceinline__ float temperature_of(const VerifyArgs &a, int s) {
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  return t > 0.0f ? t : 0.0f;
}

// Weight of a logit: the inverse temperature is 0 for a greedy row.
__device__ __forceinline__ double weight_of(float l, float top, double inv) {
  return l == top ? 1.0 : l == -INFINITY ? 0.0 : exp_neg((double(l) - double(top)) * inv);
}

constexpr int kThreads = 256, kWaves = kThreads / kWave, kEach = 32;
constexpr int kPart = kThreads * kEach;   // logits of a part

// Sums, largest and first of the largest of each part of each row.
template <class T>
__global__ __launch_bounds__(kThreads) void stats_kernel(VerifyArgs a) {
  __shared__ float tops[kWaves];
  __shared__ double sums[kWaves];
  __shared__ int firsts[kWaves];
  const int part = int(blockIdx.y), row = int(blockIdx.x), lane = threadIdx.x & (kWave - 1), wave = int(threadIdx.x) / kWave;
  const int s = sequence_of(a.offsets, a.n_seqs, row);
  if (s < 0 || row >= a.offsets[s + 1]) return;
  const T *x = static_cast<const T *>(a.logits) + size_t(row) * a.stride;
  const float t = temperature_of(a, s);
  float v[kEach], top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = part * kPart + j * kThreads + int(threadIdx.x);
    v[j] = i < a.vocab ? float(x[i]) : -INFINITY;
    nan |= v[j] != v[j];
    top = fmaxf(top, v[j]);
  }
  for (int d = kWave / 2; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
  double sum = 0.0;
  int first = 0x7FFFFFFF;
  const double inv = t > 0.0f ? 1.0 / double(t) : 0.0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (t > 0.0f) sum += weight_of(v[j], top, inv);
    else if (v[j] == top) first = min(first, part * kPart + j * kThreads + int(threadIdx.x));
  }
  if (nan || top == INFINITY) sum = __builtin_nan("");
  if (top == -INFINITY && !nan) sum = 0.0;
  sum = wave_sum(sum);
  for (int d = kWave / 2; d; d /= 2) first = min(first, __shfl_xor(first, d));
  if (lane == 0) sums[wave] = sum, firsts[wave] = first;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kWaves; ++w) sum += sums[w], first = min(first, firsts[w]);
  a.parts[size_t(row) * a.n_parts + part] = Part{sum, top, first};
}

// A row's distribution: weights over `total`.
struct Row {
  double total;   // not positive: none
  float top;
  int best;
};
__device__ __forceinline__ Row row_of(const VerifyArgs &a, int row, float t) {
  const Part *p = a.parts + size_t(row) * a.n_parts;
  const double inv = t > 0.0f ? 1.0 / double(t) : 0.0;
  Row r{0.0, -INFINITY, -1};
  for (int i = 0; i < a.n_parts; ++i) r.top = fmaxf(r.top, p[i].top);
  bool bad = false;
  for (int i = 0; i < a.n_parts; ++i) {
    bad |= p[i].sum != p[i].sum;
    if (t > 0.0f) {
      if (p[i].top > -INFINITY) r.total += p[i].sum * weight_of(p[i].top, r.top, inv);
    } else if (r.best < 0 && p[i].top == r.top) {
      r.best = p[i].best;
    }
  }
  if (t == 0.0f) r.total = 1.0;
  if (bad || r.top == -INFINITY) r.total = 0.0;
  return r;
}

template <class T>
__device__ __forceinline__ double weight_at(const VerifyArgs &a, int row, int i, const Row &r, float t) {
  if (t == 0.0f) return i == r.best ? 1.0 : 0.0;
  const float l = float((static_cast<const T *>(a.logits) + size_t(row) * a.stride)[i]);
  return weight_of(l, r.top, 1.0 / double(t));
}

// A workgroup a sequence: the first row that it stops at, and the token there.
template <class T>
__global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a) {
  __shared__ double sums[kThreads];
  const int s = int(blockIdx.x), begin = max(a.offsets[s], 0), end = min(a.offsets[s + 1], a.n_rows);
  const float t = temperature_of(a, s);
  if (begin >= end) {
    if (threadIdx.x == 0) a.accepted[s] = 0;
    return;
  }
  int row = begin;
  Row r;
  bool known;
  for (;; ++row) {
    r = row_of(a, row, t);
    const int token = a.drafts[row];
    known = token >= 0 && token < a.vocab;
    if (row == end - 1 || !known || !(r.total > 0.0)) break;
    const double q = a.probs ? double(a.probs[size_t(row) * a.probs_stride + token]) : 1.0;
    if (!(double(a.uniforms[row].x) * q * r.total < weight_at<T>(a, row, token, r, t))) break;
  }
  for (int i = begin + int(threadIdx.x); i < end; i += kThreads)
    if (i != row) a.tokens[i] = i < row ? a.drafts[i] : -1;
  if (threadIdx.x == 0) a.accepted[s] = row - begin;
  if (!(r.total > 0.0)) {
    if (threadIdx.x == 0) a.tokens[row] = -1;
    return;
  }
  const int token = a.drafts[row];
  const float *q = a.probs ? a.probs + size_t(row) * a.probs_stride : nullptr;
  bool rest = row != end - 1;
  const auto weight = [&](int i) {
    double w = weight_at<T>(a, row, i, r, t);
    if (rest) w = q ? fmax(w - double(q[i]) * r.total, 0.0) : i == token && known ? 0.0 : w;
    return w;
  };
  const double u = a.uniforms[row].y;
  const int each = (a.vocab + kThreads - 1) / kThreads, i0 = min(int(threadIdx.x) * each, a.vocab), i1 = min(i0 + each, a.vocab);
  for (;;) {
    double mine = 0.0;
    for (int i = i0; i < i1; ++i) mine += weight(i);
    sums[threadIdx.x] = mine;

    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int i = 0; i < kThreads; ++i) {
        const double w = sums[i];
        sums[i] = all;
        all += w;
      }
      sums[0] = all;
    }
    __syncthreads();
    const double all = sums[0], before = threadIdx.x == 0 ? 0.0 : sums[threadIdx.x];
    if (rest && !(all > 0.0)) {   // nothing is left: from p
      rest = false;
      __syncthreads();
      continue;
    }
    // the first past the threshold, or the last with a weight
    double upto = before;
    int mine_at = -1, last = -1;
    for (int i = i0; i < i1 && mine_at < 0; ++i) {
      const double w = weight(i);
      upto += w;
      if (w > 0.0) last = i;
      if (upto > u * all) mine_at = i;
    }
    __shared__ int at, end_at;
    if (threadIdx.x == 0) at = 0x7FFFFFFF, end_at = -1;
    __syncthreads();
    if (mine_at >= 0) atomicMin(&at, mine_at);
    if (last >= 0) atomicMax(&end_at, last);
    __syncthreads();
    if (threadIdx.x == 0) a.tokens[row] = at < 0x7FFFFFFF ? at : end_at;
    return;
  }
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

template <class T>
int launch(const VerifyArgs &a, hipStream_t st) {
  if (a.n_rows) stats_kernel<T><<<dim3(unsigned(a.n_rows), unsigned(a.n_parts)), kThreads, 0, st>>>(a);
  const int r = launch_err("verify");
  if (r) return r;
  pick_kernel<T><<<unsigned(a.n_seqs), kThreads, 0, st>>>(a);
  return launch_err("verify pick");
}

size_t parts_of(size_t vocab) { return (vocab + kPart - 1) / kPart; }

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_verify_drafts_workspace(const lmx_drafts *d, int type, size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int r = check_sizes(d, type);
  if (r) return r;
  *bytes = d->n_rows * parts_of(d->vocab) * sizeof(Part);
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
  a.parts = static_cast<Part *>(workspace), a.n_parts = int(parts_of(d->vocab));
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch<float>(a, st);
  case LMX_F16: return launch<f16>(a, st);
  default: return launch<bf16>(a, st);
  }
}

}  // extern "C"
