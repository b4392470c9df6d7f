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

// One sequence's rows of the call.
struct SeqRows {
  int seq = -1;      // -1: none
  int first = 0;     // its first work unit
  int r0 = 0, n = 0;       // first row, count
  int start = 0, len = 0;  // position of the first row (may be negative), tokens with the rows
};

// The sequence that work unit u belongs to, where sequence s begins at unit
// floor(offsets[s] * mul / size) + s * per (at least its units of `size` follow,
// and at most `per` more).  The wave looks at 64 sequences a load, with what
// else it needs of them.
__device__ __forceinline__ SeqRows unit_rows(const Kv8Args &a, int u, int mul, int per, int lane, int size) {
  SeqRows r;
  int lo = 0, n = a.n_seqs;
  while (true) {
    const int step = (n + kWave - 1) / kWave, s = min(lo + lane * step, a.n_seqs - 1);
    const int o0 = min(max(a.offsets[s], 0), a.n_rows), o1 = min(a.offsets[s + 1], a.n_rows), len = a.lengths[s];
    const int begin = o0 * mul / size + s * per;   // (below 2^31: at most 2^24 rows, 64 heads)
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane * step < n && begin <= u));
    if (c == 0) return r;
    if (step == 1) {
      const auto pick = [c](int v) { return __builtin_amdgcn_readlane(v, c - 1); };
      r.seq = lo + c - 1;
      r.first = pick(begin);
      if (r.first > u) r.seq = -1;   // (offsets that decrease)
      r.r0 = pick(o0);
      r.n = max(pick(o1), r.r0) - r.r0;
      r.len = max(pick(len), 0);
      r.start = r.len - r.n;
      return r;
    }
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
}

// First of n pages (up to 2^24) that part `part` of `parts` (up to 64) takes.
__device__ __forceinline__ int part_begin(int n, int part, int parts) { return int(unsigned(n) * unsigned(part) / unsigned(parts)); }

__device__ __forceinline__ bool page_ok(const Kv8Args &a, int page) { return page >= 0 && page < a.n_pages; }

struct AttnArgs {
  Kv8Args c;
  const void *q;
  void *out;
  size_t q_stride, out_stride;
  float scale;       // softmax scale * log2(e)
  int splits;
  float *part_o;     // [units][n_kv][splits][16][HD]
  float2 *part_ml;   // [units][n_kv][splits][16]
};

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23
// The sums of weights carry 2^kSumExp, so that V scales from 2^-100 to 2^120
// leave them in range (23 bits of weight, 2^24 tokens).
constexpr int kSumExp = -24;
constexpr float kSumUnit = 0x1p-24f;
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.0f ? 0.0f : kSumUnit / l; }

constexpr int kDigits = 3;   // signed bytes of the fixed point of queries and weights
// Digit sums (from kMagic) -> the fixed-point sum, rounded once.
__device__ __forceinline__ float join(const float (&d)[kDigits]) {
  return fmaf(d[2] - kMagic, 65536.0f, fmaf(d[1], 256.0f, -257.0f * kMagic) + d[0]);
}

// Four fixed-point values, each in the low bits of a word with kCarry added ->
// dword d of the result: their digits d.
constexpr int kCarry = 0x8080;   // 128 for every digit below the top
__device__ __forceinline__ void digit_words(const uint32_t (&u)[4], uint32_t (&w)[kDigits]) {
  const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), c = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0602u), e = __builtin_amdgcn_perm(u[3], u[2], 0x0C0C0602u);
  w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u) ^ 0x80808080u;
  w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u) ^ 0x80808080u;
  w[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
}

// A weight enters the fixed point as p 2^ex with ex its V scale's power of two,
// which the rest of the scale, scale 2^-ex, then multiplies.  Scales far below
// the largest so far (kExpSpan) share its exponent less that, so that their
// weights, small next to that reference, do not underflow in the sum of weights.
constexpr int kLeastExp = -100, kExpSpan = 60;
__device__ __forceinline__ int value_exponent(float scale) {
  return scale != 0.0f ? max(__builtin_amdgcn_frexp_expf(scale), kLeastExp) : kLeastExp;
}
template <int D>
__device__ __forceinline__ int lane_xor_int(int v, int lane) { return int(lane_xor_u32<D>(uint32_t(v), lane)); }

// Queries: |q| <= 2^kQueryBits.  Of two digits (14 bits) a head's loud channel would
// leave the others fewer bits than a 16-bit type holds (64 times as loud 8), for 1 to
// 5 % of a step.  (fp32's too lose what lies below 2^-23 of the loud one, about
// what a sum of products in fp32 loses beside it.)
constexpr int kQueryBits = 22;
// The largest weight, of three digits: weight + carry stays below 2^23, so that
// added to 2^23 it is the low bits of the float.
constexpr float kWeightUnit = 8350000.0f;

// A row's 16 contiguous elements of step m -> its digit words; f: the power of
// two of the fixed point.
__device__ __forceinline__ void query_digits(const float (&x)[16], float f, v4i (&w)[kDigits]) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t u[4], d[kDigits];
#pragma unroll
    for (int i = 0; i < 4; ++i)   // (the float's low bits are the rounded product, up to 2^22 on either side)
      u[i] = __float_as_uint(fmaf(x[4 * b + i], f, kMagic)) + (uint32_t(kCarry) - 0x4B400000u);
    digit_words(u, d);
#pragma unroll
    for (int j = 0; j < kDigits; ++j) w[j][b] = int(d[j]);
  }
}

// Many rows per sequence, 16-bit types (lmx_kv8_prompt.hip).
constexpr int kPromptRows = 256;   // rows (query heads of tokens) per workgroup
int launch_prompt(const AttnArgs &a, int type, size_t hd, size_t units, hipStream_t st);

}  // namespace lmx

#endif  // LMX_KV8_HPP
