// lmx_rotary.hip -- rotation of queries and keys to their positions (lmx_rotary):
// pairs a half of the rotated part apart or side by side, the whole head or its
// first dimensions, in either direction.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lmx_internal.hpp"
#include "lmx_types.hpp"
#include "lutmac_kv8.h"

namespace lmx {
namespace {

struct Heads {
  const void *in;
  void *out;
  size_t in_stride, out_stride;
};
struct RotaryArgs {
  Heads x[2];        // q, k
  int heads[2];
  int rows, hd, rd;
  int units;         // work units of a head: those that turn, then those that are copied
  int turning;
  uint32_t unit_inv; // ceil(2^31 / units)
  float sign;
  const int *positions;
  const float2 *rope;
  int rope_n;
};

// Half layout: a unit is E pairs, elements u E .. and those rd / 2 further on;
// interleaved: E / 2 pairs (one, for E = 1).  Behind the rotated part E elements.
template <class T, int E, bool INTER>
__device__ __forceinline__ void turn_unit(const RotaryArgs &a, const T *in, T *out, const float2 *rope, int u) {
  if (u >= a.turning) {   // behind the rotated part
    if (in == out) return;
    const int d = a.rd + (u - a.turning) * E;
    float x[E];
    load_floats<E>(in + d, x);
    store_floats<E>(out + d, x);
  } else if constexpr (INTER && E == 1) {
    const float2 c = rope[u];
    const float s = c.y * a.sign, p = float(in[2 * u]), q = float(in[2 * u + 1]);
    out[2 * u] = T(fmaf(p, c.x, -(q * s)));
    out[2 * u + 1] = T(fmaf(p, s, q * c.x));
  } else if constexpr (INTER) {
    float x[E], c[E];
    load_floats<E>(in + u * E, x);
    load_floats<E>(reinterpret_cast<const float *>(rope) + u * E, c);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float s = c[i + 1] * a.sign, p = x[i], q = x[i + 1];
      x[i] = fmaf(p, c[i], -(q * s));
      x[i + 1] = fmaf(p, s, q * c[i]);
    }
    store_floats<E>(out + u * E, x);
  } else {
    const int half = a.rd / 2;
    float x[E], y[E], c[2 * E];
    load_floats<E>(in + u * E, x);
    load_floats<E>(in + half + u * E, y);
    load_floats<2 * E>(reinterpret_cast<const float *>(rope) + 2 * u * E, c);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float s = c[2 * i + 1] * a.sign, p = x[i], q = y[i];
      x[i] = fmaf(p, c[2 * i], -(q * s));
      y[i] = fmaf(p, s, q * c[2 * i]);
    }
    store_floats<E>(out + u * E, x);
    store_floats<E>(out + half + u * E, y);
  }
}

// A workgroup a row, its up to 512 threads the units of all heads, shared evenly: bound by
// memory (16384 rows of 40 heads of 128, bf16: 61 us, 5.6 TB/s; 64 rows 2.7).  Workgroups
// lie in two dimensions, as one takes fewer than 2^32 threads.
constexpr int kGroups = 1 << 20, kThreads = 512;
template <class T, int E, bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  const int row = int(blockIdx.y) * kGroups + int(blockIdx.x);
  if (row >= a.rows) return;
  const int pos = a.positions[row];
  if (pos < 0 || pos >= a.rope_n) return;
  const float2 *rope = a.rope + size_t(pos) * (a.rd / 2);
  const int total = (a.heads[0] + a.heads[1]) * a.units;
  for (int at = int(threadIdx.x); at < total; at += int(blockDim.x)) {
    int head = int(__umulhi(uint32_t(at) * 2, a.unit_inv));
    const int u = at - head * a.units, w = head >= a.heads[0];
    if (w) head -= a.heads[0];
    const Heads &x = a.x[w];
    turn_unit<T, E, INTER>(a, static_cast<const T *>(x.in) + size_t(row) * x.in_stride + head * a.hd,
                           static_cast<T *>(x.out) + size_t(row) * x.out_stride + head * a.hd, rope, u);
  }
}

template <class T, int E, bool INTER>
int launch(RotaryArgs a, hipStream_t st) {
  a.turning = INTER && E > 1 ? a.rd / E : a.rd / 2 / E;
  a.units = a.turning + (a.hd - a.rd) / E;
  // (exact while units * at < 2^31: at most 1024 units, 2048 heads)
  a.unit_inv = ((1u << 31) + a.units - 1) / a.units;
  const size_t total = size_t(a.heads[0] + a.heads[1]) * a.units, rounds = (total + kThreads - 1) / kThreads;
  const unsigned threads = unsigned(round_up((total + rounds - 1) / rounds, kWave));
  rotary_kernel<T, E, INTER><<<dim3(unsigned(std::min(a.rows, kGroups)), unsigned((a.rows + kGroups - 1) / kGroups)), threads, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "rotary launch: %s", hipGetErrorString(e));
}

template <class T, bool INTER>
int launch(const RotaryArgs &a, int e, hipStream_t st) {
  constexpr int MOST = 16 / sizeof(T);
  if (e == MOST) return launch<T, MOST, INTER>(a, st);
  return launch<T, 1, INTER>(a, st);
}

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" int lmx_rotary(int type, const void *q, size_t q_stride, void *q_out, size_t q_out_stride, size_t n_heads,
                          const void *k, size_t k_stride, void *k_out, size_t k_out_stride, size_t n_kv_heads,
                          size_t head_dim, size_t rotary_dim, int interleaved, int inverse, const int32_t *positions,
                          size_t rows, const float *rope, size_t rope_positions, void *stream) {
  const size_t e = type_bytes(type);
  if (!e) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (!k) n_kv_heads = 0;
  if (head_dim == 0 || head_dim > 1024 || rotary_dim == 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu of %zu dimensions: head_dim 1..1024, rotary_dim even and at most that", rotary_dim, head_dim);
  if (n_heads == 0 || n_heads > 1024 || (k && n_kv_heads == 0) || n_kv_heads > 1024)
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu and %zu heads: 1..1024", n_heads, n_kv_heads);
  if (rows > (1u << 24)) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu rows: at most 2^24", rows);
  if ((interleaved | inverse) & ~1) return fail(LMX_ERR_INVALID_ARGUMENT, "interleaved and inverse are 0 or 1");
  if (rows == 0) return LMX_OK;
  if (!q || !q_out || (k && !k_out) || !positions || !rope) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (rope_positions == 0 || rope_positions >= (1u << 31) || reinterpret_cast<size_t>(rope) % 8 || reinterpret_cast<size_t>(positions) % 4)
    return fail(LMX_ERR_INVALID_ARGUMENT, "rotation table of %zu positions, or unaligned positions or table", rope_positions);
  RotaryArgs a{};
  a.x[0] = {q, q_out, q_stride, q_out_stride};
  a.x[1] = {k, k_out, k_stride, k_out_stride};
  a.heads[0] = int(n_heads), a.heads[1] = int(n_kv_heads);
  a.rows = int(rows), a.hd = int(head_dim), a.rd = int(rotary_dim);
  a.sign = inverse ? -1.0f : 1.0f;
  a.positions = positions, a.rope = reinterpret_cast<const float2 *>(rope), a.rope_n = int(rope_positions);
  const size_t most = 16 / e;   // elements of 16 bytes
  bool whole = head_dim % most == 0 && rotary_dim % (interleaved ? most : 2 * most) == 0 && reinterpret_cast<size_t>(rope) % 16 == 0;
  for (int i = 0; i < (k ? 2 : 1); ++i) {
    const Heads &x = a.x[i];
    const size_t in = reinterpret_cast<size_t>(x.in), out = reinterpret_cast<size_t>(x.out), width = size_t(a.heads[i]) * head_dim;
    if (in % e || out % e) return fail(LMX_ERR_INVALID_ARGUMENT, "%c is not aligned to its elements", i ? 'k' : 'q');
    if (rows > 1 && (x.in_stride < width || x.out_stride < width || x.in_stride >> 40 || x.out_stride >> 40))
      return fail(LMX_ERR_INVALID_ARGUMENT, "row strides %zu and %zu of rows of %zu elements", x.in_stride, x.out_stride, width);
    if (in == out && rows > 1 && x.in_stride != x.out_stride)
      return fail(LMX_ERR_INVALID_ARGUMENT, "in place with row strides %zu and %zu", x.in_stride, x.out_stride);
    whole = whole && (in | out) % 16 == 0 && (rows == 1 || (x.in_stride | x.out_stride) % most == 0);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int unit = whole ? int(most) : 1;
#define LMX_ROTARY(T) return interleaved ? launch<T, true>(a, unit, st) : launch<T, false>(a, unit, st)
  switch (type) {
  case LMX_F32: LMX_ROTARY(float);
  case LMX_F16: LMX_ROTARY(f16);
  default: LMX_ROTARY(bf16);
  }
#undef LMX_ROTARY
}
