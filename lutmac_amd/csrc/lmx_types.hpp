// lmx_types.hpp -- activation types of the 8-bit serving operators (device
// code; included by the .hip sources only): loads of a few contiguous elements
// as floats and stores rounded to nearest even.
#ifndef LMX_TYPES_HPP
#define LMX_TYPES_HPP

#include <hip/hip_runtime.h>

#include "lutmac_hip.h"

namespace lmx {

typedef _Float16 f16;
typedef __bf16 bf16;

inline size_t type_bytes(int type) { return type == LMX_F32 ? 4 : type == LMX_F16 || type == LMX_BF16 ? 2 : 0; }

// N contiguous elements (aligned to their N * sizeof(T) bytes, at most 16 a load).
template <int N, class T>
__device__ __forceinline__ void load_floats(const T *p, float (&x)[N]) {
  constexpr int V = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
  typedef T vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int i = 0; i < N; i += V) {
    const vec v = *reinterpret_cast<const vec *>(p + i);
#pragma unroll
    for (int j = 0; j < V; ++j) x[i + j] = float(v[j]);
  }
}

template <int N, class T>
__device__ __forceinline__ void store_floats(T *p, const float (&x)[N]) {
  constexpr int V = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
  typedef T vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int i = 0; i < N; i += V) {
    vec v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = T(x[i + j]);
    *reinterpret_cast<vec *>(p + i) = v;
  }
}

// a / d rounded to the nearest whole number, ties to even, for d > 0 and a
// quotient of a few bits, with r near 1 / d: the remainder of the first guess
// says whether it is the nearest.
__device__ __forceinline__ double round_quotient(double a, double d, double r) {
  double n = rint(a * r);
  const double e = fma(-n, d, a), t = fabs(e) * 2.0;
  const bool odd = (int(n) & 1) != 0;
  if (t > d || (t == d && odd)) n += copysign(1.0, e);
  return n;
}

}  // namespace lmx

#endif  // LMX_TYPES_HPP
