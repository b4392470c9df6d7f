// lmx_i8.hip -- the linear layer in 8-bit integers (lmx_linear_i8): codes of
// the activations, one scale per row, and their product with 8-bit weights on
// the matrix cores, exact in 32-bit integers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lmx_internal.hpp"
#include "lmx_lanes.hpp"
#include "lmx_types.hpp"

namespace lmx {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int kStep = 128;   // bytes of k per step; the codes' rows are padded to it with zeros

struct I8Args {
  const int8_t *w;
  size_t w_stride;
  const float *w_scale;
  const void *bias, *x;
  void *y;
  int rows, cols, batch, Kp;
  int8_t *codes;     // [batch][Kp]
  float *scales;     // [batch]
  int splits;        // parts of k, each with sums of its own to join
  int *sums;         // [splits][batch][rows]
};

// Eight neighbouring elements of a row of x (zeros past its end); vec: the row
// is 16-byte aligned.
template <class T>
__device__ __forceinline__ void load8(const T *x, int k, int cols, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= cols) {
    load_floats<8>(x + k, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (k < cols)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < cols) v[i] = float(x[k + i]);
  }
}
__device__ __forceinline__ uint32_t top8(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return top;
}
__device__ __forceinline__ uint32_t wave_top(uint32_t top, int lane) {
  top = max(top, lane_xor_u32<32>(top, lane));
  top = max(top, lane_xor_u32<16>(top, lane));
  top = max(top, lane_xor_u32<8>(top, lane));
  top = max(top, lane_xor_u32<4>(top, lane));
  top = max(top, lane_xor_u32<2>(top, lane));
  return max(top, lane_xor_u32<1>(top, lane));
}

// round(127 v / amax), exactly rounded, of a row whose largest magnitude has the
// bits `top`; zeros for a row of zeros or with a value that is not finite.
struct Rounder {
  float amax, finv;
  bool some;
  __device__ __forceinline__ explicit Rounder(uint32_t top)
      : amax(__uint_as_float(top)), some(top != 0 && top < 0x7F800000u) {
    finv = some ? 127.0f / amax : 0.0f;
  }
  __device__ __forceinline__ float scale() const { return amax < INFINITY ? amax / 127.0f : __builtin_nanf(""); }
  // The quotient in fp32 is off by at most 127 * 3 * 2^-24, far less than kSure
  // keeps it from a border between two codes; nearer ones, and those of an amax
  // so small that 127 / amax overflows, are taken in 64 bits.
  __device__ __forceinline__ uint2 codes(const float (&v)[8]) const {
    constexpr float kSure = 0.4999f;
    uint32_t w[2] = {0, 0};
    bool sure = finv < INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = v[i] * finv, n = rintf(q);
      sure = sure && fabsf(q - n) < kSure;
      w[i / 4] |= uint32_t(int(n) & 0xFF) << (8 * (i % 4));
    }
    if (some && !sure) {
      const double d = amax, inv = 1.0 / d;
      w[0] = w[1] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i / 4] |= uint32_t(int(round_quotient(double(v[i]) * 127.0, d, inv)) & 0xFF) << (8 * (i % 4));
    }
    return some ? make_uint2(w[0], w[1]) : make_uint2(0, 0);
  }
};

// The largest of a row's W / R waves.
template <int W, int R>
__device__ __forceinline__ uint32_t row_top(const uint32_t *tops, int m) {
  uint32_t t = 0;
#pragma unroll
  for (int v = 0; v < W / R; ++v) t = max(t, tops[m * (W / R) + v]);
  return t;
}

// Codes of x, zeros up to Kp: a workgroup a row, which up to K = 32 NT stays in
// registers between its maximum and them (8192 rows of 2048 bf16: 21 us; a wave
// a row took 24).
template <class T, int NT>
__global__ __launch_bounds__(NT) void i8_codes_kernel(I8Args a) {
  constexpr int KEEP = 4, R = NT * 8;   // rounds of R elements kept
  __shared__ uint32_t tops[NT / kWave];
  const int lane = threadIdx.x & (kWave - 1), row = int(blockIdx.x);
  const T *x = static_cast<const T *>(a.x) + size_t(row) * a.cols;
  const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
  float keep[KEEP][8];
  uint32_t top = 0;
  const int k0 = int(threadIdx.x) * 8;
#pragma unroll
  for (int j = 0; j < KEEP; ++j) {
    load8(x, k0 + j * R, a.cols, vec, keep[j]);
    top = top8(keep[j], top);
  }
  for (int k = k0 + KEEP * R; k < a.cols; k += R) {
    float v[8];
    load8(x, k, a.cols, vec, v);
    top = top8(v, top);
  }
  top = wave_top(top, lane);
  if (lane == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
  const Rounder r(row_top<NT / kWave, 1>(tops, 0));
  int8_t *codes = a.codes + size_t(row) * a.Kp;
#pragma unroll
  for (int j = 0; j < KEEP; ++j)
    if (k0 + j * R < a.Kp) *reinterpret_cast<uint2 *>(codes + k0 + j * R) = r.codes(keep[j]);
  for (int k = k0 + KEEP * R; k < a.Kp; k += R) {
    float v[8];
    load8(x, k, a.cols, vec, v);
    *reinterpret_cast<uint2 *>(codes + k) = r.codes(v);
  }
  if (k0 == 0) a.scales[row] = r.scale();
}

// Scales and biases of four neighbouring weight rows (past the last: its own).
struct Four { float scale[4], bias[4]; };
template <class T>
__device__ __forceinline__ Four row_factors(const I8Args &a, int n) {
  Four f;
  const T *b = static_cast<const T *>(a.bias);
  int r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = min(n + i, a.rows - 1), f.scale[i] = a.w_scale[r[i]], f.bias[i] = 0.0f;
  if (b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.bias[i] = float(b[r[i]]);
  }
  return f;
}

// Four neighbouring outputs y[m][n .. n + 3] from their integer sums; whole
// groups go out in one store where y allows it (vec).
template <class T>
__device__ __forceinline__ void store4(const I8Args &a, int m, int n, const v4i s, float xs, const Four &w, bool vec) {
  if (m >= a.batch || n >= a.rows) return;
  T *y = static_cast<T *>(a.y) + size_t(m) * a.rows + n;
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = fmaf(float(s[i]) * w.scale[i], xs, w.bias[i]);
  if (vec) {   // (then rows are whole groups)
    store_floats<4>(y, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.rows) y[i] = T(f[i]);
  }
}

template <class T>
__device__ __forceinline__ bool vector_rows(const I8Args &a) {
  return a.rows % 4 == 0 && reinterpret_cast<size_t>(a.y) % (4 * sizeof(T)) == 0;
}

// Weight rows of a workgroup as a buffer: reads past the matrix give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t weight_buffer(const I8Args &a, int row0) {
  const size_t at = size_t(row0) * a.w_stride, end = (size_t(a.rows - 1) * a.w_stride + size_t(a.cols) + 3) / 4 * 4;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(a.w) + at, 0, int(min(end - at, size_t(0x7FFFFFFF))), 0x00020000);
}

__device__ __forceinline__ void lds_barrier() {   // no wait for loads on their way, as __syncthreads makes
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// 128-byte rows in LDS: piece p (16 bytes) of row r lies at p ^ (r / 2 mod 8), so
// that the 16 lanes of a read's phase touch all 64 banks once.
__device__ __forceinline__ int piece_place(int row, int piece) { return 16 * (piece ^ (row >> 1 & 7)); }
// Where lane `lane` of a load of 8 rows reads row `row` (the last one past it).
__device__ __forceinline__ int piece_offset(int row, int last, int stride, int lane) {
  return min(row, last) * stride + piece_place(row, lane % 8);
}

// ---------------------------------------------------------------------------
// One to four rows of activations, one launch: a workgroup takes 16 weight rows,
// its W waves the k-steps w, w + W, ..., each through U LDS buffers of its own
// (see i8_few_kernel).  Every workgroup makes the codes itself, in LDS while its
// first weights are on their way (R >= batch rows, a power of two; at most 16
// values a thread, which stay in registers), which saves a launch and the trip
// through memory.
//   A (weights): lane (i, g) holds bytes 16 g .. + 15 of a 64-byte step of row i;
//   B (codes) the same of activation row j; C lane (j, g): weight rows 4 g .. + 3.
constexpr int rows_buffers(int waves) { return waves == 16 ? 3 : 4; }
template <class T, int W, int R>
__global__ __launch_bounds__(W *kWave) void i8_rows_kernel(I8Args a) {
  constexpr int U = rows_buffers(W), RB = 16 * kStep;
  __shared__ v4i part[W][kWave];
  __shared__ uint32_t tops[W];
  extern __shared__ __attribute__((aligned(1024))) char lds[];   // the waves' buffers, then codes [batch][Kp + 16]
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int i = lane & 15, g = lane >> 4, row0 = int(blockIdx.x) * 16;
  char *mine = lds + wave * (U * RB), *codes = lds + W * U * RB;
  constexpr int KEEP = 2, TR = W * kWave / R;   // threads of an activation row
  const int am = int(threadIdx.x) / TR, k0 = int(threadIdx.x) % TR * 8;
  float v[KEEP][8];
  {
    const T *x = static_cast<const T *>(a.x) + size_t(min(am, a.batch - 1)) * a.cols;
    const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) load8(x, k0 + j * TR * 8, a.cols, vec, v[j]);
  }
  const auto wbuf = weight_buffer(a, row0);
  int won[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) won[n] = piece_offset(8 * n + lane / 8, a.rows - 1 - row0, int(a.w_stride), lane);
  const int steps = a.Kp / kStep, turns = wave < steps ? (steps - 1 - wave) / W + 1 : 0;
  const auto fill = [&](int buf, int t) {
#pragma unroll
    for (int n = 0; n < 2; ++n) buffer_to_lds(wbuf, mine + buf * RB + n * 1024, won[n], (wave + t * W) * kStep);
  };
#pragma unroll
  for (int t = 0; t < U - 1; ++t)
    if (t < turns) fill(t, t);
  {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) top = top8(v[j], top);
    top = wave_top(top, lane);
    if (lane == 0) tops[wave] = top;
    lds_barrier();
    if (am < a.batch) {
      const Rounder r(row_top<W, R>(tops, am));
#pragma unroll
      for (int j = 0; j < KEEP; ++j)
        if (k0 + j * TR * 8 < a.Kp) *reinterpret_cast<uint2 *>(codes + am * (a.Kp + 16) + k0 + j * TR * 8) = r.codes(v[j]);
    }
    lds_barrier();
  }
  const int m = min(i, a.batch - 1);
  const char *xc = codes + m * (a.Kp + 16) + 16 * g;
  v4i acc = {0, 0, 0, 0};
  int buf = 0;
  for (int t = 0; t < turns; ++t) {
    if (t + U - 1 <= turns) wait_loads<(U - 2) * 2>();
    else wait_loads<0>();
    const char *at = mine + buf * RB + i * kStep;
    v4i w[2], x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = *reinterpret_cast<const v4i *>(at + piece_place(i, 4 * h + g));
      x[h] = *reinterpret_cast<const v4i *>(xc + (wave + t * W) * kStep + 64 * h);
    }
    if (t + U - 1 < turns) fill(buf == 0 ? U - 1 : buf - 1, t + U - 1);   // (the buffer of the step before)
#pragma unroll
    for (int h = 0; h < 2; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h], x[h], acc, 0, 0, 0);
    buf = buf == U - 1 ? 0 : buf + 1;
  }
  part[wave][lane] = acc;
  const Four f = row_factors<T>(a, row0 + 4 * g);
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int v = 1; v < W; ++v) acc += part[v][lane];
  store4<T>(a, i, row0 + 4 * g, acc, Rounder(row_top<W, R>(tops, m)).scale(), f, vector_rows<T>(a));
}

// ---------------------------------------------------------------------------
// Some rows of activations (up to 16 G) and so few weight rows that tiles of
// 64 x 64 leave CUs idle: 16 weight rows a workgroup, its W waves the k-steps w,
// w + W, ..., each through U LDS buffers of its own that are filled straight from
// memory U - 1 steps ahead, so that no wave waits for another before the end.
// (Straight to registers a load instruction touches 64 lines instead of 8 and
// takes as many cycles: 48 x 8960 -> 1536 24 us.)
template <class T, int W, int R, int G, int U>
__global__ __launch_bounds__(W *kWave) void i8_few_kernel(I8Args a) {
  constexpr int RB = (R + G) * 16 * kStep;   // bytes of a buffer: weights, then codes
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int i = lane & 15, g = lane >> 4, row0 = int(blockIdx.x) * (16 * R);
  const auto wbuf = weight_buffer(a, row0);
  const auto xbuf = __builtin_amdgcn_make_buffer_rsrc(a.codes, 0, a.batch * a.Kp, 0x00020000);
  int won[2 * R], xon[2 * G];   // (a load instruction: 8 rows)
#pragma unroll
  for (int n = 0; n < 2 * R; ++n) won[n] = piece_offset(8 * n + lane / 8, a.rows - 1 - row0, int(a.w_stride), lane);
#pragma unroll
  for (int n = 0; n < 2 * G; ++n) xon[n] = piece_offset(8 * n + lane / 8, a.batch - 1, a.Kp, lane);
  char *mine = lds + wave * (U * RB);
  const int steps = a.Kp / kStep, turns = wave < steps ? (steps - 1 - wave) / W + 1 : 0;
  const auto fill = [&](int buf, int t) {
    const int k = (wave + t * W) * kStep;
#pragma unroll
    for (int n = 0; n < 2 * R; ++n) buffer_to_lds(wbuf, mine + buf * RB + n * 1024, won[n], k);
#pragma unroll
    for (int n = 0; n < 2 * G; ++n) buffer_to_lds(xbuf, mine + buf * RB + (2 * R + n) * 1024, xon[n], k);
  };
#pragma unroll
  for (int t = 0; t < U - 1; ++t)
    if (t < turns) fill(t, t);
  v4i acc[R][G];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < G; ++n) acc[r][n] = v4i{0, 0, 0, 0};
  int buf = 0;
  for (int t = 0; t < turns; ++t) {
    if (t + U - 1 <= turns) wait_loads<(U - 2) * 2 * (R + G)>();
    else wait_loads<0>();
    const char *at = mine + buf * RB + i * kStep;
    v4i w[R][2], x[G][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int piece = piece_place(i, 4 * h + g);
#pragma unroll
      for (int r = 0; r < R; ++r) w[r][h] = *reinterpret_cast<const v4i *>(at + r * 16 * kStep + piece);
#pragma unroll
      for (int n = 0; n < G; ++n) x[n][h] = *reinterpret_cast<const v4i *>(at + (R + n) * 16 * kStep + piece);
    }
    if (t + U - 1 < turns) fill(buf == 0 ? U - 1 : buf - 1, t + U - 1);   // (the buffer of the step before)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < G; ++n) acc[r][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r][h], x[n][h], acc[r][n], 0, 0, 0);
    buf = buf == U - 1 ? 0 : buf + 1;
  }
  __syncthreads();   // every wave is done with its buffers
  v4i(*part)[R * G][kWave] = reinterpret_cast<v4i(*)[R * G][kWave]>(lds);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < G; ++n) part[wave][r * G + n][lane] = acc[r][n];
  __syncthreads();
  for (int q = wave; q < R * G; q += W) {
    const int r = q / G, m = 16 * (q % G) + i, row = row0 + 16 * r + 4 * g;
    const Four f = row_factors<T>(a, row);
    const float xs = a.scales[min(m, a.batch - 1)];
    v4i sum = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < W; ++v) sum += part[v][q][lane];
    store4<T>(a, m, row, sum, xs, f, vector_rows<T>(a));
  }
}

// ---------------------------------------------------------------------------
// Many rows of activations: BN weight rows x BM activation rows per workgroup,
// WN x WM waves, k in steps of BK bytes through S LDS buffers that are filled
// straight from memory S - 1 steps ahead (v_mfma_i32_32x32x32_i8).  A row's
// 16-byte pieces lie in LDS at p ^ swizzle(row), so that the 16 lanes of a
// read's phase touch all 64 banks once.  8192 x 2048 -> 16384 takes 265 us, 2.07
// POPS (8192 deep 2.3), where the library's largest product of bytes reaches 2.4.
//
// PART: workgroup (tile, part) takes part blockIdx.y of k and leaves its integer
// sums (T is int) for i8_join_kernel: where tiles are few and k is long.
template <class T, int BN, int BM, int WN, int WM, int BK, int S>
__global__ __launch_bounds__(WN *WM *kWave) __attribute__((amdgpu_waves_per_eu(BN *BM / (WN * WM) > 8192 ? 1 : 2))) void i8_tile_kernel(I8Args a) {
  constexpr bool PART = std::is_same<T, int>::value;
  constexpr int W = WN * WM, TN = BN / WN / 32, TM = BM / WM / 32;
  constexpr int RB = (BN + BM) * BK;   // bytes of a buffer: weights, then codes
  constexpr int P = BK / 16;           // pieces of a row
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const auto swizzle = [](int row) { return BK == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int wn = wave % WN, wm = wave / WN;
  // Workgroups go round the 8 XCDs, each with an L2 of its own: XCD x takes the
  // x-th eighth of the tiles, in blocks of 4 weight tiles by all activation
  // tiles, so that what its workgroups read at a time overlaps.
  const int gn = (a.rows + BN - 1) / BN, gm = (a.batch + BM - 1) / BM, share = int(gridDim.x) / 8;
  const int tile = int(blockIdx.x) % 8 * share + int(blockIdx.x) / 8;
  if (tile >= gn * gm) return;
  const int g0 = tile / (4 * gm) * 4, gw = min(4, gn - g0), in = tile - g0 * gm;
  const int row0 = (g0 + in % gw) * BN, m0 = in / gw * BM;
  const auto wbuf = weight_buffer(a, row0);
  const auto xbuf = __builtin_amdgcn_make_buffer_rsrc(a.codes + size_t(m0) * a.Kp, 0,
                                                      int(min(size_t(a.batch - m0) * a.Kp, size_t(0x7FFFFFFF))), 0x00020000);
  // One load instruction of a wave: 1 KB, 64 / P rows.
  constexpr int LR = 64 / P, LN = BN / LR / W, LM = BM / LR / W;   // rows, instructions per wave and buffer
  static_assert(LN * LR * W == BN && LM * LR * W == BM, "whole instructions");
  const int lr = lane / P, lp = lane % P;
  int won[LN], wom[LM];
#pragma unroll
  for (int j = 0; j < LN; ++j) {
    const int r = (j * W + wave) * LR + lr;
    won[j] = min(r, a.rows - 1 - row0) * int(a.w_stride) + 16 * (lp ^ swizzle(r));
  }
#pragma unroll
  for (int j = 0; j < LM; ++j) {
    const int r = (j * W + wave) * LR + lr;
    wom[j] = min(r, a.batch - 1 - m0) * a.Kp + 16 * (lp ^ swizzle(r));
  }
  const auto fill = [&](int buf, int k) {
#pragma unroll
    for (int j = 0; j < LN; ++j) buffer_to_lds(wbuf, lds + buf * RB + (j * W + wave) * 1024, won[j], k);
#pragma unroll
    for (int j = 0; j < LM; ++j) buffer_to_lds(xbuf, lds + buf * RB + BN * BK + (j * W + wave) * 1024, wom[j], k);
  };
  v16i acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[n][m][v] = 0;
  const int i = lane & 31, h = lane >> 5;
  int steps = a.Kp / BK, k0 = 0;
  if constexpr (PART) {
    const int all = steps, part = int(blockIdx.y);
    k0 = int(unsigned(all) * unsigned(part) / unsigned(a.splits));
    steps = int(unsigned(all) * unsigned(part + 1) / unsigned(a.splits)) - k0;
    k0 *= BK;
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < steps) fill(s, k0 + s * BK);
  int buf = 0;
  for (int s = 0; s < steps; ++s) {
    if (s + S - 1 <= steps) wait_loads<(S - 2) * (LN + LM)>();
    else wait_loads<0>();
    asm volatile("s_barrier" ::: "memory");   // (no wait for the loads of later steps, as __syncthreads makes)
    if (s + S - 1 < steps) fill(buf == 0 ? S - 1 : buf - 1, k0 + (s + S - 1) * BK);
    const char *wl = lds + buf * RB + (wn * (BN / WN) + i) * BK;
    const char *xl = lds + buf * RB + BN * BK + (wm * (BM / WM) + i) * BK;
#pragma unroll
    for (int q = 0; q < BK / 32; ++q) {
      const int at = 16 * ((2 * q + h) ^ swizzle(i));
      v4i wf[TN], xf[TM];
#pragma unroll
      for (int n = 0; n < TN; ++n) wf[n] = *reinterpret_cast<const v4i *>(wl + n * 32 * BK + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) xf[m] = *reinterpret_cast<const v4i *>(xl + m * 32 * BK + at);
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[n], xf[m], acc[n][m], 0, 0, 0);
    }
    buf = buf == S - 1 ? 0 : buf + 1;
  }
  // The sums leave through LDS, 32 activation rows of the wave at a time, so
  // that stores are whole lines of y (a lane's own four neighbours at a time
  // take 2 to 4 times as long).
  constexpr int NW = BN / WN, LD = NW * int(sizeof(T)) + 16;   // a row in LDS, apart by banks
  static_assert(W * 32 * LD <= S * RB, "the rows fit in the buffers");
  asm volatile("s_barrier" ::: "memory");   // every wave is done with the buffers
  char *out = lds + wave * (32 * LD);
  const int n0 = row0 + wn * NW;
  Four w[TN][4];
  if constexpr (!PART) {
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int b = 0; b < 4; ++b) w[n][b] = row_factors<T>(a, min(n0 + 32 * n + 8 * b + 4 * h, a.rows - 1));
  }
  constexpr int V = 16 / int(sizeof(T)), LPR = NW / V;   // elements of a store, lanes of a row
  T *base = PART ? reinterpret_cast<T *>(a.sums) + size_t(blockIdx.y) * a.batch * a.rows : static_cast<T *>(a.y);
  const bool vec = a.rows % V == 0 && reinterpret_cast<size_t>(base) % 16 == 0;
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int m1 = m0 + wm * (BM / WM) + 32 * m;
    if (m1 >= a.batch) break;
    const float xs = PART ? 0.0f : a.scales[min(m1 + i, a.batch - 1)];
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        T *at = reinterpret_cast<T *>(out + i * LD) + 32 * n + 8 * b + 4 * h;
        if constexpr (PART) {
          *reinterpret_cast<v4i *>(at) = v4i{acc[n][m][4 * b], acc[n][m][4 * b + 1], acc[n][m][4 * b + 2], acc[n][m][4 * b + 3]};
        } else {
          float f[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) f[v] = fmaf(float(acc[n][m][4 * b + v]) * w[n][b].scale[v], xs, w[n][b].bias[v]);
          store_floats<4>(at, f);
        }
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    T *y = base + size_t(m1) * a.rows + n0;
    if (vec) {
      typedef T vecT __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int q = 0; q < 32 * LPR / kWave; ++q) {
        const int r = q * (kWave / LPR) + lane / LPR, n = lane % LPR * V;
        if (m1 + r < a.batch && n0 + n < a.rows)
          *reinterpret_cast<vecT *>(y + size_t(r) * a.rows + n) = *reinterpret_cast<const vecT *>(out + r * LD + n * sizeof(T));
      }
    } else {
      for (int q = 0; q < 32 * NW / kWave; ++q) {
        const int at = q * kWave + lane, r = at / NW, n = at % NW;
        if (m1 + r < a.batch && n0 + n < a.rows) y[size_t(r) * a.rows + n] = *reinterpret_cast<const T *>(out + r * LD + n * sizeof(T));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// y from the parts' sums, four weight rows of an activation row per thread.
template <class T>
__global__ __launch_bounds__(256) void i8_join_kernel(I8Args a) {
  const int quads = (a.rows + 3) / 4;
  const size_t at = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= size_t(quads) * a.batch) return;
  const int m = int(at / quads), n = int(at % quads) * 4;
  const bool vec = vector_rows<T>(a);
  const float xs = a.scales[m];
  const Four w = row_factors<T>(a, n);
  const int *p = a.sums + size_t(m) * a.rows + n;
  v4i s = {0, 0, 0, 0};
#pragma unroll 8
  for (int q = 0; q < a.splits; ++q, p += size_t(a.batch) * a.rows) {
    if (a.rows % 4 == 0) {
      s += *reinterpret_cast<const v4i *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += n + i < a.rows ? p[i] : 0;
    }
  }
  store4<T>(a, m, n, s, xs, w, vec);
}

// ---- host side ----

int launch_err(const char *what) {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

// (per device: asked before each launch, 0.2 us)
int allow_lds(const void *kernel, size_t bytes) {
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_HIP, "LDS of an i8 kernel: %s", hipGetErrorString(e));
}

size_t tile_count(size_t rows, size_t batch, size_t side) { return (rows + side - 1) / side * ((batch + side - 1) / side); }

// Up to 64 activation rows go to i8_few_kernel, unless tiles of 64 x 64 are just
// one round of the CUs (us, tiles / 16 weight rows and 4 waves a workgroup / 32 and
// 4 / 64 and 2: 16 x 2048 -> 2048 11.8 / 7.4 / 7.7 / 8.8, 48 x 8960 -> 1536 16.4 /
// 13.6 / 15.1 / 22, 48 x 2048 -> 8192 13.3 / 11.5 / 10.3 / 12.0, 48 x 2048 -> 16384
// 13.1 / 18.4 / 15.1 / 14.1, 48 x 8192 -> 24576 55 / 53 / 52 / 43): more weight rows
// a workgroup read the codes less often.
enum class FewShape { none, rows16, rows32, rows64 };
FewShape few_shape(size_t rows, size_t batch) {
  const size_t tiles = tile_count(rows, batch, 64);
  if (batch > 64 || (batch > 16 && tiles >= 192 && tiles <= 256)) return FewShape::none;
  if (batch > 16 && rows > 16384) return FewShape::rows64;
  return batch > 32 && rows > 4096 ? FewShape::rows32 : FewShape::rows16;
}

// Parts of k for other calls of few tiles: as many as bring the 64 x 64 tiles to
// one per CU, of 8 steps at least, if they are three (us, in one part / in parts:
// 100 x 8960 -> 1536 in 5 28.8 / 17.8, 100 x 2048 -> 2048 in 2 11.5 / 12.1).
int split_count(size_t rows, size_t cols, size_t batch) {
  if (few_shape(rows, batch) != FewShape::none) return 1;
  const size_t tiles = tile_count(rows, batch, 64), steps = round_up(cols, kStep) / kStep;
  const size_t parts = tiles ? std::min<size_t>(256 / tiles, steps / 8) : 1;
  return parts < 3 ? 1 : int(parts);
}

// More waves share a row tile's k where the tiles alone leave CUs idle.
int rows_waves(const I8Args &a) {
  const int tiles = (a.rows + 15) / 16;
  return tiles <= 256 ? 16 : tiles <= 768 ? 8 : 4;
}

template <class T, int W, int R>
int launch_rows(const I8Args &a, hipStream_t st) {
  constexpr size_t ring = W * rows_buffers(W) * 16 * kStep, most = ring + 1024 * W + 16 * R;
  if (const int r = allow_lds(reinterpret_cast<const void *>(&i8_rows_kernel<T, W, R>), most)) return r;
  i8_rows_kernel<T, W, R><<<unsigned((a.rows + 15) / 16), W * kWave, ring + size_t(a.batch) * (a.Kp + 16), st>>>(a);
  return launch_err("i8 linear");
}
template <class T, int R>
int launch_rows(const I8Args &a, hipStream_t st) {
  switch (rows_waves(a)) {
  case 16: return launch_rows<T, 16, R>(a, st);
  case 8: return launch_rows<T, 8, R>(a, st);
  default: return launch_rows<T, 4, R>(a, st);
  }
}

// Whether every workgroup makes the codes itself: up to 4 rows, as long as that
// is two rounds of a workgroup's threads, and not too often for nothing (us,
// itself / codes in a launch before: 1 x 2048 -> 16384 8.6 / 11.4, 4 x 2048 -> 8192
// 8.5 / 8.7, 2 x 2048 -> 16384 9.9 / 11.7, 2 x 2048 -> 65536 28 / 26).
int row_slots(const I8Args &a) { return a.batch <= 2 ? a.batch : 4; }
bool in_one_launch(const I8Args &a) {
  return a.batch <= 4 && row_slots(a) * a.Kp <= 1024 * rows_waves(a) && (a.batch == 1 || a.rows <= 32768);
}

template <class T, int BN, int BM, int WN, int WM, int BK, int S>
int launch_tile(const I8Args &a, hipStream_t st) {
  constexpr size_t lds = S * (BN + BM) * BK;
  if (const int r = allow_lds(reinterpret_cast<const void *>(&i8_tile_kernel<T, BN, BM, WN, WM, BK, S>), lds)) return r;
  const size_t tiles = size_t((a.rows + BN - 1) / BN) * size_t((a.batch + BM - 1) / BM);
  if (tiles > (1u << 30)) return fail(LMX_ERR_INVALID_ARGUMENT, "%d x %d outputs", a.rows, a.batch);
  i8_tile_kernel<T, BN, BM, WN, WM, BK, S><<<dim3(unsigned(round_up(tiles, 8)), unsigned(a.splits)), WN * WM * kWave, lds, st>>>(a);
  return LMX_OK;
}

template <class T, int W, int R, int G>
int launch_few(const I8Args &a, hipStream_t st) {
  constexpr size_t lds = W * 3 * (R + G) * 16 * kStep;
  if (const int r = allow_lds(reinterpret_cast<const void *>(&i8_few_kernel<T, W, R, G, 3>), lds)) return r;
  i8_few_kernel<T, W, R, G, 3><<<unsigned((a.rows + 16 * R - 1) / (16 * R)), W * kWave, lds, st>>>(a);
  return launch_err("i8 linear");
}
template <class T>
int launch_few(const I8Args &a, hipStream_t st) {
  const int G = (a.batch + 15) / 16;
  switch (few_shape(a.rows, a.batch)) {
  case FewShape::rows64: return G == 2 ? launch_few<T, 2, 4, 2>(a, st) : G == 3 ? launch_few<T, 2, 4, 3>(a, st) : launch_few<T, 2, 4, 4>(a, st);
  case FewShape::rows32: return G == 3 ? launch_few<T, 4, 2, 3>(a, st) : launch_few<T, 4, 2, 4>(a, st);
  default:
    return G == 1 ? launch_few<T, 4, 1, 1>(a, st) : G == 2 ? launch_few<T, 4, 1, 2>(a, st) : G == 3 ? launch_few<T, 4, 1, 3>(a, st)
                                                                                      : launch_few<T, 4, 1, 4>(a, st);
  }
}

template <class T>
int launch_linear(const I8Args &a, hipStream_t st) {
  if (in_one_launch(a)) {
    switch (row_slots(a)) {
    case 1: return launch_rows<T, 1>(a, st);
    case 2: return launch_rows<T, 2>(a, st);
    default: return launch_rows<T, 4>(a, st);
    }
  }
  // (few long rows: 1024 threads a row, 48 of 8960 in 4.3 us against 6.8)
  if (a.Kp > 2048 && a.batch < 512) i8_codes_kernel<T, 1024><<<unsigned(a.batch), 1024, 0, st>>>(a);
  else i8_codes_kernel<T, 256><<<unsigned(a.batch), 256, 0, st>>>(a);
  int r = launch_err("i8 codes");
  if (r) return r;
  if (few_shape(a.rows, a.batch) != FewShape::none) return launch_few<T>(a, st);
  if (a.splits > 1) {
    if ((r = launch_tile<int, 64, 64, 2, 2, 128, 4>(a, st)) || (r = launch_err("i8 linear parts"))) return r;
    i8_join_kernel<T><<<unsigned((size_t(a.batch) * ((a.rows + 3) / 4) + 255) / 256), 256, 0, st>>>(a);
    return launch_err("i8 join");
  }
  // The largest tiles that still fill most of the CUs, as larger ones read less
  // from the L2s (us at K = 2048, 256 / 128 / 64: 2048 -> 8192 49 / 56 / 85, 1024
  // -> 8192 39 / 32 / 44, 256 -> 16384 34 / 22 / 25, 100 -> 17920 32 / 21 / 21).
  const size_t rows = a.rows, batch = a.batch;
  if (tile_count(rows, batch, 256) >= 192) r = launch_tile<T, 256, 256, 4, 2, 128, 2>(a, st);
  else if (tile_count(rows, batch, 128) >= 160) r = launch_tile<T, 128, 128, 2, 2, 128, 2>(a, st);
  else r = launch_tile<T, 64, 64, 2, 2, 128, 4>(a, st);
  return r ? r : launch_err("i8 linear");
}

// Scales, codes and, of a call that splits k, its parts' sums.
size_t codes_at(size_t batch) { return round_up(batch * sizeof(float), 256); }
size_t sums_at(size_t cols, size_t batch) { return codes_at(batch) + round_up(batch * round_up(cols, kStep), 256); }
size_t i8_workspace(size_t rows, size_t cols, size_t batch) {
  const int splits = split_count(rows, cols, batch);
  return sums_at(cols, batch) + (splits > 1 ? size_t(splits) * batch * rows * sizeof(int) : 0);
}

// Codes of an 8-bit handle from its copy for the matrix cores: byte B of word t
// of plane word kq of a 128-chunk is k = 32 kq + 8 B + 7 - t.
__global__ __launch_bounds__(256) void codes_i8_kernel(const int8_t *codes, const float *scales, int rows, int cols, int Npad,
                                                       size_t stride, int8_t *out, float *out_scales) {
  const size_t k = size_t(blockIdx.x) * 256 + threadIdx.x;
  const int r = int(blockIdx.y);
  if (k < stride) {
    const size_t ch = k / kChunk, in = k % kChunk;
    out[size_t(r) * stride + k] =
        k < size_t(cols) ? codes[(ch * Npad + r) * kChunk + in / 32 * 32 + (7 - in % 8) * 4 + in % 32 / 8] : int8_t(0);
  }
  if (k == 0) out_scales[r] = scales[r];
}

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_linear_i8_workspace(size_t rows, size_t cols, size_t batch, size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (rows == 0 || rows > (1u << 24) || cols == 0 || cols > 131072 || batch > (1u << 22))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu x %zu, %zu vectors: rows 1..2^24, cols 1..131072, at most 2^22 vectors", rows, cols, batch);
  *bytes = i8_workspace(rows, cols, batch);
  return LMX_OK;
}

int lmx_linear_i8(const int8_t *w, size_t w_stride, const float *w_scale, const void *bias, const void *x, void *y, int type,
                  size_t rows, size_t cols, size_t batch, void *workspace, size_t workspace_bytes, void *stream) {
  size_t need = 0;
  const int r = lmx_linear_i8_workspace(rows, cols, batch, &need);
  if (r) return r;
  const size_t e = type_bytes(type);
  if (!e) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (batch == 0) return LMX_OK;
  if (!w || !w_scale || !x || !y) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (reinterpret_cast<size_t>(w) % 16 || w_stride % 16 || w_stride < cols || w_stride > 262144)
    return fail(LMX_ERR_INVALID_ARGUMENT, "weight pointer and row stride (%zu) must be multiples of 16, the stride %zu..262144",
                w_stride, cols);
  if ((reinterpret_cast<size_t>(x) | reinterpret_cast<size_t>(y) | reinterpret_cast<size_t>(bias)) % e ||
      reinterpret_cast<size_t>(w_scale) % 4)
    return fail(LMX_ERR_INVALID_ARGUMENT, "x, y, bias and w_scale must be aligned to their elements");
  if (!workspace || workspace_bytes < need || reinterpret_cast<size_t>(workspace) % 16)
    return fail(LMX_ERR_INVALID_ARGUMENT, "workspace of %zu bytes at %p: %zu bytes, 16-byte aligned, are needed", workspace_bytes,
                workspace, need);
  I8Args a{};
  a.w = w, a.w_stride = w_stride, a.w_scale = w_scale, a.bias = bias, a.x = x, a.y = y;
  a.rows = int(rows), a.cols = int(cols), a.batch = int(batch), a.Kp = int(round_up(cols, kStep));
  a.scales = static_cast<float *>(workspace);
  a.codes = static_cast<int8_t *>(workspace) + codes_at(batch);
  a.splits = split_count(rows, cols, batch);
  a.sums = reinterpret_cast<int *>(static_cast<char *>(workspace) + sums_at(cols, batch));
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch_linear<float>(a, st);
  case LMX_F16: return launch_linear<f16>(a, st);
  default: return launch_linear<bf16>(a, st);
  }
}

int lmx_weight_codes_i8(const lmx_weight *w, int8_t *codes, size_t w_stride, float *scales, void *stream) {
  if (!w || !codes || !scales) return fail(LMX_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (w->format != LMX_FMT_INT8 || w->n_groups != 1 || !w->d_codes)
    return fail(LMX_ERR_UNSUPPORTED_FORMAT, "an 8-bit handle with one scale per row is needed");
  if (w_stride < w->cols || w_stride % 16 || reinterpret_cast<size_t>(codes) % 16)
    return fail(LMX_ERR_INVALID_ARGUMENT, "row stride %zu: at least %zu and, as the pointer, a multiple of 16", w_stride, w->cols);
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev != w->device)
    return fail(LMX_ERR_INVALID_ARGUMENT, "weight lives on device %d, current device is %d", w->device, dev);
  if (w->rows > 65535 * size_t(256)) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu rows", w->rows);
  // (grid.y holds 65535 rows a launch)
  for (size_t r = 0; r < w->rows; r += 65535) {
    const unsigned n = unsigned(std::min<size_t>(65535, w->rows - r));
    codes_i8_kernel<<<dim3(unsigned((w_stride + 255) / 256), n), 256, 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const int8_t *>(w->d_codes) + r * kChunk, w->d_scales + r, int(n), int(w->cols), int(w->Npad), w_stride,
        codes + r * w_stride, scales + r);
  }
  return launch_err("i8 codes of a weight");
}

}  // extern "C"
