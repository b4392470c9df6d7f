// lmx_f8.hip -- the linear layer in 8-bit floating point (lmx_linear_f8): e4m3
// weights with a scale per 128 x 128 block, activations rounded to e4m3 with a
// power of two per row and 128 columns, their products on the matrix cores.
//
// The fp8 matrix instructions align the products that they sum to the largest and
// drop what lies below 2^-13 of it: 1.3e-5 of the result for normal data, far below
// half a step of a 16-bit result (2^-9, 2^-12 on average), far above that of fp32.
// Results in fp32 therefore come from the fp16 instructions, which hold an e4m3
// number exactly and sum in fp32, at half the rate.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lmx_internal.hpp"
#include "lmx_lanes.hpp"
#include "lmx_types.hpp"

namespace lmx {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;   // columns of a block and bytes of k per step
constexpr int kLeastExp = -126;

struct F8Args {
  const uint8_t *w;
  size_t w_stride;
  const float *w_scale;   // [ceil(rows / 128)][steps]
  const void *bias, *x;
  void *y;
  int rows, cols, batch, Kp, steps;
  int Bp;            // batch padded to whole 16-byte pieces
  uint8_t *codes;    // [batch][Kp]
  float *scales;     // [steps][Bp]
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

// Eight codes of a block of 128 columns that 16 lanes hold, and its scale: the
// smallest power of two s with amax <= 448 s, 448 = 1.75 * 2^8.  (A mantissa
// above 1.75 carries into the exponent.)
__device__ __forceinline__ uint2 block_codes(const float (&v)[8], int lane, float &scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, lane_xor_u32<8>(top, lane));
  top = max(top, lane_xor_u32<4>(top, lane));
  top = max(top, lane_xor_u32<2>(top, lane));
  top = max(top, lane_xor_u32<1>(top, lane));
  if (top >= 0x7F800000u) {   // not finite: NaN codes
    scale = 1.0f;
    return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
  }
  const int e = max(int((top + 0x1FFFFFu) >> 23) - 127 - 8, kLeastExp);
  scale = __uint_as_float(uint32_t(e + 127) << 23);
  const float inv = __uint_as_float(uint32_t(127 - e) << 23);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
  return make_uint2(uint32_t(lo), uint32_t(hi));
}

// Codes and scales of x: 16 lanes a block.
template <class T>
__global__ __launch_bounds__(256) void f8_codes_kernel(F8Args a) {
  const int lane = threadIdx.x & (kWave - 1), row = int(blockIdx.x);
  const T *x = static_cast<const T *>(a.x) + size_t(row) * a.cols;
  const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
  for (int k = int(threadIdx.x) * 8; k < a.Kp; k += 256 * 8) {   // (whole groups of 16 lanes)
    float v[8], s;
    load8(x, k, a.cols, vec, v);
    const uint2 c = block_codes(v, lane, s);
    *reinterpret_cast<uint2 *>(a.codes + size_t(row) * a.Kp + k) = c;
    if (lane % 16 == 0) a.scales[size_t(k / kStep) * a.Bp + row] = s;
  }
}

// Weight rows of a workgroup as a buffer: reads past the matrix give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t weight_buffer(const F8Args &a, int row0) {
  const size_t at = size_t(row0) * a.w_stride, end = (size_t(a.rows - 1) * a.w_stride + size_t(a.cols) + 3) / 4 * 4;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.w) + at, 0, int(min(end - at, size_t(0x7FFFFFFF))), 0x00020000);
}

// Bytes from `left` on of a piece set to zero: past the last column there may be
// anything, a NaN too.
__device__ __forceinline__ v4i cut_piece(v4i p, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = left - 4 * i;
    p[i] = n >= 4 ? p[i] : n <= 0 ? 0 : p[i] & int((1u << (8 * n)) - 1);
  }
  return p;
}

__device__ __forceinline__ void lds_barrier() {   // no wait for loads on their way, as __syncthreads makes
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A uniform factor through the scalar cache.
__device__ __forceinline__ float scalar_load(const float *p) {
  return *(const __attribute__((address_space(4))) float *)(p);
}

__device__ __forceinline__ v8h halves(int lo, int hi) {   // 8 codes -> fp16, exactly
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true),
            c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Many rows of activations: BN weight rows x BM activation rows per workgroup,
// WN x WM waves, a block of 128 k per step through S LDS buffers that are filled
// straight from memory S - 1 steps ahead.  A row's 16-byte pieces lie in LDS at p ^
// (row / 2 mod 8), so that the 16 lanes of a read's phase touch all 64 banks once.
// Each step's products are summed apart and enter the result with the step's two
// scales.
template <class T, int BN, int BM, int WN, int WM, int S>
__global__ __launch_bounds__(WN *WM *kWave) __attribute__((amdgpu_waves_per_eu(BN *BM / (WN * WM) > 8192 ? 1 : 2))) void f8_tile_kernel(F8Args a) {
  constexpr bool EXACT = std::is_same<T, float>::value;
  constexpr int W = WN * WM, TN = BN / WN / 32, TM = BM / WM / 32;
  constexpr int RB = (BN + BM) * kStep;   // bytes of a buffer: weights, then codes
  static_assert(BN / WN <= kStep && kStep % (BN / WN) == 0, "a wave's weight rows share a scale");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const auto swizzle = [](int row) { return (row >> 1) & 7; };
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
  // One load instruction of a wave: 1 KB, 8 rows.
  constexpr int LN = BN / 8 / W, LM = BM / 8 / W;
  static_assert(LN * 8 * W == BN && LM * 8 * W == BM, "whole instructions");
  const int lr = lane / 8, lp = lane % 8;
  int won[LN], wom[LM];
#pragma unroll
  for (int j = 0; j < LN; ++j) {
    const int r = (j * W + wave) * 8 + lr;
    won[j] = min(r, a.rows - 1 - row0) * int(a.w_stride) + 16 * (lp ^ swizzle(r));
  }
#pragma unroll
  for (int j = 0; j < LM; ++j) {
    const int r = (j * W + wave) * 8 + lr;
    wom[j] = min(r, a.batch - 1 - m0) * a.Kp + 16 * (lp ^ swizzle(r));
  }
  const auto fill = [&](int buf, int k) {
#pragma unroll
    for (int j = 0; j < LN; ++j) buffer_to_lds(wbuf, lds + buf * RB + (j * W + wave) * 1024, won[j], k);
#pragma unroll
    for (int j = 0; j < LM; ++j) buffer_to_lds(xbuf, lds + buf * RB + BN * kStep + (j * W + wave) * 1024, wom[j], k);
  };
  v16f acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[n][m][v] = 0.0f;
  const int i = lane & 31, h = lane >> 5;
  const int n_first = row0 + wn * (BN / WN);
  const float *ws = a.w_scale + size_t(min(n_first, a.rows - 1) / kStep) * a.steps;
  int xm[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) xm[m] = min(m0 + wm * (BM / WM) + 32 * m + i, a.batch - 1);
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < a.steps) fill(s, s * kStep);
  int buf = 0;
  for (int s = 0; s < a.steps; ++s) {
    float f[TM];
    const float wf = scalar_load(ws + s);
#pragma unroll
    for (int m = 0; m < TM; ++m) f[m] = a.scales[size_t(s) * a.Bp + xm[m]] * wf;
    wait_loads<0>();
    lds_barrier();   // (a wave is there once its reads of the step before are done)
    if (s + S - 1 < a.steps) fill(buf == 0 ? S - 1 : buf - 1, (s + S - 1) * kStep);
    const char *wl = lds + buf * RB + (wn * (BN / WN) + i) * kStep;
    const char *xl = lds + buf * RB + BN * kStep + (wm * (BM / WM) + i) * kStep;
    v4i wp[TN][4], xp[TM][4];   // pieces 2 q + h
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 16 * ((2 * q + h) ^ swizzle(i));
#pragma unroll
      for (int n = 0; n < TN; ++n) wp[n][q] = *reinterpret_cast<const v4i *>(wl + n * 32 * kStep + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) xp[m][q] = *reinterpret_cast<const v4i *>(xl + m * 32 * kStep + at);
    }
    const int left = a.cols - s * kStep;
    if (left < kStep) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int n = 0; n < TN; ++n) wp[n][q] = cut_piece(wp[n][q], left - 16 * (2 * q + h));
    }
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        v16f p;
#pragma unroll
        for (int v = 0; v < 16; ++v) p[v] = 0.0f;
        if constexpr (EXACT) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int o = 0; o < 4; o += 2)
              p = __builtin_amdgcn_mfma_f32_32x32x16_f16(halves(wp[n][q][o], wp[n][q][o + 1]), halves(xp[m][q][o], xp[m][q][o + 1]), p, 0, 0, 0);
        } else {
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            const v8i w8 = __builtin_shufflevector(wp[n][q], wp[n][q + 1], 0, 1, 2, 3, 4, 5, 6, 7),
                      x8 = __builtin_shufflevector(xp[m][q], xp[m][q + 1], 0, 1, 2, 3, 4, 5, 6, 7);
            p = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, x8, p, 0, 0, 0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[n][m][v] = fmaf(p[v], f[m], acc[n][m][v]);
      }
    buf = buf == S - 1 ? 0 : buf + 1;
  }
  // The sums leave through LDS, 32 activation rows of the wave at a time, so
  // that stores are whole lines of y.
  constexpr int NW = BN / WN, LD = NW * int(sizeof(T)) + 16;   // a row in LDS, apart by banks
  static_assert(W * 32 * LD <= S * RB, "the rows fit in the buffers");
  lds_barrier();   // every wave is done with the buffers
  char *out = lds + wave * (32 * LD);
  constexpr int V = 16 / int(sizeof(T)), LPR = NW / V;   // elements of a store, lanes of a row
  T *base = static_cast<T *>(a.y);
  const T *bias = static_cast<const T *>(a.bias);
  const bool vec = a.rows % V == 0 && reinterpret_cast<size_t>(base) % 16 == 0;
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int m1 = m0 + wm * (BM / WM) + 32 * m;
    if (m1 >= a.batch) break;
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int at = 32 * n + 8 * b + 4 * h;
        float o[4];
#pragma unroll
        for (int v = 0; v < 4; ++v)
          o[v] = acc[n][m][4 * b + v] + (bias ? float(bias[min(n_first + at + v, a.rows - 1)]) : 0.0f);
        store_floats<4>(reinterpret_cast<T *>(out + i * LD) + at, o);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    T *y = base + size_t(m1) * a.rows + n_first;
    if (vec) {
      typedef T vecT __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int q = 0; q < 32 * LPR / kWave; ++q) {
        const int r = q * (kWave / LPR) + lane / LPR, n = lane % LPR * V;
        if (m1 + r < a.batch && n_first + n < a.rows)
          *reinterpret_cast<vecT *>(y + size_t(r) * a.rows + n) = *reinterpret_cast<const vecT *>(out + r * LD + n * sizeof(T));
      }
    } else {
      for (int q = 0; q < 32 * NW / kWave; ++q) {
        const int at = q * kWave + lane, r = at / NW, n = at % NW;
        if (m1 + r < a.batch && n_first + n < a.rows) y[size_t(r) * a.rows + n] = *reinterpret_cast<const T *>(out + r * LD + n * sizeof(T));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- host side ----

int launch_err(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

// (per device: asked before each launch, 0.2 us)
int allow_lds(const void *kernel, size_t bytes) {
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_HIP, "LDS of an f8 kernel: %s", hipGetErrorString(e));
}

template <class T, int BN, int BM, int WN, int WM, int S>
int launch_tile(const F8Args &a, hipStream_t st) {
  constexpr size_t lds = S * (BN + BM) * kStep;
  if (const int r = allow_lds(reinterpret_cast<const void *>(&f8_tile_kernel<T, BN, BM, WN, WM, S>), lds)) return r;
  const size_t tiles = size_t((a.rows + BN - 1) / BN) * size_t((a.batch + BM - 1) / BM);
  if (tiles > (1u << 30)) return fail(LMX_ERR_INVALID_ARGUMENT, "%d x %d outputs", a.rows, a.batch);
  f8_tile_kernel<T, BN, BM, WN, WM, S><<<unsigned(round_up(tiles, 8)), WN * WM * kWave, lds, st>>>(a);
  return launch_err("f8 linear");
}

template <class T>
int launch_linear(const F8Args &a, hipStream_t st) {
  f8_codes_kernel<T><<<unsigned(a.batch), 256, 0, st>>>(a);
  const int r = launch_err("f8 codes");
  return r ? r : launch_tile<T, 64, 64, 2, 2, 4>(a, st);
}

// Scales, then codes.
size_t padded(size_t batch) { return round_up(batch, 4); }
size_t codes_at(size_t cols, size_t batch) { return round_up(round_up(cols, kStep) / kStep * padded(batch) * sizeof(float), 256); }
size_t f8_workspace(size_t cols, size_t batch) { return codes_at(cols, batch) + batch * round_up(cols, kStep); }

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_linear_f8_workspace(size_t rows, size_t cols, size_t batch, int type, size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (rows == 0 || rows > (1u << 24) || cols == 0 || cols > 131072 || batch > (1u << 22))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu x %zu, %zu vectors: rows 1..2^24, cols 1..131072, at most 2^22 vectors", rows, cols, batch);
  *bytes = f8_workspace(cols, batch);
  return LMX_OK;
}

int lmx_linear_f8(const uint8_t *w, size_t w_stride, const float *w_scale, const void *bias, const void *x, void *y, int type,
                  size_t rows, size_t cols, size_t batch, void *workspace, size_t workspace_bytes, void *stream) {
  size_t need = 0;
  const int r = lmx_linear_f8_workspace(rows, cols, batch, type, &need);
  if (r) return r;
  if (batch == 0) return LMX_OK;
  const size_t e = type_bytes(type);
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
  F8Args a{};
  a.w = w, a.w_stride = w_stride, a.w_scale = w_scale, a.bias = bias, a.x = x, a.y = y;
  a.rows = int(rows), a.cols = int(cols), a.batch = int(batch), a.Kp = int(round_up(cols, kStep)), a.steps = a.Kp / kStep;
  a.Bp = int(padded(batch));
  a.scales = static_cast<float *>(workspace);
  a.codes = static_cast<uint8_t *>(workspace) + codes_at(cols, batch);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch_linear<float>(a, st);
  case LMX_F16: return launch_linear<f16>(a, st);
  default: return launch_linear<bf16>(a, st);
  }
}

}  // extern "C"
