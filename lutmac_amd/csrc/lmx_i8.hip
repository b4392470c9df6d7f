// lmx_i8.hip -- the linear layer in 8-bit integers (lmx_linear_i8): codes of
// the activations, one scale per row, and their product with 8-bit weights on
// the matrix cores, exact in 32-bit integers.
#include <hip/hip_runtime.h>

#include <algorithm>

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
};

// Codes of one row of x per workgroup: the largest magnitude, then
// round(127 x / amax), exactly rounded (round_quotient), zeros up to Kp.
// Up to K = 8192 the row stays in registers between the two.
template <class T>
__global__ __launch_bounds__(256) void i8_codes_kernel(I8Args a) {
  constexpr int KEEP = 4, E = 8;   // rounds of 256 x 8 elements kept
  __shared__ uint32_t tops[4];
  const int lane = threadIdx.x & (kWave - 1), row = int(blockIdx.x);
  const T *x = static_cast<const T *>(a.x) + size_t(row) * a.cols;
  const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
  const auto load = [&](int k, float (&v)[E]) {
    if (vec && k + E <= a.cols) {
      load_floats<E>(x + k, v);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = k + i < a.cols ? float(x[k + i]) : 0.0f;
    }
  };
  float keep[KEEP][E];
  uint32_t top = 0;
  const auto fold = [&top](const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  };
  const int k0 = int(threadIdx.x) * E;
#pragma unroll
  for (int j = 0; j < KEEP; ++j)
    if (k0 + j * 256 * E < a.cols) {
      load(k0 + j * 256 * E, keep[j]);
      fold(keep[j]);
    }
  for (int k = k0 + KEEP * 256 * E; k < a.cols; k += 256 * E) {
    float v[E];
    load(k, v);
    fold(v);
  }
  top = max(top, lane_xor_u32<32>(top, lane));
  top = max(top, lane_xor_u32<16>(top, lane));
  top = max(top, lane_xor_u32<8>(top, lane));
  top = max(top, lane_xor_u32<4>(top, lane));
  top = max(top, lane_xor_u32<2>(top, lane));
  top = max(top, lane_xor_u32<1>(top, lane));
  if (lane == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
  top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  const float amax = __uint_as_float(top);
  const bool some = top != 0 && top < 0x7F800000u;   // else the codes are zeros
  const double d = amax, inv = 1.0 / d;
  const auto store = [&](int k, const float (&v)[E]) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = some ? int(round_quotient(double(v[i]) * 127.0, d, inv)) : 0;
      w[i / 4] |= uint32_t(c & 0xFF) << (8 * (i % 4));
    }
    *reinterpret_cast<uint2 *>(a.codes + size_t(row) * a.Kp + k) = make_uint2(w[0], w[1]);
  };
#pragma unroll
  for (int j = 0; j < KEEP; ++j) {
    const int k = k0 + j * 256 * E;
    if (k < a.Kp) {
      if (k >= a.cols)
#pragma unroll
        for (int i = 0; i < E; ++i) keep[j][i] = 0.0f;
      store(k, keep[j]);
    }
  }
  for (int k = k0 + KEEP * 256 * E; k < a.Kp; k += 256 * E) {
    float v[E];
    load(k, v);
    store(k, v);
  }
  if (threadIdx.x == 0) a.scales[row] = top < 0x7F800000u ? amax / 127.0f : __builtin_nanf("");
}

// Four neighbouring outputs y[m][n .. n + 3] from their integer sums; whole
// groups go out in one store where y allows it (vec).
template <class T>
__device__ __forceinline__ void store4(const I8Args &a, int m, int n, const v4i s, float xs, bool vec) {
  if (m >= a.batch || n >= a.rows) return;
  T *y = static_cast<T *>(a.y) + size_t(m) * a.rows + n;
  const T *b = static_cast<const T *>(a.bias);
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = min(n + i, a.rows - 1);
    f[i] = float(s[i]) * a.w_scale[r] * xs + (b ? float(b[r]) : 0.0f);
  }
  if (vec && n + 3 < a.rows) {
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

// 16 bytes per lane from a buffer straight to LDS, lane l's at lds + 16 l (the
// host pass, which emits no device code, rejects the builtin).
__device__ __forceinline__ void buffer_to_lds(__amdgpu_buffer_rsrc_t buf, char *lds, int at, int base) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_void *)lds, 16, at, base, 0, 0);
#endif
}

// ---------------------------------------------------------------------------
// Few rows of activations (up to 16 NT): a workgroup takes 16 weight rows, its
// W waves the k-steps w, w + W, ...; every weight byte goes from memory to an
// operand register once, the codes come from the caches.
//   A (weights): lane (i, g) holds bytes 16 g .. + 15 of a 64-byte step of row i;
//   B (codes) the same of activation row j; C lane (j, g): weight rows 4 g .. + 3.
template <class T, int NT, int W>
__global__ __launch_bounds__(W *kWave) void i8_rows_kernel(I8Args a) {
  __shared__ v4i part[W > 1 ? W : 1][NT][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int i = lane & 15, g = lane >> 4, row0 = int(blockIdx.x) * 16;
  const auto wbuf = weight_buffer(a, row0);
  const int wrow = min(i, a.rows - 1 - row0) * int(a.w_stride) + 16 * g;
  const int8_t *xc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xc[t] = a.codes + size_t(min(16 * t + i, a.batch - 1)) * a.Kp + 16 * g;
  v4i acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = v4i{0, 0, 0, 0};
  for (int k = wave * kStep; k < a.Kp; k += W * kStep) {
    v4i w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(wbuf, wrow + k + 64 * h, 0, 0));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h], *reinterpret_cast<const v4i *>(xc[t] + k + 64 * h), acc[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  const bool vec = vector_rows<T>(a);
  for (int t = wave; t < NT; t += W) {
    v4i s = part[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s += part[w][t][lane];
    const int m = 16 * t + i;
    store4<T>(a, m, row0 + 4 * g, s, a.scales[min(m, a.batch - 1)], vec);
  }
}

// ---------------------------------------------------------------------------
// Many rows of activations: BN weight rows x BM activation rows per workgroup,
// WN x WM waves, k in steps of 128 bytes through two LDS buffers that are
// filled straight from memory while the other is multiplied
// (v_mfma_i32_32x32x32_i8).  A row's eight 16-byte pieces lie in LDS at p ^ (row
// / 2) % 8, so that the 16 lanes of a read's phase touch all 64 banks once.
template <class T, int BN, int BM, int WN, int WM>
__global__ __launch_bounds__(WN *WM *kWave) void i8_tile_kernel(I8Args a) {
  constexpr int W = WN * WM, TN = BN / WN / 32, TM = BM / WM / 32;
  constexpr int RB = (BN + BM) * kStep;   // bytes of a buffer: weights, then codes
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int wn = wave % WN, wm = wave / WN;
  const int row0 = int(blockIdx.x) * BN, m0 = int(blockIdx.y) * BM;
  const auto wbuf = weight_buffer(a, row0);
  const auto xbuf = __builtin_amdgcn_make_buffer_rsrc(a.codes + size_t(m0) * a.Kp, 0,
                                                      int(min(size_t(a.batch - m0) * a.Kp, size_t(0x7FFFFFFF))), 0x00020000);
  // One load instruction of a wave: 8 rows x 128 bytes.
  const int lr = lane >> 3, lp = lane & 7;
  constexpr int LN = BN / 8 / W, LM = BM / 8 / W;   // instructions per wave and buffer
  static_assert(LN * 8 * W == BN && LM * 8 * W == BM, "whole instructions");
  int won[LN], wom[LM];
#pragma unroll
  for (int j = 0; j < LN; ++j) {
    const int r = (j * W + wave) * 8 + lr;
    won[j] = min(r, a.rows - 1 - row0) * int(a.w_stride) + 16 * (lp ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int j = 0; j < LM; ++j) {
    const int r = (j * W + wave) * 8 + lr;
    wom[j] = min(r, a.batch - 1 - m0) * a.Kp + 16 * (lp ^ ((r >> 1) & 7));
  }
  const auto fill = [&](int buf, int k) {
#pragma unroll
    for (int j = 0; j < LN; ++j)
      buffer_to_lds(wbuf, lds + buf * RB + (j * W + wave) * 1024, won[j], k);
#pragma unroll
    for (int j = 0; j < LM; ++j)
      buffer_to_lds(xbuf, lds + buf * RB + BN * kStep + (j * W + wave) * 1024, wom[j], k);
  };
  v16i acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[n][m][v] = 0;
  const int i = lane & 31, h = lane >> 5;
  const int steps = a.Kp / kStep;
  fill(0, 0);
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (s + 1 < steps) fill((s + 1) & 1, (s + 1) * kStep);
    const char *wl = lds + (s & 1) * RB + (wn * (BN / WN) + i) * kStep;
    const char *xl = lds + (s & 1) * RB + BN * kStep + (wm * (BM / WM) + i) * kStep;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 16 * ((2 * q + h) ^ ((i >> 1) & 7));
      v4i wf[TN], xf[TM];
#pragma unroll
      for (int n = 0; n < TN; ++n) wf[n] = *reinterpret_cast<const v4i *>(wl + n * 32 * kStep + at);
#pragma unroll
      for (int m = 0; m < TM; ++m) xf[m] = *reinterpret_cast<const v4i *>(xl + m * 32 * kStep + at);
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[n], xf[m], acc[n][m], 0, 0, 0);
    }
  }
  const bool vec = vector_rows<T>(a);
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int mr = m0 + wm * (BM / WM) + 32 * m + i;
    const float xs = a.scales[min(mr, a.batch - 1)];
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        store4<T>(a, mr, row0 + wn * (BN / WN) + 32 * n + 8 * b + 4 * h,
                  v4i{acc[n][m][4 * b], acc[n][m][4 * b + 1], acc[n][m][4 * b + 2], acc[n][m][4 * b + 3]}, xs, vec);
  }
}

// ---- host side ----

int launch_err(const char *what) {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

template <class T, int NT>
void launch_rows(const I8Args &a, hipStream_t st) {
  const unsigned grid = unsigned((a.rows + 15) / 16);
  // more waves share a row tile's k where the tiles alone leave CUs idle
  if (grid < 512) i8_rows_kernel<T, NT, 8><<<grid, 8 * kWave, 0, st>>>(a);
  else i8_rows_kernel<T, NT, 4><<<grid, 4 * kWave, 0, st>>>(a);
}

template <class T, int BN, int BM, int WN, int WM>
int launch_tile(const I8Args &a, hipStream_t st) {
  constexpr size_t lds = 2 * (BN + BM) * kStep;
  static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&i8_tile_kernel<T, BN, BM, WN, WM>),
                                                  hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
  if (e != hipSuccess) return fail(LMX_ERR_HIP, "LDS of the i8 tile kernel: %s", hipGetErrorString(e));
  const dim3 grid(unsigned((a.rows + BN - 1) / BN), unsigned((a.batch + BM - 1) / BM));
  i8_tile_kernel<T, BN, BM, WN, WM><<<grid, WN * WM * kWave, lds, st>>>(a);
  return LMX_OK;
}

template <class T>
int launch_linear(const I8Args &a, hipStream_t st) {
  i8_codes_kernel<T><<<unsigned(a.batch), 256, 0, st>>>(a);
  int r = launch_err("i8 codes");
  if (r) return r;
  if (a.batch <= 64) {
    switch ((a.batch + 15) / 16) {
    case 1: launch_rows<T, 1>(a, st); break;
    case 2: launch_rows<T, 2>(a, st); break;
    case 3: launch_rows<T, 3>(a, st); break;
    default: launch_rows<T, 4>(a, st); break;
    }
  } else {
    const auto tiles = [&](int bn, int bm) { return size_t((a.rows + bn - 1) / bn) * size_t((a.batch + bm - 1) / bm); };
    if (tiles(256, 256) >= 256) r = launch_tile<T, 256, 256, 4, 2>(a, st);
    else r = launch_tile<T, 64, 64, 2, 2>(a, st);
  }
  return r ? r : launch_err("i8 linear");
}

size_t i8_workspace(size_t cols, size_t batch) {
  return round_up(batch * sizeof(float), 256) + batch * round_up(cols, kStep);
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
  *bytes = i8_workspace(cols, batch);
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
  a.codes = static_cast<int8_t *>(workspace) + round_up(batch * sizeof(float), 256);
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
