// lmx_f8.hip -- the linear layer in 8-bit floating point (lmx_linear_f8): e4m3
// weights with a scale per 128 x 128 block, activations rounded to e4m3 with a
// power of two per row and 128 columns, their products on the matrix cores.
//
// The products are made by the fp16 matrix instructions, which hold an e4m3 number
// exactly and sum in fp32.  The fp8 ones take half the time, but of every eight
// neighbouring k they drop what lies below 2^-13 of the largest product (measured:
// seven small ones beside a large one vanish): up to 7 * 2^-13 of a sum of one
// sign, more than half a step of fp16 and, near a border, a whole step of bf16.
// What that costs: nothing to speak of up to 64 rows, where the weights' bytes bound
// the call, a tenth to a third up to 1000, the matrix cores' factor of two beyond
// (8192 x 2048 -> 16384 275 us with the fp8 instructions, 483 so).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lmx_internal.hpp"
#include "lmx_lanes.hpp"
#include "lmx_types.hpp"

namespace lmx {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
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
  int Bp;            // batch padded to 64
  uint8_t *codes;    // [batch][Kp]
  float *scales;     // [steps][Bp]
  int splits;        // parts of k, each with sums of its own to join
  float *sums;       // [splits][batch][rows], or a few kernel's operands of sums
  unsigned *tickets; // a few kernel's, one for each of its row tiles, zeroed with the codes
  int n_tickets;
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

// Codes and scales of x: a workgroup a row, 16 lanes a block (8192 rows of 2048 bf16: 13
// to 17 us, 50 MB read and written; 48 of 8960 with 1024 threads a row 2.9).
template <class T, int NT>
__global__ __launch_bounds__(NT) void f8_codes_kernel(F8Args a) {
  const int lane = threadIdx.x & (kWave - 1), row = int(blockIdx.x);
  if (row == 0)
    for (int t = int(threadIdx.x); t < a.n_tickets; t += NT) a.tickets[t] = 0;
  const T *x = static_cast<const T *>(a.x) + size_t(row) * a.cols;
  const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
  for (int k = int(threadIdx.x) * 8; k < a.Kp; k += NT * 8) {   // (whole groups of 16 lanes)
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

// 128-byte rows in LDS: piece p (16 bytes) of row r lies at p ^ (r / 2 mod 8), so
// that the 16 lanes of a read's phase touch all 64 banks once.
__device__ __forceinline__ int piece_place(int row, int piece) { return 16 * (piece ^ (row >> 1 & 7)); }
// Where lane `lane` of a load of 8 rows reads row `row` (the last one past it).
__device__ __forceinline__ int piece_offset(int row, int last, int stride, int lane) {
  return min(row, last) * stride + piece_place(row, lane % 8);
}

// One step of 16 rows as a matrix instruction's operand: lane (i, g) holds bytes
// 16 g .. and 64 + 16 g .. of row i (any 32 bytes do, if both operands' are the same).
struct Operand {
  v4i a, b;
  __device__ __forceinline__ void cut(int left, int g) { a = cut_piece(a, left - 16 * g), b = cut_piece(b, left - 64 - 16 * g); }
};
__device__ __forceinline__ v8h halves(int lo, int hi) {   // 8 codes -> fp16, exactly
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true),
            c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The operand as the instructions take it.
struct Factor {
  v8h v[4];
  __device__ __forceinline__ explicit Factor(const Operand &o)
      : v{halves(o.a[0], o.a[1]), halves(o.a[2], o.a[3]), halves(o.b[0], o.b[1]), halves(o.b[2], o.b[3])} {}
  Factor() = default;
};
// The sums of a block of 128: lane (j, g) gets weight rows 4 g .. + 3 of activation row j.
__device__ __forceinline__ v4f products(const Factor &w, const Factor &x) {
  v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 4; ++q) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[q], x.v[q], p, 0, 0, 0);
  return p;
}
__device__ __forceinline__ void add_scaled(v4f &acc, const v4f &p, float f) {
#pragma unroll
  for (int v = 0; v < 4; ++v) acc[v] = fmaf(p[v], f, acc[v]);
}

// Biases of four neighbouring weight rows (past the last: its own).
template <class T>
__device__ __forceinline__ v4f biases(const F8Args &a, int n) {
  v4f f = {0.0f, 0.0f, 0.0f, 0.0f};
  if (const T *b = static_cast<const T *>(a.bias)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = float(b[min(n + i, a.rows - 1)]);
  }
  return f;
}
// Four neighbouring outputs y[m][n .. n + 3]; whole groups go out in one store where y allows it (vec).
template <class T>
__device__ __forceinline__ void store4(const F8Args &a, int m, int n, const v4f s, bool vec) {
  if (m >= a.batch || n >= a.rows) return;
  T *y = static_cast<T *>(a.y) + size_t(m) * a.rows + n;
  if (vec) {   // (then rows are whole groups)
    const float f[4] = {s[0], s[1], s[2], s[3]};
    store_floats<4>(y, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.rows) y[i] = T(s[i]);
  }
}
template <class T>
__device__ __forceinline__ bool vector_rows(const F8Args &a) {
  return a.rows % 4 == 0 && reinterpret_cast<size_t>(a.y) % (4 * sizeof(T)) == 0;
}

// ---------------------------------------------------------------------------
// One to four rows of activations, one launch: a workgroup takes 16 weight rows,
// its W waves the k-steps w, w + W, ..., each through U LDS buffers of its own that
// are filled straight from memory U - 1 steps ahead, so that no wave waits for
// another before the end.  Every workgroup makes the codes itself, in LDS while its
// first weights are on their way (R >= batch rows, a power of two; at most 16 values
// a thread, which stay in registers), which saves a launch and the trip through memory
// (1 x 2048 -> 16384 7.6 us, 4.4 TB/s).
constexpr int rows_buffers(int waves) { return waves == 16 ? 3 : 4; }
template <class T, int W, int R>
__global__ __launch_bounds__(W *kWave) void f8_rows_kernel(F8Args a) {
  constexpr int U = rows_buffers(W), RB = 16 * kStep;
  __shared__ v4f part[W][kWave];
  extern __shared__ __attribute__((aligned(1024))) char lds[];   // the waves' buffers, codes [batch][Kp + 16], factors [batch][steps]
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int i = lane & 15, g = lane >> 4, row0 = int(blockIdx.x) * 16;
  char *mine = lds + wave * (U * RB), *codes = lds + W * U * RB;
  float *factors = reinterpret_cast<float *>(codes + a.batch * (a.Kp + 16));
  constexpr int KEEP = 2, TR = W * kWave / R;   // threads of an activation row
  const int am = int(threadIdx.x) / TR, k0 = int(threadIdx.x) % TR * 8;
  const float *ws = a.w_scale + size_t(row0 / kStep) * a.steps;
  float v[KEEP][8], wf[KEEP];
  {
    const T *x = static_cast<const T *>(a.x) + size_t(min(am, a.batch - 1)) * a.cols;
    const bool vec = reinterpret_cast<size_t>(x) % 16 == 0;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      load8(x, k0 + j * TR * 8, a.cols, vec, v[j]);
      wf[j] = ws[min((k0 + j * TR * 8) / kStep, a.steps - 1)];
    }
  }
  const auto wbuf = weight_buffer(a, row0);
  int won[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) won[n] = piece_offset(8 * n + lane / 8, a.rows - 1 - row0, int(a.w_stride), lane);
  const int turns = wave < a.steps ? (a.steps - 1 - wave) / W + 1 : 0;
  const auto fill = [&](int buf, int t) {
#pragma unroll
    for (int n = 0; n < 2; ++n) buffer_to_lds(wbuf, mine + buf * RB + n * 1024, won[n], (wave + t * W) * kStep);
  };
#pragma unroll
  for (int t = 0; t < U - 1; ++t)
    if (t < turns) fill(t, t);
  if (am < a.batch) {
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const int k = k0 + j * TR * 8;
      if (k < a.Kp) {   // (whole groups of 16 lanes)
        float s;
        const uint2 c = block_codes(v[j], lane, s);
        *reinterpret_cast<uint2 *>(codes + am * (a.Kp + 16) + k) = c;
        if (lane % 16 == 0) factors[am * a.steps + k / kStep] = s * wf[j];
      }
    }
  }
  lds_barrier();
  const int m = min(i, a.batch - 1);
  const char *xc = codes + m * (a.Kp + 16) + 16 * g;
  const float *fc = factors + m * a.steps;
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  int buf = 0;
  for (int t = 0; t < turns; ++t) {
    if (t + U - 1 <= turns) wait_loads<(U - 2) * 2>();
    else wait_loads<0>();
    const int step = wave + t * W;
    const char *at = mine + buf * RB + i * kStep;
    Operand w = {*reinterpret_cast<const v4i *>(at + piece_place(i, g)), *reinterpret_cast<const v4i *>(at + piece_place(i, 4 + g))};
    const Operand x = {*reinterpret_cast<const v4i *>(xc + step * kStep), *reinterpret_cast<const v4i *>(xc + step * kStep + 64)};
    const float f = fc[step];
    if (t + U - 1 < turns) fill(buf == 0 ? U - 1 : buf - 1, t + U - 1);   // (the buffer of the step before, whose products are made)
    if (a.cols - step * kStep < kStep) w.cut(a.cols - step * kStep, g);
    add_scaled(acc, products(Factor(w), Factor(x)), f);
    buf = buf == U - 1 ? 0 : buf + 1;
  }
  part[wave][lane] = acc;
  const v4f bias = biases<T>(a, row0 + 4 * g);
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int v = 1; v < W; ++v) acc += part[v][lane];
  store4<T>(a, i, row0 + 4 * g, acc + bias, vector_rows<T>(a));
}

// ---------------------------------------------------------------------------
// Some rows of activations (up to 16 G) and so few weight rows that tiles of
// 64 x 64 leave CUs idle: 16 R weight rows a workgroup, its W waves the k-steps w,
// w + W, ..., each through U LDS buffers of its own as above (weights, codes, the
// codes' scales; 48 x 8960 -> 1536 9.2 us).  Where that is few workgroups, blockIdx.y takes a part of k: the parts'
// sums go past the caches, and the last workgroup of a row tile to finish adds them in
// their order.
template <class T, int W, int R, int G, int U>
__global__ __launch_bounds__(W *kWave) void f8_few_kernel(F8Args a) {
  constexpr int CB = (R + G) * 16 * kStep, RB = CB + 64 * 4;   // bytes of a buffer: weights, codes, 64 scales
  constexpr int LOADS = 2 * (R + G) + 1;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int i = lane & 15, g = lane >> 4, row0 = int(blockIdx.x) * (16 * R);
  const auto wbuf = weight_buffer(a, row0);
  const auto xbuf = __builtin_amdgcn_make_buffer_rsrc(a.codes, 0, a.batch * a.Kp, 0x00020000);
  const auto sbuf = __builtin_amdgcn_make_buffer_rsrc(a.scales, 0, a.steps * a.Bp * 4, 0x00020000);
  int won[2 * R], xon[2 * G];   // (a load instruction: 8 rows)
#pragma unroll
  for (int n = 0; n < 2 * R; ++n) won[n] = piece_offset(8 * n + lane / 8, a.rows - 1 - row0, int(a.w_stride), lane);
#pragma unroll
  for (int n = 0; n < 2 * G; ++n) xon[n] = piece_offset(8 * n + lane / 8, a.batch - 1, a.Kp, lane);
  char *mine = lds + wave * (U * RB);
  const int s0 = int(unsigned(a.steps) * blockIdx.y / gridDim.y), steps = int(unsigned(a.steps) * (blockIdx.y + 1) / gridDim.y) - s0;
  const int turns = wave < steps ? (steps - 1 - wave) / W + 1 : 0, w0 = s0 + wave;
  const auto fill = [&](int buf, int t) {
    const int k = (w0 + t * W) * kStep;
#pragma unroll
    for (int n = 0; n < 2 * R; ++n) buffer_to_lds(wbuf, mine + buf * RB + n * 1024, won[n], k);
#pragma unroll
    for (int n = 0; n < 2 * G; ++n) buffer_to_lds(xbuf, mine + buf * RB + (2 * R + n) * 1024, xon[n], k);
    buffer_to_lds<4>(sbuf, mine + buf * RB + CB, 4 * lane, (w0 + t * W) * a.Bp * 4);
  };
#pragma unroll
  for (int t = 0; t < U - 1; ++t)
    if (t < turns) fill(t, t);
  const float *ws = a.w_scale + size_t(row0 / kStep) * a.steps;
  float wf = scalar_load(ws + min(w0, a.steps - 1));
  v4f acc[R][G];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < G; ++n) acc[r][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  int buf = 0;
  for (int t = 0; t < turns; ++t) {
    if (t + U - 1 <= turns) wait_loads<(U - 2) * LOADS>();
    else wait_loads<0>();
    const int step = w0 + t * W;
    const char *at = mine + buf * RB + i * kStep;
    const int pa = piece_place(i, g), pb = piece_place(i, 4 + g);
    Operand w[R], x[G];
    float f[G];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = {*reinterpret_cast<const v4i *>(at + r * 16 * kStep + pa), *reinterpret_cast<const v4i *>(at + r * 16 * kStep + pb)};
#pragma unroll
    for (int n = 0; n < G; ++n) {
      x[n] = {*reinterpret_cast<const v4i *>(at + (R + n) * 16 * kStep + pa), *reinterpret_cast<const v4i *>(at + (R + n) * 16 * kStep + pb)};
      f[n] = *reinterpret_cast<const float *>(mine + buf * RB + CB + 4 * (16 * n + i)) * wf;
    }
    wf = scalar_load(ws + min(step + W, a.steps - 1));
    if (t + U - 1 < turns) fill(buf == 0 ? U - 1 : buf - 1, t + U - 1);   // (the buffer of the step before, whose products are made)
    if (a.cols - step * kStep < kStep)
#pragma unroll
      for (int r = 0; r < R; ++r) w[r].cut(a.cols - step * kStep, g);
    Factor wv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = Factor(w[r]);
#pragma unroll
    for (int n = 0; n < G; ++n) {
      const Factor xv(x[n]);
#pragma unroll
      for (int r = 0; r < R; ++r) add_scaled(acc[r][n], products(wv[r], xv), f[n]);
    }
    buf = buf == U - 1 ? 0 : buf + 1;
  }
  __syncthreads();   // every wave is done with its buffers
  v4f(*part)[R * G][kWave] = reinterpret_cast<v4f(*)[R * G][kWave]>(lds);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < G; ++n) part[wave][r * G + n][lane] = acc[r][n];
  __syncthreads();
  const auto outputs = [&](int q, const v4f &sum) __attribute__((always_inline)) {
    const int r = q / G, m = 16 * (q % G) + i, row = row0 + 16 * r + 4 * g;
    store4<T>(a, m, row, sum + biases<T>(a, row), vector_rows<T>(a));
  };
  const auto parts = [&](unsigned p, int q) __attribute__((always_inline)) {   // a lane's 16 bytes
    return reinterpret_cast<uint64_t *>(a.sums) + (((size_t(p) * gridDim.x + blockIdx.x) * (R * G) + q) * kWave + lane) * 2;
  };
  for (int q = wave; q < R * G; q += W) {
    v4f sum = part[0][q][lane];
#pragma unroll
    for (int v = 1; v < W; ++v) sum += part[v][q][lane];
    if (gridDim.y == 1) {
      outputs(q, sum);
    } else {
      struct Halves { uint64_t v[2]; };
      const Halves h = __builtin_bit_cast(Halves, sum);
#pragma unroll
      for (int v = 0; v < 2; ++v) __hip_atomic_store(parts(blockIdx.y, q) + v, h.v[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (gridDim.y == 1) return;
  __shared__ bool joins;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the sums are there before the ticket is taken
  __syncthreads();
  if (threadIdx.x == 0)
    joins = __hip_atomic_fetch_add(a.tickets + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.y - 1;
  __syncthreads();
  if (!joins) return;
  for (int q = wave; q < R * G; q += W) {
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (unsigned p = 0; p < gridDim.y; ++p) {
      struct Halves { uint64_t v[2]; } h;
#pragma unroll
      for (int v = 0; v < 2; ++v) h.v[v] = __hip_atomic_load(parts(p, q) + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sum += __builtin_bit_cast(v4f, h);
    }
    outputs(q, sum);
  }
}

// ---------------------------------------------------------------------------
// Many rows of activations: BN weight rows x BM activation rows per workgroup,
// WN x WM waves, a block of 128 k per step through S LDS buffers that are filled
// straight from memory S - 1 steps ahead.  Each step's products are summed apart and
// enter the result with the step's two scales.  8192 x 2048 -> 16384 takes 465 to 530 us (the
// clock falls under load), 1.2 to 1.0 PFLOP/s; matrix cores busy 0.53 and the vector unit 0.59 of
// the cycles (two thirds of it conversions to fp16).
//
// PART: workgroup (tile, part) takes part blockIdx.y of k and leaves its sums for
// f8_join_kernel: where tiles are few and k is long.
template <class T, bool PART, int BN, int BM, int WN, int WM, int S>
__global__ __launch_bounds__(WN *WM *kWave) __attribute__((amdgpu_waves_per_eu(2))) void f8_tile_kernel(F8Args a) {
  constexpr int W = WN * WM, NW = BN / WN, MW = BM / WM, TN = NW / 16, TM = MW / 16;
  constexpr int CB = (BN + BM) * kStep, RB = CB + BM * 4;   // bytes of a buffer: weights, codes, the codes' scales
  constexpr int SL = BM / 4 / W;   // lanes of a wave that load scales
  static_assert(NW <= kStep && kStep % NW == 0, "a wave's weight rows share a scale");
  static_assert(SL * 4 * W == BM && SL <= kWave, "a load for the scales");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
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
  constexpr int LN = BN / 8 / W, LM = BM / 8 / W, LOADS = LN + LM + 1;
  static_assert(LN * 8 * W == BN && LM * 8 * W == BM, "whole instructions");
  int won[LN], wom[LM];
#pragma unroll
  for (int j = 0; j < LN; ++j) won[j] = piece_offset((j * W + wave) * 8 + lane / 8, a.rows - 1 - row0, int(a.w_stride), lane);
#pragma unroll
  for (int j = 0; j < LM; ++j) wom[j] = piece_offset((j * W + wave) * 8 + lane / 8, a.batch - 1 - m0, a.Kp, lane);
  const int son = min(m0 + 4 * (wave * SL + lane), a.Bp - 4) * 4;   // (what is past the batch reaches no output)
  const auto fill = [&](int buf, int s) {
#pragma unroll
    for (int j = 0; j < LN; ++j) buffer_to_lds(wbuf, lds + buf * RB + (j * W + wave) * 1024, won[j], s * kStep);
#pragma unroll
    for (int j = 0; j < LM; ++j) buffer_to_lds(xbuf, lds + buf * RB + BN * kStep + (j * W + wave) * 1024, wom[j], s * kStep);
    const auto sbuf = __builtin_amdgcn_make_buffer_rsrc(a.scales + size_t(s) * a.Bp, 0, a.Bp * 4, 0x00020000);
    if (lane < SL) buffer_to_lds(sbuf, lds + buf * RB + CB + wave * SL * 16, son, 0);
  };
  v4f acc[TN][TM];
#pragma unroll
  for (int n = 0; n < TN; ++n)
#pragma unroll
    for (int m = 0; m < TM; ++m) acc[n][m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int i = lane & 15, g = lane >> 4;
  const int n_first = row0 + wn * NW;
  int steps = a.steps, s0 = 0;
  if constexpr (PART) {
    const int part = int(blockIdx.y);
    s0 = int(unsigned(a.steps) * unsigned(part) / unsigned(a.splits));
    steps = int(unsigned(a.steps) * unsigned(part + 1) / unsigned(a.splits)) - s0;
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < steps) fill(s, s0 + s);
  // (the weights' scales of a wave's rows, one of BN / 128 runs, wait in LDS)
  float *wsl = reinterpret_cast<float *>(lds + S * RB) + wn * NW / kStep * a.steps;
  for (int s = int(threadIdx.x); s < (BN + kStep - 1) / kStep * steps; s += W * kWave) {
    const int run = s / steps, at = s - run * steps;
    reinterpret_cast<float *>(lds + S * RB)[run * a.steps + at] =
        a.w_scale[size_t(min(row0 + run * kStep, a.rows - 1) / kStep) * a.steps + s0 + at];
  }
  int buf = 0;
  const int pa = piece_place(i, g), pb = piece_place(i, 4 + g);
  const int tail = a.cols % kStep != 0 && s0 + steps == a.steps ? steps - 1 : -1;   // the step that ends inside a block
  for (int s = 0; s < steps; ++s) {
    if (s + S - 1 <= steps) wait_loads<(S - 2) * LOADS>();
    else wait_loads<0>();
    lds_barrier();   // (a wave is there once its reads of the step before are done)
    if (s == tail) {   // past the last column there may be anything, a NaN too
      const int left = a.cols - (s0 + s) * kStep;
      for (int r = int(threadIdx.x); r < BN; r += W * kWave)
        for (int q = left / 16; q < 8; ++q) {
          v4i *piece = reinterpret_cast<v4i *>(lds + buf * RB + r * kStep + piece_place(r, q));
          *piece = cut_piece(*piece, left - 16 * q);
        }
      lds_barrier();
    }
    // What the first product needs is read first; then, in this order, an activation
    // operand ahead and matrix instructions with the vector unit's work on those before.
    const char *wl = lds + buf * RB + (wn * NW + i) * kStep, *xl = lds + buf * RB + (BN + wm * MW + i) * kStep;
    const float *sl = reinterpret_cast<const float *>(lds + buf * RB + CB) + wm * MW + i;
    const auto read = [&](const char *from, int n) __attribute__((always_inline)) {
      return Operand{*reinterpret_cast<const v4i *>(from + n * 16 * kStep + pa), *reinterpret_cast<const v4i *>(from + n * 16 * kStep + pb)};
    };
    Operand w[TN], x = read(xl, 0), ahead{};
    w[0] = read(wl, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 1; n < TN; ++n) w[n] = read(wl, n);
    float f[TM];
    const float wnow = wsl[s];
#pragma unroll
    for (int m = 0; m < TM; ++m) f[m] = sl[16 * m];
    __builtin_amdgcn_sched_barrier(0);
    v4f p[2][TN];
    Factor wv[TN];
#pragma unroll
    for (int m = 0; m <= TM; ++m) {
      if (m + 1 < TM) ahead = read(xl, m + 1);
      Factor xv{};
      if (m < TM) xv = Factor(x);
      const float fm = m > 0 ? f[m - 1] * wnow : 0.0f;
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        if (m == 0) wv[n] = Factor(w[n]);
        if (m < TM) p[m % 2][n] = products(wv[n], xv);
        if (m > 0) add_scaled(acc[n][m - 1], p[(m + 1) % 2][n], fm);
      }
      __builtin_amdgcn_sched_barrier(0);
      x = ahead;
      if (m == 0 && s + S - 1 < steps) fill(buf == 0 ? S - 1 : buf - 1, s0 + s + S - 1);
    }
    buf = buf == S - 1 ? 0 : buf + 1;
  }
  // The sums leave through LDS, 16 activation rows of the wave at a time, so that
  // stores are whole lines of y.
  typedef typename std::conditional<PART, float, T>::type Out;
  constexpr int LD = NW * int(sizeof(Out)) + 16;   // a row in LDS, apart by banks
  static_assert(W * 16 * LD <= S * RB, "the rows fit in the buffers");
  lds_barrier();   // every wave is done with the buffers
  char *out = lds + wave * (16 * LD);
  constexpr int V = 16 / int(sizeof(Out)), LPR = NW / V;   // elements of a store, lanes of a row
  Out *base = PART ? reinterpret_cast<Out *>(a.sums) + size_t(blockIdx.y) * a.batch * a.rows : static_cast<Out *>(a.y);
  v4f bias[TN];
#pragma unroll
  for (int n = 0; n < TN; ++n) bias[n] = PART ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : biases<T>(a, n_first + 16 * n + 4 * g);
  const bool vec = a.rows % V == 0 && reinterpret_cast<size_t>(base) % 16 == 0;
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int m1 = m0 + wm * MW + 16 * m;
    if (m1 >= a.batch) break;
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const v4f o = acc[n][m] + bias[n];
      const float f[4] = {o[0], o[1], o[2], o[3]};
      store_floats<4>(reinterpret_cast<Out *>(out + i * LD) + 16 * n + 4 * g, f);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    Out *y = base + size_t(m1) * a.rows + n_first;
    if (vec) {
      typedef Out vecT __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int q = 0; q < (16 * LPR + kWave - 1) / kWave; ++q) {
        const int r = q * (kWave / LPR) + lane / LPR, n = lane % LPR * V;
        if (r < 16 && m1 + r < a.batch && n_first + n < a.rows)
          *reinterpret_cast<vecT *>(y + size_t(r) * a.rows + n) = *reinterpret_cast<const vecT *>(out + r * LD + n * sizeof(Out));
      }
    } else {
      for (int q = 0; q < 16 * NW / kWave; ++q) {
        const int at = q * kWave + lane, r = at / NW, n = at % NW;
        if (m1 + r < a.batch && n_first + n < a.rows) y[size_t(r) * a.rows + n] = *reinterpret_cast<const Out *>(out + r * LD + n * sizeof(Out));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// y from the parts' sums, four weight rows of an activation row per thread.
template <class T>
__global__ __launch_bounds__(256) void f8_join_kernel(F8Args a) {
  const int quads = (a.rows + 3) / 4;
  const size_t at = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= size_t(quads) * a.batch) return;
  const int m = int(at / quads), n = int(at % quads) * 4;
  const float *p = a.sums + size_t(m) * a.rows + n;
  v4f s = biases<T>(a, n);
#pragma unroll 8
  for (int q = 0; q < a.splits; ++q, p += size_t(a.batch) * a.rows) {
    if (a.rows % 4 == 0) {
      s += *reinterpret_cast<const v4f *>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += n + i < a.rows ? p[i] : 0.0f;
    }
  }
  store4<T>(a, m, n, s, vector_rows<T>(a));
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

size_t tile_count(size_t rows, size_t batch, size_t side) { return (rows + side - 1) / side * ((batch + side - 1) / side); }

// Up to 64 activation rows go to f8_few_kernel, unless they are more than 32 and tiles of
// 64 x 64 are three quarters of a round of the CUs or more: then its 16 or 32 weight rows
// a workgroup read the codes too often.  32 read them less often than 16 where they still fill the
// chip.  (us in a graph, bf16, tiles / 16 weight rows / 32:
//   48 x 2048 ->  4096 13.9 /  7.7 /  8.7    64 x 2048 ->  4096 14.0 /  8.4 /  9.4
//   48 x 2048 ->  8192 14.4 / 11.9 /  9.9    64 x 2048 ->  8192 14.5 / 13.3 / 10.7
//   48 x 2048 -> 12288 14.8 / 16.0 / 14.7    64 x 2048 -> 12288 14.9 / 18.1 / 16.2
//   48 x 2048 -> 16384 15.7 / 20.3 / 16.1    64 x 2048 -> 16384 15.9 / 22.7 / 17.5
//   48 x 2048 -> 20000 20.4 / 24.0 / 20.4    64 x 2048 -> 20000 20.8 / 27.1 / 22.5
//   48 x 2048 -> 32768 23.5 / 36.6 / 27.2    64 x 2048 -> 32768 24.1 / 41.4 / 29.9
//   48 x 2048 -> 65536 43.6 / 68.1 / 49.5    64 x 2048 -> 65536 44.1 / 78.2 / 55.0
//   64 x 8192 -> 24576 68.2 / 85.4 / 67.8    64 x 8192 -> 32768 75.6 / 110.7 / 86.5
//   24 x 2048 -> 16384 15.4 / 14.6 / 13.5    24 x 2048 -> 32768 23.1 / 23.8 / 22.9
//   24 x 2048 -> 65536 43.0 / 40.6 / 41.2    32 x 8192 -> 32768 74.0 / 77.3 / 74.7;
// the other way: 32 x 512 -> 32768 10.2 / 13.3 / 13.2.)
enum class FewShape { none, rows16, rows32 };
FewShape few_shape(size_t rows, size_t batch) {
  if (batch > 64 || (batch > 32 && tile_count(rows, batch, 64) >= 192)) return FewShape::none;
  return batch > 16 && rows > 4096 ? FewShape::rows32 : FewShape::rows16;
}

// Parts of k for f8_few_kernel's 16 weight rows: as many as bring its workgroups to
// one per CU, of 16 steps at least (us, in one part / in parts: 48 x 8960 -> 1536 in 2
// 15.8 / 12.8, 16 x 8960 -> 1536 in 2 11.8 / 10.5, 48 x 4096 -> 2048 in 2 9.8 / 9.2, 48 x 4096 -> 1024 in
// 2 8.6 / 8.6).
int few_parts(size_t rows, size_t cols) {
  const size_t tiles = (rows + 15) / 16, steps = round_up(cols, kStep) / kStep;
  return int(std::max<size_t>(1, std::min<size_t>(256 / tiles, steps / 16)));
}

// Parts of k for other calls of few tiles: as many as bring the 64 x 64 tiles to
// one per CU, of 8 steps at least, if they are three (us, in one part / in parts:
// 100 x 8960 -> 1536 in 5 42 / 19.5, 200 x 8192 -> 1024 in 4 40 / 20.9).
int split_count(size_t rows, size_t cols, size_t batch) {
  if (few_shape(rows, batch) != FewShape::none) return few_shape(rows, batch) == FewShape::rows16 ? few_parts(rows, cols) : 1;
  const size_t tiles = tile_count(rows, batch, 64), steps = round_up(cols, kStep) / kStep;
  const size_t parts = tiles ? std::min<size_t>(256 / tiles, steps / 8) : 1;
  return parts < 3 ? 1 : int(parts);
}

// More waves share a row tile's k where the tiles alone leave CUs idle (us, 4 / 8 /
// 16 waves: 1 x 8192 -> 2048 - / 7.3 / 7.0, 1 x 2048 -> 8192 6.1 / 5.9 / 7.5, 1 x 2048 ->
// 16384 9.1 / 10.4 / 13.3).
int rows_waves(const F8Args &a) {
  const int tiles = (a.rows + 15) / 16;
  return tiles <= 256 ? 16 : tiles <= 768 ? 8 : 4;
}

template <class T, int W, int R>
int launch_rows(const F8Args &a, hipStream_t st) {
  constexpr size_t ring = W * rows_buffers(W) * 16 * kStep, most = ring + 1024 * W + 16 * R + 4 * R * 1024 * W / R / kStep;
  if (const int r = allow_lds(reinterpret_cast<const void *>(&f8_rows_kernel<T, W, R>), most)) return r;
  f8_rows_kernel<T, W, R><<<unsigned((a.rows + 15) / 16), W * kWave, ring + size_t(a.batch) * (a.Kp + 16 + 4 * a.steps), st>>>(a);
  return launch_err("f8 linear");
}
template <class T, int R>
int launch_rows(const F8Args &a, hipStream_t st) {
  switch (rows_waves(a)) {
  case 16: return launch_rows<T, 16, R>(a, st);
  case 8: return launch_rows<T, 8, R>(a, st);
  default: return launch_rows<T, 4, R>(a, st);
  }
}

// Whether every workgroup makes the codes itself: up to 4 rows, as long as that
// is two rounds of a workgroup's threads, and not too often for nothing (us,
// itself / codes in a launch before: 1 x 2048 -> 16384 9.2 / 11.8, 2 x 2048 -> 16384 11.1 /
// 12.0, 4 x 2048 -> 2048 4.0 / 5.7, 2 x 2048 -> 65536 33.3 / 31.8).
int row_slots(const F8Args &a) { return a.batch <= 2 ? a.batch : 4; }
bool in_one_launch(const F8Args &a) {
  return a.batch <= 4 && row_slots(a) * a.Kp <= 1024 * rows_waves(a) && (a.batch == 1 || a.rows <= 32768);
}

template <class T, bool PART, int BN, int BM, int WN, int WM, int S>
int launch_tile(const F8Args &a, hipStream_t st) {
  const size_t lds = S * ((BN + BM) * kStep + BM * 4) + (BN + kStep - 1) / kStep * a.steps * 4;   // (at most 8 KB of scales)
  const auto kernel = &f8_tile_kernel<T, PART, BN, BM, WN, WM, S>;
  if (const int r = allow_lds(reinterpret_cast<const void *>(kernel), lds)) return r;
  const size_t tiles = size_t((a.rows + BN - 1) / BN) * size_t((a.batch + BM - 1) / BM);
  if (tiles > (1u << 30)) return fail(LMX_ERR_INVALID_ARGUMENT, "%d x %d outputs", a.rows, a.batch);
  kernel<<<dim3(unsigned(round_up(tiles, 8)), unsigned(a.splits)), WN * WM * kWave, lds, st>>>(a);
  return launch_err("f8 linear");
}

template <class T, int W, int R, int G>
int launch_few(const F8Args &a, hipStream_t st) {
  constexpr size_t lds = W * 3 * ((R + G) * 16 * kStep + 256);
  if (const int r = allow_lds(reinterpret_cast<const void *>(&f8_few_kernel<T, W, R, G, 3>), lds)) return r;
  f8_few_kernel<T, W, R, G, 3><<<dim3(unsigned((a.rows + 16 * R - 1) / (16 * R)), unsigned(a.splits)), W * kWave, lds, st>>>(a);
  return launch_err("f8 linear");
}
template <class T>
int launch_few(const F8Args &a, hipStream_t st) {
  const int G = (a.batch + 15) / 16;
  if (few_shape(a.rows, a.batch) == FewShape::rows32)
    return G == 2 ? launch_few<T, 4, 2, 2>(a, st) : G == 3 ? launch_few<T, 4, 2, 3>(a, st) : launch_few<T, 4, 2, 4>(a, st);
  return G == 1 ? launch_few<T, 4, 1, 1>(a, st) : G == 2 ? launch_few<T, 4, 1, 2>(a, st) : G == 3 ? launch_few<T, 4, 1, 3>(a, st)
                                                                                            : launch_few<T, 4, 1, 4>(a, st);
}

template <class T>
int launch_linear(const F8Args &a, hipStream_t st) {
  if (in_one_launch(a)) {
    switch (row_slots(a)) {
    case 1: return launch_rows<T, 1>(a, st);
    case 2: return launch_rows<T, 2>(a, st);
    default: return launch_rows<T, 4>(a, st);
    }
  }
  // (few long rows: 1024 threads a row)
  if (a.Kp > 2048 && a.batch < 512) f8_codes_kernel<T, 1024><<<unsigned(a.batch), 1024, 0, st>>>(a);
  else f8_codes_kernel<T, 256><<<unsigned(a.batch), 256, 0, st>>>(a);
  int r = launch_err("f8 codes");
  if (r) return r;
  if (few_shape(a.rows, a.batch) != FewShape::none) return launch_few<T>(a, st);
  if (a.splits > 1) {
    if ((r = launch_tile<T, true, 64, 64, 2, 2, 4>(a, st))) return r;
    f8_join_kernel<T><<<unsigned((size_t(a.batch) * ((a.rows + 3) / 4) + 255) / 256), 256, 0, st>>>(a);
    return launch_err("f8 join");
  }
  // The larger tiles where they are not half empty and still fill most of the CUs, as they read less from the
  // L2s (us, bf16, 128 / 64: 2048 x 2048 -> 8192 70 / 106, 1024 x 2048 -> 8192 40 / 58, 256 x
  // 2048 -> 16384 28 / 33, 512 x 2048 -> 4096 26 / 19.6, 517 x 1400 -> 3001 21 / 15.7, 64 x 2048 -> 32768 30 / 24; 256 x
  // 128 take 498 for 8192 x 2048 -> 16384 where 128 x 128 take 500).
  if (a.batch > 64 && tile_count(a.rows, a.batch, 128) >= 160) return launch_tile<T, false, 128, 128, 2, 2, 2>(a, st);
  return launch_tile<T, false, 64, 64, 2, 2, 4>(a, st);
}

// Scales, codes and, of a call that splits k, its parts' sums.
size_t padded(size_t batch) { return round_up(batch, 64); }
size_t codes_at(size_t cols, size_t batch) { return round_up(round_up(cols, kStep) / kStep * padded(batch) * sizeof(float), 256); }
size_t sums_at(size_t cols, size_t batch) { return codes_at(cols, batch) + round_up(batch * round_up(cols, kStep), 256); }
size_t sum_bytes(size_t rows, size_t cols, size_t batch) {
  const int splits = split_count(rows, cols, batch);
  if (splits == 1) return 0;
  // (a few kernel's: whole tiles of 16 x 16)
  return size_t(splits) * (few_shape(rows, batch) == FewShape::none ? batch * rows : round_up(batch, 16) * round_up(rows, 16)) * sizeof(float);
}
size_t tickets_at(size_t rows, size_t cols, size_t batch) { return sums_at(cols, batch) + round_up(sum_bytes(rows, cols, batch), 16); }
size_t ticket_count(size_t rows, size_t cols, size_t batch) {
  return few_shape(rows, batch) != FewShape::none && split_count(rows, cols, batch) > 1 ? (rows + 15) / 16 : 0;
}
size_t f8_workspace(size_t rows, size_t cols, size_t batch) {
  return tickets_at(rows, cols, batch) + ticket_count(rows, cols, batch) * sizeof(unsigned);
}

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_linear_f8_workspace(size_t rows, size_t cols, size_t batch, int type, size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (rows == 0 || rows > (1u << 24) || cols == 0 || cols > 131072 || batch > (1u << 22))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu x %zu, %zu vectors: rows 1..2^24, cols 1..131072, at most 2^22 vectors", rows, cols, batch);
  *bytes = f8_workspace(rows, cols, batch);
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
  a.splits = split_count(rows, cols, batch);
  a.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + sums_at(cols, batch));
  a.tickets = reinterpret_cast<unsigned *>(static_cast<char *>(workspace) + tickets_at(rows, cols, batch));
  a.n_tickets = int(ticket_count(rows, cols, batch));
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch_linear<float>(a, st);
  case LMX_F16: return launch_linear<f16>(a, st);
  default: return launch_linear<bf16>(a, st);
  }
}

}  // extern "C"
