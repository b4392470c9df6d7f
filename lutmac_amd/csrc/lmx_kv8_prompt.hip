// lmx_kv8_prompt.hip -- attention of many rows per sequence over the 8-bit
// paged cache (include/lutmac_kv8.h), for 16-bit activations.
#include "lmx_kv8.hpp"

namespace lmx {
namespace {

typedef int v16i __attribute__((ext_vector_type(16)));

// Bytes from memory straight to LDS, 16 per lane, lane l's at lds + 16 l.
__device__ __forceinline__ void memory_to_lds(const int8_t *from, char *lds) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) const void global_void;
  __builtin_amdgcn_global_load_lds((global_void *)from, (lds_void *)lds, 16, 0, 0);
#endif
}

template <class T, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv8_prompt_kernel(AttnArgs a) {
  constexpr int W = 4, M = HD / 32, D = HD / 32, KB = kPage * HD;
  constexpr float E = 11.98f, kRoom = 3.0f;
  __shared__ __attribute__((aligned(1024))) char buf[2][2 * KB];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int j = lane & 31, h = lane >> 5;
  const int kvh = int(blockIdx.y), group = a.c.group;
  int first = 0;
  // the last tiles, which see the most, first
  const int unit = int(gridDim.x) - 1 - int(blockIdx.x);
  const int seq = unit_sequence(a.c, unit, group, 1, lane, first, kPromptRows);
  if (seq < 0) return;
  const SeqRows r(a.c, seq);
  const int tile0 = (unit - first) * kPromptRows, rows = r.n * group;
  if (tile0 >= rows) return;
  const int see = min(r.len, a.c.max_pages * kPage) - 1;
  const int i0 = tile0 + 32 * wave, i = min(i0 + j, rows - 1);
  const int first_pos = min(r.start + min(i0, rows - 1) / group, see);              // of the wave's rows
  const int last_pos = min(r.start + min(i0 + 31, rows - 1) / group, see);
  const int tile_last = min(r.start + min(tile0 + kPromptRows - 1, rows - 1) / group, see);   // of the workgroup's
  const int limit = min(r.start + i / group, see);
  const int n_pages = tile_last < 0 ? 0 : tile_last / kPage + 1;
  const int part = int(blockIdx.z);
  const int p0 = int((long long)n_pages * part / a.splits), p1 = int((long long)n_pages * (part + 1) / a.splits);

  // query digits: this lane's 16 dimensions of every 32-dimension step
  v4i qd[M][2];
  float qs;
  {
    const T *q = static_cast<const T *>(a.q) + size_t(r.r0 + i / group) * a.q_stride + size_t(kvh * group + i % group) * HD;
    float x[M][16];
    uint32_t top = 0;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      load_floats<16>(q + 32 * m + 16 * h, x[m]);
#pragma unroll
      for (int d = 0; d < 16; ++d) top = max(top, __float_as_uint(x[m][d]) & 0x7FFFFFFFu);
    }
    top = max(top, lane_xor_u32<32>(top, lane));
    const bool finite = top < 0x7F800000u;
    const int e = max(int(top >> 23), 29) - 126;
    const float f = finite ? __builtin_amdgcn_ldexpf(1.0f, Digits<2>::q_bits - e) : 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int d = 0; d < 16; ++d) x[m][d] = finite ? x[m][d] : 0.0f;
      query_digits<2>(x[m], f, qd[m]);
    }
    qs = finite ? __builtin_amdgcn_ldexpf(a.scale, e - Digits<2>::q_bits) : __builtin_nanf("");
  }

  // LDS: 16-byte piece c of key token t at piece c ^ swizzle(t) of its row, of
  // value dimension d at c ^ (d / 4) % 4: the 16 lanes of a read's phase touch
  // all banks once.
  const auto key_swizzle = [](int t) {
    return HD == 128 ? ((t >> 1) & 3) | ((t >> 4) & 1) << 2 : ((t >> 2) & 1) | ((t >> 4) & 1) << 1;
  };
  constexpr int KP = HD / 16;            // pieces of a key row
  constexpr int LOADS = KB / 1024 / W;   // load instructions per wave, of keys and of values
  int kfrom[LOADS], vfrom[LOADS];
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const int at = (n * W + wave) * 64 + lane;   // 16-byte piece of the page
    const int t = at / KP, d = at / 4;
    kfrom[n] = t * HD + 16 * ((at % KP) ^ key_swizzle(t));
    vfrom[n] = d * kPage + 16 * ((at % 4) ^ ((d >> 2) & 3));
  }
  const auto stage = [&](int page, int b) {
    const size_t at = (size_t(page) * a.c.n_kv + kvh) * KB;
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      memory_to_lds(a.c.k + at + kfrom[n], buf[b] + (n * W + wave) * 1024);
      memory_to_lds(a.c.v + at + vfrom[n], buf[b] + KB + (n * W + wave) * 1024);
    }
  };
  // operand reads: key row i = 8 b + 4 h' + r of a 32-token tile is token 16 h'
  // + 4 b + r, so that lane half h ends with the 16 tokens of block h in order
  const int tok = 16 * ((j >> 2) & 1) + 4 * (j >> 3) + (j & 3);
  int koff[M], voff[2];
#pragma unroll
  for (int m = 0; m < M; ++m) koff[m] = tok * HD + 16 * ((2 * m + h) ^ key_swizzle(tok));
#pragma unroll
  for (int t = 0; t < 2; ++t) voff[t] = KB + j * kPage + 16 * ((2 * t + h) ^ ((j >> 2) & 3));

  const int *table = a.c.pages + size_t(seq) * a.c.max_pages;
  v16i acc[D][2];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[d][n][v] = 0;
  v16i zero;
#pragma unroll
  for (int v = 0; v < 16; ++v) zero[v] = __float_as_int(kMagic);
  float mref = 0.0f, l = 0.0f, thr = -INFINITY;
  int exmax = kLeastExp + kExpSpan;

  // acc and l by 2^-s (s <= 16 a round)
  const auto scale_down = [&](int s) {
    for (; __builtin_amdgcn_ballot_w64(s > 0) != 0; s -= 16) {
      const int n = min(max(s, 0), 16);
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int hi = acc[d][1][v], rest = hi & ((1 << n) - 1);
          acc[d][1][v] = hi >> n;
          acc[d][0][v] = (acc[d][0][v] >> n) + ((rest << 8) >> n);
        }
      l = __builtin_amdgcn_ldexpf(l, -n);
    }
  };

  int page = p0 < p1 ? __builtin_amdgcn_readfirstlane(table[p0]) : -1;
  if (page_ok(a.c, page)) stage(page, 0);
  for (int p = p0; p < p1; ++p) {
    const int here = page, b = (p - p0) & 1;
    page = p + 1 < p1 ? __builtin_amdgcn_readfirstlane(table[p + 1]) : -1;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (page_ok(a.c, page)) stage(page, b ^ 1);
    if (!page_ok(a.c, here) || p * kPage > last_pos) continue;   // (uniform over the wave)
    const size_t sc = (size_t(here) * a.c.n_kv + kvh) * kPageBlocks + h;
    const char *kl = buf[b];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int t0 = p * kPage + 32 * t + 16 * h;   // this lane's first token
      float ks = a.c.k_scale[sc + 2 * t], vs = a.c.v_scale[sc + 2 * t];
      v16i s[2] = {zero, zero};
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const v4i k = *reinterpret_cast<const v4i *>(kl + koff[m] + t * 32 * HD);
        s[0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, qd[m][0], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, qd[m][1], s[1], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (t0 > last_pos) ks = 0.0f, vs = 0.0f;
      int ex = value_exponent(vs);
      exmax = max(exmax, max(ex, lane_xor_int<32>(ex, lane)));
      ex = max(ex, exmax - kExpSpan);
      const float mant = __builtin_amdgcn_ldexpf(vs, -ex), c = qs * ks;
      const float off = float(ex) - mref + E;
      float y[16], top = -INFINITY;
      const bool masked = p * kPage + 32 * t + 31 > first_pos;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float d[2] = {__int_as_float(s[0][v]), __int_as_float(s[1][v])};
        y[v] = fmaf(join<2>(d), c, off);
        if (masked && t0 + v > limit) y[v] = -INFINITY;
        top = fmaxf(top, y[v]);
      }
      if (__builtin_amdgcn_ballot_w64(top > thr) != 0) {   // a row's maximum outgrows its reference
        top = fmaxf(top, lane_xor<32>(top, lane));
        if (top > thr) {
          const float now = ceilf(top - E + mref), by = now - mref;
          const int sh = thr == -INFINITY ? 0 : int(fminf(by, 1000.0f));
#pragma unroll
          for (int v = 0; v < 16; ++v) y[v] -= by;
          mref = now, thr = E + kRoom;
          top = __int_as_float(sh);
        } else {
          top = 0.0f;
        }
        scale_down(__float_as_int(top));
      }
      v4i pd[2];
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t w[4], dw[2];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float e = __builtin_amdgcn_exp2f(y[4 * u + v]);
          sum += e;
          w[v] = __float_as_uint(fmaf(e, mant, kMagic + float(Digits<2>::carry)));
        }
        digit_words<2>(w, dw);
        pd[0][u] = int(dw[0]), pd[1][u] = int(dw[1]);
      }
      const float unit_l = vs - vs == 0.0f ? __builtin_amdgcn_ldexpf(1.0f, kSumExp - ex) : __builtin_nanf("");
      if (sum != 0.0f) l = fmaf(sum, unit_l, l);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const v4i v = *reinterpret_cast<const v4i *>(kl + voff[t] + d * 32 * kPage);
        acc[d][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(v, pd[0], acc[d][0], 0, 0, 0);
        acc[d][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(v, pd[1], acc[d][1], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // a page adds at most 2^20 to a sum of digit products
    if (((p - p0) & 1023) == 1023) {
      scale_down(1);
      mref += 1.0f;
    }
  }
  l += lane_xor<32>(l, lane);
  if (a.splits > 1) {
    const size_t at = ((size_t(unit) * a.c.n_kv + kvh) * a.splits + part) * kPromptRows + 32 * wave + j;
    if (h == 0) a.part_ml[at] = make_float2(thr == -INFINITY ? -INFINITY : mref, l);
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float f[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) f[v] = fmaf(float(acc[d][1][4 * b + v]), 256.0f, float(acc[d][0][4 * b + v]));
        store_floats<4>(a.part_o + at * HD + 32 * d + 8 * b + 4 * h, f);
      }
    return;
  }
  if (i0 + j >= rows) return;
  const float inv = inverse_sum(l);
  T *out = static_cast<T *>(a.out) + size_t(r.r0 + i / group) * a.out_stride + size_t(kvh * group + i % group) * HD;
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      float f[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) f[v] = fmaf(float(acc[d][1][4 * b + v]), 256.0f, float(acc[d][0][4 * b + v])) * inv;
      store_floats<4>(out + 32 * d + 8 * b + 4 * h, f);
    }
}

template <class T>
void launch(const AttnArgs &a, size_t hd, dim3 grid, hipStream_t st) {
  if (hd == 64) kv8_prompt_kernel<T, 64><<<grid, dim3(256), 0, st>>>(a);
  else kv8_prompt_kernel<T, 128><<<grid, dim3(256), 0, st>>>(a);
}

}  // namespace

int launch_prompt(const AttnArgs &a, int type, size_t hd, size_t units, hipStream_t st) {
  const dim3 grid(unsigned(units), unsigned(a.c.n_kv), unsigned(a.splits));
  if (type == LMX_F16) launch<f16>(a, hd, grid, st);
  else launch<bf16>(a, hd, grid, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "kv8 prompt attention launch: %s", hipGetErrorString(e));
}

}  // namespace lmx
