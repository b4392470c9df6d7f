// lmx_kv8_prompt.hip -- attention of many rows per sequence over the 8-bit
// paged cache (include/lutmac_kv8.h), for 16-bit activations.
//
// 8 waves take 32 rows (a row: one query head of one token) of one KV head each
// and share its pages, which pass through LDS as fp16: codes are whole numbers
// below 2^8 and queries, scaled by a power of two, have at most 11 bits, so both
// are exact, and v_mfma_f32_32x32x16_f16 sums their products in fp32.
//   S^T = K Q^T: key row i = 8 b + 4 h' + r of a 32-token tile is its token 16 h'
//     + 4 b + r, so lane (row j, h) ends with the 16 tokens of block h in order:
//     one K and one V scale per lane, and P^T's operand in place;
//   O^T = V^T P^T with weights p 2^E in fp16: 11 bits each, which moves an fp16
//     output by about its own rounding and a bf16 one by an eighth of that (with
//     byte digits, as steps have them, the kernel took 1052 us).
// p is relative to a running reference of score + log2(V scale), raised only
// when a row outgrows it by 2^kRoom: then, seldom, the sums are scaled down.
//
// What bounds it is the vector unit (about 100 operations and 16 exponentials a
// tile and wave, next to 16 matrix instructions), so a wave keeps three tiles in
// flight: while the matrix cores sum the values of the tile before, the scores
// of this one are scaled, and while they make the scores of the next, its
// weights.  Two sequences of 4096 rows after 4096, 32 query and 8 KV heads of 128:
// 863 to 882 us by card, 930 to 950 TFLOP/s (CUs busy 0.95 of the time, of that the
// vector unit 0.62 and the matrix cores 0.45; operands read three or four steps
// ahead instead of two change nothing).
#include "lmx_kv8.hpp"

namespace lmx {
namespace {

typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef f16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// 16 signed bytes -> fp16, exactly: 0x64xx is 1024 + xx.
__device__ __forceinline__ void codes_to_f16(v4u x, v4u &lo, v4u &hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = x[i] ^ 0x80808080u;
    const v2h off = {f16(-1152.0f), f16(-1152.0f)};
    const v2h a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    const v2h b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
    v4u &w = i < 2 ? lo : hi;
    w[2 * (i & 1)] = __builtin_bit_cast(uint32_t, a);
    w[2 * (i & 1) + 1] = __builtin_bit_cast(uint32_t, b);
  }
}

constexpr int kPromptWaves = kPromptRows / 32;

template <class T, int HD>
__global__ __launch_bounds__(kPromptWaves *kWave) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv8_prompt_kernel(AttnArgs a) {
  constexpr int M = HD / 16, D = HD / 32, KB = kPage * HD * 2;   // KB: bytes of a page's keys (or values) in LDS
  constexpr float E = 8.0f, kRoom = 7.0f;                         // weights up to 2^15
  extern __shared__ __attribute__((aligned(1024))) char buf[];    // keys of two pages, values of three
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int j = lane & 31, h = lane >> 5;
  const int kvh = int(blockIdx.x) % a.c.n_kv, group = a.c.group;
  // the last tiles, which see the most, first, of all heads: what is left at the
  // end is short (heads one after another left CUs idle for a sixth of the time)
  const int unit = int(gridDim.x - 1 - blockIdx.x) / a.c.n_kv;
  const SeqRows r = unit_rows(a.c, unit, group, 1, lane, kPromptRows);
  const int tile0 = (unit - r.first) * kPromptRows, rows = r.n * group;
  if (r.seq < 0 || tile0 >= rows) return;
  const int see = min(r.len, a.c.max_pages * kPage) - 1;
  const int i0 = tile0 + 32 * wave, i = min(i0 + j, rows - 1);
  const int first_pos = min(r.start + min(i0, rows - 1) / group, see);              // of the wave's rows
  const int last_pos = min(r.start + min(i0 + 31, rows - 1) / group, see);
  const int tile_last = min(r.start + min(tile0 + kPromptRows - 1, rows - 1) / group, see);   // of the workgroup's
  const int limit = min(r.start + i / group, see);
  const int n_pages = tile_last < 0 ? 0 : tile_last / kPage + 1;
  const int part = int(blockIdx.z);
  const int p0 = part_begin(n_pages, part, a.splits), p1 = part_begin(n_pages, part + 1, a.splits);

  // the row's query: this lane's 8 dimensions of every 16-dimension step
  v8h qf[M];
  float qs;
  {
    const T *q = static_cast<const T *>(a.q) + size_t(r.r0 + i / group) * a.q_stride + size_t(kvh * group + i % group) * HD;
    float x[M][8];
    uint32_t top = 0;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      load_floats<8>(q + 16 * m + 8 * h, x[m]);
#pragma unroll
      for (int d = 0; d < 8; ++d) top = max(top, __float_as_uint(x[m][d]) & 0x7FFFFFFFu);
    }
    top = max(top, lane_xor_u32<32>(top, lane));
    const bool finite = top < 0x7F800000u;
    const int e = max(int(top >> 23), 29) - 126;   // |x| < 2^e
    const float f = finite ? __builtin_amdgcn_ldexpf(1.0f, 14 - e) : 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int d = 0; d < 8; ++d) qf[m][d] = finite ? f16(x[m][d] * f) : f16(0.0f);
    qs = finite ? __builtin_amdgcn_ldexpf(a.scale, e - 14) : __builtin_nanf("");
  }

  // LDS: 16-byte piece c of key token t lies at piece c ^ key_swizzle(t) of its
  // row, of value dimension d at c ^ (d / 2) % 8: the 16 lanes of a read's phase
  // touch all banks once.
  const auto key_swizzle = [](int t) {
    return HD == 128 ? (t & 7) | ((t >> 4) & 1) << 3 : ((t >> 1) & 3) | ((t >> 4) & 1) << 2;
  };
  // Loads: 16 codes each, a page's keys by the first KC of them
  constexpr int KC = kPage * HD / 16, LOADS = 2 * KC / (kPromptWaves * kWave);
  static_assert(LOADS * kPromptWaves * kWave == 2 * KC, "whole rounds");
  int from[LOADS], to[LOADS][2];
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const int at = (n * int(kPromptWaves * kWave) + int(threadIdx.x)) % KC;
    from[n] = 16 * at;
    const int t = at / (HD / 16), d = at / 4;
#pragma unroll
    for (int w = 0; w < 2; ++w)
      to[n][w] = n * kPromptWaves * kWave + wave * kWave < KC ? t * 2 * HD + 16 * ((2 * (at % (HD / 16)) + w) ^ key_swizzle(t))
                                                           : d * 2 * kPage + 16 * ((2 * (at % 4) + w) ^ ((d >> 1) & 7));
  }
  const int tok = 16 * ((j >> 2) & 1) + 4 * (j >> 3) + (j & 3);
  int koff[M], voff[4];   // of the lane's key row, and of its value row's four pieces (tile, step)
#pragma unroll
  for (int m = 0; m < M; ++m) koff[m] = tok * 2 * HD + 16 * ((2 * m + h) ^ key_swizzle(tok));
#pragma unroll
  for (int t = 0; t < 4; ++t) voff[t] = j * 2 * kPage + 16 * ((4 * (t >> 1) + 2 * h + (t & 1)) ^ ((j >> 1) & 7));

  const int *table = a.c.pages + size_t(r.seq) * a.c.max_pages;
  v16f acc[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[d][v] = 0.0f;
  float mref = 0.0f, l = 0.0f, thr = -INFINITY, vmax = 0x1p-40f;

  // A page's codes on their way to LDS, and the scales of this lane's two
  // blocks; a page outside the pool has zeros, and no token of it is seen.
  struct Page {
    v4u code[LOADS];
    float k[2], v[2];
    bool ok;
  };
  // (the table's entry is read a page before it is needed)
  int entry = p0 < p1 ? table[p0] : -1;
  const auto request = [&](int p) {
    const int page = p < p1 ? __builtin_amdgcn_readfirstlane(entry) : -1;
    entry = table[min(p + 1, p1 - 1)];
    Page g;
    g.ok = page_ok(a.c, page);
#pragma unroll
    for (int n = 0; n < LOADS; ++n) g.code[n] = v4u{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t) g.k[t] = g.v[t] = 0.0f;
    if (!g.ok) return g;
    const size_t ph = size_t(page) * a.c.n_kv + kvh;
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      const int8_t *src = n * kPromptWaves * kWave + wave * kWave < KC ? a.c.k : a.c.v;
      g.code[n] = *reinterpret_cast<const v4u *>(src + ph * (kPage * HD) + from[n]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      g.k[t] = a.c.k_scale[ph * kPageBlocks + h + 2 * t];
      g.v[t] = a.c.v_scale[ph * kPageBlocks + h + 2 * t];
    }
    return g;
  };
  const auto deposit = [&](const Page &g, int n) {   // page n of this part
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      char *dst = buf + (i * kPromptWaves * kWave + wave * kWave < KC ? (n & 1) * KB : (2 + n % 3) * KB);
      v4u lo, hi;
      codes_to_f16(g.code[i], lo, hi);
      *reinterpret_cast<v4u *>(dst + to[i][0]) = lo;
      *reinterpret_cast<v4u *>(dst + to[i][1]) = hi;
    }
  };

  v16f s;        // scores of the tile to come
  v8h pf[2];     // weights of the tile that was
  float y[16];   // scores of the tile at hand, relative to mref
  float top;     // their largest
  v8h fr[2];     // operands read ahead

  // What a page's scales make of its two tiles' scores and weights' sums.  V
  // scales below 2^-60 of the largest so far count as that.
  struct Factors { float c[2], off[2], sum[2]; };
  const auto factors = [&](const Page &g, int p) {
    Factors f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float ks = g.k[t], vs = g.v[t];
      if (p * kPage + 32 * t + 16 * h > last_pos) ks = 0.0f, vs = 0.0f;   // (scales behind the end may hold anything)
      vmax = fmaxf(vmax, fmaxf(vs, lane_xor<32>(vs, lane)));
      const float ve = fmaxf(vs, vmax * 0x1p-60f);
      f.sum[t] = __builtin_amdgcn_rcpf(ve) * kSumUnit;
      f.c[t] = qs * ks;
      f.off[t] = (__builtin_amdgcn_logf(ve) + E) + (vs - vs);   // (vs - vs: NaN where the scale is not finite)
    }
    return f;
  };
  const auto read = [](const char *at) { return *reinterpret_cast<const v8h *>(at); };
  const auto pin = []() { __builtin_amdgcn_sched_barrier(0); };
  const auto key_ahead = [&](const char *kl) { fr[0] = read(kl + koff[0]), fr[1] = read(kl + koff[1]); };
  const auto value_at = [&](const char *vl, int t, int st) { return vl + voff[2 * t + st / D] + st % D * 64 * kPage; };
  const auto value_ahead = [&](const char *vl, int t) { fr[0] = read(value_at(vl, t, 0)), fr[1] = read(value_at(vl, t, 1)); };
  // Scores of the next tile (key rows kl; its first operands read ahead), and
  // beside each matrix instruction a share of this tile's weights.
  const auto scores_weights = [&](const char *kl, float lunit, bool some) {
    float sum = 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      v16f z;
#pragma unroll
      for (int v = 0; v < 16; ++v) z[v] = 0.0f;
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[m & 1], qf[m], m ? s : z, 0, 0, 0);
      if (m + 2 < M) fr[m & 1] = read(kl + koff[m + 2]);
      if (some) {
#pragma unroll
        for (int v = m * 16 / M; v < (m + 1) * 16 / M; ++v) {
          const float e = __builtin_amdgcn_exp2f(y[v]);
          sum += e;
          pf[v / 8][v % 8] = f16(e);
        }
      }
      pin();
    }
    if (some) l = fmaf(sum, lunit, l);
  };
  // Value sums of the tile before (tile t of the page at vl), and beside each
  // matrix instruction a share of this tile's scores, relative.
  const auto values_scores = [&](const char *vl, int t, float c, float off, bool some) {
    top = -INFINITY;
#pragma unroll
    for (int st = 0; st < 2 * D; ++st) {
      acc[st % D] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[st & 1], pf[st / D], acc[st % D], 0, 0, 0);
      if (st + 2 < 2 * D) fr[st & 1] = read(value_at(vl, t, st + 2));
      if (some) {
#pragma unroll
        for (int v = st * 16 / (2 * D); v < (st + 1) * 16 / (2 * D); ++v) {
          y[v] = fmaf(s[v], c, off);
          top = fmaxf(top, y[v]);
        }
      }
      pin();
    }
  };
  // Masks tile t of page p where its tokens are not seen; raises the reference of
  // rows whose scores outgrow it, and takes what was summed so far to it.
  const auto mask_reference = [&](int p, int t, bool seen) {
    if (!seen || p * kPage + 32 * t + 31 > first_pos) {
      const int lim = seen ? limit - (p * kPage + 32 * t + 16 * h) : -1;
      top = -INFINITY;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        y[v] = v > lim ? -INFINITY : y[v];
        top = fmaxf(top, y[v]);
      }
      pin();
    }
    if (__builtin_amdgcn_ballot_w64(top > thr) == 0) return;
    top = fmaxf(top, lane_xor<32>(top, lane));
    if (top > thr) {
      const float by = ceilf(top - E);
#pragma unroll
      for (int v = 0; v < 16; ++v) y[v] -= by;
      const float root = thr == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-0.5f * by), f = root * root;
      l = l * root * root;   // (f alone may underflow where l is large)
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[d][v] *= f;
      mref += by;
      thr = E + kRoom;
    }
  };

  if (p0 < p1) {
    Page g = request(p0), next = request(p0 + 1);
    deposit(g, 0);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int v = 0; v < 8; ++v) pf[q][v] = f16(0.0f);
    __syncthreads();
    key_ahead(buf);
    scores_weights(buf, 0.0f, false);
    value_ahead(buf + 2 * KB, 1);
    for (int p = p0, n = 0; p < p1; ++p, ++n) {
      const char *kl = buf + (n & 1) * KB, *vl = buf + (2 + n % 3) * KB;
      const Factors f = factors(g, p);
      // (the first page finds weights of zero, and sums its own values with them)
      values_scores(n ? buf + (2 + (n + 2) % 3) * KB : vl, 1, f.c[0], f.off[0] - mref, true);
      key_ahead(kl + 64 * HD);
      mask_reference(p, 0, g.ok);
      scores_weights(kl + 64 * HD, f.sum[0], true);
      value_ahead(vl, 0);
      pin();
      values_scores(vl, 0, f.c[1], f.off[1] - mref, true);
      // the next page's codes, requested a page ago
      deposit(next, n + 1);
      mask_reference(p, 1, g.ok);
      __syncthreads();   // it is there; this page's keys and the values before it are done with
      const char *after = buf + ((n + 1) & 1) * KB;
      key_ahead(after);
      g = next;
      next = request(p + 2);
      scores_weights(after, f.sum[1], true);
      value_ahead(vl, 1);
      pin();
    }
    values_scores(buf + (2 + (p1 - p0 - 1) % 3) * KB, 1, 0.0f, 0.0f, false);
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
        for (int v = 0; v < 4; ++v) f[v] = acc[d][4 * b + v];
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
      for (int v = 0; v < 4; ++v) f[v] = acc[d][4 * b + v] * inv;
      store_floats<4>(out + 32 * d + 8 * b + 4 * h, f);
    }
}

template <class T, int HD>
int launch(const AttnArgs &a, dim3 grid, hipStream_t st) {
  constexpr int lds = 5 * kPage * HD * 2;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&kv8_prompt_kernel<T, HD>),
                                                  hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return fail(LMX_ERR_LAUNCH_FAILED, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  kv8_prompt_kernel<T, HD><<<grid, dim3(kPromptWaves * kWave), lds, st>>>(a);
  return LMX_OK;
}

}  // namespace

int launch_prompt(const AttnArgs &a, int type, size_t hd, size_t units, hipStream_t st) {
  if (units * a.c.n_kv >= (1u << 31)) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu tiles of rows for %d KV heads", units, a.c.n_kv);
  const dim3 grid(unsigned(units * a.c.n_kv), 1, unsigned(a.splits));
  int r;
  if (type == LMX_F16) r = hd == 64 ? launch<f16, 64>(a, grid, st) : launch<f16, 128>(a, grid, st);
  else r = hd == 64 ? launch<bf16, 64>(a, grid, st) : launch<bf16, 128>(a, grid, st);
  if (r) return r;
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "kv8 prompt attention launch: %s", hipGetErrorString(e));
}

}  // namespace lmx
