// lmx_kv8.hip -- the 8-bit paged KV cache (include/lutmac_kv8.h): rotation and
// append, and attention of a few rows per sequence over it.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "lmx_kv8.hpp"

namespace lmx {
namespace {

// ---------------------------------------------------------------------------
// Append.  A unit is one page of a sequence that receives rows; a workgroup
// takes one unit of one KV head's keys, of one KV head's values, or of kHeads
// query heads.  Keys and values: a wave takes a 16-token block (4 lanes a
// token), whose scale needs every value before any code, so the values wait in
// registers.  Scales and codes are those of 64-bit arithmetic: what lies next to
// a border between two codes falls on the right side whatever the order of
// operations.  They are reached in fp32, which is off by far less than kSure
// keeps a quotient from a border and kNear a value from the largest; the few
// elements nearer than that, and blocks with a value that is not finite in fp32,
// are done again in 64 bits (doing all of them so costs a third of the call).
// Values are turned (4 x 4 bytes at a time, between lanes) into the page's order
// and leave through LDS, whole rows of 64 tokens.
// Long prompts are bound by memory (4 of 4096, 32 + 8 heads of 128, bf16: 91 us,
// 4.1 TB/s, where a copy reaches 4.9), short calls by the chain of loads from
// the offsets over the table to the block (64 rows: 6.7 us).
struct AppendArgs {
  Kv8Args c;
  const void *k, *v, *q;
  void *q_out;
  size_t k_stride, v_stride, q_stride, q_out_stride;
  const float2 *rope;
  int rope_n;
};
constexpr int kHeads = 8;

// The pairs (a[i], b[i]) of elements d0 + i and d0 + i + HD / 2, rotated.
template <int E, int HD, class F>
__device__ __forceinline__ void turned(const float (&a)[E], const float (&b)[E], const float2 *rope, int pos, int d0, F (&x)[E],
                                       F (&y)[E]) {
  if (rope) {
    const float2 *t = rope + size_t(pos) * (HD / 2) + d0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const F c = t[i].x, s = t[i].y;
      x[i] = F(a[i]) * c - F(b[i]) * s;
      y[i] = F(a[i]) * s + F(b[i]) * c;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = a[i], y[i] = b[i];
  }
}
template <int E, class T, int HD, class F>
__device__ __forceinline__ void rotated(const T *row, const float2 *rope, int pos, int d0, F (&x)[E], F (&y)[E]) {
  float a[E], b[E];
  load_floats<E>(row + d0, a);
  load_floats<E>(row + d0 + HD / 2, b);
  turned<E, HD>(a, b, rope, pos, d0, x, y);
}

// Element d (of the pair d, d + HD / 2: h) of a row, rotated, in 64 bits.
template <class T, int HD>
__device__ double exact_element(const T *row, const float2 *rope, int pos, int d, int h) {
  double x[1], y[1];
  rotated<1, T, HD>(row, rope, pos, d, x, y);
  return h ? y[0] : x[0];
}

__device__ __forceinline__ float wave_max(float v, int lane) { return lane_max<32>(v, lane); }

// The block's scale from its new values' largest magnitude.
__device__ __forceinline__ float block_scale(double top, bool finite, float was, bool kept) {
  float now = fmaxf(float(top / 127.0), 0x1p-100f);
  if (kept) now = was != was ? was : fmaxf(now, was);
  return finite && now < INFINITY ? now : __builtin_nanf("");
}

// (a NaN scale leaves the codes 0)
__device__ __forceinline__ int code_of(double x, double scale) {
  return scale == scale ? int(round_quotient(x, scale, 1.0 / scale)) : 0;
}

// Codes of four values, a byte each; false: one lies next to a border.
constexpr float kSure = 0.4999f, kNear = 1.0f - 0x1p-18f;
__device__ __forceinline__ bool sure_codes(const float *x, float inverse, uint32_t &w) {
  bool sure = true;
  w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float q = x[j] * inverse, n = rintf(q);
    sure = sure && fabsf(q - n) < kSure;
    w |= uint32_t(int(n) & 0xFF) << (8 * j);
  }
  return sure;
}

// Four codes of a block whose scale grew.
__device__ __forceinline__ uint32_t rescaled(uint32_t old, float was, float now) {
  const auto code = [old](int j) { return int(old << (24 - 8 * j)) >> 24; };
  const float x[4] = {float(code(0)), float(code(1)), float(code(2)), float(code(3))};
  uint32_t w;
  if (!sure_codes(x, was / now, w)) {
    w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= uint32_t(code_of(double(code(j)) * double(was), now) & 0xFF) << (8 * j);
  }
  return w;
}
// A word's first n bytes (none below 1, all from 4 on).
__device__ __forceinline__ uint32_t low_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; }

// A block's part in a call: tokens [kept, last) of it are rows of the call,
// those below kept the sequence's earlier ones.
struct BlockRows { int kept, last; };

template <class T, int HD>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
  constexpr int E = HD / 8, VE = HD / 4, LD = kPage + 16;   // pairs and values of a lane; a value row in LDS
  __shared__ __attribute__((aligned(16))) uint8_t cod[HD][LD];
  __shared__ float scales[kPageBlocks][2];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const SeqRows r = unit_rows(a.c, int(blockIdx.x), 1, 2, lane, kPage);
  const int from = max(r.start, 0);   // rows before position 0 have no place
  const int end = a.rope ? min(r.len, a.rope_n) : r.len;   // (rows past the rotation table are left out)
  const int pi = from / kPage + (int(blockIdx.x) - r.first);
  if (r.seq < 0 || end <= from || pi > (end - 1) / kPage) return;
  const int t0 = pi * kPage;   // (at most 2^31 - kPage, whatever the length: t0 + kPage may be past int)
  const int role = int(blockIdx.y), n_kv = a.c.n_kv;
  if (role >= 2 * n_kv) {   // query heads: 8 lanes a row and head
    constexpr int QE = 8, QL = HD / 2 / QE, SLOTS = 256 / QL;
    const int h0 = (role - 2 * n_kv) * kHeads, heads = min(kHeads, a.c.n_heads - h0);
    const int first = max(from, t0), items = (min(end - t0, kPage) - (first - t0)) * heads;
    const int slot = int(threadIdx.x) / QL, d0 = int(threadIdx.x) % QL * QE;
    const int inverse = 65536 / heads + 1;   // (item / heads, exactly for the up to 512)
    constexpr int U = sizeof(T) == 4 ? 1 : 4;   // rows of a lane on their way
    for (int n = slot; n < items; n += U * SLOTS) {
      float f[U][QE], g[U][QE];
      const T *q[U];
      size_t to[U];
      int pos[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int item = min(n + u * SLOTS, items - 1), t = item * inverse >> 16, h = h0 + item - t * heads;
        pos[u] = first + t;
        const size_t row = size_t(r.r0 + (pos[u] - r.start));
        q[u] = static_cast<const T *>(a.q) + row * a.q_stride + size_t(h) * HD;
        to[u] = row * a.q_out_stride + size_t(h) * HD + d0;
        load_floats<QE>(q[u] + d0, f[u]);
        load_floats<QE>(q[u] + d0 + HD / 2, g[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (n + u * SLOTS >= items) break;
        if constexpr (sizeof(T) == 4) {
          double x[QE], y[QE];
          turned<QE, HD>(f[u], g[u], a.rope, pos[u], d0, x, y);
#pragma unroll
          for (int i = 0; i < QE; ++i) f[u][i] = float(x[i]), g[u][i] = float(y[i]);
        } else {   // (rounded to 16 bits: fp32 leaves at most 2^-22 of the pair's larger)
          float x[QE], y[QE];
          turned<QE, HD>(f[u], g[u], a.rope, pos[u], d0, x, y);
#pragma unroll
          for (int i = 0; i < QE; ++i) f[u][i] = x[i], g[u][i] = y[i];
        }
        T *out = static_cast<T *>(a.q_out) + to[u];
        store_floats<QE>(out, f[u]);
        store_floats<QE>(out + HD / 2, g[u]);
      }
    }
    return;
  }
  if (pi >= a.c.max_pages) return;
  const int page = a.c.pages[size_t(r.seq) * a.c.max_pages + pi];
  if (!page_ok(a.c, page)) return;
  const int tk = lane >> 2, part = lane & 3;
  const auto block_rows = [&](int b) {
    return BlockRows{min(max(from - t0 - b * kBlock, 0), kBlock), min(max(end - t0 - b * kBlock, 0), kBlock)};
  };
  const BlockRows br = block_rows(wave);
  const bool some = br.last > br.kept, live = tk >= br.kept && tk < br.last;
  const int pos = t0 + wave * kBlock + tk;
  const size_t row = size_t(r.r0 + ((live ? pos : from) - r.start));
  if (role < n_kv) {
    if (!some) return;
    const size_t ph = size_t(page) * n_kv + role;
    float *scale = a.c.k_scale + ph * kPageBlocks + wave;
    const float was = *scale;
    const T *src = static_cast<const T *>(a.k) + row * a.k_stride + size_t(role) * HD;
    int8_t *dst = a.c.k + (ph * kPage + wave * kBlock + tk) * HD + part * E;
    typedef uint32_t words __attribute__((ext_vector_type(E / 4)));
    words old[2] = {};   // (fetched before they are known to be needed)
    if (tk < br.kept) {
#pragma unroll
      for (int h = 0; h < 2; ++h) old[h] = *reinterpret_cast<const words *>(dst + h * (HD / 2));
    }
    float x[2][E], most = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) x[0][i] = x[1][i] = 0.0f;
    if (live) rotated<E, T, HD>(src, a.rope, pos, part * E, x[0], x[1]);
    bool in_range = true;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      most = fmaxf(most, fmaxf(fabsf(x[0][i]), fabsf(x[1][i])));
      in_range = in_range && fabsf(x[0][i]) < INFINITY && fabsf(x[1][i]) < INFINITY;
    }
    most = wave_max(most, lane);
    const bool fast = __builtin_amdgcn_ballot_w64(!in_range) == 0;
    // the largest in 64 bits: of the elements that can be it (all, !fast)
    double top = 0.0;
    bool finite = true;
    if (live) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!fast || fmaxf(fabsf(x[0][i]), fabsf(x[1][i])) >= most * kNear) {
          double u[1], v[1];
          rotated<1, T, HD>(src, a.rope, pos, part * E + i, u, v);
          top = fmax(top, fmax(fabs(u[0]), fabs(v[0])));
          finite = finite && fabs(u[0]) < INFINITY && fabs(v[0]) < INFINITY;
        }
      }
    }
    // (of numbers >= 0 the largest has the largest bits; what is not finite goes by itself)
    top = __longlong_as_double(static_cast<long long>(wave_max_key(static_cast<unsigned long long>(__double_as_longlong(top)), lane)));
    const float now = block_scale(top, __builtin_amdgcn_ballot_w64(!finite) == 0, was, br.kept > 0);
    if (live) {
      const float finv = 1.0f / now;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        words c;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          uint32_t w;
          if (!sure_codes(x[h] + 4 * i, finv, w) || !fast) {
            w = 0;
            for (int j = 0; j < 4; ++j)
              w |= uint32_t(code_of(exact_element<T, HD>(src, a.rope, pos, part * E + 4 * i + j, h), now) & 0xFF) << (8 * j);
          }
          c[i] = now == now ? w : 0u;
        }
        *reinterpret_cast<words *>(dst + h * (HD / 2)) = c;
      }
    } else if (tk < br.kept && now == now && now != was) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        words c;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) c[i] = rescaled(old[h][i], was, now);
        *reinterpret_cast<words *>(dst + h * (HD / 2)) = c;
      }
    }
    if (lane == 0) *scale = now;
    return;
  }
  const size_t ph = size_t(page) * n_kv + (role - n_kv);
  // a thread's dimension and block (two of head_dim 128), of which it writes the
  // row of 16 tokens in the end; what is there now, for blocks not written whole
  typedef uint32_t words __attribute__((ext_vector_type(kBlock / 4)));
  constexpr int ROUNDS = HD * kPageBlocks / 256;
  words old[ROUNDS] = {};
#pragma unroll
  for (int n = 0; n < ROUNDS; ++n) {
    const int d = (n * 256 + int(threadIdx.x)) / kPageBlocks, b = int(threadIdx.x) % kPageBlocks;
    const BlockRows w = block_rows(b);
    if (w.last > w.kept && (w.kept > 0 || w.last < kBlock))
      old[n] = *reinterpret_cast<const words *>(a.c.v + (ph * HD + d) * kPage + b * kBlock);
  }
  if (some) {
    float *scale = a.c.v_scale + ph * kPageBlocks + wave;
    const float was = *scale;
    float x[VE], most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = 0.0f;
    if (live) load_floats<VE>(static_cast<const T *>(a.v) + row * a.v_stride + size_t(role - n_kv) * HD + part * VE, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      most = fmaxf(most, fabsf(x[i]));
      finite = finite && fabsf(x[i]) < INFINITY;
    }
    const float now = block_scale(wave_max(most, lane), __builtin_amdgcn_ballot_w64(!finite) == 0, was, br.kept > 0);
    const float finv = 1.0f / now;
    // four dimensions of four tokens at a time: lane (token 4 n + q, part) ends
    // with dimension 4 i + q of its part, the tokens 4 n .. 4 n + 3
    const int q = tk & 3;
#pragma unroll
    for (int i = 0; i < VE / 4; ++i) {
      uint32_t w;
      if (!sure_codes(x + 4 * i, finv, w)) {
        w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= uint32_t(code_of(x[4 * i + j], now) & 0xFF) << (8 * j);
      }
      w = now == now ? w : 0u;
      // the words of the lanes 4, 8 and 12 places on (row of 16 lanes = 4 tokens x 4 parts)
      const uint32_t w1 = dpp_u32<0x12C>(w), w2 = dpp_u32<0x128>(w), w3 = dpp_u32<0x124>(w);
      // byte q of each, tokens q, q + 1, q + 2, q + 3 (mod 4), turned to begin with token 0
      const uint32_t b0 = w >> (8 * q) & 0xFF, b1 = w1 >> (8 * q) & 0xFF, b2 = w2 >> (8 * q) & 0xFF, b3 = w3 >> (8 * q) & 0xFF;
      const uint32_t turned = b0 | b1 << 8 | b2 << 16 | b3 << 24;
      const uint32_t out = q ? turned << (8 * q) | turned >> (32 - 8 * q) : turned;
      *reinterpret_cast<uint32_t *>(&cod[part * VE + 4 * i + q][wave * kBlock + 4 * (tk >> 2)]) = out;
    }
    if (lane == 0) {
      scales[wave][0] = was, scales[wave][1] = now;
      *scale = now;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < ROUNDS; ++n) {
    const int d = (n * 256 + int(threadIdx.x)) / kPageBlocks, b = int(threadIdx.x) % kPageBlocks;
    const BlockRows w = block_rows(b);
    if (w.last <= w.kept) continue;
    words c = *reinterpret_cast<const words *>(&cod[d][b * kBlock]);
    if (w.kept > 0 || w.last < kBlock) {   // earlier tokens are rescaled, later places left
      const float was = scales[b][0], now = scales[b][1];
      const bool rescale = now == now && now != was;
#pragma unroll
      for (int i = 0; i < kBlock / 4; ++i) {
        const uint32_t kept = low_bytes(w.kept - 4 * i), rows = low_bytes(w.last - 4 * i) & ~kept;
        c[i] = (c[i] & rows) | (old[n][i] & ~(rows | kept)) | ((rescale && kept ? rescaled(old[n][i], was, now) : old[n][i]) & kept);
      }
    }
    *reinterpret_cast<words *>(a.c.v + (ph * HD + d) * kPage + b * kBlock) = c;
  }
}

// ---------------------------------------------------------------------------
// Attention of up to 16 rows (a row: one query head of one token) of one KV
// head per workgroup, on the 8-bit matrix cores with exact products.
//
// A query row becomes fixed point of three signed-byte digits relative to a power
// of two; S^T = K Q^T digit by digit (v_mfma_i32_16x16x64_i8, sums from the bits
// of 1.5 * 2^23, so the sum is a float that differs from it by the sum); the
// weights p become fixed point the same way, and O^T = V^T P^T.  No code is
// converted, and cache bytes go from memory straight into the operand
// registers:
//   K operand, tile t: lane (i, g) holds dimensions 64 m + 16 g .. + 15 of token
//     16 (i / 4) + 4 t + i % 4, so that of S^T tile t lane (column j, g) gets the
//     tokens 16 g + 4 t + 0..3 -- over the four tiles the 16 tokens of block g,
//     in order: one K and one V scale per lane, and P^T's operand in place.
//   V operand: lane (i, g) holds tokens 16 g .. + 15 of dimension 16 h + i.
// Weights are relative to their page's largest score + log2 of the V scale's
// power of two (what bounds the fixed point), so that a heavy token takes bits
// from its own page alone; the page's sums are brought to the running reference
// as they are added.  The rest of the scale is multiplied in as the digits are
// made (see value_exponent).  (Relative to the running reference, weights far
// below a heavy first token counted in their sum and not in the values': a tenth
// of the output lost with 15 bits, 1e-4 with 23.  Two digits instead of three
// would save up to 7 % of a step, and leave the other tokens of a page whose
// heaviest has 0.99 of the weight some 5 steps each.)
//
// The 4 waves take pages in turn, grid.z parts ("splits") a share of them;
// (m, l, o) of the waves merge in LDS, of the parts in kv8_merge_kernel.
// Bound by the cache's bytes where contexts are long (32 sequences of 20 to 33
// thousand tokens, 8 KV heads of 128, bf16: 349 us, 5.0 TB/s, what a copy reaches),
// else by the chain of loads (offsets, table, page, and each further page of a
// wave; one row of 320 tokens: 5.9 us) and some 450 vector and 48 matrix
// instructions a page of head_dim 128 (64 sequences of up to 2048 tokens, fp32: 14.5
// us and 4 for the merge): table entries
// come 64 at a time, and a page's keys and values are requested as soon as the
// registers of the page before are free of theirs.
//
// With head_dim 128 the registers are those of two workgroups a CU for fp32 and
// fp16, of three for bf16 (us, two / three: 64 sequences of up to 2048 tokens 18.4 /
// 19.8, 16 of 4000 32.4 / 30.3, 32 of 20 to 33 thousand 380 / 354).
template <class T>
constexpr bool kThree = std::is_same<T, bf16>::value;
template <class T, int HD>
__global__ __launch_bounds__(4 * kWave) __attribute__((amdgpu_waves_per_eu(HD == 128 && !kThree<T> ? 2 : 3))) void kv8_rows_kernel(AttnArgs a) {
  constexpr int W = 4, M = HD / 64, H = HD / 16;
  __shared__ float os[W][16][HD + 4];
  __shared__ float ms[W][16], ls[W][16];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int j = lane & 15, g = lane >> 4;
  const int kvh = int(blockIdx.y), group = a.c.group;
  const SeqRows r = unit_rows(a.c, int(blockIdx.x), group, 1, lane, 16);
  const int tile0 = (int(blockIdx.x) - r.first) * 16, rows = r.n * group;   // (< 2^31: checked by the host)
  if (r.seq < 0 || tile0 >= rows) return;
  // row i of the sequence: query head kvh * group + i % group of token i / group
  const int i = tile0 + j;
  const int t = min(i, rows - 1) / group;
  const int see = min(r.len, a.c.max_pages * kPage) - 1;   // the last token with a place
  const int first_pos = min(r.start + tile0 / group, see), last_pos = min(r.start + min(tile0 + 15, rows - 1) / group, see);
  const int limit = min(r.start + t, see);
  const int n_pages = last_pos < 0 ? 0 : last_pos / kPage + 1;
  const int part = int(blockIdx.z);
  const int p0 = part_begin(n_pages, part, a.splits), p1 = part_begin(n_pages, part + 1, a.splits);

  float mref = -INFINITY, l = 0.0f;
  int exmax = kLeastExp + kExpSpan;
  float o[H][4];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int v = 0; v < 4; ++v) o[h][v] = 0.0f;
  const v4i zero = {__float_as_int(kMagic), __float_as_int(kMagic), __float_as_int(kMagic), __float_as_int(kMagic)};
  const int *table = a.c.pages + size_t(r.seq) * a.c.max_pages;
  int entries = 0;   // lane n: the table's entry of the wave's page n (of 64)
  const auto read_entries = [&](int p) { entries = table[min(p + W * lane, p1 - 1)]; };
  if (p0 + wave < p1) read_entries(p0 + wave);
  // the row's query: this lane's 16 dimensions of every 64-dimension step
  const T *q = static_cast<const T *>(a.q) + size_t(r.r0 + t) * a.q_stride + size_t(kvh * group + min(i, rows - 1) % group) * HD;
  float x[M][16];
#pragma unroll
  for (int m = 0; m < M; ++m) load_floats<16>(q + 64 * m + 16 * g, x[m]);
  v4i kb[4][M], vb[H];
  float ks = 0.0f, vs = 0.0f;   // the scales of the page whose keys were requested last
  int page = -1;
  // (through buffers of a page's size, or of none: then nothing is fetched, and
  // no register waits behind a branch)
  const auto buffer = [](const void *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00020000);
  };
  const int kat = (16 * (j >> 2) + (j & 3)) * HD + 16 * g, vat = j * kPage + 16 * g;
  const auto request_keys = [&](int p, int n) {   // page p, the wave's n-th
    page = p < p1 ? __builtin_amdgcn_readlane(entries, n & (kWave - 1)) : -1;
    const bool ok = page_ok(a.c, page);
    const size_t ph = size_t(ok ? page : 0) * a.c.n_kv + kvh;
    const auto kbuf = buffer(a.c.k + ph * kPage * HD, ok ? kPage * HD : 0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int m = 0; m < M; ++m)
        kb[u][m] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(kbuf, kat + 4 * u * HD + 64 * m, 0, 0));
    ks = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer(a.c.k_scale + ph * kPageBlocks, ok ? 16 : 0), 4 * g, 0, 0));
    vs = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer(a.c.v_scale + ph * kPageBlocks, ok ? 16 : 0), 4 * g, 0, 0));
  };
  const auto request_values = [&]() {
    const bool ok = page_ok(a.c, page);
    const auto vbuf = buffer(a.c.v + (size_t(ok ? page : 0) * a.c.n_kv + kvh) * (kPage * HD), ok ? kPage * HD : 0);
#pragma unroll
    for (int h = 0; h < H; ++h)
      vb[h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(vbuf, vat + h * 16 * kPage, 0, 0));
  };
  if (p0 + wave < p1) {
    request_keys(p0 + wave, 0);
    request_values();
  }
  // (its digits are made while the first page is on its way)
  v4i qd[M][kDigits];
  float qs;
  {
    uint32_t top = 0;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int d = 0; d < 16; ++d) top = max(top, __float_as_uint(x[m][d]) & 0x7FFFFFFFu);
    top = max(top, lane_xor_u32<16>(top, lane));
    top = max(top, lane_xor_u32<32>(top, lane));
    const bool finite = top < 0x7F800000u;
    const int e = max(int(top >> 23), 29) - 126;   // |x| < 2^e
    const float f = finite ? __builtin_amdgcn_ldexpf(1.0f, kQueryBits - e) : 0.0f;
#pragma unroll
    for (int m = 0; m < M; ++m) query_digits(x[m], f, qd[m]);   // (anything where not finite: qs is NaN then)
    qs = finite ? __builtin_amdgcn_ldexpf(a.scale, e - kQueryBits) : __builtin_nanf("");
  }

  for (int p = p0 + wave, n = 0; p < p1; p += W, ++n) {
    const bool ok = page_ok(a.c, page);
    float ksp = ks, vsp = vs;
    if ((n & (kWave - 1)) == kWave - 1 && p + W < p1) read_entries(p + W);
    const int t0 = p * kPage + 16 * g;   // this lane's first token
    if (t0 > last_pos || !ok) ksp = 0.0f, vsp = 0.0f;   // nothing of the block is seen: its scales may hold anything
    // (of a block whose scale is not finite nothing is summed: rows that see it get
    // NaN below, the tile's others are not to find its scale in their digits)
    const bool finite = vsp - vsp == 0.0f;
    if (!finite) vsp = 0.0f;
    int ex = value_exponent(vsp);
    exmax = max(exmax, max(ex, lane_xor_int<16>(ex, lane)));
    exmax = max(exmax, lane_xor_int<32>(exmax, lane));
    ex = max(ex, exmax - kExpSpan);
    const float mant = __builtin_amdgcn_ldexpf(vsp, -ex) * kWeightUnit, fex = float(ex), c = qs * ksp;
    float y[4][4], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v4i s[kDigits];
#pragma unroll
      for (int d = 0; d < kDigits; ++d) {
        s[d] = zero;
#pragma unroll
        for (int m = 0; m < M; ++m) s[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kb[u][m], qd[m][d], s[d], 0, 0, 0);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float d[kDigits];
#pragma unroll
        for (int n = 0; n < kDigits; ++n) d[n] = __int_as_float(s[n][v]);
        y[u][v] = fmaf(join(d), c, fex);
      }
    }
    request_keys(p + W, n + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (!ok || p * kPage + kPage - 1 > first_pos) {
      const int lim = ok ? limit - t0 : -1;
#pragma unroll
      for (int v = 0; v < 16; ++v) y[v / 4][v % 4] = v > lim ? -INFINITY : y[v / 4][v % 4];
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) top = fmaxf(top, y[v / 4][v % 4]);
    top = fmaxf(top, lane_xor<16>(top, lane));
    top = fmaxf(top, lane_xor<32>(top, lane));
    // weights relative to the page's largest; `share` brings its sums to the
    // running reference, and where that rises the sums so far follow it
    const float base = top == -INFINITY ? 0.0f : top, was = mref;
    mref = fmaxf(mref, top);
    if (n > 0 && __builtin_amdgcn_ballot_w64(mref > was) != 0) {
      const float root = mref > was ? __builtin_amdgcn_exp2f(0.5f * (was - mref)) : 1.0f, keep = root * root;
      l = l * root * root;   // (keep alone may underflow where l is large)
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int v = 0; v < 4; ++v) asm("v_mul_f32 %0, %0, %1" : "+v"(o[h][v]) : "v"(keep));
    }
    const float root = __builtin_amdgcn_exp2f(0.5f * (top - (mref == -INFINITY ? 0.0f : mref))), share = root * root;
    v4i pd[kDigits];
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t w[4], dw[kDigits];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float e = __builtin_amdgcn_exp2f(y[u][v] - base);
        sum += e;
        w[v] = __float_as_uint(fmaf(e, mant, 0x1p23f + float(kCarry)));
      }
      digit_words(w, dw);
#pragma unroll
      for (int d = 0; d < kDigits; ++d) pd[d][u] = int(dw[d]);
    }
    l = fmaf(sum * root, __builtin_amdgcn_ldexpf(kWeightUnit, kSumExp - ex) * root, l);
    if (!finite && t0 <= limit) l = __builtin_nanf("");
#pragma unroll
    for (int h = 0; h < H; ++h) {
      v4i s[kDigits];
#pragma unroll
      for (int d = 0; d < kDigits; ++d) s[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vb[h], pd[d], zero, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float d[kDigits];
#pragma unroll
        for (int n = 0; n < kDigits; ++n) d[n] = __int_as_float(s[n][v]);
        // (in place: as a plain fma the compiler makes another register of it and
        // copies all of them back, a tenth of the loop)
        const float sum = join(d);
        asm("v_fma_f32 %0, %1, %2, %0" : "+v"(o[h][v]) : "v"(sum), "v"(share));
      }
    }
    request_values();
    __builtin_amdgcn_sched_barrier(0);
  }
  l += lane_xor<16>(l, lane);
  l += lane_xor<32>(l, lane);
  if (g == 0) ms[wave][j] = mref, ls[wave][j] = l;
#pragma unroll
  for (int h = 0; h < H; ++h)
    *reinterpret_cast<float4 *>(&os[wave][j][16 * h + 4 * g]) = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
  __syncthreads();
  // thread (row, its share of the dimensions) merges the waves
  constexpr int TR = W * kWave / 16, E = HD / TR;   // threads of a row, dimensions of a thread
  const int row = int(threadIdx.x) / TR, d0 = int(threadIdx.x) % TR * E;
  float mx = ms[0][row];
#pragma unroll
  for (int w = 1; w < W; ++w) mx = fmaxf(mx, ms[w][row]);
  float sum = 0.0f, acc[E];
#pragma unroll
  for (int d = 0; d < E; ++d) acc[d] = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    // (1: a sum that is NaN stays so)
    const float root = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(0.5f * (ms[w][row] - mx)), f = root * root;
    sum += ls[w][row] * root * root;
#pragma unroll
    for (int d = 0; d < E; ++d) acc[d] = fmaf(f, os[w][row][d0 + d], acc[d]);
  }
  if (a.splits > 1) {
    const size_t at = ((size_t(blockIdx.x) * a.c.n_kv + kvh) * a.splits + part) * 16 + row;
    if (int(threadIdx.x) % TR == 0) a.part_ml[at] = make_float2(mx, sum);
    store_floats<E>(a.part_o + at * HD + d0, acc);
    return;
  }
  if (tile0 + row >= rows) return;
  const float inv = inverse_sum(sum);
#pragma unroll
  for (int d = 0; d < E; ++d) acc[d] *= inv;
  T *out = static_cast<T *>(a.out) + size_t(r.r0 + (tile0 + row) / group) * a.out_stride +
           size_t(kvh * group + (tile0 + row) % group) * HD + d0;
  store_floats<E>(out, acc);
}

// The parts of a split unit: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s,
// eight parts' loads at a time in flight.
template <class T, int HD, int ROWS>
__global__ __launch_bounds__(256) void kv8_merge_kernel(AttnArgs a) {
  constexpr int E = HD / 16, S = 8;
  const int lane = threadIdx.x & (kWave - 1), kvh = int(blockIdx.y), group = a.c.group;
  const int row = int(blockIdx.z) * 16 + (int(threadIdx.x) >> 4), d0 = (int(threadIdx.x) & 15) * E;
  const SeqRows r = unit_rows(a.c, int(blockIdx.x), group, 1, lane, ROWS);
  const int i = (int(blockIdx.x) - r.first) * ROWS + row;
  if (r.seq < 0 || i >= r.n * group) return;
  const size_t at = (size_t(blockIdx.x) * a.c.n_kv + kvh) * a.splits * ROWS + row;
  float mx = -INFINITY, sum = 0.0f, acc[E];
#pragma unroll
  for (int d = 0; d < E; ++d) acc[d] = 0.0f;
  for (int s0 = 0; s0 < a.splits; s0 += S) {
    float2 ml[S];
    float o[S][E];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const size_t n = at + size_t(min(s0 + s, a.splits - 1)) * ROWS;
      ml[s] = a.part_ml[n];
      load_floats<E>(a.part_o + n * HD + d0, o[s]);
    }
    float now = mx;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s0 + s >= a.splits) ml[s] = make_float2(-INFINITY, 0.0f);
      now = fmaxf(now, ml[s].x);
    }
    // (1: a sum that is NaN stays so)
    const float r0 = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(0.5f * (mx - now));
    sum = sum * r0 * r0;
#pragma unroll
    for (int d = 0; d < E; ++d) acc[d] *= r0 * r0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const float root = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(0.5f * (ml[s].x - now)), f = root * root;
      sum += ml[s].y * root * root;
#pragma unroll
      for (int d = 0; d < E; ++d)
        if (s0 + s < a.splits) acc[d] = fmaf(f, o[s][d], acc[d]);
    }
    mx = now;
  }
  const float inv = inverse_sum(sum);
#pragma unroll
  for (int d = 0; d < E; ++d) acc[d] *= inv;
  store_floats<E>(static_cast<T *>(a.out) + size_t(r.r0 + i / group) * a.out_stride + size_t(kvh * group + i % group) * HD + d0,
                  acc);
}

// ---- host side ----

int launch_err(const char *what) {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? LMX_OK : fail(LMX_ERR_LAUNCH_FAILED, "%s launch: %s", what, hipGetErrorString(e));
}

int check_sizes(const lmx_kv8_cache *c, const lmx_kv8_batch *b, size_t n_heads) {
  if (!c || !b) return fail(LMX_ERR_INVALID_ARGUMENT, "cache or batch is NULL");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(LMX_ERR_INVALID_ARGUMENT, "head_dim %zu must be 64 or 128", c->head_dim);
  if (c->n_kv_heads == 0 || c->n_kv_heads > 512) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu KV heads", c->n_kv_heads);
  if (c->n_pages == 0 || c->n_pages >= (1u << 31)) return fail(LMX_ERR_INVALID_ARGUMENT, "%zu pages", c->n_pages);
  if (b->n_seqs > (1u << 20) || b->max_pages > (1u << 24) || b->n_rows > (1u << 24))
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu sequences of up to %zu pages, %zu rows: at most 2^20, 2^24, 2^24", b->n_seqs,
                b->max_pages, b->n_rows);
  if (n_heads == 0 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 64)
    return fail(LMX_ERR_INVALID_ARGUMENT, "%zu query heads must be a multiple of %zu KV heads, at most 64 times", n_heads,
                c->n_kv_heads);
  return LMX_OK;
}

int check_pointers(const lmx_kv8_cache *c, const lmx_kv8_batch *b) {
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(LMX_ERR_INVALID_ARGUMENT, "cache pointer is NULL");
  if (!b->offsets || !b->lengths || (b->max_pages && !b->pages)) return fail(LMX_ERR_INVALID_ARGUMENT, "batch pointer is NULL");
  if ((reinterpret_cast<size_t>(c->k) | reinterpret_cast<size_t>(c->v)) % 16)
    return fail(LMX_ERR_INVALID_ARGUMENT, "cache codes must be 16-byte aligned");
  return LMX_OK;
}

// A row array: 16-byte aligned rows that do not run into each other.
int check_rows(const char *what, const void *p, size_t stride, size_t width, int type, size_t rows) {
  if (!p) return fail(LMX_ERR_INVALID_ARGUMENT, "%s is NULL", what);
  if (reinterpret_cast<size_t>(p) % 16 || stride * type_bytes(type) % 16)
    return fail(LMX_ERR_INVALID_ARGUMENT, "%s: pointer and row stride must be multiples of 16 bytes", what);
  if (stride < width && rows > 1) return fail(LMX_ERR_INVALID_ARGUMENT, "%s: row stride %zu is less than a row's %zu", what, stride, width);
  return LMX_OK;
}

Kv8Args kv8_args(const lmx_kv8_cache *c, const lmx_kv8_batch *b, size_t n_heads) {
  Kv8Args a{};
  a.k = c->k, a.v = c->v, a.k_scale = c->k_scale, a.v_scale = c->v_scale;
  a.offsets = b->offsets, a.lengths = b->lengths, a.pages = b->pages;
  a.n_pages = int(c->n_pages), a.n_kv = int(c->n_kv_heads);
  a.n_seqs = int(b->n_seqs), a.max_pages = int(b->max_pages), a.n_rows = int(b->n_rows);
  a.n_heads = int(n_heads), a.group = int(n_heads / c->n_kv_heads);
  return a;
}

// How a call is split over the device, from its sizes alone (lengths are known
// to the kernels only).
struct Plan {
  size_t rows;     // of a work unit: 16 (kv8_rows_kernel) or kPromptRows
  size_t units;    // at most
  int splits;      // parts of a unit's pages
};

Plan plan(const lmx_kv8_cache *c, const lmx_kv8_batch *b, size_t n_heads, int type) {
  const size_t group = n_heads / c->n_kv_heads;
  const size_t each = (b->n_rows + b->n_seqs - 1) / b->n_seqs * group;   // rows of a sequence, if they have equal shares
  const auto tiles = [&](size_t rows) { return b->n_seqs * ((each + rows - 1) / rows) * c->n_kv_heads; };
  // 256 rows a workgroup, of 16-bit types, where their tiles are not mostly empty
  // and tiles of 16 would be four a CU and more, each of them with the pages to read
  // (us, 16 / 256 rows a workgroup, bf16, KV heads: 16 tokens x 4 heads after 500, 8
  // of 128, 13 / 25; 606 x 4 after 300, 8 of 64, 21 / 28; 64 sequences of 16 x 4 after
  // 4000, 8 of 64, 160 / 201, of 24 x 4 after 0 22 / 20; 8 of 130 x 2 after 300, 8 of 128,
  // 25 / 26; 27 of 54 x 2, 8 of 128, 18 / 13; 43 of 68 x 4 after 6000, 4 of 128, 450 / 394.
  // It is wrong for fewer tiles of long contexts: 8 of 28 x 8 after 6000, 8 of 128,
  // 181 / 116.  Over 110 calls of 1 to 91 sequences this rule's times are 3 % above
  // the better kernel's; those of 256 rows from 64 a sequence on were 20 %.)
  Plan p{};
  p.rows = type != LMX_F32 && each >= 96 && tiles(16) >= 1024 ? kPromptRows : 16;
  p.units = b->n_rows * group / p.rows + b->n_seqs;
  // As many parts as fill the device once (three workgroups per CU; two of fp32
  // and fp16 with head_dim 128 and of prompts: a workgroup more runs a second round),
  // of four pages at least, one per wave (prompts: 8).
  const size_t room = p.rows > 16 || (type != LMX_BF16 && c->head_dim == 128) ? 512 : 768;
  const size_t s = std::min<size_t>(room / tiles(p.rows), b->max_pages / (p.rows == 16 ? 4 : 8));
  p.splits = int(std::max<size_t>(1, std::min<size_t>(s, 64)));
  return p;
}

size_t workspace_bytes(const lmx_kv8_cache *c, const lmx_kv8_batch *b, size_t n_heads, int type) {
  if (b->n_seqs == 0 || b->n_rows == 0) return 0;
  const Plan p = plan(c, b, n_heads, type);
  if (p.splits == 1) return 0;
  return p.units * c->n_kv_heads * size_t(p.splits) * p.rows * (c->head_dim + 2) * sizeof(float);
}

template <class T, int HD>
int launch_attention(const AttnArgs &a, int type, const Plan &p, hipStream_t st) {
  const dim3 grid(unsigned(p.units), unsigned(a.c.n_kv), unsigned(a.splits));
  int r;
  if (p.rows == 16) {
    kv8_rows_kernel<T, HD><<<grid, dim3(256), 0, st>>>(a);
    r = launch_err("kv8 attention");
  } else {
    r = launch_prompt(a, type, HD, p.units, st);
  }
  if (r || a.splits == 1) return r;
  if (p.rows == 16) kv8_merge_kernel<T, HD, 16><<<dim3(grid.x, grid.y, 1), dim3(256), 0, st>>>(a);
  else kv8_merge_kernel<T, HD, kPromptRows><<<dim3(grid.x, grid.y, kPromptRows / 16), dim3(256), 0, st>>>(a);
  return launch_err("kv8 merge");
}

template <class T>
int launch_append(const AppendArgs &a, size_t hd, dim3 grid, hipStream_t st) {
  if (hd == 64) kv8_append_kernel<T, 64><<<grid, dim3(256), 0, st>>>(a);
  else kv8_append_kernel<T, 128><<<grid, dim3(256), 0, st>>>(a);
  return launch_err("kv8 append");
}

}  // namespace
}  // namespace lmx

using namespace lmx;

extern "C" {

int lmx_kv8_append(const lmx_kv8_cache *cache, const lmx_kv8_batch *batch, int type, const void *k, size_t k_stride,
                   const void *v, size_t v_stride, const void *q, size_t q_stride, void *q_out, size_t q_out_stride,
                   size_t n_heads, const float *rope, size_t rope_positions, void *stream) {
  int r = check_sizes(cache, batch, q ? n_heads : cache ? cache->n_kv_heads : 1);
  if (r) return r;
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (batch->n_seqs == 0 || batch->n_rows == 0) return LMX_OK;
  const size_t kvw = cache->n_kv_heads * cache->head_dim, qw = n_heads * cache->head_dim, rows = batch->n_rows;
  if ((r = check_pointers(cache, batch)) || (r = check_rows("k", k, k_stride, kvw, type, rows)) ||
      (r = check_rows("v", v, v_stride, kvw, type, rows)))
    return r;
  if (q && ((r = check_rows("q", q, q_stride, qw, type, rows)) || (r = check_rows("q_out", q_out, q_out_stride, qw, type, rows))))
    return r;
  if (rope && (rope_positions == 0 || rope_positions >= (1u << 31) || reinterpret_cast<size_t>(rope) % 8))
    return fail(LMX_ERR_INVALID_ARGUMENT, "rotation table of %zu positions, or not 8-byte aligned", rope_positions);
  AppendArgs a{};
  a.c = kv8_args(cache, batch, q ? n_heads : cache->n_kv_heads);
  a.k = k, a.v = v, a.q = q, a.q_out = q_out;
  a.k_stride = k_stride, a.v_stride = v_stride, a.q_stride = q_stride, a.q_out_stride = q_out_stride;
  a.rope = reinterpret_cast<const float2 *>(rope);
  a.rope_n = rope ? int(rope_positions) : 0;
  // a sequence of n rows touches at most n / 64 + 2 pages, rounded down
  const dim3 grid(unsigned(rows / kPage + 2 * batch->n_seqs),
                  unsigned(2 * cache->n_kv_heads + (q ? (n_heads + kHeads - 1) / kHeads : 0)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (type) {
  case LMX_F32: return launch_append<float>(a, cache->head_dim, grid, st);
  case LMX_F16: return launch_append<f16>(a, cache->head_dim, grid, st);
  default: return launch_append<bf16>(a, cache->head_dim, grid, st);
  }
}

int lmx_kv8_attention_workspace(const lmx_kv8_cache *cache, const lmx_kv8_batch *batch, int type, size_t n_heads,
                                size_t *bytes) {
  if (!bytes) return fail(LMX_ERR_INVALID_ARGUMENT, "bytes is NULL");
  const int r = check_sizes(cache, batch, n_heads);
  if (r) return r;
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  *bytes = workspace_bytes(cache, batch, n_heads, type);
  return LMX_OK;
}

int lmx_kv8_attention(const lmx_kv8_cache *cache, const lmx_kv8_batch *batch, int type, const void *q, size_t q_stride,
                      size_t n_heads, float scale, void *out, size_t out_stride, void *workspace, size_t workspace_size,
                      void *stream) {
  int r = check_sizes(cache, batch, n_heads);
  if (r) return r;
  if (!type_bytes(type)) return fail(LMX_ERR_UNSUPPORTED_FORMAT, "unknown element type %d", type);
  if (!(scale > 0.0f) || !(scale < INFINITY)) return fail(LMX_ERR_INVALID_ARGUMENT, "scale %g must be positive and finite", double(scale));
  if (batch->n_seqs == 0 || batch->n_rows == 0) return LMX_OK;
  const size_t qw = n_heads * cache->head_dim, need = workspace_bytes(cache, batch, n_heads, type);
  if ((r = check_pointers(cache, batch)) || (r = check_rows("q", q, q_stride, qw, type, batch->n_rows)) ||
      (r = check_rows("out", out, out_stride, qw, type, batch->n_rows)))
    return r;
  if (need && (!workspace || workspace_size < need || reinterpret_cast<size_t>(workspace) % 16))
    return fail(LMX_ERR_INVALID_ARGUMENT, "workspace of %zu bytes at %p: %zu bytes, 16-byte aligned, are needed", workspace_size,
                workspace, need);
  AttnArgs a{};
  a.c = kv8_args(cache, batch, n_heads);
  a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
  a.scale = scale * 1.44269504088896340736f;
  const Plan p = plan(cache, batch, n_heads, type);
  a.splits = p.splits;
  if (a.splits > 1) {
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + p.units * cache->n_kv_heads * size_t(a.splits) * p.rows * cache->head_dim);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
#define LMX_KV8_ATTENTION(T) \
  return cache->head_dim == 64 ? launch_attention<T, 64>(a, type, p, st) : launch_attention<T, 128>(a, type, p, st)
  switch (type) {
  case LMX_F32: LMX_KV8_ATTENTION(float);
  case LMX_F16: LMX_KV8_ATTENTION(f16);
  default: LMX_KV8_ATTENTION(bf16);
  }
#undef LMX_KV8_ATTENTION
}

}  // extern "C"
