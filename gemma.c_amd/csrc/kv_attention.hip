// kv_attention.hip -- attention over the paged 8-bit cache: single tokens,
// prompt rows and shared prefixes of a ragged batch.
//
// Both products run on the f16 matrix cores.  A code (int8, or e4m3 down to its
// subnormals) is exact in f16, so only the fp32 operands are split: q, scaled by a
// power of two, and the softmax weights are each two f16 pieces (22 significant
// bits), and every product is the sum of two piece products with fp32
// accumulation.  A position's scales stay out of the products: K's goes into its
// score, V's into its weight.
//
// With c = asc log2 e, s the scaled score in octaves, and a whole number M per
// query: w = 2^(s - M) vs, l = sum 2^(s - M), out = sum w code / l.  M follows the
// largest s + log2 vs, not the largest s: what must fit f16 is w.  It has some
// octaves of slack, so that the sums are rescaled rarely and by powers of two.
// Weights are kept to 2^-31 of the largest beside them and have all their 22 bits
// down to 2^-20 of it.
//
// A wave computes S^T = K Q^T (rows: 16 keys, columns: 16 queries) and O^T = V^T
// P^T (rows: 16 dims) with 16x16x32 products.  Operand layout: lane l holds row (or
// column) l % 16 and eight values of the summed axis, number 8 (l / 16) and up; its
// results are rows 4 (l / 16) .. + 3 of column l % 16.  Which dim or key a number of
// the summed axis stands for is free as long as both operands agree:
//  - scores: lane group g takes dims 64 j + 16 g .. + 15 of its key, one 16-byte load;
//  - values: the numbers 8 g .. + 7 are keys 4 g .. + 3 of both 16-key halves of a
//    tile, those whose weights the lane has from its scores.  So weights never
//    change lanes, and V's codes are transposed by byte permutations within a lane
//    (its eight keys are eight loads).
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kTile = 32;             // keys of a tile
constexpr int kStepRows = 16;         // query vectors (rows x heads of a kv head) of a step tile
constexpr float kFloor = -0x1p55f;    // M of a query that has seen no key
constexpr float kSlack = 14.0f;       // weights stay below 2^15 ...
constexpr float kSet = 7.0f;          // ... and a moved M puts the largest at 2^6 .. 2^8
constexpr float kLeastVs = -60.0f;    // octaves that a scale counts at least
constexpr float kLog2e = 1.44269502162933349609375f;

// How a call is cut into workgroups: the same on the host, which sizes the
// workspace by it, and in the kernels.
struct KvPlan {
  int group;                    // heads per kv head
  int step, step_ns, step_tpc;  // single tokens: on or off, key chunks, tiles of a chunk
  int step_rows;                // query vectors of a sequence and kv head, at most
  int rows_ns, rows_tpc;        // prompt rows (0 chunks: off)
  int pre_ns, pre_tpc;          // shared prefix (0: none)
  int qb;                       // 16-query blocks of a wave of the prompt kernel
  size_t step_o, step_m, rows_o, rows_m, pre_o, pre_m, bytes;  // workspace
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// tanh(x) to about an ulp: its odd series below 0.35, else from e^-2|x|.
__device__ __forceinline__ float tanh32(float x) {
  const float z = fabsf(x), y = x * x;
  float s = fmaf(y, -1382.0f / 155925.0f, 62.0f / 2835.0f);
  s = fmaf(y, s, -17.0f / 315.0f);
  s = fmaf(y, s, 2.0f / 15.0f);
  s = fmaf(y, s, -1.0f / 3.0f);
  const float small = fmaf(x * y, s, x);
  const float e = __builtin_amdgcn_exp2f(z * (-2.0f * kLog2e));
  const float large = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  return z < 0.35f ? small : copysignf(large, x);
}

// Codes to f16 pairs.  int8: the byte with its top bit flipped is the low byte of
// an f16 of 1024 and up (0x64..), 1152 above the code.
__device__ __forceinline__ uint32_t flip(uint32_t x) { return x ^ 0x80808080u; }
template <uint32_t SEL>
__device__ __forceinline__ h2 magic(uint32_t x) {  // bytes SEL of x, an f16 each
  const uint32_t t = __builtin_amdgcn_perm(0x64646464u, x, SEL);
  return __builtin_bit_cast(h2, t) - h2{(_Float16)1152.0f, (_Float16)1152.0f};
}
template <bool HI>
__device__ __forceinline__ h2 from_e4m3(uint32_t x) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HI));
}
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// eight codes in a row
template <int TYPE>
__device__ __forceinline__ h8 codes8(uint32_t a, uint32_t b) {
  if constexpr (TYPE == kKvI8) {
    a = flip(a);
    b = flip(b);
    return join(magic<0x04010400u>(a), magic<0x04030402u>(a), magic<0x04010400u>(b),
                magic<0x04030402u>(b));
  } else {
    return join(from_e4m3<false>(a), from_e4m3<true>(a), from_e4m3<false>(b), from_e4m3<true>(b));
  }
}
// x: a dword (four dims) of each of eight keys; f[i]: dim i of the eight keys
template <int TYPE>
__device__ __forceinline__ void codes_t(const uint32_t (&x)[8], h8 (&f)[4]) {
  h2 p[4][4];  // [dim][pair of keys]
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a = x[2 * j], b = x[2 * j + 1];
    if (TYPE == kKvI8) {
      a = flip(a);
      b = flip(b);
    }
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u);  // a0 b0 a1 b1
    const uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07030602u);  // a2 b2 a3 b3
    if constexpr (TYPE == kKvI8) {
      p[0][j] = magic<0x04010400u>(lo);
      p[1][j] = magic<0x04030402u>(lo);
      p[2][j] = magic<0x04010400u>(hi);
      p[3][j] = magic<0x04030402u>(hi);
    } else {
      p[0][j] = from_e4m3<false>(lo);
      p[1][j] = from_e4m3<true>(lo);
      p[2][j] = from_e4m3<false>(hi);
      p[3][j] = from_e4m3<true>(hi);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = join(p[i][0], p[i][1], p[i][2], p[i][3]);
}

__device__ __forceinline__ v4f mma(h8 a, h8 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// What a lane's query sees: keys lo .. hi.
struct KvSee {
  int lo, hi;
};

// The scales of a lane's eight keys of a tile: keys 16 u + 4 g + i.
struct Scales {
  v4f k[2], v[2];
};

// The running softmax of a query: M, and the sum of the weights of the keys that
// the lane has.
struct Soft {
  float m, l;
};

// A query of HD dims in operand order (dims 64 j + 16 g + 8 h .. + 7 are piece
// number 2 j + h), in two f16 pieces; the exponent it was scaled by comes back.
template <int HD>
__device__ __forceinline__ int load_q(const float *row, int g, h8 (&hi)[HD / 32],
                                      h8 (&lo)[HD / 32]) {
  float x[HD / 32][8], amax = 0.0f;
#pragma unroll
  for (int s = 0; s < HD / 32; ++s)
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const v4f t =
          *reinterpret_cast<const v4f *>(row + 64 * (s / 2) + 16 * g + 8 * (s % 2) + e);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[s][e + u] = t[u];
        amax = fmaxf(amax, finite_abs(t[u]));
      }
    }
  amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
  amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
  const int eq = amax > 0.0f ? ilogbf(amax) - 14 : 0;
#pragma unroll
  for (int s = 0; s < HD / 32; ++s)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float a = ldexpf(x[s][e], -eq), b = ldexpf(x[s][e + 1], -eq);
      const h2 p = cvt_pk_f16(a, b);
      const h2 r = cvt_pk_f16(a - (float)p[0], b - (float)p[1]);
      hi[s][e] = p[0];
      hi[s][e + 1] = p[1];
      lo[s][e] = r[0];
      lo[s][e + 1] = r[1];
    }
  return eq;
}

// A query's score scale: raw dot products times c times a key's scale are octaves;
// with a cap, z times the key's scale goes through the tanh.
struct Score {
  float c, z, cap;
  __device__ __forceinline__ Score(float asc, float sc_att, int eq) {
    z = ldexpf(asc, eq) / (sc_att != 0.0f ? sc_att : 1.0f);
    c = ldexpf(asc * kLog2e, eq);
    cap = sc_att * kLog2e;
  }
};

// Scores of a tile to weights.  d: raw dot products; p: the weights' pieces.
// live: bit 4 u + i is set where the key is seen (used when some isn't).
template <bool CAP, class F>
__device__ __forceinline__ void weights(const v4f (&d)[2], const Scales &sc, const Score &q,
                                        bool masked, unsigned live, Soft &s, h8 &phi, h8 &plo,
                                        F &&rescale) {
  float x[8], a[8], vs[8];
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float ks = sc.k[e / 4][e % 4];
    vs[e] = sc.v[e / 4][e % 4];
    if constexpr (CAP) {
      x[e] = tanh32(d[e / 4][e % 4] * (q.z * ks));
      a[e] = q.cap;
    } else {
      x[e] = d[e / 4][e % 4];
      a[e] = q.c * ks;
    }
  }
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int ev = (int)(__float_as_uint(vs[e]) >> 23 & 255) - 127;
    t[e] = fmaf(x[e], a[e], fmaxf((float)ev, kLeastVs));
  }
  if (masked) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!(live >> e & 1)) {
        t[e] = -INFINITY;
        x[e] = -INFINITY;
        a[e] = 1.0f;
        vs[e] = 0.0f;
      }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, t[e]);
  if (__any(top > s.m + kSlack)) {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m = top > s.m + kSlack ? ceilf(top) - kSet : s.m;
    const float f = __builtin_amdgcn_exp2f(s.m - m);
    s.m = m;
    s.l *= f;
    rescale(f);
  }
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(x[e], a[e], -s.m));
    const float p1 = __builtin_amdgcn_exp2f(fmaf(x[e + 1], a[e + 1], -s.m));
    sum += p0 + p1;
    const float w0 = p0 * vs[e], w1 = p1 * vs[e + 1];
    const h2 h = cvt_pk_f16(w0, w1);
    const h2 r = cvt_pk_f16(w0 - (float)h[0], w1 - (float)h[1]);
    phi[e] = h[0];
    phi[e + 1] = h[1];
    plo[e] = r[0];
    plo[e + 1] = r[1];
  }
  s.l += sum;
}

// Which of a lane's eight keys of the tile at key0 are seen.
__device__ __forceinline__ unsigned seen(int key0, int g, KvSee see, bool ok0, bool ok1) {
  unsigned live = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int key = key0 + 16 * (e / 4) + 4 * g + e % 4;
    if (key >= see.lo && key <= see.hi && (e < 4 ? ok0 : ok1)) live |= 1u << e;
  }
  return live;
}

// Where the two halves of the tile at key0 lie (wave-uniform): pages hold whole
// halves.  A half that isn't there (past the end, or on a bad page) reads page 0.
struct Half {
  size_t slot;
  bool ok;
};
__device__ __forceinline__ Half half_at(const KvCache &c, const int *pages, int width, int key,
                                        int len, int hk) {
  const int id = pages[min(key >> c.shift, width - 1)];
  Half h;
  h.ok = key < len && (unsigned)id < (unsigned)c.npages;
  const int page = h.ok ? id : 0;
  h.slot = (((size_t)page * c.nkv + hk) << c.shift) + (key & ((1 << c.shift) - 1));
  return h;
}

__device__ __forceinline__ int wave_max_all(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// ---- single tokens ------------------------------------------------------------
// A workgroup takes up to 16 query vectors of one sequence and kv head, and a chunk
// of its keys, whose tiles its four waves share out.  Codes go straight from memory
// to registers, a tile ahead of their use; 24 KB and more in flight a wave.  Bound by
// the cache's bytes: per 32 keys (16 KB) a wave spends about 1000 cycles of products and
// 1500 of vector work on what takes 1200 to arrive at the card's rate.

// The keys that a sequence's rows see: tiles t0 .. t1 - 1, from `from` on.
struct KvRange {
  int t0, t1;
};
__device__ __forceinline__ KvRange key_range(int first_pos, int last_pos, int len, int slide,
                                             int dense, int from) {
  const KvSpan a = kv_span(first_pos, len, slide, dense), b = kv_span(last_pos, len, slide, dense);
  const int lo = max(max(a.lo, 0), from), hi = b.hi;
  if (hi < lo) return {0, 0};
  return {lo / kTile, hi / kTile + 1};
}

constexpr int kStepWaves = 4;

template <int HD, int TYPE, bool CAP>
__global__ __launch_bounds__(64 * kStepWaves, 2) void kv_step_kernel(KvAttn a, KvPlan pl) {
  constexpr int KS = HD / 32, ND = HD / 16, NJ = HD / 64, VW = HD / 64;
  constexpr int LS = HD + 4;  // floats of a query in LDS
  __shared__ float part[kStepWaves][kStepRows][LS];
  __shared__ float sm[kStepWaves][kStepRows], sl[kStepWaves][kStepRows];
  const int chunk = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const KvSeq s = kv_seq(a.b, b);
  const int rows = s.n * pl.group;
  if (s.n == 0 || rows > kStepRows) return;
  const int p0 = s.len - s.n;
  const KvRange kr = key_range(p0, s.len - 1, s.len, a.slide, a.dense, a.shared);
  const int t0 = kr.t0 + chunk * pl.step_tpc, t1 = min(kr.t1, t0 + pl.step_tpc);
  if (t0 >= t1 && chunk > 0) return;

  // the lane's query
  const int j = min(n, rows - 1), row = s.r0 + j / pl.group, head = hk * pl.group + j % pl.group;
  const KvSpan span = kv_span(p0 + j / pl.group, s.len, a.slide, a.dense);
  const KvSee see{max(span.lo, a.shared), span.hi};
  const int f_lo = wave_max_all(see.lo), f_hi = -wave_max_all(-see.hi);
  h8 qhi[KS], qlo[KS];
  const int eq = load_q<HD>(a.q + (size_t)row * a.q_stride + head * HD, g, qhi, qlo);
  const Score score(a.asc, a.cap, eq);

  v4f o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i] = v4f{};
  Soft soft{kFloor, 0.0f};

  typedef uint32_t vreg __attribute__((ext_vector_type(VW)));
  const int *pages = a.b.pages + (size_t)b * a.b.width;
  u4 kreg[2][NJ];
  vreg vval[2][4];
  Scales sc;
  auto halves = [&](int t, Half (&h)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      h[u] = half_at(a.c, pages, a.b.width, kTile * t + 16 * u, s.len, hk);
  };
  auto load_k = [&](const Half (&h)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t *p = a.c.k + (h[u].slot + n) * HD + 16 * g;
#pragma unroll
      for (int i = 0; i < NJ; ++i) kreg[u][i] = *reinterpret_cast<const u4 *>(p + 64 * i);
      sc.k[u] = *reinterpret_cast<const v4f *>(a.c.ks + h[u].slot + 4 * g);
    }
  };
  auto load_v = [&](const Half (&h)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t *p = a.c.v + (h[u].slot + 4 * g) * HD + (HD / 16) * n;
#pragma unroll
      for (int i = 0; i < 4; ++i) vval[u][i] = *reinterpret_cast<const vreg *>(p + HD * i);
      sc.v[u] = *reinterpret_cast<const v4f *>(a.c.vs + h[u].slot + 4 * g);
    }
  };

  int t = t0 + wave;
  if (t < t1) {
    Half cur[2], nxt[2];
    halves(t, cur);
    load_k(cur);
    load_v(cur);
    for (; t < t1; t += kStepWaves) {
      const int tn = min(t + kStepWaves, t1 - 1);  // past the last: loaded, not used
      halves(tn, nxt);
      v4f dh[2] = {}, dl[2] = {};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u4 x = kreg[u][i / 2];
          const h8 f = codes8<TYPE>(x[2 * (i % 2)], x[2 * (i % 2) + 1]);
          dl[u] = mma(f, qlo[i], dl[u]);
          dh[u] = mma(f, qhi[i], dh[u]);
        }
      const v4f d[2] = {dh[0] + dl[0], dh[1] + dl[1]};
      Scales now = sc;
      __builtin_amdgcn_sched_barrier(0);
      load_k(nxt);
      __builtin_amdgcn_sched_barrier(0);
      const int key0 = kTile * t;
      const bool masked =
          key0 < f_lo || key0 + kTile - 1 > f_hi || !cur[0].ok || !cur[1].ok;  // wave-uniform
      unsigned live = 0xff;
      if (masked) {
        live = seen(key0, g, see, cur[0].ok, cur[1].ok);
        // what lies past a sequence's end may be a NaN's code, times a weight of 0
        if (TYPE == kKvE4m3)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (key0 + 16 * (e / 4) + 4 * g + e % 4 >= s.len || !cur[e / 4].ok)
              vval[e / 4][e % 4] = vreg(0u);
      }
      h8 phi, plo;
      weights<CAP>(d, now, score, masked, live, soft, phi, plo, [&](float f) {
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= f;
      });
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = vval[e / 4][e % 4][w];
        h8 f[4];
        codes_t<TYPE>(x, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[4 * w + i] = mma(f[i], plo, o[4 * w + i]);
          o[4 * w + i] = mma(f[i], phi, o[4 * w + i]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_v(nxt);
      cur[0] = nxt[0];
      cur[1] = nxt[1];
    }
  }

  // the waves' sums, by the largest M
  soft.l += __shfl_xor(soft.l, 16, 64);
  soft.l += __shfl_xor(soft.l, 32, 64);
  if (g == 0) {
    sm[wave][n] = soft.m;
    sl[wave][n] = soft.l;
  }
  __syncthreads();
  if (n < rows) {
    float m = kFloor;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) m = fmaxf(m, sm[w][n]);
    const float f = __builtin_amdgcn_exp2f(soft.m - m);
    // o[i][r]: dim 16 (4 g + r) + i of 256, 8 (4 g + r) + i of 128
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < ND; i += 4)
        *reinterpret_cast<v4f *>(&part[wave][n][ND * (4 * g + r) + i]) =
            v4f{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]} * f;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (HD / 4); e += 64 * kStepWaves) {
    const int q = e / (HD / 4), d = 4 * (e % (HD / 4));
    float m = kFloor, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) m = fmaxf(m, sm[w][q]);
    v4f x = {};
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) {
      l += sl[w][q] * __builtin_amdgcn_exp2f(sm[w][q] - m);
      x += *reinterpret_cast<const v4f *>(&part[w][q][d]);
    }
    if (pl.step_ns == 1 && pl.pre_ns == 0) {
      float *out = a.out + ((size_t)(s.r0 + q / pl.group) * a.n_heads + hk * pl.group +
                            q % pl.group) * HD + d;
      *reinterpret_cast<v4f *>(out) = l != 0.0f ? x / l : v4f{};
    } else {
      const size_t at = (((size_t)b * a.c.nkv + hk) * pl.step_ns + chunk) * pl.step_rows + q;
      *reinterpret_cast<v4f *>((float *)(a.work + pl.step_o) + at * HD + d) = x;
      if (d == 0) ((float2 *)(a.work + pl.step_m))[at] = float2{m, l};
    }
  }
}

// ---- prompt rows and shared prefixes ---------------------------------------------
// A workgroup takes 64 QB query vectors of a kv head, 16 QB a wave, and a chunk of
// their keys; PRE: the rows of all sequences, over the shared prefix.  Each tile's
// codes are made f16 once, a share by each wave, and reach the others through LDS in
// operand order.

template <int HD, int TYPE, bool CAP, int QB, bool PRE>
__global__ __launch_bounds__(256) void kv_rows_kernel(KvAttn a, KvPlan pl) {
  constexpr int KS = HD / 32, ND = HD / 16;
  constexpr int TR = 64 * QB;
  __shared__ h8 kf[2 * KS][64], vf[ND][64];
  const int ns = PRE ? pl.pre_ns : pl.rows_ns, tpc = PRE ? pl.pre_tpc : pl.rows_tpc;
  const int chunk = blockIdx.x % ns, tile = blockIdx.x / ns, hk = blockIdx.y;
  const int b = PRE ? 0 : blockIdx.z;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  KvSeq s = kv_seq(a.b, b);
  int len = s.len;
  if (PRE) {
    s.r0 = kv_clamp(a.b.row0[0], 0, a.b.rows);
    s.n = kv_clamp(a.b.row0[a.b.batch], s.r0, a.b.rows) - s.r0;
    len = a.shared;
  } else if (pl.step && s.n * pl.group <= kStepRows) {
    return;
  }
  const int rows = s.n * pl.group, at = tile * TR;
  if (at >= rows) return;

  // the lane's queries
  KvSee see[QB];
  int qrow[QB], qhead[QB];
  h8 qhi[QB][KS], qlo[QB][KS];
  float cq[QB], zq[QB];
  int f_lo = 0, f_hi = INT_MAX, any_lo = INT_MAX, any_hi = -1;
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int j = at + 16 * (QB * wave + q) + n;
    const int jj = min(j, rows - 1);
    qrow[q] = s.r0 + jj / pl.group;
    qhead[q] = hk * pl.group + jj % pl.group;
    KvSpan span{0, -1};
    if (PRE) {
      const int i = kv_find(a.b.row0, a.b.batch, qrow[q]);
      if (i >= 0) {
        const KvSeq o = kv_seq(a.b, i);
        span = kv_span(o.len - o.n + (qrow[q] - o.r0), o.len, a.slide, a.dense);
      }
      see[q] = {span.lo, min(span.hi, a.shared - 1)};
    } else {
      span = kv_span(s.len - s.n + jj / pl.group, s.len, a.slide, a.dense);
      see[q] = {max(span.lo, a.shared), span.hi};
    }
    if (see[q].hi >= see[q].lo) {
      any_lo = min(any_lo, see[q].lo);
      any_hi = max(any_hi, see[q].hi);
    }
    f_lo = max(f_lo, see[q].lo);
    f_hi = min(f_hi, see[q].hi);
    const int eq = load_q<HD>(a.q + (size_t)qrow[q] * a.q_stride + qhead[q] * HD, g, qhi[q],
                              qlo[q]);
    const Score sc(a.asc, a.cap, eq);
    cq[q] = sc.c;
    zq[q] = sc.z;
  }
  f_lo = wave_max_all(f_lo);
  f_hi = -wave_max_all(-f_hi);
  int t0, t1;
  if (PRE) {  // chunks of the whole prefix
    t0 = chunk * tpc;
    t1 = min(ceil_div(a.shared, kTile), t0 + tpc);
  } else {
    const int i0 = at / pl.group, i1 = min(s.n - 1, (at + TR - 1) / pl.group);
    const KvRange kr = key_range(s.len - s.n + i0, s.len - s.n + i1, s.len, a.slide, a.dense,
                                 a.shared);
    t0 = kr.t0 + chunk * tpc;
    t1 = min(kr.t1, t0 + tpc);
    if (t0 >= t1 && chunk > 0) return;
  }

  v4f o[QB][ND];
  Soft soft[QB];
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    soft[q] = {kFloor, 0.0f};
#pragma unroll
    for (int i = 0; i < ND; ++i) o[q][i] = v4f{};
  }
  const int *pages = a.b.pages + (size_t)b * a.b.width;
  for (int t = t0; t < t1; ++t) {
    Half h[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      h[u] = half_at(a.c, pages, a.b.width, kTile * t + 16 * u, len, hk);
    Scales sc;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc.k[u] = *reinterpret_cast<const v4f *>(a.c.ks + h[u].slot + 4 * g);
      sc.v[u] = *reinterpret_cast<const v4f *>(a.c.vs + h[u].slot + 4 * g);
    }
    __syncthreads();
    for (int f = wave; f < HD / 32; f += 4) {  // halves and 64-dim blocks of K
      const int u = f % 2, jc = f / 2;
      const u4 x = *reinterpret_cast<const u4 *>(a.c.k + (h[u].slot + n) * HD + 64 * jc + 16 * g);
      kf[u * KS + 2 * jc][lane] = codes8<TYPE>(x[0], x[1]);
      kf[u * KS + 2 * jc + 1][lane] = codes8<TYPE>(x[2], x[3]);
    }
    for (int f = wave; f < HD / 64; f += 4) {  // 64-dim blocks of V
      uint32_t x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = *reinterpret_cast<const uint32_t *>(
            a.c.v + (h[e / 4].slot + 4 * g + e % 4) * HD + 64 * f + 4 * (4 * (n & 3) + (n >> 2)));
        if (kTile * t + 16 * (e / 4) + 4 * g + e % 4 >= len || !h[e / 4].ok) x[e] = 0;
      }
      h8 fr[4];
      codes_t<TYPE>(x, fr);
#pragma unroll
      for (int i = 0; i < 4; ++i) vf[4 * f + i][lane] = fr[i];
    }
    __syncthreads();
    const int key0 = kTile * t;
    const bool masked = key0 < f_lo || key0 + kTile - 1 > f_hi || !h[0].ok || !h[1].ok;
    h8 phi[QB], plo[QB];
#pragma unroll
    for (int q = 0; q < QB; ++q) {
      v4f dh[2] = {}, dl[2] = {};
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          dl[u] = mma(kf[u * KS + i][lane], qlo[q][i], dl[u]);
          dh[u] = mma(kf[u * KS + i][lane], qhi[q][i], dh[u]);
        }
      const v4f d[2] = {dh[0] + dl[0], dh[1] + dl[1]};
      Score score(0.0f, a.cap, 0);
      score.c = cq[q];
      score.z = zq[q];
      const unsigned live = masked ? seen(key0, g, see[q], h[0].ok, h[1].ok) : 0xff;
      weights<CAP>(d, sc, score, masked, live, soft[q], phi[q], plo[q], [&](float f) {
#pragma unroll
        for (int i = 0; i < ND; ++i) o[q][i] *= f;
      });
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const h8 f = vf[i][lane];
#pragma unroll
      for (int q = 0; q < QB; ++q) {
        o[q][i] = mma(f, plo[q], o[q][i]);
        o[q][i] = mma(f, phi[q], o[q][i]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    soft[q].l += __shfl_xor(soft[q].l, 16, 64);
    soft[q].l += __shfl_xor(soft[q].l, 32, 64);
    if (at + 16 * (QB * wave + q) + n >= rows) continue;
    const size_t vec = (size_t)qrow[q] * a.n_heads + qhead[q];
    const bool whole = !PRE && ns == 1 && pl.pre_ns == 0;
    const size_t pt = (size_t)chunk * a.b.rows * a.n_heads + vec;
    float *dst = whole ? a.out + vec * HD
                       : (float *)(a.work + (PRE ? pl.pre_o : pl.rows_o)) + pt * HD;
    const float f = !whole ? 1.0f : soft[q].l != 0.0f ? 1.0f / soft[q].l : 0.0f;
    // o[4 w + i][r]: dim 64 w + 16 r + 4 g + i
#pragma unroll
    for (int w = 0; w < HD / 64; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v4f x = v4f{o[q][4 * w][r], o[q][4 * w + 1][r], o[q][4 * w + 2][r], o[q][4 * w + 3][r]};
        x = f != 0.0f ? x * f : v4f{};
        *reinterpret_cast<v4f *>(dst + 64 * w + 16 * r + 4 * g) = x;
      }
    if (!whole && g == 0)
      ((float2 *)(a.work + (PRE ? pl.pre_m : pl.rows_m)))[pt] = float2{soft[q].m, soft[q].l};
  }
}

// ---- the chunks' sums together ------------------------------------------------------
// One workgroup per row and head, its waves sharing out the chunks.

template <int HD>
__global__ __launch_bounds__(1024) void kv_merge_kernel(KvAttn a, KvPlan pl) {
  constexpr int E = HD / 64;
  __shared__ float so[16][HD], sm[16], sl[16];
  const int b = blockIdx.z, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const KvSeq s = kv_seq(a.b, b);
  const int i = blockIdx.x, head = blockIdx.y;
  if (i >= s.n) return;
  const int hk = head / pl.group, j = i * pl.group + head % pl.group, p0 = s.len - s.n;
  const bool step = pl.step && s.n * pl.group <= kStepRows;
  const size_t vec = (size_t)(s.r0 + i) * a.n_heads + head;
  // this row's own chunks: number, first partial and the step to the next
  int n;
  size_t first, stride;
  const float *po;
  const float2 *pm;
  if (step) {
    const KvRange kr = key_range(p0, s.len - 1, s.len, a.slide, a.dense, a.shared);
    n = max(1, ceil_div(kr.t1 - kr.t0, pl.step_tpc));
    if (pl.step_ns == 1 && pl.pre_ns == 0) return;
    first = ((size_t)b * a.c.nkv + hk) * pl.step_ns * pl.step_rows + j;
    stride = pl.step_rows;
    po = (const float *)(a.work + pl.step_o);
    pm = (const float2 *)(a.work + pl.step_m);
  } else {
    const int tr = 64 * pl.qb, at = j / tr * tr;
    const int i0 = at / pl.group, i1 = min(s.n - 1, (at + tr - 1) / pl.group);
    const KvRange kr = key_range(p0 + i0, p0 + i1, s.len, a.slide, a.dense, a.shared);
    n = max(1, ceil_div(kr.t1 - kr.t0, pl.rows_tpc));
    if (pl.rows_ns == 1 && pl.pre_ns == 0) return;
    first = vec;
    stride = (size_t)a.b.rows * a.n_heads;
    po = (const float *)(a.work + pl.rows_o);
    pm = (const float2 *)(a.work + pl.rows_m);
  }
  const int total = n + pl.pre_ns;
  auto where = [&](int c, const float **o) {
    size_t at;
    float2 v;
    if (c < n) {
      at = first + c * stride;
      *o = po + at * HD;
      v = pm[at];
    } else {
      at = (size_t)(c - n) * a.b.rows * a.n_heads + vec;
      *o = (const float *)(a.work + pl.pre_o) + at * HD;
      v = ((const float2 *)(a.work + pl.pre_m))[at];
    }
    return v;
  };
  float m = kFloor, l = 0.0f, x[E] = {};
  for (int c = wave; c < total; c += nw) {
    const float *o;
    const float2 v = where(c, &o);
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = o[E * lane + e];
    const float mn = fmaxf(m, v.x);
    const float f = __builtin_amdgcn_exp2f(m - mn), h = __builtin_amdgcn_exp2f(v.x - mn);
    m = mn;
    l = l * f + v.y * h;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * f + y[e] * h;
  }
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[wave][E * lane + e] = x[e];
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float mm = kFloor, ll = 0.0f, sum = 0.0f;
  for (int w = 0; w < nw; ++w) mm = fmaxf(mm, sm[w]);
  for (int w = 0; w < nw; ++w) {
    const float f = __builtin_amdgcn_exp2f(sm[w] - mm);
    ll += sl[w] * f;
    sum += so[w][threadIdx.x] * f;
  }
  a.out[vec * HD + threadIdx.x] = ll != 0.0f ? sum / ll : 0.0f;
}

KvPlan plan(const KvAttn &a, const DeviceInfo &dev) {
  KvPlan p{};
  p.group = a.n_heads / a.c.nkv;
  const int most = a.b.max_rows * p.group;  // query vectors of a sequence and kv head
  p.step = p.group <= kStepRows && (most <= kStepRows || a.b.batch > 1);
  const bool rows = !p.step || most > kStepRows;
  // tiles that a sequence's rows see behind the prefix: by the window where there is one
  const int own = a.b.max_len - a.shared;
  auto tiles = [&](int n) {  // n neighbouring rows
    const int keys = a.slide > 0 ? (int)std::min<long>(own, (long)a.slide + n) : own;
    return std::max(1, ceil_div(keys, kTile) + 1);
  };
  auto cut = [](int tiles, int ns, int unit, int *out_ns, int *out_tpc) {
    ns = std::max(1, std::min({ns, ceil_div(tiles, unit), 256}));
    *out_tpc = ceil_div(ceil_div(tiles, ns), unit) * unit;
    *out_ns = ceil_div(tiles, *out_tpc);
  };
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  const size_t vecs = (size_t)a.b.rows * a.n_heads;
  if (p.step) {
    p.step_rows = std::min(kStepRows, most);
    const int n = std::min(a.b.max_rows, kStepRows / p.group);
    cut(tiles(n), 4 * dev.cus / std::max(1, a.b.batch * a.c.nkv), kStepWaves, &p.step_ns,
        &p.step_tpc);
  }
  p.qb = (long)a.b.rows * p.group > 64 ? 2 : 1;
  const int blocks = (int)std::max<long>(1, ((long)a.b.rows * p.group + 64 * p.qb - 1) /
                                                (64 * p.qb)) * a.c.nkv;
  if (rows) cut(tiles(ceil_div(64 * p.qb, p.group) + 1), dev.cus / blocks, 4, &p.rows_ns, &p.rows_tpc);
  if (a.shared > 0)
    cut(ceil_div(a.shared, kTile), dev.cus / blocks, 4, &p.pre_ns, &p.pre_tpc);
  if (p.step && (p.step_ns > 1 || p.pre_ns > 0)) {
    const size_t n = (size_t)a.b.batch * a.c.nkv * p.step_ns * p.step_rows;
    p.step_o = take(n * a.c.hdim * 4);
    p.step_m = take(n * 8);
  }
  if (p.rows_ns > 1 || (p.rows_ns > 0 && p.pre_ns > 0)) {
    p.rows_o = take(p.rows_ns * vecs * a.c.hdim * 4);
    p.rows_m = take(p.rows_ns * vecs * 8);
  }
  if (p.pre_ns > 0) {
    p.pre_o = take(p.pre_ns * vecs * a.c.hdim * 4);
    p.pre_m = take(p.pre_ns * vecs * 8);
  }
  p.bytes = at;
  // every key of a dense row, in as many chunks
  if (a.dense && a.slide > 0) {
    const int all = std::max(1, ceil_div(own, kTile) + 1);
    if (p.step) p.step_tpc = ceil_div(ceil_div(all, p.step_ns), kStepWaves) * kStepWaves;
    if (p.rows_ns) p.rows_tpc = ceil_div(all, p.rows_ns);
  }
  return p;
}

template <int HD, int TYPE, bool CAP>
void launch_typed(const KvAttn &a, const KvPlan &p, hipStream_t stream) {
  const int nkv = a.c.nkv, batch = a.b.batch;
  if (p.step)
    kv_step_kernel<HD, TYPE, CAP>
        <<<dim3(p.step_ns, nkv, batch), 64 * kStepWaves, 0, stream>>>(a, p);
  auto rows = [&](auto kernel, int vecs, int ns, int z) {
    kernel<<<dim3(ceil_div(vecs, 64 * p.qb) * ns, nkv, z), 256, 0, stream>>>(a, p);
  };
  if (p.rows_ns > 0) {
    const int vecs = a.b.max_rows * p.group;
    if (p.qb == 2)
      rows(kv_rows_kernel<HD, TYPE, CAP, 2, false>, vecs, p.rows_ns, batch);
    else
      rows(kv_rows_kernel<HD, TYPE, CAP, 1, false>, vecs, p.rows_ns, batch);
  }
  if (p.pre_ns > 0) {
    const int vecs = a.b.rows * p.group;
    if (p.qb == 2)
      rows(kv_rows_kernel<HD, TYPE, CAP, 2, true>, vecs, p.pre_ns, 1);
    else
      rows(kv_rows_kernel<HD, TYPE, CAP, 1, true>, vecs, p.pre_ns, 1);
  }
  const int most = std::max(p.step ? p.step_ns : 0, p.rows_ns) + p.pre_ns;
  if (most > 1)
    kv_merge_kernel<HD><<<dim3(a.b.max_rows, a.n_heads, batch), most > 16 ? 1024 : 256, 0, stream>>>(
        a, p);
}

template <int HD>
void launch_hd(const KvAttn &a, const KvPlan &p, hipStream_t stream) {
  if (a.c.type == kKvI8)
    a.cap != 0.0f ? launch_typed<HD, kKvI8, true>(a, p, stream)
                  : launch_typed<HD, kKvI8, false>(a, p, stream);
  else
    a.cap != 0.0f ? launch_typed<HD, kKvE4m3, true>(a, p, stream)
                  : launch_typed<HD, kKvE4m3, false>(a, p, stream);
}

}  // namespace

size_t kv_attention_work(const KvAttn &a, const DeviceInfo &dev) { return plan(a, dev).bytes; }

hipError_t launch_kv_attention(const KvAttn &a, const DeviceInfo &dev, hipStream_t stream) {
  const KvPlan p = plan(a, dev);
  if (a.c.hdim == 256)
    launch_hd<256>(a, p, stream);
  else
    launch_hd<128>(a, p, stream);
  return hipGetLastError();
}

}  // namespace gh
