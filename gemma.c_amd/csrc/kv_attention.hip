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
// query: p = 2^(s - M), w = p vs 2^-24, l = sum p, out = 2^24 sum w code / l.  M follows
// the largest s + log2 vs, not the largest s: what must fit f16 is w.  It has twelve
// octaves of slack, so that the sums are rescaled rarely and by powers of two.  A weight w
// in its two pieces is off by at most 2^-23 of itself, or by 2^-25 where that is more, and the
// largest of a query is 2 or more.  Where it may not be (M doesn't follow scales below 2^-60,
// nor scores past 2^23 octaves) the query is done over in 64 bits: wide_query().
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
#include <type_traits>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kTile = 32;             // keys of a tile
constexpr int kLongRun = 16;          // tiles by 64 query vectors of a compute unit: see plan()
constexpr int kBothTiles = 64;         // tiles of own keys, at most, of single tokens that share
                                      // a launch with their prefix
constexpr int kStepRows = 16;         // query vectors (rows x heads of a kv head) of a step tile
constexpr float kFloor = -0x1p126f;   // M of a query that has seen no key
constexpr float kFar = 0x1p23f;       // |M| from which on fp32 can't hold M and M + kSlack apart
constexpr float kVsUnit = 0x1p-24f;   // V's scales enter the weights in units of 2^24, so that
constexpr float kVsOctaves = 24.0f;   // l keeps its terms beside the largest scales
constexpr float kSlack = 14.0f + kVsOctaves;  // weights stay below 2^15 ...
constexpr float kSet = 2.0f + kVsOctaves;     // ... and a moved M puts the largest at 2 .. 2^3
constexpr float kLeastVs = -60.0f;    // octaves that a scale counts at least ...
constexpr float kMostVs = 121.0f;     // ... and at most (its own largest; for a NaN)
constexpr float kLog2e = 1.44269502162933349609375f;

// How a call is cut into workgroups: the same on the host, which sizes the
// workspace by it, and in the kernels.
struct KvPlan {
  int group;                    // heads per kv head
  uint32_t inv_group;           // 2^21 / group, rounded up
  int step, step_ns;            // single tokens: on or off, key chunks at most
  int step_rows;                // query vectors of a sequence and kv head, at most
  int rows_ns;                  // prompt rows (0 chunks: off)
  int pre_ns, pre_tpc;          // shared prefix (0: none), tiles of a chunk
  int pre_blocks;               // its tiles of rows, where one launch takes it and the single
                                // tokens (0: not)
  int qb, pre_qb;               // 16-query blocks of a wave of the prompt kernel
  size_t step_o, step_m, rows_o, rows_m, pre_o, pre_m, bytes;  // workspace
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Tiles of a chunk, at least, and the whole number of them that a chunk has: what rows see is
// cut evenly into ns chunks or fewer, by the lengths on the device, of which the host only
// knows a bound.
constexpr int kChunkTiles = 4;
__host__ __device__ inline int chunk_tiles(int tiles, int ns) {
  const int n = ceil_div(ceil_div(tiles, ns), kChunkTiles) * kChunkTiles;
  return n > 0 ? n : kChunkTiles;
}

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
// A dword (four dims) of each of eight keys, transposed: dim(i) is dim i of the eight
// keys.  Two keys at a time.
struct Transposed {
  h2 p[4][4];  // [dim][pair of keys]
  __device__ __forceinline__ h8 dim(int i) const { return join(p[i][0], p[i][1], p[i][2], p[i][3]); }
};
template <int TYPE, int J>
__device__ __forceinline__ void transpose_pair(const uint32_t (&x)[8], Transposed &t) {
  const uint32_t a = x[2 * J], b = x[2 * J + 1];
  uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u);  // a0 b0 a1 b1
  uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07030602u);  // a2 b2 a3 b3
  if constexpr (TYPE == kKvI8) {
    lo = flip(lo);
    hi = flip(hi);
    t.p[0][J] = magic<0x04010400u>(lo);
    t.p[1][J] = magic<0x04030402u>(lo);
    t.p[2][J] = magic<0x04010400u>(hi);
    t.p[3][J] = magic<0x04030402u>(hi);
  } else {
    t.p[0][J] = from_e4m3<false>(lo);
    t.p[1][J] = from_e4m3<true>(lo);
    t.p[2][J] = from_e4m3<false>(hi);
    t.p[3][J] = from_e4m3<true>(hi);
  }
}

// ... of two of the four dims, by sel
struct TransposedHalf {
  h2 p[2][4];
  __device__ __forceinline__ h8 dim(int i) const { return join(p[i][0], p[i][1], p[i][2], p[i][3]); }
};
constexpr uint32_t kDims01 = 0x05010400u, kDims23 = 0x07030602u;
template <int TYPE, int J>
__device__ __forceinline__ void transpose_pair(const uint32_t (&x)[8], uint32_t sel,
                                               TransposedHalf &t) {
  uint32_t a = __builtin_amdgcn_perm(x[2 * J + 1], x[2 * J], sel);
  if constexpr (TYPE == kKvI8) {
    a = flip(a);
    t.p[0][J] = magic<0x04010400u>(a);
    t.p[1][J] = magic<0x04030402u>(a);
  } else {
    t.p[0][J] = from_e4m3<false>(a);
    t.p[1][J] = from_e4m3<true>(a);
  }
}

// f(0) .. f(N - 1), the numbers as constants.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F &&f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

__device__ __forceinline__ v4f mma(h8 a, h8 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// What a lane's query sees: keys lo .. hi.
struct KvSee {
  int lo, hi;
};

// The scales of a lane's eight keys of a tile: keys 16 u + 4 g + i.
typedef float v8f __attribute__((ext_vector_type(8)));
struct Scales {
  v8f k, v;
};
__device__ __forceinline__ v8f eight(v4f a, v4f b) {
  return v8f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// The running softmax of a query: M, and the sum of the weights of the keys that
// the lane has.
struct Soft {
  float m, l;
};

// A query of HD dims in operand order (dims 64 j + 16 g + 8 h .. + 7 are step 2 j + h).
template <int HD>
struct Query {
  v4f x[HD / 16];
  __device__ __forceinline__ void load(const float *row, int g) {
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
      x[e] = *reinterpret_cast<const v4f *>(row + 64 * (e / 4) + 16 * g + 4 * (e % 4));
  }
  // in two f16 pieces; the exponent that it was scaled by comes back
  __device__ __forceinline__ int split(h8 (&hi)[HD / 32], h8 (&lo)[HD / 32]) const {
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
#pragma unroll
      for (int u = 0; u < 4; ++u) amax = fmaxf(amax, finite_abs(x[e][u]));
    amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
    const int eq = amax > 0.0f ? max(ilogbf(amax) - 14, -126) : 0;
    const float down = ldexpf(1.0f, -eq);
#pragma unroll
    for (int s = 0; s < HD / 32; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = x[2 * s + e / 4][e % 4] * down, b = x[2 * s + e / 4][e % 4 + 1] * down;
        const h2 p = cvt_pk_f16(a, b);
        const h2 r = cvt_pk_f16(a - (float)p[0], b - (float)p[1]);
        hi[s][e] = p[0];
        hi[s][e + 1] = p[1];
        lo[s][e] = r[0];
        lo[s][e + 1] = r[1];
      }
    return eq;
  }
};

// A query's score scale: raw dot products times c times a key's scale are octaves;
// with a cap, z times the key's scale goes through the tanh.
struct Score {
  float c, z, cap;
  Score() = default;
  __device__ __forceinline__ Score(float asc, float sc_att, int eq) {
    z = ldexpf(asc, eq) / (sc_att != 0.0f ? sc_att : 1.0f);
    c = ldexpf(asc * kLog2e, eq);
    cap = sc_att * kLog2e;
  }
};

// Octaves that the values of a lane's eight keys may add to a weight, from their scales in
// units of 2^24.
__device__ __forceinline__ void scale_octaves(const v8f &vs, float (&lv)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int ev = (int)(__float_as_uint(vs[e]) >> 23 & 255) - 127 + (int)kVsOctaves;
    lv[e] = fminf(fmaxf((float)ev, kLeastVs), kMostVs);
  }
}

// A raw dot product to a score in octaves.
template <bool CAP>
__device__ __forceinline__ float score_of(float x, float ks, const Score &q) {
  return CAP ? tanh32(x * (q.z * ks)) * q.cap : x * (q.c * ks);
}
// The scores of keys that aren't seen (live: a bit per key) become -inf; the largest
// s + log2 vs of the lane's keys comes back.
__device__ __forceinline__ float top_of(v4f (&d)[2], const float (&lv)[8], bool masked,
                                        unsigned live) {
  if (masked) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!(live >> e & 1)) d[e / 4][e % 4] = -INFINITY;
  }
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, d[e / 4][e % 4] + lv[e]);
  return top;
}

// l by another M, `by` octaves above its own (a whole number, 0 or below).  In one step: beside
// values of very different sizes l may be 2^98 where 2^by alone is 0.  An infinite l stays so.
__device__ __forceinline__ float lowered(float l, float by) {
  return ldexpf(l, (int)fmaxf(by, -400.0f));
}

__device__ __forceinline__ bool far(float m) { return fabsf(m) >= kFar && m > kFloor; }

// Moves a query's M where the tile's largest weight needs it.  An M that was too far out leaves
// an infinite l: the sums may be anything.
template <class F>
__device__ __forceinline__ void settle(float top, Soft &s, F &&rescale) {
  if (!__any(top > s.m + kSlack)) return;
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const float m = top > s.m + kSlack ? ceilf(top) - kSet : s.m;
  const float f = __builtin_amdgcn_exp2f(s.m - m);
  s.l = m != s.m && far(s.m) ? INFINITY : lowered(s.l, s.m - m);
  s.m = m;
  rescale(f);
}

// a b, 0 where a is 0, whatever b (v_mul_legacy_f32; as the compiler's own
// instruction, so that it keeps its distance from the exponential before it).
__device__ float mul_legacy(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

// Scores 2 j and 2 j + 1 to weights' pieces.  The product by a value's scale is 0 for
// a weight of 0, whatever the scale.
__device__ __forceinline__ void weigh(int j, const v4f (&x)[2], const v8f &vs, Soft &s, h8 &phi,
                                      h8 &plo) {
  const int e = 2 * j;
  const float p0 = __builtin_amdgcn_exp2f(x[e / 4][e % 4] - s.m);
  const float p1 = __builtin_amdgcn_exp2f(x[e / 4][e % 4 + 1] - s.m);
  s.l += p0 + p1;
  const float w0 = mul_legacy(p0, vs[e]);
  const float w1 = mul_legacy(p1, vs[e + 1]);
  const h2 h = cvt_pk_f16(w0, w1);
  const h2 r = cvt_pk_f16(fmaf((float)h[0], -1.0f, w0), fmaf((float)h[1], -1.0f, w1));
  phi[e] = h[0];
  phi[e + 1] = h[1];
  plo[e] = r[0];
  plo[e + 1] = r[1];
}

// Which of a lane's eight keys of the tile at key0 are seen.
__device__ __forceinline__ unsigned seen(int key0, int g, KvSee see, int ok) {
  unsigned live = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int key = key0 + 16 * (e / 4) + 4 * g + e % 4;
    if (key >= see.lo && key <= see.hi && (ok >> (e / 4) & 1)) live |= 1u << e;
  }
  return live;
}

// Where the halves (16 keys) of a tile lie: number of the first position's row in the
// cache, wave-uniform (pages hold whole halves).  One that isn't there (past the end, or on
// a bad page) reads page 0.
struct Halves {
  size_t slot0, slot1;
  int ok;  // bits 0 and 1: the halves that are there
};

// The halves of a wave's tiles first, first + step, ... in turn.  Lane i works out half i
// of 32 tiles at a time, the next ones' page ids loaded ahead of their use; by vector
// loads, since waits for a scalar load would be waits for all of the wave's LDS reads too.
struct Pager {
  const int *pages;
  int width, shift, npages, nkv, hk, len, first, step;
  int next, slot_lo, slot_hi;
  unsigned long long there;
  __device__ __forceinline__ Pager(const KvAttn &a, int seq, int length, int head, int t0, int dt)
      : pages(a.b.pages + (size_t)seq * a.b.width), width(a.b.width), shift(a.c.shift),
        npages(a.c.npages), nkv(a.c.nkv), hk(head), len(length), first(t0), step(dt) {
    next = load(0);  // place(0) waits for it
  }
  __device__ __forceinline__ int key(int from) const {
    const int lane = threadIdx.x & 63;
    return kTile * (first + step * (from + lane / 2)) + 16 * (lane & 1);
  }
  __device__ __forceinline__ int load(int from) const {
    return pages[min(key(from) >> shift, width - 1)];
  }
  __device__ __forceinline__ void place(int from) {
    const int k = key(from);
    const bool ok = k < len && (unsigned)next < (unsigned)npages;
    const size_t slot = (((size_t)(ok ? next : 0) * nkv + hk) << shift) + (k & ((1 << shift) - 1));
    slot_lo = (int)slot;
    slot_hi = (int)(slot >> 32);
    there = __ballot(ok);
    next = load(from + 32);
  }
  __device__ __forceinline__ size_t slot(int i) const {
    return (size_t)(uint32_t)__builtin_amdgcn_readlane(slot_hi, i) << 32 |
           (uint32_t)__builtin_amdgcn_readlane(slot_lo, i);
  }
  // the j-th tile's halves; prepare() is called before, for each j from 0 up
  __device__ __forceinline__ void prepare(int j) {
    if ((j & 31) == 0 && j > 0) place(j);
  }
  __device__ __forceinline__ Halves get(int j) const {
    const int i = 2 * (j & 31);
    return Halves{slot(i), slot(i + 1), (int)(there >> i) & 3};
  }
};

// The lane's value at a wave-uniform address and an offset of its own, in bytes.
template <class T, class P>
__device__ __forceinline__ T at_offset(const P *base, uint32_t off) {
  return *reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + off);
}

// One load from memory straight to LDS: each lane's 16 bytes at base + off land at lds +
// 16 lane (base and lds wave-uniform).  The compiler doesn't see it: who reads it waits
// first (dma_wait).  m0 has no other user in the kernel that calls this.
__device__ __forceinline__ void dma16(const void *base, uint32_t off, const void *lds) {
  const uint32_t m = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)lds;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(m), "v"(off),
               "s"(base)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// ... from an address of each lane's own
__device__ __forceinline__ void dma16_at(const void *src, const void *lds) {
  const uint32_t m = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)lds;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m), "v"(src)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// Waits until at most N of the wave's loads, the newest, are under way.
template <int N>
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ int wave_max_all(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// ---- queries whose weights f16 doesn't hold ----------------------------------------
// Whether, of a sequence's keys first .. last, any has a scale that counted as kLeastVs for more
// than it is, and any a value (not so: nothing but zeros was written there); by a whole wave.
__device__ bool any_small(const KvAttn &a, int b, int hk, int first, int last) {
  bool small = false, value = false;
  for (int key = first + (threadIdx.x & 63); key <= last; key += 64) {
    const long slot = kv_slot(a.c, a.b, b, key, hk);
    const float vs = slot >= 0 ? fabsf(a.c.vs[slot]) : 1.0f;
    small = small || vs < 0x1p-60f;
    value = value || (slot >= 0 && vs != 0.0f);
  }
  return __any(small) && __any(value);
}

// A query's l, infinite where its sums have lost what counts: M is far, or has been, or was set
// by a key of a small scale, or of zeros, among the wave's first .. last.  M lies 25 to 38
// octaves below the largest s + log2 vs of its keys.  Where that key's log2 vs is its own, its w
// is 2 or more; where it is kLeastVs instead, its p = 2^(s - M) is 2^85 or more, and so is l.
// (l is that large, too, where all scales are below 2^-45 or so, or 0.)  The inner loops pay
// nothing for it; a test of w itself, for each key, made them 2 to 5% slower.
//
// A query with an infinite l is done over by whoever has its sums last: the merge, for a chunk,
// or the kernel where there is no merge.
__device__ __forceinline__ float marked(const KvAttn &a, const Soft &s, int b, int hk, int first,
                                        int last) {
  float l = far(s.m) ? INFINITY : s.l;
  const bool large = l >= 0x1p84f;
  if (__any(large && l < INFINITY) && any_small(a, b, hk, first, last) && large) l = INFINITY;
  return l;
}

__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <int TYPE>
__device__ __forceinline__ void codes4(uint32_t x, float (&f)[4]) {
  if constexpr (TYPE == kKvI8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(x >> (8 * e));
  } else {
    f[0] = __builtin_amdgcn_cvt_f32_fp8(x, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8(x, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8(x, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8(x, 3);
  }
}

// A query's softmax sums in fp64: the largest score in octaves, and, by that, the sum of
// weights and the lane's dims (HD / 64 lane and up) of the sum of weighted values.
template <int HD>
struct Wide {
  double m = -INFINITY, l = 0.0, x[HD / 64] = {};
};

// One query over keys lo .. hi of sequence b, all in fp64, whose exponents hold any weight times
// any scale; by a whole wave: a key a lane for the scores, HD / 64 dims a lane for the values.
template <int HD, int TYPE>
__device__ Wide<HD> wide_query(const KvAttn &a, int b, int hk, const float *q, int lo, int hi) {
  constexpr int E = HD / 64;
  constexpr double log2e = 0x1.71547652b82fep+0;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // nothing of this is worked out ahead, beside an inner loop
  Wide<HD> r;
  for (int base = lo; base <= hi; base += 64) {
    const int key = base + lane;
    const long slot = key <= hi ? kv_slot(a.c, a.b, b, key, hk) : -1;
    const unsigned long long live = __ballot(slot >= 0);
    if (live == 0) continue;
    double s = -INFINITY, vs = 0.0;
    if (slot >= 0) {
      const uint32_t *codes = reinterpret_cast<const uint32_t *>(a.c.k + (size_t)slot * HD);
      double dot = 0.0;
#pragma unroll 1  // (registers count here, time less)
      for (int d = 0; d < HD; d += 16) {
        const u4 x = *reinterpret_cast<const u4 *>(codes + d / 4);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float f[4];
          codes4<TYPE>(x[u], f);
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = fma((double)q[d + 4 * u + e], (double)f[e], dot);
        }
      }
      s = dot * (double)a.c.ks[slot] * (double)a.asc;
      if (a.cap != 0.0f) s = tanh(s / (double)a.cap) * (double)a.cap;
      s *= log2e;
      if (!(fabs(s) < INFINITY)) s = NAN;
      vs = (double)a.c.vs[slot];
    }
    const double m = fmax(r.m, wave_max_f64(s)), f = exp2(r.m - m);
    const double p = slot >= 0 ? exp2(s - m) : 0.0, w = slot >= 0 ? p * vs : 0.0;
    r.m = m;
    r.l = r.l * f + wave_sum_f64(p);
#pragma unroll
    for (int e = 0; e < E; ++e) r.x[e] *= f;
#pragma unroll 1
    for (int i0 = 0; i0 < 64; i0 += 4) {
      typedef std::conditional_t<E == 4, uint32_t, uint16_t> T;
      T v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // (a key that isn't there: any row, not used)
        const long at = max(slot, 0l);
        const size_t row = (size_t)__builtin_amdgcn_readlane((int)(at >> 32), i0 + u) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)at, i0 + u);
        v[u] = *reinterpret_cast<const T *>(a.c.v + row * HD + E * lane);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (!(live >> (i0 + u) & 1)) continue;
        const double wi = readlane_f64(w, i0 + u);
        float c[4];
        codes4<TYPE>(v[u], c);
#pragma unroll
        for (int e = 0; e < E; ++e) r.x[e] = fma(wi, (double)c[e], r.x[e]);
      }
    }
  }
  return r;
}

// ... to an output row.
template <int HD>
__device__ __forceinline__ void wide_out(const Wide<HD> &r, float *out) {
  constexpr int E = HD / 64;
#pragma unroll
  for (int e = 0; e < E; ++e)
    out[E * (threadIdx.x & 63) + e] = r.l != 0.0 ? (float)(r.x[e] / r.l) : 0.0f;
}

// ... to a chunk's sums, by an M that keeps both of them in fp32: l and the largest of the
// others at equal distances from 1.  Past 2^29 octaves fp32 has no M for that and past 2^30 none
// for the score either: chunks are then weighed by what their largest scores round to.
template <int HD>
__device__ __forceinline__ float2 wide_part(const Wide<HD> &r, float (&x)[HD / 64]) {
  double most = 0.0;
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) most = fmax(most, fabs(r.x[e]));
  most = wave_max_f64(most);
  const bool both = most > 0.0 && r.l > 0.0 && fabs(r.m) < 0x1p29;
  // (past 2^-90 of l the others round to zeros, which is what they are beside it)
  const double by =
      both ? fmin(rint(0.5 * (kVsOctaves - log2(r.l) - log2(most))), 90.0) : 0.0;
  const float m = fabs(r.m) < INFINITY ? (float)rint(r.m - by) : kFloor;
  double up = r.m - (double)m;
  if (!(fabs(up - by) <= 32.0)) up = by;
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) x[e] = (float)(r.x[e] * exp2(up - kVsOctaves));
  return float2{m, (float)(r.l * exp2(up))};
}

// ---- single tokens ------------------------------------------------------------
// A workgroup takes up to 16 query vectors of one sequence and kv head, and a chunk
// of its keys, whose tiles its four waves share out.  Codes go straight from memory
// to registers, a tile (16 KB of 256 dims) ahead of their use.  Bound by the cache's bytes
// where there are many: 32 gemma-3-4b tokens of up to 8192 int8 positions (335 MB) take 75
// us, 4.5 TB/s of the 5.1 that a large copy reaches; two gemma-3-1b ones of 131072 e4m3
// positions (136 MB) 30 us.  256 dims take all of the 256 registers that two workgroups a
// compute unit leave a lane, and 13 to 28 more that wait in scratch, most of them read outside
// the inner loop.  Few keys are a chain of round trips to memory (tables, page ids,
// the query and codes, each about a microsecond) and code fetched cold: one token of 1001
// positions takes 9 to 10 us.

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

template <int HD>
struct StepLds {
  float part[kStepWaves][kStepRows][HD + 4];
  float sm[kStepWaves][kStepRows], sl[kStepWaves][kStepRows];
};

// WHOLE: one chunk and no prefix, so that what comes out is the output.
template <int HD, int TYPE, bool CAP, bool WHOLE>
__device__ __forceinline__ void step_keys(const KvAttn &a, const KvPlan &pl, int chunk, int hk,
                                          int b, StepLds<HD> &lds) {
  constexpr int KS = HD / 32, ND = HD / 16, NJ = HD / 64, VW = HD / 64;
  auto &part = lds.part;
  auto &sm = lds.sm;
  auto &sl = lds.sl;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const KvSeq s = kv_seq(a.b, b);
  const int rows = s.n * pl.group;
  if (s.n == 0 || rows > kStepRows) return;
  const int p0 = s.len - s.n;
  const KvRange kr = key_range(p0, s.len - 1, s.len, a.slide, a.dense, a.shared);
  const int tpc = chunk_tiles(kr.t1 - kr.t0, pl.step_ns);
  const int t0 = kr.t0 + chunk * tpc, t1 = min(kr.t1, t0 + tpc);
  if (t0 >= t1 && chunk > 0) return;

  // the lane's query
  const int j = min(n, rows - 1), row = s.r0 + j / pl.group, head = hk * pl.group + j % pl.group;
  const KvSpan span = kv_span(p0 + j / pl.group, s.len, a.slide, a.dense);
  const KvSee see{max(span.lo, a.shared), span.hi};
  const int f_lo = wave_max_all(see.lo), f_hi = -wave_max_all(-see.hi);
  h8 qhi[KS], qlo[KS];

  v4f o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i] = v4f{};
  Soft soft{kFloor, 0.0f};

  typedef uint32_t vreg __attribute__((ext_vector_type(VW)));
  const uint32_t koff = n * HD + 16 * g, voff = 4 * g * HD + (HD / 16) * n, soff = 16 * g;
  u4 kreg[2][NJ];
  vreg vval[2][4];
  Scales sc;
  auto load_k = [&](const Halves &h) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < NJ; ++i)
        kreg[u][i] = at_offset<u4>(a.c.k + (u ? h.slot1 : h.slot0) * HD + 64 * i, koff);
    }
    sc.k = eight(at_offset<v4f>(a.c.ks + h.slot0, soff), at_offset<v4f>(a.c.ks + h.slot1, soff));
  };
  auto load_v = [&](const Halves &h) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vval[u][i] = at_offset<vreg>(a.c.v + ((u ? h.slot1 : h.slot0) + i) * HD, voff);
    }
    sc.v = eight(at_offset<v4f>(a.c.vs + h.slot0, soff), at_offset<v4f>(a.c.vs + h.slot1, soff));
  };

  int t = t0 + wave;
  if (t < t1) {  // (there may be no page table where there is no key)
    // page ids, then the query, then codes are asked for before the first of them is needed
    Pager pager(a, b, s.len, hk, t, kStepWaves);
    Query<HD> raw;
    raw.load(a.q + (size_t)row * a.q_stride + head * HD, g);
    pager.place(0);
    Halves cur = pager.get(0);
    load_k(cur);
    load_v(cur);
    const Score score(a.asc, a.cap, raw.split(qhi, qlo));
    for (int k = 1; t < t1; t += kStepWaves, ++k) {
      pager.prepare(k);
      const Halves nxt = pager.get(k);  // past the last: of this sequence or page 0, loaded and not used
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
      v4f d[2] = {dh[0] + dl[0], dh[1] + dl[1]};
      Scales now = sc;
      now.v *= kVsUnit;
      __builtin_amdgcn_sched_barrier(0);
      load_k(nxt);
      __builtin_amdgcn_sched_barrier(0);
      const int key0 = kTile * t;
      const bool masked =
          key0 < f_lo || key0 + kTile - 1 > f_hi || cur.ok != 3;  // wave-uniform
      unsigned live = 0xff;
      if (masked) {
        live = seen(key0, g, see, cur.ok);
        // what lies past a sequence's end may be a NaN's code, times a weight of 0
        if (TYPE == kKvE4m3)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (key0 + 16 * (e / 4) + 4 * g + e % 4 >= s.len ||
                !(cur.ok >> (e / 4) & 1))
              vval[e / 4][e % 4] = vreg(0u);
      }
      float lv[8];
      scale_octaves(now.v, lv);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        d[e / 4][e % 4] = score_of<CAP>(d[e / 4][e % 4], now.k[e], score);
      settle(top_of(d, lv, masked, live), soft, [&](float f) {
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= f;
      });
      h8 phi, plo;
#pragma unroll
      for (int j = 0; j < 4; ++j) weigh(j, d, now.v, soft, phi, plo);
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = vval[e / 4][e % 4][w];
        Transposed v;
        each<4>([&](auto J) { transpose_pair<TYPE, J>(x, v); });
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * w + i] = mma(v.dim(i), plo, o[4 * w + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * w + i] = mma(v.dim(i), phi, o[4 * w + i]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_v(nxt);
      cur = nxt;
    }
  }

  // the waves' sums, by the largest M
  soft.l += __shfl_xor(soft.l, 16, 64);
  soft.l += __shfl_xor(soft.l, 32, 64);
  soft.l = marked(a, soft, b, hk, kTile * t0, min(kTile * t1, s.len) - 1);
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
  auto out_of = [&](int q) {
    return a.out + ((size_t)(s.r0 + q / pl.group) * a.n_heads + hk * pl.group + q % pl.group) * HD;
  };
  unsigned again = 0;  // a bit for each query that is done over here
  if (WHOLE) {
    static_assert(kStepWaves * kStepRows == 64, "a lane each");
    const unsigned long long marks = __ballot((&sl[0][0])[lane] == INFINITY);
    again = (unsigned)(marks | marks >> 32);
    again = (again | again >> 16) & ((1u << rows) - 1);
  }
  for (int e = threadIdx.x; e < rows * (HD / 4); e += 64 * kStepWaves) {
    const int q = e / (HD / 4), d = 4 * (e % (HD / 4));
    if (WHOLE && (again >> q & 1)) continue;
    float m = kFloor, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) m = fmaxf(m, sm[w][q]);
    v4f x = {};
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) {
      l += lowered(sl[w][q], sm[w][q] - m);
      x += *reinterpret_cast<const v4f *>(&part[w][q][d]);
    }
    if (WHOLE) {
      *reinterpret_cast<v4f *>(out_of(q) + d) = l != 0.0f ? x / (l * kVsUnit) : v4f{};
    } else {
      const size_t at = (((size_t)b * a.c.nkv + hk) * pl.step_ns + chunk) * pl.step_rows + q;
      *reinterpret_cast<v4f *>((float *)(a.work + pl.step_o) + at * HD + d) = x;
      if (d == 0) ((float2 *)(a.work + pl.step_m))[at] = float2{m, l};
    }
  }
  if (WHOLE && again != 0)
    for (int q = wave; q < rows; q += kStepWaves) {
      if (!(again >> q & 1)) continue;
      const KvSpan sees = kv_span(p0 + q / pl.group, s.len, a.slide, a.dense);
      const float *from = a.q + (size_t)(s.r0 + q / pl.group) * a.q_stride +
                          (hk * pl.group + q % pl.group) * HD;
      wide_out(wide_query<HD, TYPE>(a, b, hk, from, sees.lo, sees.hi), out_of(q));
    }
}

template <int HD, int TYPE, bool CAP, bool WHOLE>
__global__ __launch_bounds__(64 * kStepWaves, 2) void kv_step_kernel(KvAttn a, KvPlan pl) {
  __shared__ StepLds<HD> lds;
  step_keys<HD, TYPE, CAP, WHOLE>(a, pl, blockIdx.x, blockIdx.y, blockIdx.z, lds);
}

// ---- prompt rows and shared prefixes ---------------------------------------------
// A workgroup of NW waves takes 16 NW QB query vectors of a kv head, 16 QB a wave, and a
// chunk of their keys; PRE: the rows of all sequences, over the shared prefix.  Each
// tile's codes are made f16 once, a share by each wave, and reach the others through LDS in
// operand order (16-byte reads of 64 lanes in a row: no conflicts).  128 vectors of 256
// dims are eight waves of 16: two a SIMD hide more of each other's waits than one of 32
// vectors (two 2048-token gemma-3-4b prompts in a window of 1024: 85 us, 93 with four waves, both
// in a kernel trace, under which this kernel takes a tenth longer: calls in turn 75 us).
// Their 4100 cycles a tile are 2050 of products, about 2600 of LDS traffic (every wave
// reads all of a tile's fragments) and 1800 of vector work, which overlap in part; a third
// of the whole is the card's wait for the workgroups that have the most keys.
//
// Tiles are pipelined so that the vector unit works while the matrix cores do: the
// scores of tile t + 1 run with the weights of tile t, the value products of tile t with
// the conversion of K of tile t + 2 and of V of tile t + 1, whose codes were loaded an
// iteration before.  One barrier a tile; K and V each have two buffers.

// A wave's share of a tile: K's half tiles by 64 dims, both of a block or one; 64 dims of
// V or 32, of which a lane transposes VD.
template <int HD, int NW>
struct RowsLds {
  static constexpr int NB = HD / 64;  // blocks of 64 dims
  static_assert(NW == NB || NW == 2 * NB, "shares");
  static constexpr int KS = HD / 32, ND = HD / 16, KU = NW == NB ? 2 : 1, VD = NW == NB ? 4 : 2,
                       VL = VD / 2;
  h8 kf[2][2 * KS][64], vf[2][ND][64];
  v4f scales[4][64];  // of which the first 16 are read; all waves write the same
  u4 raw_k[NW][3][KU][64], raw_v[NW][3][VL][64];
};

// Prompt rows are cut into tiles of tr query vectors, sequence by sequence and the last rows,
// which see most, first.  Where the id-th lies; false past the last.  By each wave, 64
// sequences at a time: a grid of all sequences by the longest one's tiles would be mostly
// workgroups that find nothing to do (a 2048-row prompt beside 200 single tokens: 255 us).
__device__ __forceinline__ bool find_tile(const KvAttn &a, const KvPlan &pl, int tr, int id, int *b,
                                          int *tile) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.b.batch; base += 64) {
    int sum = 0;
    if (base + lane < a.b.batch) {
      const int rows = kv_seq(a.b, base + lane).n * pl.group;
      sum = pl.step && rows <= kStepRows ? 0 : (rows + tr - 1) / tr;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(sum, off, 64);
      if (lane >= off) sum += t;
    }
    const unsigned long long past = __ballot(sum > id);
    if (past != 0) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
      *b = base + l;
      *tile = __builtin_amdgcn_readlane(sum, l) - 1 - id;
      return true;
    }
    id -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// block_x: of nblocks, the chunks of a tile of rows one after the other.
template <int HD, int TYPE, bool CAP, int QB, int NW, bool PRE>
__device__ __forceinline__ void rows_keys(const KvAttn &a, const KvPlan &pl, int block_x,
                                          int nblocks, int hk, RowsLds<HD, NW> &lds) {
  typedef RowsLds<HD, NW> L;
  constexpr int NB = L::NB, KS = L::KS, ND = L::ND, KU = L::KU, VD = L::VD, VL = L::VL;
  constexpr int TR = 16 * NW * QB, VP = 4;  // VP: value fragments read ahead
  constexpr int LOADS = KU + VL + 1;
  auto &kf = lds.kf;
  auto &vf = lds.vf;
  auto &scales = lds.scales;
  auto &raw_k = lds.raw_k;
  auto &raw_v = lds.raw_v;
  const int ns = PRE ? pl.pre_ns : pl.rows_ns;
  const int chunk = block_x % ns;
  int b = 0, tile = nblocks / ns - 1 - block_x / ns;
  if (!PRE && !find_tile(a, pl, TR, block_x / ns, &b, &tile)) return;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  KvSeq s = kv_seq(a.b, b);
  int len = s.len;
  if (PRE) {
    s.r0 = kv_clamp(a.b.row0[0], 0, a.b.rows);
    s.n = kv_clamp(a.b.row0[a.b.batch], s.r0, a.b.rows) - s.r0;
    len = a.shared;
  }
  const int rows = s.n * pl.group, at = tile * TR;
  if (at >= rows) return;

  // the rows' sequences are looked up in LDS, where the table fits: a search in memory is
  // as many round trips as it has steps
  constexpr int kFind = (int)(sizeof(kf) / 4);
  int *const row0 = reinterpret_cast<int *>(&kf[0][0][0]);
  if (PRE && a.b.batch < kFind) {
    for (int i = threadIdx.x; i <= a.b.batch; i += 64 * NW) row0[i] = a.b.row0[i];
    __syncthreads();
  }

  // the lane's queries: loads first
  KvSee see[QB];
  int qrow[QB], qhead[QB];
  Query<HD> raw[QB];
  const int base_row = at / pl.group, base_head = at % pl.group;
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    const int j = base_head + min(16 * (QB * wave + q) + n, rows - 1 - at);
    const int i = (int)((uint32_t)j * pl.inv_group >> 21);  // j / group: j is below group + 128
    qrow[q] = s.r0 + base_row + i;
    qhead[q] = hk * pl.group + j - i * pl.group;
    raw[q].load(a.q + (size_t)qrow[q] * a.q_stride + qhead[q] * HD, g);
  }
  int f_lo = 0, f_hi = INT_MAX;
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    if (PRE) {
      KvSpan span{0, -1};
      const int i = a.b.batch < kFind ? kv_find(row0, a.b.batch, qrow[q])
                                      : kv_find(a.b.row0, a.b.batch, qrow[q]);
      if (i >= 0) {
        const KvSeq o = kv_seq(a.b, i);
        span = kv_span(o.len - o.n + (qrow[q] - o.r0), o.len, a.slide, a.dense);
      }
      see[q] = {span.lo, min(span.hi, a.shared - 1)};
    } else {
      const KvSpan span = kv_span(s.len - s.n + qrow[q] - s.r0, s.len, a.slide, a.dense);
      see[q] = {max(span.lo, a.shared), span.hi};
    }
    f_lo = max(f_lo, see[q].lo);
    f_hi = min(f_hi, see[q].hi);
  }
  h8 qhi[QB][KS], qlo[QB][KS];
  Score score[QB];
  auto split_queries = [&]() {
#pragma unroll
    for (int q = 0; q < QB; ++q) score[q] = Score(a.asc, a.cap, raw[q].split(qhi[q], qlo[q]));
  };
  f_lo = wave_max_all(f_lo);
  f_hi = -wave_max_all(-f_hi);
  if (PRE) __syncthreads();  // the search is over, its table goes
  int t0, t1;
  if (PRE) {  // chunks of the whole prefix
    t0 = chunk * pl.pre_tpc;
    t1 = min(ceil_div(a.shared, kTile), t0 + pl.pre_tpc);
  } else {
    const int i0 = at / pl.group, i1 = min(s.n - 1, (at + TR - 1) / pl.group);
    const KvRange kr = key_range(s.len - s.n + i0, s.len - s.n + i1, s.len, a.slide, a.dense,
                                 a.shared);
    const int tpc = chunk_tiles(kr.t1 - kr.t0, ns);
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
  // Codes wait in LDS, three tiles of them, for the wave that loaded them: in registers, two
  // tiles ahead, they don't fit.
  const int block = wave % NB, part = wave / NB, khalf = KU == 2 ? 0 : part;
  const uint32_t koff = n * HD + 16 * g;
  // row r of 16 lanes' LDS holds key 4 (r % 4) + r / 4, so that the four lane groups, which
  // read keys 4 g + e at a time, meet different banks
  const int vrow = VD == 4 ? lane >> 2 : lane >> 1 & 15;
  const uint32_t voff = (4 * (vrow & 3) + (vrow >> 2)) * HD + 16 * (lane & (VD - 1));
  const uint8_t *const k_base = a.c.k + 64 * block;
  const uint8_t *const v_base = a.c.v + 64 * block + (VD == 4 ? 0 : 32 * part);
  auto load_k = [&](int r, const Halves &h) {  // r: the buffer, tile modulo 3
#pragma unroll
    for (int i = 0; i < KU; ++i) {
      const size_t slot = khalf + i != 0 ? h.slot1 : h.slot0;
      dma16(k_base + slot * HD, koff, raw_k[wave][r][i]);
    }
  };
  auto load_v = [&](int r, size_t slot0, size_t slot1) {
    if constexpr (VD == 4) {
      dma16(v_base + slot0 * HD, voff, raw_v[wave][r][0]);
      dma16(v_base + slot1 * HD, voff, raw_v[wave][r][VL - 1]);
    } else {
      dma16_at(v_base + (lane < 32 ? slot0 : slot1) * HD + voff, raw_v[wave][r][0]);
    }
  };
  const float *const scale_base = (lane & 8 ? a.c.vs : a.c.ks) + 4 * (lane & 3);
  auto load_scales = [&](int t, size_t slot0, size_t slot1) {
    dma16_at(scale_base + (lane & 4 ? slot1 : slot0), scales[t & 3]);
  };
  auto scales_k = [&](int t) { return eight(scales[t & 3][g], scales[t & 3][4 + g]); };
  auto scales_v = [&](int t) {
    return eight(scales[t & 3][8 + g], scales[t & 3][12 + g]) * kVsUnit;
  };
  auto read_k = [&](int r, u4 (&x)[KU]) {
#pragma unroll
    for (int i = 0; i < KU; ++i) x[i] = raw_k[wave][r][i][lane];
  };
  auto store_k = [&](int buf, int i, int half, const u4 (&x)[KU]) {
    kf[buf][(khalf + i) * KS + 2 * block + half][lane] =
        codes8<TYPE>(x[i][2 * half], x[i][2 * half + 1]);
  };
  // A lane of 64 dims: the four of row n of its block's fragments; of 32: two of four, so
  // that lanes n and n + 8 share dims
  const int vquad = VD == 4 ? 4 * (n & 3) + (n >> 2) : n & 7;
  const uint32_t vsel = n < 8 ? kDims01 : kDims23;
  auto read_v = [&](int r, uint32_t (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t *raw = reinterpret_cast<const uint32_t *>(raw_v[wave][r][VD == 4 ? e / 4 : 0]);
      x[e] = VD == 4 ? raw[16 * (4 * (e % 4) + g) + vquad]
                     : raw[8 * (16 * (e / 4) + 4 * (e % 4) + g) + vquad];
    }
  };
  typedef std::conditional_t<VD == 4, Transposed, TransposedHalf> VT;
  auto turn = [&](auto J, const uint32_t (&x)[8], VT &v) {
    if constexpr (VD == 4)
      transpose_pair<TYPE, J>(x, v);
    else
      transpose_pair<TYPE, J>(x, vsel, v);
  };
  const int vfrag = 4 * block + (VD == 4 ? 0 : 2 * (n >> 3));
  const int vlane = VD == 4 ? lane : 16 * g + 4 * (n & 3) + 2 * part + (n >> 2 & 1);
  auto store_v = [&](int buf, int i, const VT &v) { vf[buf][vfrag + i][vlane] = v.dim(i); };
  // what lies past the end may be a NaN's code, times a weight of 0 (ok: bits 0 and 1, the
  // halves that are there)
  auto clear_v = [&](int t, int ok, uint32_t (&x)[8]) {
    if (TYPE != kKvE4m3 || (kTile * (t0 + t) + kTile <= len && (ok & 3) == 3)) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (kTile * (t0 + t) + 16 * (e / 4) + 4 * g + e % 4 >= len || !(ok >> (e / 4) & 1)) x[e] = 0;
  };
  // step i of the scores; f: K's fragments
  auto score_step = [&](auto I, const h8 (&f)[2], v4f (&d)[QB][2]) {
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
      for (int u = 0; u < 2; ++u) d[q][u] = mma(f[u], qlo[q][I], d[q][u]);
#pragma unroll
    for (int q = 0; q < QB; ++q)
#pragma unroll
      for (int u = 0; u < 2; ++u) d[q][u] = mma(f[u], qhi[q][I], d[q][u]);
  };

  if (t0 < t1) {
    Pager pager(a, b, len, hk, t0, 1);  // tiles past the last are loaded and not used
    pager.place(0);
    int there = 0;  // bits 2 i and 2 i + 1: the halves of tile t + i that are there
    size_t v_slot0, v_slot1;  // where tile t + 3 lies
    uint32_t rv[8];  // codes of V of tile t + 1
    {
      const Halves h0 = pager.get(0), h1 = pager.get(1), h2 = pager.get(2), h3 = pager.get(3);
      there = h0.ok | h1.ok << 2 | h2.ok << 4 | h3.ok << 6;
      v_slot0 = h3.slot0;
      v_slot1 = h3.slot1;
      load_k(0, h0);
      load_v(0, h0.slot0, h0.slot1);
      load_scales(0, h0.slot0, h0.slot1);
      load_k(1, h1);
      load_scales(1, h1.slot0, h1.slot1);
      load_k(2, h2);
      load_v(1, h1.slot0, h1.slot1);
      split_queries();
      dma_wait<LOADS - 1>();
      u4 rk[KU];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        read_k(t, rk);
#pragma unroll
        for (int i = 0; i < KU; ++i) {
          store_k(t, i, 0, rk);
          store_k(t, i, 1, rk);
        }
      }
      read_v(0, rv);
      clear_v(0, there, rv);
      VT v;
      each<4>([&](auto J) { turn(J, rv, v); });
      each<VD>([&](auto I) { store_v(0, I, v); });
      lds_barrier();
      load_k(0, h3);
      load_v(2, h2.slot0, h2.slot1);
      load_scales(2, h2.slot0, h2.slot1);
      dma_wait<LOADS>();
      read_v(1, rv);
    }
    v4f d[QB][2] = {};
    each<KS>([&](auto I) {
      const h8 f[2] = {kf[0][I][lane], kf[0][KS + I][lane]};
      score_step(I, f, d);
    });
    float top[QB];
    v8f vs = scales_v(0);
    {
      const v8f ks = scales_k(0);
      float lv[8];
      scale_octaves(vs, lv);
#pragma unroll
      for (int q = 0; q < QB; ++q) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          d[q][e / 4][e % 4] = score_of<CAP>(d[q][e / 4][e % 4], ks[e], score[q]);
        top[q] = top_of(d[q], lv, false, 0);
      }
    }
    lds_barrier();
    int t = 0, r = 0;  // the tile, from t0 on; its number modulo 3
    // Hides what queries of tile t don't see; whether some query's M has to move.  That
    // rarely happens, and lies outside the inner loop: in it the value sums are touched by
    // the matrix cores alone and stay in the accumulation registers.
    auto begin = [&]() {
      int key0 = kTile * (t0 + t);
      pager.prepare(t + 4);
      if (key0 < f_lo || key0 + kTile - 1 > f_hi || (there & 3) != 3) {  // wave-uniform
        asm volatile("" : "+s"(key0));  // the compiler would have all tiles work out the masks
        float lv[8];
        scale_octaves(vs, lv);
#pragma unroll
        for (int q = 0; q < QB; ++q)
          top[q] = top_of(d[q], lv, true, seen(key0, g, see[q], there));
      }
      clear_v(t + 1, there >> 2, rv);
      bool moves = false;
#pragma unroll
      for (int q = 0; q < QB; ++q) moves = moves || top[q] > soft[q].m + kSlack;
      return __any(moves);
    };
    // One tile.  Each chunk of products takes its share of the vector work; what a later
    // chunk reads from LDS is asked for one or two chunks before.
    auto tile = [&]() {
      const int cur = t & 1, nxt = cur ^ 1, r1 = r == 2 ? 0 : r + 1, r2 = 3 - r - r1;
      h8 phi[QB], plo[QB], kpre[2] = {kf[nxt][0][lane], kf[nxt][KS][lane]}, vpre[VP];
      v4f dn[QB][2] = {};
      u4 rk[KU];
      v8f ks, vn;
      VT v;
      const Halves h4 = pager.get(t + 4);
      // scores of tile t + 1; weights of tile t, V of tile t + 1, loads of tiles t + 3 and
      // t + 4 (into the buffers that the iteration before was done with)
      each<KS>([&](auto I) {
        constexpr int i = I;
        const h8 f[2] = {kpre[0], kpre[1]};
        if constexpr (i + 1 < KS) {
          kpre[0] = kf[nxt][i + 1][lane];
          kpre[1] = kf[nxt][KS + i + 1][lane];
        } else {
          read_k(r2, rk);
          each<VP>([&](auto V) { vpre[V] = vf[cur][V][lane]; });
          ks = scales_k(t + 1);
          vn = scales_v(t + 1);
        }
        score_step(I, f, dn);
        constexpr int j0 = 4 * QB * i / KS, j1 = 4 * QB * (i + 1) / KS;
        each<j1 - j0>([&](auto J) {
          constexpr int j = j0 + J, q = j / 4;
          weigh(j % 4, d[q], vs, soft[q], phi[q], plo[q]);
        });
        if constexpr (KS == 8) {
          if constexpr (i < 4)
            turn(I, rv, v);
          else if constexpr (i - 4 < VD)
            store_v(nxt, i - 4, v);
        } else {
          turn(I, rv, v);
          if constexpr (i == KS - 1) each<VD>([&](auto D) { store_v(nxt, D, v); });
        }
        if constexpr (i == KS / 2 - 1) load_k(r1, h4);
        if constexpr (i == KS / 2) load_v(r, v_slot0, v_slot1);
        if constexpr (i == KS / 2 + 1) load_scales(t + 3, v_slot0, v_slot1);
        __builtin_amdgcn_sched_barrier(0);
      });
      // value products of tile t; scores and K of tiles t + 1 and t + 2
      constexpr int NC = ND / 2;  // chunks of two blocks of dims
      float lv[8];
      each<NC>([&](auto I) {
        constexpr int i = I;
        const h8 f[2] = {vpre[2 * i % VP], vpre[(2 * i + 1) % VP]};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * i + e + VP < ND) vpre[(2 * i + e) % VP] = vf[cur][2 * i + e + VP][lane];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int q = 0; q < QB; ++q) o[q][2 * i + e] = mma(f[e], plo[q], o[q][2 * i + e]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int q = 0; q < QB; ++q) o[q][2 * i + e] = mma(f[e], phi[q], o[q][2 * i + e]);
        if constexpr (i == 0) scale_octaves(vn, lv);
        constexpr int k0 = 2 * KU * i / NC, k1 = 2 * KU * (i + 1) / NC;
        each<k1 - k0>([&](auto J) {
          constexpr int j = k0 + J;
          store_k(cur, j / 2, j % 2, rk);
        });
        constexpr int e0 = i > 0 ? 8 * QB * (i - 1) / (NC - 1) : 0, e1 = 8 * QB * i / (NC - 1);
        each<e1 - e0>([&](auto E) {
          constexpr int e = (e0 + E) % 8, q = (e0 + E) / 8;
          float x = score_of<CAP>(dn[q][e / 4][e % 4], ks[e], score[q]);
          asm volatile("" : "+v"(x));  // here, not behind the barrier
          d[q][e / 4][e % 4] = x;
          top[q] = e == 0 ? x + lv[e] : fmaxf(top[q], x + lv[e]);
        });
        if constexpr (i == NC - 2) {
          // what was loaded an iteration ago is in
          dma_wait<LOADS>();
          read_v(r2, rv);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
#pragma unroll
      for (int q = 0; q < QB; ++q) asm volatile("" : "+v"(top[q]));
      vs = vn;
      there = there >> 2 | h4.ok << 6;
      v_slot0 = h4.slot0;
      v_slot1 = h4.slot1;
      r = r1;
      lds_barrier();
    };
    const int nt = t1 - t0;
    begin();
    for (;;) {
#pragma unroll
      for (int q = 0; q < QB; ++q)
        settle(top[q], soft[q], [&](float f) {
#pragma unroll
          for (int i = 0; i < ND; ++i) o[q][i] *= f;
        });
      bool moves = false;
      do {
        tile();
        if (++t == nt) break;
        moves = begin();
      } while (!moves);
      if (t == nt) break;
    }
  }
#pragma unroll
  for (int q = 0; q < QB; ++q) {
    soft[q].l += __shfl_xor(soft[q].l, 16, 64);
    soft[q].l += __shfl_xor(soft[q].l, 32, 64);
    soft[q].l = marked(a, soft[q], b, hk, kTile * t0, min(kTile * t1, len) - 1);
    const bool there = at + 16 * (QB * wave + q) + n < rows;
    const bool whole = !PRE && ns == 1 && pl.pre_ns == 0;
    unsigned again = 0;  // a bit for each query that is done over here
    if (!PRE && whole) again = (unsigned)__ballot(there && soft[q].l == INFINITY) & 0xffff;
    if (there && !(again >> n & 1)) {
      const size_t vec = (size_t)qrow[q] * a.n_heads + qhead[q];
      const size_t pt = (size_t)chunk * a.b.rows * a.n_heads + vec;
      float *dst = whole ? a.out + vec * HD
                         : (float *)(a.work + (PRE ? pl.pre_o : pl.rows_o)) + pt * HD;
      const float f = !whole ? 1.0f : soft[q].l != 0.0f ? 1.0f / (soft[q].l * kVsUnit) : 0.0f;
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
    for (; again != 0; again &= again - 1) {
      const int i = __ffs(again) - 1;
      const size_t row = __builtin_amdgcn_readlane(qrow[q], i);
      const int head = __builtin_amdgcn_readlane(qhead[q], i);
      wide_out(wide_query<HD, TYPE>(a, b, hk, a.q + row * a.q_stride + head * HD,
                                    __builtin_amdgcn_readlane(see[q].lo, i),
                                    __builtin_amdgcn_readlane(see[q].hi, i)),
               a.out + (row * a.n_heads + head) * HD);
    }
  }
}

template <int HD, int TYPE, bool CAP, int QB, int NW, bool PRE>
__global__ __launch_bounds__(64 * NW) void kv_rows_kernel(KvAttn a, KvPlan pl) {
  __shared__ RowsLds<HD, NW> lds;
  rows_keys<HD, TYPE, CAP, QB, NW, PRE>(a, pl, blockIdx.x, gridDim.x, blockIdx.y, lds);
}

// The shared prefix and what single tokens' sequences have of their own in one launch: each
// leaves most of its time to latencies, and neither fills the card for long.  The prefix's
// workgroups, which take longest, come first.
template <int HD, int TYPE, bool CAP>
__global__ __launch_bounds__(64 * kStepWaves) void kv_both_kernel(KvAttn a, KvPlan pl) {
  constexpr int NW = kStepWaves;
  __shared__ union {
    RowsLds<HD, NW> rows;
    StepLds<HD> step;
  } lds;
  const int blocks = pl.pre_blocks * pl.pre_ns, id = blockIdx.x;
  if (id < blocks * a.c.nkv) {
    rows_keys<HD, TYPE, CAP, 1, NW, true>(a, pl, id % blocks, blocks, id / blocks, lds.rows);
  } else {
    const int i = id - blocks * a.c.nkv;  // one chunk
    step_keys<HD, TYPE, CAP, false>(a, pl, 0, i % a.c.nkv, i / a.c.nkv, lds.step);
  }
}

// ---- the chunks' sums together ------------------------------------------------------
// SHARE waves take a query vector and share out its chunks; STEP: vectors of single tokens,
// else of prompt rows, which may have very different numbers of both.  Bound by the partial
// sums' bytes where there are many vectors.

constexpr int kMergeWaves = 4;  // of a workgroup, at least

template <int HD, int TYPE, int SHARE, bool STEP>
__global__ __launch_bounds__(64 * (SHARE > kMergeWaves ? SHARE : kMergeWaves)) void kv_merge_kernel(
    KvAttn a, KvPlan pl) {
  constexpr int E = HD / 64, W = SHARE > kMergeWaves ? SHARE : kMergeWaves;
  __shared__ float so[SHARE][HD], sm[SHARE], sl[SHARE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % SHARE;
  // single tokens: of sequence blockIdx.y; prompt rows: of all sequences, one after the other
  const int v = blockIdx.x * (W / SHARE) + wave / SHARE, head = v % a.n_heads;
  const int b = STEP ? blockIdx.y : kv_find_wave(a.b, v / a.n_heads);
  const KvSeq s = kv_seq(a.b, b);
  const int i = v / a.n_heads - (STEP ? 0 : s.r0);
  const bool step = pl.step && s.n * pl.group <= kStepRows;
  if (i < 0 || i >= s.n || step != STEP) return;  // (a whole workgroup's, where its waves share)
  const int hk = head / pl.group, j = i * pl.group + head % pl.group, p0 = s.len - s.n;
  const size_t vec = (size_t)(s.r0 + i) * a.n_heads + head;
  // this row's own chunks: number, first partial and the step to the next; their tiles
  int n, t0, tpc;
  size_t first, stride;
  const float *po;
  const float2 *pm;
  if (STEP) {
    const KvRange kr = key_range(p0, s.len - 1, s.len, a.slide, a.dense, a.shared);
    tpc = chunk_tiles(kr.t1 - kr.t0, pl.step_ns);
    t0 = kr.t0;
    n = max(1, ceil_div(kr.t1 - kr.t0, tpc));
    first = ((size_t)b * a.c.nkv + hk) * pl.step_ns * pl.step_rows + j;
    stride = pl.step_rows;
    po = (const float *)(a.work + pl.step_o);
    pm = (const float2 *)(a.work + pl.step_m);
  } else {
    const int tr = 64 * pl.qb, at = j / tr * tr;
    const int i0 = at / pl.group, i1 = min(s.n - 1, (at + tr - 1) / pl.group);
    const KvRange kr = key_range(p0 + i0, p0 + i1, s.len, a.slide, a.dense, a.shared);
    tpc = chunk_tiles(kr.t1 - kr.t0, pl.rows_ns);
    t0 = kr.t0;
    n = max(1, ceil_div(kr.t1 - kr.t0, tpc));
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
  auto add = [&](float2 v, const float (&y)[E]) {
    const float mn = fmaxf(m, v.x);
    const float f = __builtin_amdgcn_exp2f(m - mn), h = __builtin_amdgcn_exp2f(v.x - mn);
    l = lowered(l, m - mn) + lowered(v.y, v.x - mn);
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] * f + y[e] * h;
  };
  constexpr int A = SHARE == 16 ? 8 : 4;  // chunks loaded at a time
  for (int c = part; c < total; c += A * SHARE) {
    float2 v[A];
    float y[A][E];
#pragma unroll
    for (int u = 0; u < A; ++u) {
      if (c + u * SHARE >= total) break;
      const float *o;
      v[u] = where(c + u * SHARE, &o);
#pragma unroll
      for (int e = 0; e < E; ++e) y[u][e] = o[E * lane + e];
    }
#pragma unroll
    for (int u = 0; u < A; ++u) {
      if (c + u * SHARE >= total) break;
      add(v[u], y[u]);
    }
  }
  if (__any(!(l < INFINITY))) {  // some chunk is to be done over: all once more
    m = kFloor;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.0f;
    const float *from = a.q + (size_t)(s.r0 + i) * a.q_stride + head * HD;
    const KvSpan sees = kv_span(p0 + i, s.len, a.slide, a.dense);
    for (int c = part; c < total; c += SHARE) {
      const float *o;
      float2 v = where(c, &o);
      float y[E];
      if (v.y == INFINITY) {
        const bool own = c < n;
        const int first = kTile * (own ? t0 + c * tpc : (c - n) * pl.pre_tpc);
        const int lo = max(own ? max(sees.lo, a.shared) : sees.lo, first);
        const int hi = min(own ? sees.hi : min(sees.hi, a.shared - 1),
                           first + kTile * (own ? tpc : pl.pre_tpc) - 1);
        v = wide_part(wide_query<HD, TYPE>(a, own ? b : 0, hk, from, lo, hi), y);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = o[E * lane + e];
      }
      add(v, y);
    }
  }
  if constexpr (SHARE == 1) {
    const float unit = l * kVsUnit;
#pragma unroll
    for (int e = 0; e < E; ++e) a.out[vec * HD + E * lane + e] = l != 0.0f ? x[e] / unit : 0.0f;
  } else {
    if (lane == 0) {
      sm[part] = m;
      sl[part] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) so[part][E * lane + e] = x[e];
    __syncthreads();
    if (threadIdx.x >= HD) return;
    float mm = kFloor, ll = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < SHARE; ++w) mm = fmaxf(mm, sm[w]);
#pragma unroll
    for (int w = 0; w < SHARE; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w] - mm);
      ll += lowered(sl[w], sm[w] - mm);
      sum += so[w][threadIdx.x] * f;
    }
    a.out[vec * HD + threadIdx.x] = ll != 0.0f ? sum / (ll * kVsUnit) : 0.0f;
  }
}

KvPlan plan(const KvAttn &a, const DeviceInfo &dev) {
  KvPlan p{};
  p.group = a.n_heads / a.c.nkv;
  p.inv_group = ((1 << 21) + p.group - 1) / p.group;
  const int most = a.b.max_rows * p.group;  // query vectors of a sequence and kv head
  // (a batch whose rows add up to max_rows of each has no single tokens)
  p.step = p.group <= kStepRows &&
           (most <= kStepRows || a.b.rows < (long)a.b.batch * a.b.max_rows);
  const bool rows = !p.step || most > kStepRows;
  // tiles that a sequence's rows see behind the prefix: by the window where there is one
  const int own = a.b.max_len - a.shared;
  auto tiles = [&](int n) {  // n neighbouring rows
    const int keys = a.slide > 0 ? (int)std::min<long>(own, (long)a.slide + n) : own;
    return std::max(1, ceil_div(keys, kTile) + 1);
  };
  // chunks: so many, if there are tiles enough
  auto cut = [](int tiles, int ns) {
    return std::max(1, std::min({ns, ceil_div(tiles, kChunkTiles), 256}));
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
    // two workgroups a compute unit are resident: more than that is rounds of them.  32
    // sequences of up to 8192 keys and 4 kv heads: 72 us with 2, 73 with 1, 82 with 4
    // ... and few keys are one chunk, without a merge: a tile more a wave is 0.85 us of 256 dims,
    // the merge about 2.  A token over 200 positions 10.2 us and 10.7 (split), over 330 11.8
    // and 11.2; of 128 dims over 330 7.2 and 7.8, over 460 8.1 and 7.6 (int8; e4m3 7.5 and 7.7)
    const bool few = tiles(n) * a.c.hdim <= 8 * 256;
    p.step_ns = cut(tiles(n), few ? 1 : 2 * dev.cus / std::max(1, a.b.batch * a.c.nkv));
  }
  const long vecs_kv = (long)a.b.rows * p.group;  // query vectors of a kv head
  auto blocks = [&](int qb) {
    return (int)std::max<long>(1, (vecs_kv + 64 * qb - 1) / (64 * qb)) * a.c.nkv;
  };
  // (All figures are of 256 dims; 128 take the same rules, not measured on both sides, though two
  // of their workgroups of 64 vectors fit a compute unit.)
  // A workgroup of 128 vectors of 256 dims takes 4100 cycles a tile and 25000 to begin, one
  // of 64 3000 and 16000, and writes half as much for the merge where there are chunks:
  // short runs take 64.  gemma-3-1b behind 16384 positions, merge included: 256 vectors (8
  // tiles by 64 vectors a compute unit) 30 us with 64 and 35 with 128, 512 vectors (16) 42
  // and 42; a 613-row chunk (10) 39 and 44, 1024 rows of gemma-3-4b (16) 46 and 44
  auto block_rows = [&](int tiles) {
    return vecs_kv > 64 && (long)blocks(1) * tiles > (long)kLongRun * dev.cus ? 2 : 1;
  };
  const int own_tiles = tiles(std::min(a.b.max_rows, kStepRows / std::min(p.group, kStepRows)));
  auto rows_tiles = [&](int qb) { return tiles(ceil_div(64 * qb, p.group) + 1); };
  p.qb = block_rows(rows_tiles(1));
  if (rows) p.rows_ns = cut(rows_tiles(p.qb), dev.cus / blocks(p.qb));
  if (a.shared > 0) {
    const int all = ceil_div(a.shared, kTile);
    p.pre_qb = block_rows(all);
    int ns = cut(all, dev.cus / blocks(p.pre_qb));
    const long seqs = (long)a.b.batch * a.c.nkv;
    if (p.step && !rows && p.pre_qb == 1 && own_tiles <= kBothTiles && seqs <= 2 * dev.cus) {
      // One launch for both, one workgroup a compute unit at a time.  In 1000 cycles a
      // prefix's takes 16 and 3 a tile, a sequence's (in one chunk) 18 and 1 / 2: chunks such
      // that the sequences find room beside the prefix
      long best = LONG_MAX;
      for (int n = 1, most_ns = ns; n <= most_ns; ++n) {
        const long room = dev.cus - (long)n * blocks(1), pre = 16 + 3 * ceil_div(all, n);
        const long step = 18 + own_tiles / 2;
        const long t = room > 0 ? std::max(pre, (seqs + room - 1) / room * step)
                                : pre + (seqs + dev.cus - 1) / dev.cus * step;
        if (t < best) {
          best = t;
          ns = n;
        }
      }
      p.pre_blocks = blocks(1) / a.c.nkv;
      p.step_ns = 1;
    }
    p.pre_tpc = ceil_div(all, ns);
    p.pre_ns = ceil_div(all, p.pre_tpc);
  }
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
  return p;
}

// Waves share a vector where it has many chunks: 2452 vectors of 6 chunks take 6.5 us with a
// wave each and 8.4 with four, 256 of 64 chunks 6.1 with 16.
template <int HD, int TYPE, bool STEP>
void launch_merge(const KvAttn &a, const KvPlan &p, int chunks, int rows, hipStream_t stream) {
  const int vecs = rows * a.n_heads, batch = STEP ? a.b.batch : 1;
  if (chunks > 16)
    kv_merge_kernel<HD, TYPE, 16, STEP><<<dim3(vecs, batch), 1024, 0, stream>>>(a, p);
  else if (chunks > 8)
    kv_merge_kernel<HD, TYPE, 4, STEP><<<dim3(vecs, batch), 64 * kMergeWaves, 0, stream>>>(a, p);
  else if (chunks > 1)
    kv_merge_kernel<HD, TYPE, 1, STEP>
        <<<dim3(ceil_div(vecs, kMergeWaves), batch), 64 * kMergeWaves, 0, stream>>>(a, p);
}

// 64 B query vectors a workgroup.
template <int HD, int TYPE, bool CAP, int B, bool PRE>
void launch_rows(const KvAttn &a, const KvPlan &p, hipStream_t stream) {
  constexpr int NW = B == 2 && HD == 256 ? 8 : 4, QB = B * 4 / NW;
  const int vecs = a.b.rows * p.group;
  // tiles: one more than the whole ones for each sequence, of which there are so many
  const int tiles = PRE ? ceil_div(vecs, 64 * B)
                        : vecs / (64 * B) +
                              std::min(a.b.batch, vecs / (p.step ? kStepRows + 1 : p.group));
  if (tiles > 0)
    kv_rows_kernel<HD, TYPE, CAP, QB, NW, PRE>
        <<<dim3(tiles * (PRE ? p.pre_ns : p.rows_ns), a.c.nkv), 64 * NW, 0, stream>>>(a, p);
}

template <int HD, int TYPE, bool CAP>
void launch_typed(const KvAttn &a, const KvPlan &p, hipStream_t stream) {
  const int nkv = a.c.nkv, batch = a.b.batch;
  if (p.pre_blocks > 0)
    kv_both_kernel<HD, TYPE, CAP>
        <<<(p.pre_blocks * p.pre_ns + batch) * nkv, 64 * kStepWaves, 0, stream>>>(a, p);
  else if (p.step && p.step_ns == 1 && p.pre_ns == 0)
    kv_step_kernel<HD, TYPE, CAP, true>
        <<<dim3(1, nkv, batch), 64 * kStepWaves, 0, stream>>>(a, p);
  else if (p.step)
    kv_step_kernel<HD, TYPE, CAP, false>
        <<<dim3(p.step_ns, nkv, batch), 64 * kStepWaves, 0, stream>>>(a, p);
  if (p.rows_ns > 0) {
    if (p.qb == 2)
      launch_rows<HD, TYPE, CAP, 2, false>(a, p, stream);
    else
      launch_rows<HD, TYPE, CAP, 1, false>(a, p, stream);
  }
  if (p.pre_ns > 0 && p.pre_blocks == 0) {
    if (p.pre_qb == 2)
      launch_rows<HD, TYPE, CAP, 2, true>(a, p, stream);
    else
      launch_rows<HD, TYPE, CAP, 1, true>(a, p, stream);
  }
  if (p.step)
    launch_merge<HD, TYPE, true>(a, p, p.step_ns + p.pre_ns,
                                 std::min(a.b.max_rows, kStepRows / p.group), stream);
  if (p.rows_ns > 0) launch_merge<HD, TYPE, false>(a, p, p.rows_ns + p.pre_ns, a.b.rows, stream);
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
