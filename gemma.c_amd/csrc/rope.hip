// rope.hip -- rotary positions, by themselves and on the way into the paged cache.
//
// Pair j of a head's first `rot` values (x, y) becomes (x c - y s, y c + x s), c and s amp times
// the cosine and sine of pos f_j; the others stay.  Before that comes, if asked for, the head's
// norm x / sqrt(mean x^2 + eps) (w + 1).  Both in fp64, rounded to fp32 once: a far position's
// angle needs more than fp32.  What is off before that is 1e-15 of the head's largest value and
// the rounding of pos f_j, 2^-53 of the angle: up to 7e-12 by position 131071.  The keys' codes that
// follow are the exact ones but where a border between two codes is hit to that (an fp32 rounding
// in between moves one in 10^5).
//
// Few rows, and heads of any size: a head is hdim / 4 lanes' (16, 32 or 64 of them), four values a
// lane: pairs 2l and 2l + 1 of lane l, then what doesn't turn.
//
// Many rows of heads of 64, 128 or 256 values: a row is hdim / 16 lanes', which take one head after
// the other and have all the angles of their values from the start.  That is a quarter of the sums
// over lanes, scales and addresses: 16 values a lane instead of 4.  9342 rows of 8 + 4 + 4 heads of
// 256 (249 MB) take 59 us, 4.2 TB/s, with 76 vector instructions a head; with 4 values a lane
// 199, which bounded it (66 us).  Other heads and rotations take four values a lane however many rows
// there are, 24 or 18 of 32 lanes at work for heads of 96 or 72: 4096 rows of 16 heads 13 us (96, 50
// MB) and 12 (72, 38 MB).
#include <type_traits>

#include "dec_common.h"
#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kThreads = 256;

typedef float v2f __attribute__((ext_vector_type(2)));

// Sum and largest over each aligned group of G lanes, the same in all of them.
template <int G>
__device__ __forceinline__ double group_sum_f64(double v) {
  if (G == 64) return wave_sum_f64(v);
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  v += dpp_f64<kDppMirror>(v);
  if (G == 32) v += __shfl_xor(v, 16, 64);
  return v;
}
template <int G>
__device__ __forceinline__ int group_max_i32(int v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  return v;
}

template <int CTRL>
__device__ __forceinline__ int dpp_i32(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}

// 1 / sqrt(v) for v > 0: the instruction's approximation and a step of third order
__device__ __forceinline__ double rsqrt_f64(double v) {
  const double y = __builtin_amdgcn_rsq(v);
  const double e = fma(-v * y, y, 1.0);
  return v < INFINITY ? fma(y * e, fma(e, 0.375, 0.5), y) : y;
}

// Cosine and sine of an angle of up to some 2^40, to fp64 rounding: the nearest multiple of pi/2
// taken off (in two parts), Taylor polynomials of degree 15 and 16 on what is left, at most pi/4
// (the terms left out are below 7e-17).
__device__ __forceinline__ void cos_sin(double angle, double *c, double *s) {
  const double shift = fma(angle, 0x1.45f306dc9c883p-1, 0x1.8p52);  // 2 / pi
  const double k = shift - 0x1.8p52;
  double r = fma(-k, 0x1.921fb54442d18p0, angle);
  r = fma(-k, 0x1.1a62633145c07p-54, r);
  const double z = r * r;
  double p = fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0);
  p = fma(z, p, -1.0 / 39916800.0);
  p = fma(z, p, 1.0 / 362880.0);
  p = fma(z, p, -1.0 / 5040.0);
  p = fma(z, p, 1.0 / 120.0);
  p = fma(z, p, -1.0 / 6.0);
  const double sine = fma(r * z, p, r);
  double q = fma(z, 1.0 / 20922789888000.0, -1.0 / 87178291200.0);
  q = fma(z, q, 1.0 / 479001600.0);
  q = fma(z, q, -1.0 / 3628800.0);
  q = fma(z, q, 1.0 / 40320.0);
  q = fma(z, q, -1.0 / 720.0);
  q = fma(z, q, 1.0 / 24.0);
  q = fma(z, q, -0.5);
  const double cosine = fma(z, q, 1.0);
  const int turn = (int)__double_as_longlong(shift) & 3;
  const double a = turn & 1 ? sine : cosine, b = turn & 1 ? cosine : sine;
  *c = turn == 1 || turn == 2 ? -a : a;
  *s = turn & 2 ? -b : b;
}

// Where a lane's four values lie in its head: two and two neighbours at `a` and `b`, or, with
// PAIRS, four from `a`; turns: they are pairs f and f + 1.
struct Place {
  int a, b, f;
  bool there, turns;
};
template <bool PAIRS>
__device__ __forceinline__ Place place_of(int lane, int hdim, int rot) {
  Place p;
  p.there = 4 * lane < hdim;
  p.turns = 4 * lane < rot;
  p.f = 2 * lane;
  p.a = PAIRS ? 4 * lane : p.turns ? 2 * lane : 4 * lane;
  p.b = PAIRS ? 4 * lane + 2 : p.turns ? rot / 2 + 2 * lane : 4 * lane + 2;
  return p;
}

// x[0], x[2] and x[1], x[3] are the lane's pairs
template <bool PAIRS>
__device__ __forceinline__ void head_load(const float *p, const Place &at, float (&x)[4]) {
  if (PAIRS) {
    const v4f v = *reinterpret_cast<const v4f *>(p + at.a);
    x[0] = v[0], x[2] = v[1], x[1] = v[2], x[3] = v[3];
  } else {
    const v2f a = *reinterpret_cast<const v2f *>(p + at.a);
    const v2f b = *reinterpret_cast<const v2f *>(p + at.b);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  }
}
template <bool PAIRS>
__device__ __forceinline__ void head_store(float *p, const Place &at, const float (&x)[4]) {
  if (PAIRS) {
    *reinterpret_cast<v4f *>(p + at.a) = v4f{x[0], x[2], x[1], x[3]};
  } else {
    *reinterpret_cast<v2f *>(p + at.a) = v2f{x[0], x[1]};
    *reinterpret_cast<v2f *>(p + at.b) = v2f{x[2], x[3]};
  }
}

// A lane's cosines and sines at a position.
struct Turn {
  double c[2], s[2];
};
__device__ __forceinline__ Turn turn_at(const Rotary &r, const Place &at, const double (&f)[2],
                                        int pos) {
  Turn t = {{1.0, 1.0}, {0.0, 0.0}};
  if (!at.turns) return t;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    double angle = f[e] * (double)pos;
    if (r.angle32) angle = (double)((float)f[e] * (float)pos);
    cos_sin(angle, &t.c[e], &t.s[e]);
    if (r.angle32) t.c[e] = (double)(float)t.c[e], t.s[e] = (double)(float)t.s[e];
    t.c[e] *= (double)r.amp;
    t.s[e] *= (double)r.amp;
  }
  return t;
}

// The norm (weights w1 are w + 1), where the lane's group has one (some: any group has), and the
// turn of a lane's values.
template <int G>
__device__ __forceinline__ void head_turn(float (&x)[4], bool some, bool norm,
                                          const double (&w1)[4], int hdim, float eps, bool turns,
                                          const Turn &t) {
  double d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] = (double)x[e];
  if (some) {
    const double ss = fma(d[0], d[0], d[1] * d[1]) + fma(d[2], d[2], d[3] * d[3]);
    const double m = rsqrt_f64(fma(group_sum_f64<G>(ss), 1.0 / (double)hdim, (double)eps));
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = norm ? d[e] * (m * w1[e]) : d[e];
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const double a = d[e], b = d[e + 2];
    x[e] = (float)(turns ? a * t.c[e] - b * t.s[e] : a);
    x[e + 2] = (float)(turns ? b * t.c[e] + a * t.s[e] : b);
  }
}

template <bool PAIRS>
__device__ __forceinline__ void weights_load(const float *w, const Place &at, double (&w1)[4]) {
  float x[4] = {};
  if (w != nullptr && at.there) head_load<PAIRS>(w, at, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) w1[e] = (double)x[e] + 1.0;
}
__device__ __forceinline__ void freq_load(const Rotary &r, const Place &at, double (&f)[2]) {
  f[0] = f[1] = 0.0;
  if (at.turns) f[0] = r.freq[at.f], f[1] = r.freq[at.f + 1];
}

// H heads of a row for each group of G lanes; a wave's groups take neighbouring ones
template <int G, bool PAIRS, int H>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeRows a) {
  constexpr int PER = 64 / G * H;  // heads of a wave
  const int lane = threadIdx.x % G, group = threadIdx.x % 64 / G;
  const int parts = (a.heads + PER - 1) / PER;
  const long unit = (long)blockIdx.x * (kThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r = (int)(unit / parts), h0 = (int)(unit % parts) * PER + group;
  if (r >= a.rows) return;
  const Place at = place_of<PAIRS>(lane, a.hdim, a.rot.rot);
  float x[H][4];
#pragma unroll
  for (int j = 0; j < H; ++j) {
    const int h = min(h0 + j * (64 / G), a.heads - 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[j][e] = 0.0f;
    if (at.there) head_load<PAIRS>(a.src + r * a.src_stride + h * a.hdim, at, x[j]);
  }
  double w1[4], f[2];
  weights_load<PAIRS>(a.w, at, w1);
  freq_load(a.rot, at, f);
  const Turn t = turn_at(a.rot, at, f, a.pos[r]);
#pragma unroll
  for (int j = 0; j < H; ++j) {
    const int h = h0 + j * (64 / G);
    head_turn<G>(x[j], a.w != nullptr, a.w != nullptr, w1, a.hdim, a.eps, at.turns, t);
    if (at.there && h < a.heads)
      head_store<PAIRS>(a.dst + r * a.dst_stride + h * a.hdim, at, x[j]);
  }
}

// A head of a row, its values at their places in x, as codes and a scale: cache_write's arithmetic.
template <int G, int TYPE, bool PAIRS>
__device__ __forceinline__ void head_code(const KvCache &c, bool isv, long slot, const Place &at,
                                          const float (&x)[4], int lane) {
  int top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_int(x[e]) & 0x7fffffff);
  top = group_max_i32<G>(top);
  if (slot < 0) return;
  const bool finite = top < 0x7f800000;
  const float amax = finite ? daz(__int_as_float(top)) : 0.0f;
  uint32_t q = 0;  // codes of x[0], x[1], x[2], x[3]
  float scale = 0.0f;
  if (amax > 0.0f) {
    if (TYPE == kKvI8) {
      const QuantParams qp = quant_params(amax);
      scale = qp.scale;
      q = pack4(quant_one(x[0], qp.inv), quant_one(x[1], qp.inv), quant_one(x[2], qp.inv),
                quant_one(x[3], qp.inv));
    } else {
      scale = mul_ftz(amax, 1.0f / 448.0f);
      const float inv = (float)(448.0 / (double)amax);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaxf(-448.0f, fminf(448.0f, daz(x[e]) * inv));
      const int t = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      q = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], t, true);
    }
  }
  uint8_t *dst = (isv ? c.v : c.k) + (size_t)slot * (4 * G);
  if (PAIRS) {
    *reinterpret_cast<uint32_t *>(dst + at.a) = __builtin_amdgcn_perm(q, q, 0x03010200u);
  } else {
    *reinterpret_cast<uint16_t *>(dst + at.a) = (uint16_t)q;
    *reinterpret_cast<uint16_t *>(dst + at.b) = (uint16_t)(q >> 16);
  }
  if (lane == 0) (isv ? c.vs : c.ks)[slot] = finite ? scale : __int_as_float(0x7fc00000);
}

// H of a row's heads (q's, then k's, then v's) for each group of G lanes
template <int G, int TYPE, bool PAIRS, int H>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppend a) {
  constexpr int PER = 64 / G * H, HD = 4 * G;
  const int lane = threadIdx.x % G, group = threadIdx.x % 64 / G;
  const int nq = a.q != nullptr ? a.n_heads : 0, nk = a.c.nkv, all = nq + 2 * nk;
  const int parts = (all + PER - 1) / PER;
  const long unit = (long)blockIdx.x * (kThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r = (int)(unit / parts), h0 = (int)(unit % parts) * PER + group;
  if (r >= a.b.rows) return;
  const Place at = place_of<PAIRS>(lane, HD, a.rot.rot);
  float x[H][4];
#pragma unroll
  for (int j = 0; j < H; ++j) {
    const int h = min(h0 + j * (64 / G), all - 1);
    const float *row = h < nq        ? a.q + r * a.q_stride + h * HD
                       : h < nq + nk ? a.k + r * a.k_stride + (h - nq) * HD
                                     : a.v + r * a.v_stride + (h - nq - nk) * HD;
    head_load<PAIRS>(row, at, x[j]);
  }
  double wq[4], wk[4], f[2];
  weights_load<PAIRS>(a.nq, at, wq);
  weights_load<PAIRS>(a.nk, at, wk);
  freq_load(a.rot, at, f);
  const KvRow row = kv_row_wave<true>(a.b, r);
  if (row.i < 0) return;
  const Turn t = turn_at(a.rot, at, f, row.pos);
#pragma unroll
  for (int j = 0; j < H; ++j) {
    const int h = h0 + j * (64 / G);
    const bool isq = h < nq, isk = !isq && h < nq + nk, there = h < all;
    if (__any(isq || isk)) {
      double w1[4];
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w1[e] = isq ? wq[e] : wk[e], y[e] = x[j][e];
      head_turn<G>(y, a.nq != nullptr || a.nk != nullptr, isq ? a.nq != nullptr : a.nk != nullptr,
                   w1, HD, a.eps, at.turns, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = isq || isk ? y[e] : x[j][e];
    }
    if (isq) head_store<PAIRS>(a.q_out + r * a.out_stride + h * HD, at, x[j]);
    if (__any(!isq && there)) {
      const bool isv = !isq && !isk;
      const int kv = isv ? h - nq - nk : h - nq;
      const long slot = isq || !there || row.pos < 0 ? -1 : kv_slot(a.c, a.b, row.i, row.pos, kv);
      head_code<G, TYPE, PAIRS>(a.c, isv, slot, at, x[j], lane);
    }
  }
}

// ---- many rows ---------------------------------------------------------------------

// A lane's 16 values of a head: chunks of four at 4 (l + G j), G lanes a head.  NT chunks turn (4 or
// fewer, the first ones): within themselves with PAIRS, else j with j + NT / 2, NT 2 or 4.
template <int G, bool PAIRS>
struct Wide {
  static constexpr int HD = 16 * G;
  double c[8], s[8];  // of the lane's pairs
  int nt, lane;

  __device__ __forceinline__ Wide(const Rotary &r, int pos, int lane_) : lane(lane_) {
    nt = r.rot / (4 * G);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int j = PAIRS ? n / 2 : n / 4;
      if (j >= (PAIRS ? nt : nt / 2)) break;
      const int f = PAIRS ? 2 * (lane + G * j) + n % 2 : 4 * (lane + G * j) + n % 4;
      double angle = r.freq[f] * (double)pos;
      if (r.angle32) angle = (double)((float)r.freq[f] * (float)pos);
      cos_sin(angle, &c[n], &s[n]);
      if (r.angle32) c[n] = (double)(float)c[n], s[n] = (double)(float)s[n];
      c[n] *= (double)r.amp;
      s[n] *= (double)r.amp;
    }
  }
  // ONCE: past the caches' order of use, for rows that are read once and don't fit
  template <bool ONCE = false>
  __device__ __forceinline__ void load(const float *p, v4f (&x)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v4f *at = reinterpret_cast<const v4f *>(p + 4 * (lane + G * j));
      x[j] = ONCE ? __builtin_nontemporal_load(at) : *at;
    }
  }
  __device__ __forceinline__ void store(float *p, const v4f (&x)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<v4f *>(p + 4 * (lane + G * j)) = x[j];
  }
  // through the norm (weights w, applied as w + 1; norm is the same in the whole wave) and the turn
  __device__ __forceinline__ void turn(v4f (&x)[4], bool norm, const v4f (&w)[4], float eps) const {
    double d[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[j][e] = (double)x[j][e];
    if (norm) {
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fma(d[j][e], d[j][e], ss);
      ss += dpp_f64<kDppXor1>(ss);
      ss += dpp_f64<kDppXor2>(ss);
      if (G >= 8) ss += dpp_f64<kDppHalfMirror>(ss);
      if (G >= 16) ss += dpp_f64<kDppMirror>(ss);
      const double m = rsqrt_f64(fma(ss, 1.0 / HD, (double)eps));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[j][e] *= m * ((double)w[j][e] + 1.0);
    }
    auto pair = [&](double &a, double &b, int n) {
      const double t = a * c[n] - b * s[n];
      b = fma(b, c[n], a * s[n]);
      a = t;
    };
    if (PAIRS) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < nt) {
          pair(d[j][0], d[j][1], 2 * j);
          pair(d[j][2], d[j][3], 2 * j + 1);
        }
    } else if (nt == 4) {
#pragma unroll
      for (int n = 0; n < 8; ++n) pair(d[n / 4][n % 4], d[n / 4 + 2][n % 4], n);
    } else if (nt == 2) {
#pragma unroll
      for (int n = 0; n < 4; ++n) pair(d[0][n], d[1][n], n);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = (float)d[j][e];
  }
  // As codes and a scale into the cache's row `slot` of HD codes (negative: none), as cache_write
  // makes them.
  template <int TYPE>
  __device__ __forceinline__ void code(const v4f (&x)[4], uint8_t *codes, float *scales,
                                       long slot) const {
    int top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, __float_as_int(x[j][e]) & 0x7fffffff);
    top = max(top, dpp_i32<kDppXor1>(top));
    top = max(top, dpp_i32<kDppXor2>(top));
    if (G >= 8) top = max(top, dpp_i32<kDppHalfMirror>(top));
    if (G >= 16) top = max(top, dpp_i32<kDppMirror>(top));
    const bool finite = top < 0x7f800000;
    const float amax = finite ? daz(__int_as_float(top)) : 0.0f;
    float scale = 0.0f;
    uint32_t q[4] = {};
    if (TYPE == kKvI8) {
      const QuantParams qp = quant_params(amax);
      scale = amax > 0.0f ? qp.scale : 0.0f;
      if (__all(finite && (amax == 0.0f || amax > 1e-30f))) {
        // 127 / amax is finite and no code leaves -127 .. 127: quant_one without its clamps
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = x[j][e] * qp.inv;
            t[e] = (uint32_t)(int)(y + copysignf(0.5f, y));
          }
          q[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400u),
                                       __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u), 0x05040100u);
        }
      } else if (amax > 0.0f) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[j] = pack4(quant_one(x[j][0], qp.inv), quant_one(x[j][1], qp.inv),
                       quant_one(x[j][2], qp.inv), quant_one(x[j][3], qp.inv));
      }
    } else if (amax > 0.0f) {
      scale = mul_ftz(amax, 1.0f / 448.0f);
      const float inv = (float)(448.0 / (double)amax);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaxf(-448.0f, fminf(448.0f, daz(x[j][e]) * inv));
        const int t = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], t, true);
      }
    }
    if (slot < 0) return;
    uint32_t *dst = reinterpret_cast<uint32_t *>(codes + (size_t)slot * HD) + lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[G * j] = q[j];
    if (lane == 0) scales[slot] = finite ? scale : __int_as_float(0x7fc00000);
  }
};

// Whether rows go by Wide: whole chunks turn.
bool wide(int hdim, const Rotary &r) {
  return (hdim == 64 || hdim == 128 || hdim == 256) && r.rot % (r.pairs ? hdim / 4 : hdim / 2) == 0;
}

// `per` heads of 64 / G rows a wave
template <int G, bool PAIRS>
__global__ __launch_bounds__(kThreads) void rope_wide_kernel(RopeRows a, int per) {
  const long wave = (long)blockIdx.x * (kThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int parts = (a.heads + per - 1) / per;
  const int h0 = (int)(wave % parts) * per, h1 = min(h0 + per, a.heads);
  const long first = wave / parts * (64 / G);
  if (first >= a.rows) return;
  const int r = (int)first + threadIdx.x % 64 / G;
  const bool there = r < a.rows;
  const int row = there ? r : a.rows - 1;
  const float *src = a.src + row * a.src_stride;
  float *dst = a.dst + row * a.dst_stride;
  const Wide<G, PAIRS> t(a.rot, a.pos[row], threadIdx.x % G);
  v4f w[4] = {}, x[4], next[4];
  if (a.w != nullptr) t.load(a.w, w);
  t.load(src + h0 * (16 * G), next);
  for (int h = h0; h < h1; ++h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = next[j];
    t.load(src + min(h + 1, h1 - 1) * (16 * G), next);
    t.turn(x, a.w != nullptr, w, a.eps);
    if (there) t.store(dst + h * (16 * G), x);
  }
}

// `per` heads (q's, then k's, then v's) of 64 / G rows a wave
template <int G, int TYPE, bool PAIRS>
__global__ __launch_bounds__(kThreads) void kv_append_wide_kernel(KvAppend a, int per) {
  constexpr int HD = 16 * G, ROWS = 64 / G;
  const long wave = (long)blockIdx.x * (kThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int nq = a.q != nullptr ? a.n_heads : 0, nk = a.c.nkv, all = nq + 2 * nk;
  const int parts = (all + per - 1) / per;
  const int h0 = (int)(wave % parts) * per, h1 = min(h0 + per, all);
  const long first = wave / parts * ROWS;
  if (first >= a.b.rows) return;
  const int group = threadIdx.x % 64 / G, r = min((int)first + group, a.b.rows - 1);
  KvRow row = {-1, 0};
  kv_rows_wave<ROWS>(a.b, (int)first, [&](int i, KvRow of) {
    if (i == group) row = of;
  });
  if ((int)first + group >= a.b.rows) row.i = -1;
  const bool there = row.i >= 0;
  // the row's place in the first head of its page
  const long place = there && row.pos >= 0 ? kv_slot(a.c, a.b, row.i, row.pos, 0) : -1;
  const Wide<G, PAIRS> t(a.rot, row.pos, threadIdx.x % G);
  const float *q = nq > 0 ? a.q + r * a.q_stride : nullptr;
  const float *k = a.k + r * a.k_stride, *v = a.v + r * a.v_stride;
  float *out = nq > 0 ? a.q_out + r * a.out_stride : nullptr;
  auto from = [&](int h) {
    return h < nq ? q + h * HD : h < nq + nk ? k + (h - nq) * HD : v + (h - nq - nk) * HD;
  };
  v4f w[4] = {}, x[4], next[4];
  t.template load<true>(from(h0), next);
  for (int h = h0; h < h1; ++h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = next[j];
    t.template load<true>(from(min(h + 1, h1 - 1)), next);
    const bool isq = h < nq;
    if (h < nq + nk) {
      const float *norm = isq ? a.nq : a.nk;
      if (norm != nullptr && (h == h0 || h == nq)) t.load(norm, w);
      t.turn(x, norm != nullptr, w, a.eps);
    }
    if (isq) {
      if (there) t.store(out + h * HD, x);
    } else {
      const bool isv = h >= nq + nk;
      const int head = isv ? h - nq - nk : h - nq;
      t.template code<TYPE>(x, isv ? a.c.v : a.c.k, isv ? a.c.vs : a.c.ks,
                            place < 0 ? -1 : place + ((long)head << a.c.shift));
    }
  }
}

// Heads in a call up to which lanes take one each, so that a few rows are one trip to memory; beyond,
// rows go by Wide where they can and if that leaves every SIMD two heads to do, else lanes take four
// heads, which share the row's angles and table look-ups.  us of q, k and v appended (16 heads of
// 256 a row) by one, by four and by Wide: 512 rows 8.7, 8.5, 6.8, 2048 rows 26, 18, 18, 8192 rows 96,
// 57, 50; of 1024 rows (8 heads of 128) 5.6, 5.5, 6.5, 2048 rows 8.7, 7.4, 7.4.
constexpr long kFewHeads = 8192;
// Calls of Wide: `rows` waves' worth of rows, `per` heads of them a wave, `waves` in all.
struct WideCall {
  long waves;
  int per;
};
// most: heads a wave, if that leaves every SIMD two waves.  Rows for the cache take up to 8, as each
// wave looks their places up; rope two (32768 rows of 8 heads of 256: 51 us, with eight 57).
WideCall wide_call(int nrows, int heads, int g, int most, const DeviceInfo &dev) {
  const long rows = (nrows + 64 / g - 1l) / (64 / g), all = rows * heads;
  if (all < 8l * dev.cus) return WideCall{0, 0};
  const long per = all / (8l * dev.cus);
  const int p = (int)(per < 2 ? 2 : per > most ? most : per);
  return WideCall{rows * ((heads + p - 1) / p), p};
}

}  // namespace

hipError_t launch_rope(const RopeRows &a, const DeviceInfo &dev, hipStream_t stream) {
  auto go = [&](auto g, auto pairs, auto h) {
    constexpr int PER = 64 / g() * h();
    const long units = (long)a.rows * ((a.heads + PER - 1) / PER);
    rope_kernel<g(), pairs(), h()><<<(unsigned)((units + 3) / 4), kThreads, 0, stream>>>(a);
  };
  auto heads = [&](auto g, auto pairs) {
    constexpr int G = g() / 4;
    const WideCall w = wide_call(a.rows, a.heads, G, 2, dev);
    if (w.waves > 0 && wide(a.hdim, a.rot))
      rope_wide_kernel<G, pairs()>
          <<<(unsigned)((w.waves + 3) / 4), kThreads, 0, stream>>>(a, w.per);
    else if ((long)a.rows * a.heads <= kFewHeads)
      go(g, pairs, std::integral_constant<int, 1>());
    else
      go(g, pairs, std::integral_constant<int, 4>());
  };
  auto pairs = [&](auto g) {
    a.rot.pairs ? heads(g, std::true_type()) : heads(g, std::false_type());
  };
  a.hdim <= 64    ? pairs(std::integral_constant<int, 16>())
  : a.hdim <= 128 ? pairs(std::integral_constant<int, 32>())
                  : pairs(std::integral_constant<int, 64>());
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppend &a, const DeviceInfo &dev, hipStream_t stream) {
  const int all = (a.q != nullptr ? a.n_heads : 0) + 2 * a.c.nkv;
  auto go = [&](auto g, auto type, auto pairs, auto h) {
    constexpr int PER = 64 / g() * h();
    const long units = (long)a.b.rows * ((all + PER - 1) / PER);
    kv_append_kernel<g(), type(), pairs(), h()>
        <<<(unsigned)((units + 3) / 4), kThreads, 0, stream>>>(a);
  };
  auto heads = [&](auto g, auto type, auto pairs) {
    constexpr int G = g() / 4;
    const WideCall w = wide_call(a.b.rows, all, G, 8, dev);
    if (w.waves > 0 && wide(a.c.hdim, a.rot))
      kv_append_wide_kernel<G, type(), pairs()>
          <<<(unsigned)((w.waves + 3) / 4), kThreads, 0, stream>>>(a, w.per);
    else if ((long)a.b.rows * all <= kFewHeads)
      go(g, type, pairs, std::integral_constant<int, 1>());
    else
      go(g, type, pairs, std::integral_constant<int, 4>());
  };
  auto pairs = [&](auto g, auto type) {
    a.rot.pairs ? heads(g, type, std::true_type()) : heads(g, type, std::false_type());
  };
  auto type = [&](auto g) {
    a.c.type == kKvI8 ? pairs(g, std::integral_constant<int, kKvI8>())
                      : pairs(g, std::integral_constant<int, kKvE4m3>());
  };
  a.c.hdim == 256 ? type(std::integral_constant<int, 64>())
                  : type(std::integral_constant<int, 32>());
  return hipGetLastError();
}

}  // namespace gh
