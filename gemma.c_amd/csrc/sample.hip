// sample.hip -- the next token of each row of logits: temperature, top-k, top-p
// and min-p, from a given uniform random number.
//
// Let z = l log2(e) / temperature be a token's logit in octaves, w = 2^z its weight.
// The kept tokens are a prefix of the row in the order of falling logit (ties by
// rising index), and so is what each filter keeps and what lies before the token
// drawn: each step finds the first token of that order up to which a running
// count or a running weight reaches a target.  No row is sorted for that: tokens
// are counted, and weighed, in 512 bins of 1/16 octave below the row's largest (the
// last bin holds all the rest), and only the bins in which a target may be reached
// are looked into.
//
// Weights are fp64.  A bin's tokens weigh 1 to 1.044 times its lower end: what a token
// adds is 1 and a fraction in whole multiples of 2^-39, count and fraction in one
// 64-bit sum, exact in any order.  What the last bin's add is whole multiples of 2^-44 of the
// bin's upper end, some 2^-75 of the row's largest weight.  Sums over bins and workgroups are
// fp64 in one order.
// So equal calls give equal bits.  What a token adds is the same wherever it is summed, so that
// sums over equal logits meet a target (top-p's, the draw's) where exact ones do: at or past it
// within kTie.
//
// Up to kWholeVocab columns a workgroup does a row by itself, from registers.  Longer rows
// take four launches: each 8192-column chunk's bins, from its own largest logit down so that
// one reading does (sample_bins_kernel); their sum and the bins that matter
// (sample_decide_kernel); these bins' tokens (sample_collect_kernel; chunks that hold none
// are not read again); and the targets inside them (sample_pick_kernel).
//
// Of 16000 columns one row by top-k 64 and top-p 0.95 takes 17 us, 64 rows with settings of
// all kinds 22 (24 and 37 when the bins' tokens are looked for in the row, not in a list).
// Of 262144 columns, us: the one row 8 + 13 + 5 + 8, four chains of round trips and of code
// fetched cold; the 64 rows (67 MB) 26 + 13 + 18 + 28: the first by its vector instructions (47
// a logit, a fifth of them fp64 arithmetic, keep the vector units busy for three quarters of
// the time and more; LDS, conflicts included, for two fifths; 2.6 TB/s), the last by the rows that
// cut deep into a flat part, a workgroup each.
#include <float.h>
#include <limits.h>

#include "dec_common.h"
#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

typedef unsigned long long u64;

constexpr int kBins = 512;
constexpr double kPerOctave = 16.0;
constexpr int kChunk = 8192;       // columns of a workgroup of the long rows' kernels
constexpr int kChunkThreads = 512;
constexpr int kPer = kChunk / kChunkThreads;
constexpr int kThreads = 1024;     // ... of the kernels that see whole rows
constexpr int kWholeVocab = 16384;
constexpr int kWholeList = 4096;   // their tokens that are put into LDS, at most
constexpr int kRanked = 256;       // tokens that are put in order by comparing all pairs
constexpr int kSubs = 1024;        // parts of a bin with more
constexpr int kList = 32768;       // tokens of a row's bins that are collected, at most
constexpr int kFrac = 39;          // a bin's sum: fractions in 2^-39 below, the count above
constexpr int kCountAt = 49;       // (2^14 tokens of fractions below 0.0443 stay below 2^49)
constexpr int kUnit = 44;          // a weight's units within its bin: 2^-44 of the bin's octave
constexpr double kTie = 0x1p-46;   // of a target: sums as near count as equal to it
constexpr double kInfZ = 0x1p1000;  // an infinite logit, far above any other's octaves

// A token's place in the order: rising.  NaN and -inf have none.
__device__ __forceinline__ bool has_place(float l) { return l > -INFINITY; }
__device__ __forceinline__ u64 place(float l, int index) {
  const uint32_t b = l == 0.0f ? 0u : __float_as_uint(l);
  const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)~up << 32 | (uint32_t)index;
}
__device__ __forceinline__ float logit_at(u64 place) {
  const uint32_t up = ~(uint32_t)(place >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

__device__ __forceinline__ double octaves(float l, double c) {
  return l == INFINITY ? kInfZ : (double)l * c;
}
// ... times kPerOctave (c16 is c times that, a power of two: the same to the bit); INF: some
// logit may be infinite
template <bool INF>
__device__ __forceinline__ double steps(float l, double c16) {
  return INF && l == INFINITY ? kInfZ * kPerOctave : (double)l * c16;
}

// 2^x in fp64 for x <= 0 (0 below -1000): x = e + j / 128 + r, the table's 2^(j/128)
// (exp_tab_load) and the Taylor polynomial of 2^r, |r| <= 2^-8 (truncation below
// 2e-18).
__device__ __forceinline__ double pow2(double x, const double *tab) {
  x = fmax(x, -1000.0);
  const double kf = rint(x * 128.0);
  const double r = fma(kf, -0x1p-7, x);
  double p = fma(r, 0x1.5d87fe78a6731p-10, 0x1.3b2ab6fba4e77p-7);  // (ln 2)^i / i!
  p = fma(r, p, 0x1.c6b08d704a0c0p-5);
  p = fma(r, p, 0x1.ebfbdff82c58fp-3);
  p = fma(r, p, 0x1.62e42fefa39efp-1);
  p = fma(r, p, 1.0);
  const int k = (int)kf;
  return ldexp(tab[k & 127] * p, k >> 7);
}
// ... rounded to a whole number of units 2^-bits, bits <= 51
__device__ __forceinline__ u64 units(double w, int bits) {
  const double magic = 0x1p52;
  return (u64)(__double_as_longlong(ldexp(w, bits) + magic) - __double_as_longlong(magic));
}

// A row's settings; a temperature of 0 is top-k 1.
struct Settings {
  double c;  // octaves of a logit
  int k;     // 0: all
  double p;  // 1: all
  double m;  // 0: all
  double u;
};
__device__ __forceinline__ double octave_scale(const Sample &a, int row) {
  constexpr double log2e = 0x1.71547652b82fep+0;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  return t > 0.0f ? log2e / (double)t : log2e;
}
__device__ __forceinline__ Settings settings(const Sample &a, int row) {
  Settings s;
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  s.c = octave_scale(a, row);
  s.k = a.top_k != nullptr ? max(a.top_k[row], 0) : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  s.p = p < 1.0f ? (double)p : 1.0;
  const float m = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  s.m = m > 0.0f ? (double)m : 0.0;
  const float u = a.u[row];
  s.u = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
  if (!(t > 0.0f)) {
    s.k = 1;
    s.p = 1.0;
    s.m = 0.0;
  }
  return s;
}

// Where bins lie: bin i holds 16 z in [gmax - i, gmax - i + 1), the last one all below;
// weights are relative to the first one's lower end.
struct Grid {
  double gmax;
};
__device__ __forceinline__ Grid grid_of(double zmax) { return {floor(zmax * kPerOctave)}; }
__device__ __forceinline__ int bin_at(double y, double gmax) {  // y: z kPerOctave
  const double d = gmax - floor(y);
  return d >= kBins - 1 ? kBins - 1 : (int)d;
}
__device__ __forceinline__ int bin_of(double z, double gmax) {
  return bin_at(z * kPerOctave, gmax);
}
// The power of two that no weight of the last bin exceeds.
__device__ __forceinline__ double rest_top(const Grid &g) {
  return ceil((g.gmax - (kBins - 1) + 1.0) / kPerOctave);
}

// What a token r of a bin's width above the bin's lower end adds to the bin's sum: 1 and
// 2^(r / 16) - 1 in units of 2^-kFrac, by its Taylor polynomial (what it leaves out is below
// 2^-43), whose coefficients hold the units and whose last step rounds to a whole number.
__device__ __forceinline__ u64 bin_term(double r) {
  constexpr double q = 0x1.62e42fefa39efp-5;  // ln 2 / 16
  constexpr double unit = (double)(1ull << kFrac);
  constexpr double c1 = q * unit, c2 = c1 * q / 2.0, c3 = c2 * q / 3.0, c4 = c3 * q / 4.0,
                   c5 = c4 * q / 5.0, c6 = c5 * q / 6.0;
  double p = fma(r, c6, c5);
  p = fma(r, p, c4);
  p = fma(r, p, c3);
  p = fma(r, p, c2);
  p = fma(r, p, c1);
  p = fma(r, p, 0x1p52);
  return ((u64)__double_as_longlong(p) & ((1ull << kCountAt) - 1)) | 1ull << kCountAt;
}

// What a token of a bin (its z kPerOctave: y) adds to the bin's sum, in the bin's units ...
__device__ __forceinline__ u64 token_units(double y, int bin, const Grid &g, const double *tab) {
  if (bin < kBins - 1) return (bin_term(y - floor(y)) & ((1ull << kCountAt) - 1)) + (1ull << kFrac);
  const double x = y * (1.0 / kPerOctave) - rest_top(g);
  return x > -64.0 ? units(pow2(x, tab), kUnit) : 0;
}
// ... and these units.
__device__ __forceinline__ double bin_unit(int bin, const Grid &g, const double *tab) {
  return bin < kBins - 1 ? pow2(bin * (-1.0 / kPerOctave), tab) * 0x1p-39
                         : pow2(rest_top(g) - g.gmax * (1.0 / kPerOctave), tab) * 0x1p-44;
}
static_assert(kFrac == 39 && kUnit == 44, "bin_unit's");

constexpr uint32_t kNone = ~0u;
constexpr int kPerLane = kBins / 64;
// Arrays of which a lane reads neighbouring entries have a gap after every eight: without
// them all lanes would meet in one LDS bank.
__device__ __forceinline__ constexpr int gap(int i) { return i + (i >> 3); }
constexpr int kBinsGap = kBins + kBins / 8, kSubsGap = kSubs + kSubs / 8;
// A row's bins, running sums from the largest logits down, and where the tokens of
// the bins that matter have been collected.
struct Row {
  Grid g;
  double zmax;
  u64 sum_m[kBinsGap];       // (doubles) running weight ...
  uint32_t sum_c[kBinsGap];  // ... and count, each bin's own included
  uint32_t at[kBinsGap];     // list position of the bin's tokens, kNone: not collected
  uint32_t fill[kBinsGap];   // tokens of the bin in the list so far
  uint32_t listed;        // tokens of the bins that matter, kNone: more than the list takes
  uint32_t last;          // the last of them
  __device__ double weight(int i) const { return __longlong_as_double((long long)sum_m[gap(i)]); }
  __device__ double weight_before(int i) const { return i > 0 ? weight(i - 1) : 0.0; }
  __device__ uint32_t count_before(int i) const { return i > 0 ? sum_c[gap(i - 1)] : 0u; }
  __device__ uint32_t count_of(int i) const { return sum_c[gap(i)] - count_before(i); }
};

// A row's running sums, a lane's bins in its registers: each wave searches them alone.
struct Bins {
  uint32_t before, c[kPerLane];  // count before the lane's bins, and up to each
  double w[kPerLane];
  __device__ __forceinline__ explicit Bins(const Row &r) {
    const int lane = threadIdx.x & 63;
    before = r.count_before(kPerLane * lane);
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      c[e] = r.sum_c[gap(kPerLane * lane + e)];
      w[e] = r.weight(kPerLane * lane + e);
    }
  }
  // the first bin with tokens for which f holds, the last one with tokens if none
  template <class F>
  __device__ __forceinline__ int first(F &&f) const {
    int hit = kPerLane, some = -1;
#pragma unroll
    for (int e = kPerLane - 1; e >= 0; --e) {
      if (c[e] == (e > 0 ? c[e > 0 ? e - 1 : 0] : before)) continue;
      some = max(some, e);
      if (f(c[e], w[e])) hit = e;
    }
    const u64 any = __ballot(hit < kPerLane), full = __ballot(some >= 0);
    if (any != 0) {
      const int l = __ffsll(any) - 1;
      return kPerLane * l + __shfl(hit, l, 64);
    }
    const int l = full != 0 ? 63 - __clzll(full) : 0;
    return kPerLane * l + max(0, __shfl(some, l, 64));
  }
  __device__ __forceinline__ int by_weight(double target) const {
    return first([&](uint32_t, double x) { return x >= target; });
  }
  __device__ __forceinline__ int past_weight(double target) const {
    return first([&](uint32_t, double x) { return x > target; });
  }
  __device__ __forceinline__ int by_count(uint32_t target) const {
    return first([&](uint32_t x, double) { return x >= target; });
  }
};
// Bins in which min-p's border may lie: [0], the first of them, to [1].
__device__ __forceinline__ void min_p_bins(const Row &r, double m, int (&b)[2]) {
  const double z = r.zmax + log2(m);
  const double slack = 1e-9 * (1.0 + fabs(r.zmax));
  b[0] = z + slack >= r.zmax ? 0 : bin_of(z + slack, r.g.gmax);
  b[1] = z - slack >= r.zmax ? 0 : bin_of(z - slack, r.g.gmax);
}

// What a running sum has to reach to be at least t, or to exceed it.
__device__ __forceinline__ double at_least(double t) { return t - t * kTie; }
__device__ __forceinline__ double past(double t) { return t + t * kTie; }

// Running sums over the bins, by wave 0 (count, then weight).
__device__ __forceinline__ void sum_bins(const uint32_t *count, const double *mass, Row &r) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  uint32_t c[kPerLane], cs = 0;
  double m[kPerLane], ms = 0.0;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    c[e] = cs += count[gap(kPerLane * lane + e)];
    m[e] = ms += mass[gap(kPerLane * lane + e)];
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t ct = __shfl_up(cs, off, 64);
    const double mt = __shfl_up(ms, off, 64);
    if (lane >= off) {
      cs += ct;
      ms += mt;
    }
  }
  const uint32_t cb = cs - c[kPerLane - 1];
  const double before = __shfl_up(ms, 1, 64);  // not ms less the own: sums must not fall
  const double mb = lane > 0 ? before : 0.0;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    r.sum_c[gap(kPerLane * lane + e)] = cb + c[e];
    r.sum_m[gap(kPerLane * lane + e)] = (u64)__double_as_longlong(fmin(mb + m[e], ms));
  }
}

// Marks the bins that pick() may look into, by wave 0.  A target that is a share of
// a sum which itself depends on a border inside a bin lies between the shares of
// that bin's ends.
__device__ __forceinline__ void decide(const Settings &st, Row &r) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  const Bins bins(r);
  const uint32_t n = r.sum_c[gap(kBins - 1)];
  bool need[kPerLane] = {};
  auto mark = [&](int lo, int hi) {
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) need[e] = need[e] || (kPerLane * lane + e >= lo && kPerLane * lane + e <= hi);
  };
  int cut_lo = kBins - 1, cut_hi = kBins - 1;
  double s_lo = r.weight(kBins - 1), s_hi = s_lo;
  if (st.k > 0 && (uint32_t)st.k < n) {
    cut_lo = cut_hi = bins.by_count(st.k);
    s_hi = r.weight(cut_hi);
    s_lo = r.weight_before(cut_lo);
    if (r.sum_c[gap(cut_hi)] == (uint32_t)st.k)
      s_lo = s_hi;
    else
      mark(cut_lo, cut_hi);
  }
  if (st.p < 1.0) {
    const int lo = bins.by_weight(at_least(st.p * s_lo));
    const int hi = bins.by_weight(at_least(st.p * s_hi));
    mark(min(lo, cut_lo), min(hi, cut_hi));
    cut_lo = min(cut_lo, lo);
    cut_hi = min(cut_hi, hi);
    s_lo = fmin(s_lo, r.weight_before(cut_lo));
    s_hi = fmin(s_hi, r.weight(cut_hi));
  }
  if (st.m > 0.0) {
    int b[2];
    min_p_bins(r, st.m, b);
    if (b[0] <= cut_hi) {
      mark(b[0], min(b[1], cut_hi));
      cut_lo = min(cut_lo, b[0]);
      cut_hi = min(cut_hi, b[1]);
      s_lo = fmin(s_lo, r.weight_before(cut_lo));
      s_hi = fmin(s_hi, r.weight(cut_hi));
    }
  }
  mark(bins.past_weight(past(st.u * s_lo)), min(bins.past_weight(past(st.u * s_hi)), cut_hi));
  // list positions
  uint32_t own[kPerLane], sum = 0;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    own[e] = sum;
    sum += need[e] ? r.count_of(kPerLane * lane + e) : 0u;
  }
  uint32_t run = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t t = __shfl_up(run, off, 64);
    if (lane >= off) run += t;
  }
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) {
    r.at[gap(kPerLane * lane + e)] = need[e] ? run - sum + own[e] : kNone;
    r.fill[gap(kPerLane * lane + e)] = 0;
  }
  int last = 0;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e)
    if (need[e]) last = kPerLane * lane + e;
  const u64 some = __ballot(last > 0);
  last = __shfl(last, some != 0 ? 63 - __clzll(some) : 0, 64);
  if (lane == 63) {
    r.listed = run <= kList ? run : kNone;
    r.last = last;
  }
}

// Working memory of pick() and of what it calls.
struct Lds {
  Row row;
  double tab[128];
  u64 mass[kSubsGap];
  uint32_t count[kSubsGap];
  u64 place[kRanked], sorted[kRanked];
  double weight[kRanked];
  double wred[kThreads / 64];
  u64 red[3];
  uint32_t n;
};

// A token's weight, relative to the first bin's lower end.
__device__ __forceinline__ double weight_of(const Settings &st, const Row &r, u64 place,
                                            const double *tab) {
  return pow2(octaves(logit_at(place), st.c) - r.g.gmax * (1.0 / kPerOctave), tab);
}

// A token found: how many tokens of its bin come before it, the weight of the bin up
// to and with it, and its own.
struct Found {
  u64 place;
  uint32_t before;
  double upto, own;
};

// Where pick() finds the tokens of the bins that matter: in the row's list, of which one
// bin at a time is brought to LDS (staged; null: the list is there already); null: in the
// row alone.
constexpr int kStaged = 8192;
struct Source {
  const u64 *list;
  u64 *staged;  // LDS
};

// Brings a bin's tokens to LDS, if they are listed and fit: then true (barriers around it
// are the caller's).
__device__ __forceinline__ bool stage(const Source &src, const Row &r, int bin) {
  constexpr int kAhead = 8;
  const uint32_t n = r.count_of(bin);
  if (src.staged == nullptr || r.listed == kNone || r.at[gap(bin)] == kNone || n > kStaged) return false;
  const u64 *from = src.list + r.at[gap(bin)];
  u64 p[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e) p[e] = from[min(threadIdx.x + e * kThreads, n - 1)];
#pragma unroll
  for (int e = 0; e < kAhead; ++e)
    if (threadIdx.x + e * kThreads < n) src.staged[threadIdx.x + e * kThreads] = p[e];
  static_assert(kAhead * kThreads == kStaged, "all of it");
  return true;
}

// Calls f(place) for the tokens of a bin.
template <class F>
__device__ __forceinline__ void each_of_bin(const Sample &a, int row, const Settings &st,
                                            const Source &src, const Row &r, int bin, bool staged,
                                            F &&f) {
  const uint32_t n = r.count_of(bin);
  if (staged) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) f(src.staged[i]);
  } else if (src.list != nullptr && r.listed != kNone && r.at[gap(bin)] != kNone) {
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) f(src.list[r.at[gap(bin)] + i]);
  } else {
    const float *l = a.logits + row * a.stride;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float x = l[i];
      if (has_place(x) && bin_of(octaves(x, st.c), r.g.gmax) == bin) f(place(x, i));
    }
  }
}

// The first part of an array of counts and weights (units) at which the running count
// or weight reaches the target, or the last that isn't empty: into red[] as part,
// count before, weight before.  By wave 0, first over N / 64 parts a lane, then over those
// of the lane found, one each; barriers around it are the caller's.
template <int N>
__device__ __forceinline__ void find_part(Lds &s, bool by_count, double target, bool strict,
                                          double unit, uint32_t count0, u64 mass0) {
  const int lane = threadIdx.x;
  if (lane >= 64) return;
  constexpr int P = N / 64;
  uint32_t c = 0;
  u64 m = 0;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    c += s.count[gap(P * lane + e)];
    m += s.mass[gap(P * lane + e)];
  }
  // the lane found; then c and m are the sums before its own
  auto first = [&]() {
    uint32_t cs = c;
    u64 ms = m;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t ct = __shfl_up(cs, off, 64);
      const u64 mt = __shfl_up(ms, off, 64);
      if (lane >= off) {
        cs += ct;
        ms += mt;
      }
    }
    const double v = by_count ? (double)(count0 + cs) : (double)(mass0 + ms) * unit;
    const u64 some = __ballot(c != 0);
    const u64 hits = __ballot(c != 0 && (strict ? v > target : v >= target));
    const int who = hits ? __ffsll(hits) - 1 : some ? 63 - __clzll(some) : 0;
    count0 += __shfl(cs - c, who, 64);
    mass0 += __shfl(ms - m, who, 64);
    return who;
  };
  const int lot = first();
  c = lane < P ? s.count[gap(P * lot + lane % P)] : 0;
  m = lane < P ? s.mass[gap(P * lot + lane % P)] : 0;
  const int at = first();
  if (lane == 0) {
    s.red[0] = P * lot + at;
    s.red[1] = count0;
    s.red[2] = mass0;
  }
}

// The first token of a bin up to which the bin's running count, or `base` plus its
// running weight, reaches (strict: exceeds) the target; its last one where none
// does.  By the whole workgroup.
//  - Up to 256 tokens: all pairs compared.
//  - More: counted and weighed in 1024 parts of the bin, then the part's tokens.
//  - Where a part has more than that (equal logits): digit by digit of the place.
__device__ __forceinline__ Found locate(const Sample &a, int row, const Settings &st,
                                        const Source &src, Lds &s, int bin, bool by_count,
                                        double target, bool strict, double base) {
  const Row &r = s.row;
  const int tid = threadIdx.x;
  const double unit = bin_unit(bin, r.g, s.tab);
  if (!by_count) target -= base;
  auto weigh = [&](u64 p) {
    return token_units(octaves(logit_at(p), st.c) * kPerOctave, bin, r.g, s.tab);
  };
  // the part of the bin that a token falls into: any that falls as logits rise does; of the
  // last bin, 1/16 octave each
  const double edge = r.g.gmax - bin;  // 16 z of the bin's lower end
  auto part = [&](u64 p) {
    const double y = octaves(logit_at(p), st.c) * kPerOctave - edge;  // in [0, 1); the last: < 1
    const double d = bin < kBins - 1 ? (1.0 - y) * kSubs : 1.0 - y;
    return min(kSubs - 1, max(0, (int)fmin(d, 1e6)));
  };
  int only = -1;  // the part to look at, all if -1
  uint32_t count0 = 0;
  u64 mass0 = 0;
  uint32_t n = r.count_of(bin);
  __syncthreads();
  const bool staged = stage(src, r, bin);
  if (n > kRanked) {
    for (int i = tid; i < kSubsGap; i += kThreads) s.count[i] = s.mass[i] = 0;
    __syncthreads();
    each_of_bin(a, row, st, src, r, bin, staged, [&](u64 p) {
      const int i = gap(part(p));
      atomicAdd(&s.count[i], 1u);
      atomicAdd(&s.mass[i], weigh(p));
    });
    __syncthreads();
    find_part<kSubs>(s, by_count, target, strict, unit, 0, 0);
    __syncthreads();
    only = (int)s.red[0];
    count0 = (uint32_t)s.red[1];
    mass0 = s.red[2];
    n = s.count[gap(only)];
  }
  if (n > kRanked) {
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < gap(256); i += kThreads) s.count[i] = s.mass[i] = 0;
      __syncthreads();
      each_of_bin(a, row, st, src, r, bin, staged, [&](u64 p) {
        if (part(p) != only || (shift < 56 && (p >> (shift + 8)) != prefix)) return;
        const int d = gap((int)(p >> shift) & 255);
        atomicAdd(&s.count[d], 1u);
        atomicAdd(&s.mass[d], weigh(p));
      });
      __syncthreads();
      find_part<256>(s, by_count, target, strict, unit, count0, mass0);
      __syncthreads();
      prefix = prefix << 8 | s.red[0];
      count0 = (uint32_t)s.red[1];
      mass0 = s.red[2];
    }
    return Found{prefix, count0, base + (double)(mass0 + weigh(prefix)) * unit,
                 weight_of(st, r, prefix, s.tab)};
  }
  // gather, rank, sum in order
  if (tid == 0) s.n = 0;
  __syncthreads();  // (what was staged is there, too)
  each_of_bin(a, row, st, src, r, bin, staged, [&](u64 p) {
    if (only >= 0 && part(p) != only) return;
    const uint32_t i = atomicAdd(&s.n, 1u);
    if (i < kRanked) s.place[i] = p;
  });
  if (tid < kRanked) s.count[tid] = 0;
  __syncthreads();
  n = min(s.n, (uint32_t)kRanked);
  {
    constexpr int S = kThreads / kRanked;
    const uint32_t i = tid % kRanked, q = tid / kRanked;
    if (i < n) {
      const u64 mine = s.place[i];
      uint32_t rank = 0;
      for (uint32_t e = q; e < n; e += S) rank += s.place[e] < mine;
      atomicAdd(&s.count[i], rank);
    }
  }
  __syncthreads();
  if (tid < kRanked) s.weight[tid] = 0.0;
  __syncthreads();
  if (tid < (int)n) {
    const uint32_t at = s.count[tid];
    s.sorted[at] = s.place[tid];
    s.weight[at] = (double)weigh(s.place[tid]) * unit;
  }
  __syncthreads();
  if (tid < 64) {
    constexpr int P = kRanked / 64;
    double w[P], sum = 0.0;
    for (int e = 0; e < P; ++e) sum += w[e] = s.weight[P * tid + e];
    double run = sum;
    for (int off = 1; off < 64; off <<= 1) {
      const double t = __shfl_up(run, off, 64);
      if (tid >= off) run += t;
    }
    const double prev = __shfl_up(run, 1, 64);
    run = (double)mass0 * unit + (tid > 0 ? prev : 0.0);
    int hit = -1;
    double upto = 0.0;
    for (int e = 0; e < P; ++e) {
      const int i = P * tid + e;
      run += w[e];
      if (hit >= 0 || i >= (int)n) continue;
      const double v = by_count ? (double)(count0 + i + 1) : run;
      if (strict ? v > target : v >= target) {
        hit = i;
        upto = run;
      } else if (i == (int)n - 1) {
        upto = run;  // the last one, for want of another
      }
    }
    const u64 hits = __ballot(hit >= 0);
    const int who = hits ? __ffsll(hits) - 1 : (int)(n - 1) / P;
    if (tid == who) {
      s.red[0] = hits ? hit : (int)n - 1;
      s.wred[0] = upto;
    }
  }
  __syncthreads();
  const uint32_t at = (uint32_t)s.red[0];
  return Found{s.sorted[at], count0 + at, base + s.wred[0],
               weight_of(st, r, s.sorted[at], s.tab)};
}

// Where a bin's tokens are put in order once for all targets: those of all bins that
// matter, up to kRanked, in s.sorted with running weights (over all of them) in s.weight.
__device__ __forceinline__ void rank_all(const Settings &st, u64 mine_, Lds &s) {
  const Row &r = s.row;
  const uint32_t n = r.listed, tid = threadIdx.x;
  if (tid < kRanked) {
    s.place[tid] = tid < n ? mine_ : ~0ull;
    s.count[tid] = 0;
  }
  __syncthreads();
  constexpr uint32_t S = kThreads / kRanked, E = kRanked / S;  // parts of the pairs, tokens of one
  const uint32_t i = tid % kRanked, q = tid / kRanked;
  if (i < n && q * E < n) {
    const u64 mine = s.place[i];
    uint32_t rank = 0;
#pragma unroll 8
    for (uint32_t e = q * E; e < (q + 1) * E; ++e) rank += s.place[e] < mine;
    atomicAdd(&s.count[i], rank);
  }
  __syncthreads();
  if (tid < n) {
    const u64 p = s.place[tid];
    const double y = octaves(logit_at(p), st.c) * kPerOctave;
    const int bin = bin_at(y, r.g.gmax);
    s.sorted[s.count[tid]] = p;
    s.weight[s.count[tid]] =
        (double)token_units(y, bin, r.g, s.tab) * bin_unit(bin, r.g, s.tab);
  } else if (tid < kRanked) {
    s.weight[tid] = 0.0;
  }
  __syncthreads();
  if (tid < 64) {
    constexpr int P = kRanked / 64;
    double w[P], sum = 0.0;
#pragma unroll
    for (int e = 0; e < P; ++e) w[e] = sum += s.weight[P * tid + e];
    double run = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double t = __shfl_up(run, off, 64);
      if ((int)tid >= off) run += t;
    }
    const double before = __shfl_up(run, 1, 64);
#pragma unroll
    for (int e = 0; e < P; ++e) s.weight[P * tid + e] = (tid > 0 ? before : 0.0) + w[e];
  }
  __syncthreads();
}

// locate() among ranked tokens, by each wave alone.
__device__ __forceinline__ Found locate_ranked(const Settings &st, const Lds &s, int bin,
                                               bool by_count, double target, bool strict,
                                               double base) {
  const Row &r = s.row;
  const int lane = threadIdx.x & 63;
  const uint32_t from = r.at[gap(bin)], n = r.count_of(bin);
  const double start = from > 0 ? s.weight[from - 1] : 0.0;
  uint32_t at = n - 1;
  if (by_count) {
    at = min(n, (uint32_t)target) - 1;
  } else {
    uint32_t hit = kNone;
    for (uint32_t i = lane; i < n; i += 64) {
      const double v = base + (s.weight[from + i] - start);
      if (strict ? v > target : v >= target) {
        hit = i;
        break;
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) hit = min(hit, (uint32_t)__shfl_xor((int)hit, off, 64));
    at = min(at, hit);
  }
  const u64 p = s.sorted[from + at];
  return Found{p, at, base + (s.weight[from + at] - start), weight_of(st, r, p, s.tab)};
}

// The token, from the row's bins.
// listed: the list's threadIdx.x-th.
// (Inlined, as all that it calls and decide() are: calls would go through scratch, 8 to 45% of a
// short row.)
__device__ __forceinline__ void pick(const Sample &a, int row, const Settings &st,
                                     const Source &src, u64 listed, Lds &s) {
  const Row &r = s.row;
  const Bins bins(r);
  const uint32_t total = r.sum_c[gap(kBins - 1)];
  uint32_t n = total;  // what is kept: so many, weighing so much
  double sum = r.weight(kBins - 1);
  const bool ranked = src.list != nullptr && r.listed <= kRanked;
  if (ranked) rank_all(st, listed, s);
  // sums stay between the bins' own, whatever they were rounded to
  auto within = [&](double w, int bin) { return fmin(fmax(w, r.weight_before(bin)), r.weight(bin)); };
  auto in_bin = [&](int bin, bool by_count, double target, bool strict)
      __attribute__((always_inline)) {
    const double base = r.weight_before(bin);
    Found f = ranked && r.at[gap(bin)] != kNone
                  ? locate_ranked(st, s, bin, by_count, target, strict, base)
                  : locate(a, row, st, src, s, bin, by_count, target, strict, base);
    f.upto = within(f.upto, bin);
    return f;
  };
  if (st.k > 0 && (uint32_t)st.k < n) {
    n = st.k;
    const int bin = bins.by_count(n);
    sum = r.sum_c[gap(bin)] == n ? r.weight(bin)
                                 : in_bin(bin, true, n - r.count_before(bin), false).upto;
  }
  if (st.p < 1.0) {
    const double target = at_least(st.p * sum);
    const int bin = bins.by_weight(target);
    const Found f = in_bin(bin, false, target, false);
    const uint32_t np = r.count_before(bin) + f.before + 1;
    if (np < n) {
      n = np;
      sum = f.upto;
    }
  }
  if (st.m > 0.0) {
    int b[2];
    min_p_bins(r, st.m, b);
    for (int bin = b[0]; bin <= b[1] && r.count_before(bin) < n; ++bin) {
      uint32_t kept = 0;
      double weight = r.weight_before(bin);
      const uint32_t in = r.count_of(bin);
      auto enough = [&](u64 p) {
        const double z = octaves(logit_at(p), st.c);
        return z >= r.zmax || pow2(z - r.zmax, s.tab) >= st.m;
      };
      if (in != 0 && ranked && r.at[gap(bin)] != kNone) {
        const uint32_t from = r.at[gap(bin)];
        for (uint32_t i = threadIdx.x & 63; i < (in + 63) / 64 * 64; i += 64)
          kept += __popcll(__ballot(i < in && enough(s.sorted[from + min(i, in - 1)])));
        if (kept > 0)
          weight += s.weight[from + kept - 1] - (from > 0 ? s.weight[from - 1] : 0.0);
      } else if (in != 0) {
        uint32_t c = 0;
        u64 w = 0;
        each_of_bin(a, row, st, src, r, bin, false, [&](u64 p) {
          if (!enough(p)) return;
          ++c;
          w += token_units(octaves(logit_at(p), st.c) * kPerOctave, bin, r.g, s.tab);
        });
        __syncthreads();
        if (threadIdx.x == 0) s.red[0] = s.red[1] = 0;
        __syncthreads();
        atomicAdd(&s.red[0], (u64)c);
        atomicAdd(&s.red[1], w);
        __syncthreads();
        kept = (uint32_t)s.red[0];
        weight += (double)s.red[1] * bin_unit(bin, r.g, s.tab);
        __syncthreads();
      }
      if (kept == in && bin < b[1]) continue;
      if (r.count_before(bin) + kept < n) {  // at least the largest logit is
        n = r.count_before(bin) + kept;
        sum = within(weight, bin);
      }
      break;
    }
  }
  const double target = past(st.u * sum);
  int bin = min(bins.past_weight(target), bins.by_count(n));
  Found f = in_bin(bin, false, target, true);
  // where a rounding took the draw past the last token kept
  if (r.count_before(bin) + f.before + 1 > n) {
    bin = bins.by_count(n);
    f = in_bin(bin, true, n - r.count_before(bin), false);
  }
  if (threadIdx.x == 0) {
    a.tokens[row] = (int)(uint32_t)f.place;
    if (a.probs != nullptr) a.probs[row] = (float)(f.own / sum);
  }
}

__device__ __forceinline__ void pick_none(const Sample &a, int row) {
  if (threadIdx.x == 0) {
    a.tokens[row] = -1;
    if (a.probs != nullptr) a.probs[row] = 0.0f;
  }
}

// The largest of a workgroup's values (-inf: none), by waves through red[].
template <int NT>
__device__ __forceinline__ float block_most(float v, float *red) {
  v = wave_max_dpp(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, red[w]);
  return m;
}

// Counts and weighs tokens into bins; the last bin's, which most tokens of a peaked
// row share, in registers first (weights of all sizes: count, and units of 2^-kUnit of
// the bin's octave).
struct Rest {
  u64 mass;
  uint32_t count;
};
struct Binner {
  u64 *bins;
  Rest *rest;
  uint32_t rest_c = 0;
  u64 rest_m = 0;
  __device__ __forceinline__ Binner(u64 *b, Rest *r) : bins(b), rest(r) {}
  template <bool INF>
  __device__ __forceinline__ void add(float l, double c16, const Grid &g, const double *tab) {
    if (!has_place(l)) return;
    const double y = steps<INF>(l, c16), f = floor(y), d = g.gmax - f;
    if (d < kBins - 1) {
      atomicAdd(&bins[(int)d], bin_term(y - f));
    } else {
      ++rest_c;
      rest_m += token_units(y, kBins - 1, g, tab);
    }
  }
  // a thread's logits, of which `most` is the workgroup's largest
  template <int N>
  __device__ __forceinline__ void add_all(const float (&x)[N], float most, double c, const Grid &g,
                                          const double *tab) {
    const double c16 = c * kPerOctave;
    if (most == INFINITY) {
#pragma unroll 1
      for (int e = 0; e < N; ++e) add<true>(x[e], c16, g, tab);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) add<false>(x[e], c16, g, tab);
    }
  }
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      rest_c += __shfl_xor(rest_c, off, 64);
      rest_m += __shfl_xor(rest_m, off, 64);
    }
    if ((threadIdx.x & 63) == 0 && rest_c != 0) {
      atomicAdd(&rest->count, rest_c);
      atomicAdd(&rest->mass, rest_m);
    }
  }
};
__device__ __forceinline__ uint32_t bin_count(u64 b) { return (uint32_t)(b >> kCountAt); }
// ... and weight, relative to the bin's lower end
__device__ __forceinline__ double bin_weight(u64 b) {
  return (double)bin_count(b) + ldexp((double)(b & ((1ull << kCountAt) - 1)), -kFrac);
}
// A bin's lower end, relative to the first one's.
__device__ __forceinline__ double bin_end(int bin, const double *tab) {
  return pow2(bin * (-1.0 / kPerOctave), tab);
}

// ---- short rows: a workgroup each -----------------------------------------------

__global__ __launch_bounds__(kThreads) void sample_whole_kernel(Sample a) {
  __shared__ Lds s;
  __shared__ float red[kThreads / 64];
  __shared__ double mass[kBinsGap];
  __shared__ Rest rest;
  __shared__ u64 list[kWholeList];
  const int row = blockIdx.x, tid = threadIdx.x;
  const float *l = a.logits + row * a.stride;
  const Settings st = settings(a, row);
  exp_tab_load(s.tab);
  if (tid < kBins) s.mass[tid] = 0;
  if (tid == 0) rest = Rest{0, 0};
  float most = -INFINITY;
  constexpr int kWhole = kWholeVocab / kThreads;
  float x[kWhole];
#pragma unroll
  for (int e = 0; e < kWhole; ++e) {
    x[e] = l[min(tid + e * kThreads, a.vocab - 1)];
    if (tid + e * kThreads >= a.vocab) x[e] = -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < kWhole; ++e) most = fmaxf(most, x[e]);
  most = block_most<kThreads>(most, red);
  if (!has_place(most)) return pick_none(a, row);
  const Grid g = grid_of(octaves(most, st.c));
  Binner bins(s.mass, &rest);
  bins.add_all(x, most, st.c, g, s.tab);
  bins.finish();
  if (tid == 0) {
    s.row.g = g;
    s.row.zmax = octaves(most, st.c);
  }
  __syncthreads();
  if (tid < kBins) {
    s.count[gap(tid)] = tid < kBins - 1 ? bin_count(s.mass[tid]) : rest.count;
    mass[gap(tid)] = tid < kBins - 1 ? bin_weight(s.mass[tid]) * bin_end(tid, s.tab)
                                     : (double)rest.mass * bin_unit(tid, g, s.tab);
  }
  __syncthreads();
  sum_bins(s.count, mass, s.row);
  __syncthreads();
  decide(st, s.row);
  __syncthreads();
  const bool fits = s.row.listed <= kWholeList;
  if (fits) {
#pragma unroll
    for (int e = 0; e < kWhole; ++e) {
      if (!has_place(x[e])) continue;
      const int bin = gap(bin_of(octaves(x[e], st.c), g.gmax));
      if (s.row.at[bin] == kNone) continue;
      const uint32_t i = s.row.at[bin] + atomicAdd(&s.row.fill[bin], 1u);
      if (i < kWholeList) list[i] = place(x[e], tid + e * kThreads);
    }
  }
  __syncthreads();
  pick(a, row, st, Source{fits ? list : nullptr, nullptr}, list[min(tid, kRanked - 1)], s);
}

// ---- long rows --------------------------------------------------------------------

// A chunk's bins, from its own largest logit down.
struct Chunk {
  Grid g;  // gmax -inf: no token
  double zmax;
  Rest rest;
  u64 bins[kBins];
};

struct Work {
  Chunk *chunks;  // [rows][nchunk]
  Row *rows;      // [rows]
  u64 *list;      // [rows][kList]
};
__host__ __device__ inline int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

__device__ __forceinline__ void load_chunk(const Sample &a, int row, float (&x)[kPer]) {
  const float *l = a.logits + row * a.stride;
  const int base = blockIdx.x * kChunk + threadIdx.x;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = base + e * kChunkThreads;
    x[e] = l[min(i, a.vocab - 1)];
    x[e] = i < a.vocab ? x[e] : -INFINITY;
  }
}

__global__ __launch_bounds__(kChunkThreads) void sample_bins_kernel(Sample a, Work w) {
  __shared__ double tab[128];
  __shared__ u64 count[kBins];
  __shared__ Rest rest;
  __shared__ float red[kChunkThreads / 64];
  const int row = blockIdx.y, tid = threadIdx.x;
  float x[kPer];
  load_chunk(a, row, x);
  const double c = octave_scale(a, row);
  exp_tab_load(tab);
  count[tid] = 0;
  if (tid == 0) rest = Rest{0, 0};
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < kPer; ++e) most = fmaxf(most, x[e]);
  most = block_most<kChunkThreads>(most, red);
  Chunk *out = w.chunks + (size_t)row * gridDim.x + blockIdx.x;
  if (!has_place(most)) {
    if (tid == 0) out->g.gmax = -INFINITY;
    return;
  }
  const Grid g = grid_of(octaves(most, c));
  Binner bins(count, &rest);
  bins.add_all(x, most, c, g, tab);
  bins.finish();
  __syncthreads();
  out->bins[tid] = count[tid];
  if (tid == 0) {
    out->g = g;
    out->zmax = octaves(most, c);
    out->rest = rest;
  }
}

// The chunks' bins summed into the row's: thread (bin, part) takes one bin of each chunk of
// its part, all loaded before the row's largest logit is known.  Counts and fractions are
// whole numbers and their sums exact in any order; so are those of bins that fall into
// the row's last one, in units.
constexpr int kMaxChunks = (kSampleMaxVocab + kChunk - 1) / kChunk;
__global__ __launch_bounds__(kThreads) void sample_decide_kernel(Sample a, Work w, int nchunk) {
  constexpr int kParts = kThreads / kBins, kAhead = 16;
  static_assert(kMaxChunks <= 64, "a lane per chunk");
  __shared__ Row r;
  __shared__ double tab[128], mass[kBinsGap];
  __shared__ uint32_t count[kBinsGap];
  __shared__ u64 frac[kBins];
  __shared__ Rest rest;
  const int row = blockIdx.x, tid = threadIdx.x, bin = tid % kBins, lane = tid & 63;
  const int part = __builtin_amdgcn_readfirstlane(tid / kBins);
  const Chunk *ch = w.chunks + (size_t)row * nchunk;
  const Chunk *mine = ch + min(lane, nchunk - 1);  // a lane per chunk
  const double gm = mine->g.gmax, zm = mine->zmax;
  const Rest mr = mine->rest;
  const Settings st = settings(a, row);
  u64 b[kAhead];
  auto load = [&](int c) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) b[e] = ch[min(c + kParts * e, nchunk - 1)].bins[bin];
  };
  load(part);
  exp_tab_load(tab);
  if (tid < kBins) {
    count[gap(tid)] = 0;
    frac[tid] = 0;
  }
  if (tid == 0) rest = Rest{0, 0};
  double z = gm > -INFINITY ? zm : -INFINITY;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) z = fmax(z, __shfl_xor(z, off, 64));
  Row *out = w.rows + row;
  if (!(z > -INFINITY)) {
    if (tid == 0) out->zmax = -INFINITY;
    return;
  }
  const Grid g = grid_of(z);
  const double top = rest_top(g);
  // chunks without a token, and past the last, are shifted out
  const int shift =
      lane < nchunk && gm > -INFINITY ? (int)fmin(g.gmax - gm, (double)kBins) : 2 * kBins;
  __syncthreads();
  uint32_t rest_n = 0;
  u64 rest_m = 0;
  for (int c = part; c < nchunk; c += kParts * kAhead) {
    if (c != part) load(c);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int i = c + kParts * e;
      if (i >= nchunk || bin >= kBins - 1 || b[e] == 0) continue;
      const int s = __builtin_amdgcn_readlane(shift, i);
      if (s > kBins) continue;
      if (bin + s < kBins - 1) {
        atomicAdd(&count[gap(bin + s)], bin_count(b[e]));
        atomicAdd(&frac[bin + s], b[e] & ((1ull << kCountAt) - 1));
      } else {
        const double end = (readlane_f64(gm, i) - bin) * (1.0 / kPerOctave) - top;
        // (more than units() takes: up to 2^14 weights)
        rest_n += bin_count(b[e]);
        if (end > -64.0)
          rest_m += (u64)rint(ldexp(bin_weight(b[e]) * pow2(end, tab), kUnit));
      }
    }
  }
  if (tid < nchunk && shift <= kBins && mr.count != 0) {
    const double down = top - rest_top(Grid{gm});
    rest_n += mr.count;
    rest_m += down < 64.0 ? mr.mass >> (int)down : 0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    rest_n += __shfl_xor(rest_n, off, 64);
    rest_m += __shfl_xor(rest_m, off, 64);
  }
  if (lane == 0 && rest_n != 0) {
    atomicAdd(&rest.count, rest_n);
    atomicAdd(&rest.mass, rest_m);
  }
  __syncthreads();
  if (tid < kBins - 1) {
    mass[gap(tid)] =
        ((double)count[gap(tid)] + ldexp((double)frac[tid], -kFrac)) * bin_end(tid, tab);
  } else if (tid == kBins - 1) {
    mass[gap(tid)] = (double)rest.mass * bin_unit(tid, g, tab);
    count[gap(tid)] = rest.count;
  }
  if (tid == 0) {
    r.g = g;
    r.zmax = z;
  }
  __syncthreads();
  sum_bins(count, mass, r);
  __syncthreads();
  decide(st, r);
  __syncthreads();
  for (int i = tid; i < (int)(sizeof(Row) / 8); i += kThreads) ((u64 *)out)[i] = ((u64 *)&r)[i];
}

// The tokens of the bins that matter, into the row's list: each workgroup takes room
// for a bin's at once.
__global__ __launch_bounds__(kChunkThreads) void sample_collect_kernel(Sample a, Work w) {
  __shared__ uint32_t at[kBins], count[kBins];
  const int row = blockIdx.y, tid = threadIdx.x;
  Row *r = w.rows + row;
  const Chunk *ch = w.chunks + (size_t)row * gridDim.x + blockIdx.x;
  const Grid g = r->g;
  const double cmax = ch->g.gmax;
  if (!(r->zmax > -INFINITY) || !(cmax > -INFINITY) || r->listed == kNone) return;
  at[tid] = r->at[gap(tid)];
  count[tid] = 0;
  __syncthreads();
  // whether the chunk has any of them
  const int shift = (int)fmin(g.gmax - cmax, (double)kBins);
  const bool here = (tid < kBins - 1 ? bin_count(ch->bins[tid]) : ch->rest.count) != 0 &&
                    at[min(tid + shift, kBins - 1)] != kNone;
  if (!__syncthreads_or(here)) return;
  float x[kPer];
  load_chunk(a, row, x);
  // logits below the last of these bins are most of a row's: told by a bound a little lower
  const double c16 = octave_scale(a, row) * kPerOctave;
  const uint32_t last = r->last;
  const double end = (g.gmax - last) / c16;  // (0 / 0 of a row of equal weights: no bound)
  const float least = last < kBins - 1 ? (float)(end - fabs(end) * 0x1p-22) : -INFINITY;
  int bin[kPer];
  uint32_t slot[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    bin[e] = -1;
    if (!has_place(x[e]) || x[e] < least) continue;
    const int i = bin_at(steps<true>(x[e], c16), g.gmax);
    if (at[i] == kNone) continue;
    bin[e] = i;
    slot[e] = atomicAdd(&count[i], 1u);
  }
  __syncthreads();
  if (count[tid] != 0) at[tid] += atomicAdd(&r->fill[gap(tid)], count[tid]);
  __syncthreads();
  u64 *list = w.list + (size_t)row * kList;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (bin[e] < 0) continue;
    const uint32_t i = at[bin[e]] + slot[e];
    if (i < kList) list[i] = place(x[e], blockIdx.x * kChunk + tid + e * kChunkThreads);
  }
}

__global__ __launch_bounds__(kThreads) void sample_pick_kernel(Sample a, Work w) {
  __shared__ Lds s;
  __shared__ u64 staged[kStaged];
  const int row = blockIdx.x, tid = threadIdx.x;
  const Row *r = w.rows + row;
  const u64 *list = w.list + (size_t)row * kList;
  const Settings st = settings(a, row);
  const u64 listed = list[min(tid, kRanked - 1)];  // before it is known how many there are
  const double zmax = r->zmax;
  u64 x[(sizeof(Row) / 8 + kThreads - 1) / kThreads];
#pragma unroll
  for (int e = 0; e < (int)(sizeof(x) / 8); ++e)
    x[e] = ((const u64 *)r)[min(tid + e * kThreads, (int)(sizeof(Row) / 8) - 1)];
  exp_tab_load(s.tab);
  if (!(zmax > -INFINITY)) return pick_none(a, row);
#pragma unroll
  for (int e = 0; e < (int)(sizeof(x) / 8); ++e)
    if (tid + e * kThreads < (int)(sizeof(Row) / 8)) ((u64 *)&s.row)[tid + e * kThreads] = x[e];
  __syncthreads();
  pick(a, row, st, Source{list, staged}, listed, s);
}

static_assert(sizeof(Row) % 8 == 0 && kBins == kChunkThreads, "layout");

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t sample_work(int rows, int vocab) {
  if (vocab <= kWholeVocab) return 0;
  return align256((size_t)rows * chunks_of(vocab) * sizeof(Chunk)) +
         align256((size_t)rows * sizeof(Row)) + align256((size_t)rows * kList * 8);
}

hipError_t launch_sample(const Sample &a, hipStream_t stream) {
  if (a.vocab <= kWholeVocab) {
    sample_whole_kernel<<<a.rows, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  }
  const int n = chunks_of(a.vocab);
  Work w;
  w.chunks = (Chunk *)a.work;
  w.rows = (Row *)(a.work + align256((size_t)a.rows * n * sizeof(Chunk)));
  w.list = (u64 *)((char *)w.rows + align256((size_t)a.rows * sizeof(Row)));
  const dim3 grid(n, a.rows);
  sample_bins_kernel<<<grid, kChunkThreads, 0, stream>>>(a, w);
  sample_decide_kernel<<<a.rows, kThreads, 0, stream>>>(a, w, n);
  sample_collect_kernel<<<grid, kChunkThreads, 0, stream>>>(a, w);
  sample_pick_kernel<<<a.rows, kThreads, 0, stream>>>(a, w);
  return hipGetLastError();
}

}  // namespace gh
