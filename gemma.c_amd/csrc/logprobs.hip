// logprobs.hip -- what rows of logits say: log probabilities and ranks of given tokens, the
// entropy, and the likeliest tokens.
//
// Let z = l log2(e) / temperature.  With any reference m, S = sum 2^(z - m), T = sum (z - m)
// 2^(z - m): log2 p = z - m - log2 S, and the entropy is log2 S - T / S octaves; sums by
// different references join when one is moved to the other's.  A token's rank is 1 and the
// count of those above it.  The n likeliest lie in the n runs of 64 columns with the largest
// largest logits (equals by index): a token of another run has n above it.
//
// So one reading does: a wave takes 2048 columns, 32 a lane in registers, and leaves S and T by
// its own largest logit (fp32, the exponents' errors below 2^-22), the given tokens' counts and its 32
// runs' largest logits.  A second launch joins a row's (fp64) and looks into the n runs that
// matter.  256 rows of 262144 (268 MB) take 56 + 9 us by themselves: the reading at 4.8 TB/s, the join
// a chain of two trips to memory and two searches; one row 5 + 9.  Short rows are bound by that chain,
// not by their bytes: 4000 rows of 1500 38 us (24 MB, 5 at a copy's rate), 256 of 32000 14.4 (33, 6).
#include <float.h>
#include <type_traits>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

typedef unsigned long long u64;

constexpr int kRun = 64;                  // columns of a run
constexpr int kLoads = 8;                 // 256 columns each
constexpr int kTile = 256 * kLoads;       // columns of a wave
constexpr int kTileRuns = kTile / kRun;
constexpr int kThreads = 256;
constexpr int kMaxTiles = (kSampleMaxVocab + kTile - 1) / kTile;
constexpr int kMost = kMaxTiles * kTileRuns;  // runs of a row
constexpr float kFar = -160.0f;  // octaves; a weight there is 0 in fp32

// rows of logits may begin anywhere
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

// What a wave leaves: its largest logit, S and T by it.
struct Part {
  float m, s, t;
};

// A row's parts, runs and counts in the workspace.
struct Layout {
  size_t parts, runs, counts, all;
};
__host__ __device__ inline int tiles_of(int vocab) { return (vocab + kTile - 1) / kTile; }
__host__ __device__ inline Layout layout_of(int rows, int vocab, int targets, int ntop) {
  const size_t tiles = (size_t)rows * tiles_of(vocab);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l;
  l.parts = 0;
  l.runs = up(tiles * sizeof(Part));
  l.counts = l.runs + (ntop > 0 ? up(tiles * kTileRuns * 4) : 0);
  l.all = l.counts + up(tiles * targets * 4);
  return l;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float no_nan(float l) { return fmaxf(l, -INFINITY); }

// How many octaves l lies above m (l <= m) by a temperature: fma(h, l, -h m) c, h a power of two that
// keeps both factors in fp32.  Finite logits may lie more than FLT_MAX apart, so where a logit is less
// than an octave they are halved.  Where it is more than FLT_MAX octaves, h is 2^64 as long as m is
// below 2^60: what this takes past FLT_MAX is further below m than any weight reaches; so is all that
// isn't m itself about larger m, where FLT_MAX will do.  Anywhere else the bits are those of (l - m) c.
struct Octaves {
  float h, c;
  __device__ __forceinline__ Octaves about(float m) const {
    return h > 1.0f && !(fabsf(m) < 0x1p60f) ? Octaves{1.0f, FLT_MAX} : *this;
  }
};
// c 0 where the temperature is 0 or none: all on the largest
__device__ __forceinline__ Octaves octaves_of(const float *temperature, int r) {
  const float t = temperature != nullptr ? temperature[r] : 1.0f;
  if (!(t > 0.0f)) return Octaves{1.0f, 0.0f};
  const double c = 0x1.71547652b82fep+0 / (double)t;
  const float h = c < 1.0 ? 0.5f : c > (double)FLT_MAX ? 0x1p64f : 1.0f;
  return Octaves{h, (float)(c * (h == 0.5f ? 2.0 : h > 1.0f ? 0x1p-64 : 1.0))};
}

// The least float above l (l not NaN); of +inf: NaN, which nothing reaches.
__device__ __forceinline__ float next_up(float l) {
  if (l == 0.0f) return __int_as_float(1);
  const int b = __float_as_int(l);
  return __int_as_float(b > 0 ? b + 1 : b - 1);
}

// A tile of row r by a wave; its part, runs (if TOP) and counts.
template <bool TOP>
__device__ __forceinline__ void scan_tile(const Logprobs &a, int r, int tile, Part *part,
                                          float *runs, int *counts) {
  const int lane = threadIdx.x & 63, c0 = tile * kTile;
  const float *row = a.logits + r * a.stride;
  float l[kLoads][4];
  if (c0 + kTile <= a.vocab) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      // past the caches' order of use: read once
      const v4f_any v = __builtin_nontemporal_load(
          reinterpret_cast<const v4f_any *>(row + c0 + 256 * j + 4 * lane));
#pragma unroll
      for (int e = 0; e < 4; ++e) l[j][e] = v[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = c0 + 256 * j + 4 * lane + e;
        l[j][e] = c < a.vocab ? row[c] : -INFINITY;
      }
  }
  const Octaves octaves = octaves_of(a.temperature, r);
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    float top = fmaxf(fmaxf(no_nan(l[j][0]), l[j][1]), fmaxf(no_nan(l[j][2]), l[j][3]));
    m = fmaxf(m, top);
    if (TOP) {  // 16 lanes' columns are a run
      top = fmaxf(top, dpp_f32<kDppXor1>(top));
      top = fmaxf(top, dpp_f32<kDppXor2>(top));
      top = fmaxf(top, dpp_f32<kDppHalfMirror>(top));
      top = fmaxf(top, dpp_f32<kDppMirror>(top));
      if ((lane & 15) == 0) runs[4 * j + lane / 16] = top;
    }
  }
  // S and T of a lane by its largest, then of the wave by the wave's
  float s = 0.0f, t = 0.0f;
  const Octaves by = octaves.about(m);
  const float hm = by.h * m;
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = fmaxf(fmaf(by.h, l[j][e], -hm) * by.c, kFar);  // NaN and -inf are far off
      const float w = exp2_fast(x);
      s += w;
      t = fmaf(w, x, t);
    }
  const float top = wave_max_dpp(m);
  if (top == INFINITY) {  // infinite logits share everything
    s = t = 0.0f;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += l[j][e] == INFINITY ? 1.0f : 0.0f;
  } else {
    const Octaves by = octaves.about(top);
    const float x = fmaxf(fmaf(by.h, m, -(by.h * top)) * by.c, kFar);
    const float w = exp2_fast(x);
    t = w * fmaf(s, x, t);
    s = w * s;
  }
  s = group_sum_f32<64>(s);
  t = group_sum_f32<64>(t);
  if (lane == 0) *part = Part{top, s, t};
  for (int k = 0; k < a.targets; ++k) {
    const int id = a.ids[(size_t)r * a.targets + k];
    int above = 0;
    if ((unsigned)id < (unsigned)a.vocab) {
      const float mine = no_nan(row[id]), more = next_up(mine);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int first = c0 + 256 * j;
        if (id < first || id >= first + 256) {
          const float least = id < first ? more : mine;
#pragma unroll
          for (int e = 0; e < 4; ++e) above += __popcll(__ballot(no_nan(l[j][e]) >= least));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            above += __popcll(
                __ballot(no_nan(l[j][e]) >= (first + 4 * lane + e < id ? mine : more)));
        }
      }
    }
    if (lane == 0) counts[k] = above;
  }
}

template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_scan_kernel(Logprobs a, Layout at) {
  const int tiles = tiles_of(a.vocab);
  const long unit = (long)blockIdx.x * (kThreads / 64) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r = (int)(unit / tiles), tile = (int)(unit % tiles);
  if (r >= a.rows) return;
  scan_tile<TOP>(a, r, tile, reinterpret_cast<Part *>(a.work + at.parts) + unit,
                 reinterpret_cast<float *>(a.work + at.runs) + unit * kTileRuns,
                 reinterpret_cast<int *>(a.work + at.counts) + unit * a.targets);
}

// Tokens and runs in the order of falling logit, then rising index, as falling whole numbers;
// 0: none.
__device__ __forceinline__ u64 key_of(float l, int index) {
  if (!(l > -INFINITY)) return 0;
  const uint32_t b = l == 0.0f ? 0u : __float_as_uint(l);
  const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)up << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float logit_of(u64 key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// The join's workgroups have 1024 threads, as one row's time is the length of a wave's program, or
// 256 where rows are many and their sum counts; keys are looked at by 256 groups of one or four.
constexpr int kGroups = 256;
constexpr int kListed = kMost / kGroups * kLogprobsMaxTop;
struct JoinShared {
  u64 most[kGroups];
  u64 list[kListed + 16];
  u64 best[kLogprobsMaxTop];
  u64 least;
  double logs;
  float top;
  int count;
  int above[kLogprobsMaxTargets];
  float given[kLogprobsMaxTargets];
};

// How many of n keys in LDS are above `mine`; sixteen are asked for at a time, behind the last too.
__device__ __forceinline__ int above_in(const u64 *keys, int n, u64 mine) {
  int above = 0;
  for (int j = 0; j < n; j += 16)
#pragma unroll
    for (int i = 0; i < 16; ++i) above += keys[j + i] > mine && j + i < n;
  return above;
}

template <int CTRL>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
  return (u64)__double_as_longlong(dpp_f64<CTRL>(__longlong_as_double((long long)v)));
}

// Keys (no two alike but 0) of all threads into sh.list, their number into sh.count: the n largest
// at least (all but 0 where there are fewer), and not many more.  One wave looks for a bound that the
// largest keys of n groups reach, or a few more, bit by bit from the highest (with
// every wave doing so, 3 us went by instead of 1), and what reaches it is listed: at most 64
// groups' keys.
template <int NT, int PER>
__device__ __forceinline__ void list_largest(JoinShared &sh, int n, const u64 (&keys)[PER]) {
  constexpr int GROUP = NT / kGroups;
  static_assert(GROUP == 1 || GROUP == 4, "a group is a lane or a quad");
  static_assert(kListed >= kLogprobsMaxTop * GROUP * PER, "the list holds 64 groups' keys");
  const int tid = threadIdx.x;
  u64 own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) own = max(own, keys[j]);
  u64 most = own;
  if (GROUP == 4) {
    most = max(most, dpp_u64<kDppXor1>(most));
    most = max(most, dpp_u64<kDppXor2>(most));
  }
  if (tid % GROUP == 0) sh.most[tid / GROUP] = most;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  if (tid < 64) {
    const int enough = min(n + 8, kLogprobsMaxTop);
    u64 other[kGroups / 64];
    uint32_t high[kGroups / 64], bound = 0;
#pragma unroll
    for (int j = 0; j < kGroups / 64; ++j) {
      other[j] = sh.most[tid + 64 * j];
      high[j] = (uint32_t)(other[j] >> 32);
    }
    bool found = false;
    for (int bit = 31; bit >= 0 && !found; --bit) {
      const uint32_t next = bound | 1u << bit;
      int reach = 0;
#pragma unroll
      for (int j = 0; j < kGroups / 64; ++j) reach += __popcll(__ballot(high[j] >= next));
      bound = reach >= n ? next : bound;
      found = reach >= n && reach <= enough;
    }
    u64 least = (u64)bound << 32;
    for (int bit = 31; bit >= 0 && !found; --bit) {  // equals, by their indices
      const u64 next = least | 1ull << bit;
      int reach = 0;
#pragma unroll
      for (int j = 0; j < kGroups / 64; ++j) reach += __popcll(__ballot(other[j] >= next));
      least = reach >= n ? next : least;
      found = reach >= n && reach <= enough;
    }
    if (tid == 0) sh.least = max(least, (u64)1);  // (0: fewer than n)
  }
  __syncthreads();
  const u64 least = sh.least;
  if (own >= least) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) mine += keys[j] >= least;
    int at = atomicAdd(&sh.count, mine);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (keys[j] >= least) sh.list[at++] = keys[j];
  }
  __syncthreads();
}

// The list's n largest, in order, into sh.best, 0 where there are fewer.
template <int NT>
__device__ __forceinline__ void rank_list(JoinShared &sh, int n) {
  const int count = sh.count;
  for (int i = threadIdx.x; i < count; i += NT) {
    const u64 mine = sh.list[i];
    const int rank = above_in(sh.list, count, mine);
    if (rank < n) sh.best[rank] = mine;
  }
  if ((int)threadIdx.x >= count && (int)threadIdx.x < n) sh.best[threadIdx.x] = 0;
  __syncthreads();
}

// S and T of the row's parts by its largest logit, by one wave; c: octaves a logit.
template <int PARTS>
__device__ __forceinline__ void join_parts(JoinShared &sh, const Part (&p)[PARTS], bool drawn,
                                           double c, float *entropy) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < PARTS; ++j) top = fmaxf(top, p[j].m);
  top = wave_max_dpp(top);
  double s = 0.0, t = 0.0;
#pragma unroll
  for (int j = 0; j < PARTS; ++j) {
    if (!(p[j].m > -INFINITY)) continue;
    double x = top == p[j].m ? 0.0 : ((double)p[j].m - (double)top) * c;  // (-inf below +inf)
    x = fmax(x, -1000.0);
    // 2^x: e^y for what is left of the nearest whole number, by Taylor's polynomial (y^9 / 9! is
    // below 3e-10)
    const double whole = rint(x), y = (x - whole) * 0x1.62e42fefa39efp-1;
    double e = fma(y, 1.0 / 40320.0, 1.0 / 5040.0);
    e = fma(y, e, 1.0 / 720.0);
    e = fma(y, e, 1.0 / 120.0);
    e = fma(y, e, 1.0 / 24.0);
    e = fma(y, e, 1.0 / 6.0);
    e = fma(y, e, 0.5);
    e = fma(y, e, 1.0);
    const double w = ldexp(fma(y, e, 1.0), (int)whole);
    s = fma(w, (double)p[j].s, s);
    t = fma(w, (double)p[j].t + (double)p[j].s * x, t);
  }
  s = wave_sum_f64(s);
  t = wave_sum_f64(t);
  const double ln2 = 0x1.62e42fefa39efp-1, logs = log(s);
  if ((threadIdx.x & 63) != 0) return;
  sh.top = top;
  sh.logs = logs;
  if (entropy != nullptr)
    *entropy = drawn && top > -INFINITY ? (float)fmax(0.0, logs - ln2 * t / s) : 0.0f;
}

// A row's answers from its tiles' parts, runs and counts; RUNS: of a thread, at most.  It is mostly
// waiting, so it takes two trips to memory: for the runs and what else is there, and then for the
// columns of the runs that matter, while one wave joins the parts and the others look up the given
// tokens.
template <int NT, int RUNS>
__device__ __forceinline__ void join_row(const Logprobs &a, int r, JoinShared &sh,
                                         const Part *parts, const float *runs,
                                         const int *counts) {
  constexpr int kWaves = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, tiles = tiles_of(a.vocab);
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const float *row = a.logits + r * a.stride;
  const int nruns = a.ntop > 0 ? (a.vocab + kRun - 1) / kRun : 0;
  float most[RUNS];
#pragma unroll
  for (int j = 0; j < RUNS; ++j) {
    const int i = tid + j * NT;
    most[j] = i < nruns ? runs[i] : -INFINITY;
  }
  const float temp = a.temperature != nullptr ? a.temperature[r] : 1.0f;
  const bool drawn = temp > 0.0f, joins = wave == kWaves - 1;
  constexpr int kParts = (RUNS * NT / kTileRuns + 63) / 64;  // of a lane
  Part part[kParts];
#pragma unroll
  for (int j = 0; j < kParts; ++j) {
    const int i = lane + 64 * j;
    part[j] = joins && i < tiles ? parts[i] : Part{-INFINITY, 0.0f, 0.0f};
  }
  int id = !joins && wave < a.targets ? a.ids[(size_t)r * a.targets + wave] : -1;
  // the runs that matter, as they were listed unless they are too many
  int chosen = 0;
  bool few = true;
  if (a.ntop > 0) {
    u64 keys[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) keys[j] = key_of(most[j], tid + j * NT);
    list_largest<NT>(sh, a.ntop, keys);
    few = sh.count <= kLogprobsMaxTop;
    if (!few) rank_list<NT>(sh, a.ntop);
    chosen = few ? sh.count : a.ntop;
  }
  // a wave a run: its columns are the threads' keys
  float l[kLogprobsMaxTop / kWaves];
  int col[kLogprobsMaxTop / kWaves];
#pragma unroll
  for (int j = 0; j < kLogprobsMaxTop / kWaves; ++j) {
    const int i = j * kWaves + wave;
    l[j] = -INFINITY, col[j] = 0;
    if (i >= chosen) continue;
    col[j] = index_of(few ? sh.list[i] : sh.best[i]) * kRun + lane;
    if (col[j] < a.vocab) l[j] = row[col[j]];
  }
  if (joins) {
    const double c = drawn ? 0x1.71547652b82fep+0 / (double)temp : 0.0;
    join_parts(sh, part, drawn, c, a.entropy != nullptr ? a.entropy + r : nullptr);
  } else {
    for (int k = wave; k < a.targets; k += kWaves - 1) {
      if (k != wave) id = a.ids[(size_t)r * a.targets + k];
      const bool there = (unsigned)id < (unsigned)a.vocab;
      const float given = there ? no_nan(row[id]) : -INFINITY;
      int above = 0;
      for (int j = lane; j < tiles; j += 64) above += counts[(size_t)j * a.targets + k];
      above = group_sum_i32<64>(above);
      if (lane == 0) sh.above[k] = there ? above : -1, sh.given[k] = given;
    }
  }
  __syncthreads();
  if (a.ntop > 0) {
    u64 mine[kLogprobsMaxTop / kWaves];
#pragma unroll
    for (int j = 0; j < kLogprobsMaxTop / kWaves; ++j) mine[j] = key_of(l[j], col[j]);
    list_largest<NT>(sh, a.ntop, mine);
    rank_list<NT>(sh, a.ntop);
  }
  const float top = sh.top;
  const double logs = sh.logs;
  const double per = 1.0 / (double)temp;
  // log p of a logit that isn't NaN; first: whether it is the row's first largest
  auto logp = [&](float l, bool first) -> float {
    if (!(l > -INFINITY)) return -INFINITY;
    if (!drawn) return first ? 0.0f : -INFINITY;
    if (l == top) return (float)(0.0 - logs);
    if (top == INFINITY) return -INFINITY;
    return (float)(((double)l - (double)top) * per - logs);
  };
  if (tid < a.targets) {
    const size_t to = (size_t)r * a.targets + tid;
    const int above = sh.above[tid];
    if (a.rank != nullptr) a.rank[to] = above + 1;
    if (a.logp != nullptr) a.logp[to] = logp(sh.given[tid], above == 0);
  }
  if (tid < a.ntop) {
    const u64 k = sh.best[tid];
    const size_t to = (size_t)r * a.ntop + tid;
    if (a.top != nullptr) a.top[to] = k != 0 ? index_of(k) : -1;
    if (a.top_logp != nullptr)
      a.top_logp[to] = k != 0 ? logp(logit_of(k), tid == 0) : -INFINITY;
  }
}

template <int NT, int RUNS>
__global__ __launch_bounds__(NT) void logprobs_join_kernel(Logprobs a, Layout at) {
  __shared__ JoinShared sh;
  const int r = blockIdx.x;
  const size_t first = (size_t)r * tiles_of(a.vocab);
  join_row<NT, RUNS>(a, r, sh, reinterpret_cast<const Part *>(a.work + at.parts) + first,
                     reinterpret_cast<const float *>(a.work + at.runs) + first * kTileRuns,
                     reinterpret_cast<const int *>(a.work + at.counts) + first * a.targets);
}

// Short rows by one workgroup, which keeps in LDS what the tiles leave: a launch (3.7 us on the host)
// and a trip less.
constexpr int kShortTiles = 16, kShortVocab = kShortTiles * kTile;
template <int NT>
__global__ __launch_bounds__(NT) void logprobs_short_kernel(Logprobs a) {
  __shared__ JoinShared sh;
  __shared__ Part parts[kShortTiles];
  __shared__ float runs[kShortTiles * kTileRuns];
  __shared__ int counts[kShortTiles * kLogprobsMaxTargets];
  const int r = blockIdx.x, tiles = tiles_of(a.vocab);
  for (int i = __builtin_amdgcn_readfirstlane(threadIdx.x / 64); i < tiles; i += NT / 64)
    scan_tile<true>(a, r, i, parts + i, runs + i * kTileRuns, counts + i * a.targets);
  __syncthreads();
  join_row<NT, (kShortTiles * kTileRuns + NT - 1) / NT>(a, r, sh, parts, runs, counts);
}

}  // namespace

size_t logprobs_work(int rows, int vocab, int targets, int ntop) {
  return layout_of(rows, vocab, targets, ntop).all;
}

namespace {
bool many_rows(int rows, const DeviceInfo &dev) { return rows > 2 * dev.cus; }
}  // namespace

// Short rows by one launch, but not many that leave most of a workgroup's waves without a tile: us by
// two launches and by one, 11 rows of 2511 10.4, 8.5, 256 of 32000 17.7, 14.4, 2048 of 32000 74, 61,
// 600 of 8000 19.6, 16.8, 2433 of 3023 32, 35.
bool logprobs_one_launch(int rows, int vocab, const DeviceInfo &dev) {
  return vocab <= kShortVocab && (!many_rows(rows, dev) || tiles_of(vocab) >= 4);
}

hipError_t launch_logprobs(const Logprobs &a, const DeviceInfo &dev, hipStream_t stream) {
  const bool many = many_rows(a.rows, dev);
  if (logprobs_one_launch(a.rows, a.vocab, dev)) {
    many ? logprobs_short_kernel<256><<<a.rows, 256, 0, stream>>>(a)
         : logprobs_short_kernel<1024><<<a.rows, 1024, 0, stream>>>(a);
    return hipGetLastError();
  }
  const Layout at = layout_of(a.rows, a.vocab, a.targets, a.ntop);
  const long units = (long)a.rows * tiles_of(a.vocab);
  const unsigned grid = (unsigned)((units + 3) / 4);
  a.ntop > 0 ? logprobs_scan_kernel<true><<<grid, kThreads, 0, stream>>>(a, at)
             : logprobs_scan_kernel<false><<<grid, kThreads, 0, stream>>>(a, at);
  using std::integral_constant;
  const auto join = [&](auto nt, auto runs) {
    logprobs_join_kernel<nt(), runs()><<<a.rows, nt(), 0, stream>>>(a, at);
  };
  const auto by = [&](auto nt) {
    const int runs = (a.vocab + kRun * nt() - 1) / (kRun * nt());
    if constexpr (nt() > 256) {
      if (runs <= 1) return join(nt, integral_constant<int, 1>());
    }
    runs <= 4              ? join(nt, integral_constant<int, 4>())
    : runs <= kMost / 1024 ? join(nt, integral_constant<int, kMost / 1024>())
                           : join(nt, integral_constant<int, kMost / nt()>());
  };
  many ? by(integral_constant<int, 256>()) : by(integral_constant<int, 1024>());
  return hipGetLastError();
}

}  // namespace gh
