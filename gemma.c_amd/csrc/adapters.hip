// adapters.hip -- low-rank adapters of many requests on one batch of rows.
//
//   u = scale[id] A[id] x  (rank values a job),  dst = base + B[id] u
//
// id is that of the row's sequence; jobs are projections side by side (q, k, v; gate, up).  A launch
// for the first product, whose results lie in the workspace, and one for the second; single tokens
// with little to read take both in one.
//
// Rows of prompts go 16 at a time through the bf16 matrix cores: an fp32 value is the sum of three
// bf16 pieces, a bf16 weight is one, an f16 weight the sum of two and an fp32 weight of three, and
// of the piece products those are summed whose orders add up to at most 2 (3, 5 or 6 of
// them: what is left out is below 2^-22 of a product).  Where pieces can't make a value up, an
// infinity or one that rounds to an infinite bf16, the sums with it aren't finite, and such sums are
// done over in fp32 as they are for single tokens.  A tile is one sequence's: with tiles across
// sequences, which took a pass for each adapter, the few that had two set the time.
//
// The products are small; what bounds these kernels is how x, base and dst get in and out.  A load
// whose neighbouring lanes have a row each, as the matrix instructions want them, takes 64 cycles
// (4096 rows of 2560 with 48 values of u so: 23 us, by whole runs and LDS 15), so all tiles but B's of
// short sequences are read by runs and turned in LDS.  4096 rows of 2560 by rank 16 on 4096 columns: first
// product 16 us (42 MB, 8 at a copy's rate), second 26 (134 MB, 26), 42 a call in bf16, 45 in f16 and
// 52 in fp32; 851 rows of 2560 by rank 64 on 20480 columns, f16: 14 and 36 (139 MB, 27).  Single
// tokens beside a chunk of a prompt each have a tile, which a workgroup takes for itself: 63 beside
// 512 rows by rank 16 on 20480 columns 84 us (106 MB, 21).
#include <type_traits>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kThreads = 256;
constexpr int kNone = -1, kOutside = -2;  // a row's id: no adapter, in no sequence
constexpr float kBf16Most = 0x1.fep127f;

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
// the largest magnitude of x and v; NaN if there is one
__device__ __forceinline__ float largest(float x, v4f v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x = __builtin_elementwise_maximum(x, fabsf(v[e]));
  return x;
}

// ---- weights ---------------------------------------------------------------------

template <int TYPE>
constexpr int kPieces = TYPE == kAdapterBf16 ? 1 : TYPE == kAdapterF16 ? 2 : 3;

// eight neighbouring weights as they lie in memory
template <int TYPE>
struct Raw8 {
  u4 v[TYPE == kAdapterF32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> raw8(const void *p, size_t at) {
  Raw8<TYPE> w;
  if (TYPE == kAdapterF32) {
    w.v[0] = *reinterpret_cast<const u4 *>((const float *)p + at);
    w.v[TYPE == kAdapterF32] = *reinterpret_cast<const u4 *>((const float *)p + at + 4);
  } else {
    w.v[0] = *reinterpret_cast<const u4 *>((const uint16_t *)p + at);
  }
  return w;
}
template <int TYPE>
__device__ __forceinline__ void floats8(const Raw8<TYPE> &w, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (TYPE == kAdapterF32) {
      f[e] = __uint_as_float(w.v[0][e]);
      f[e + 4] = __uint_as_float(w.v[TYPE == kAdapterF32][e]);
    } else if (TYPE == kAdapterBf16) {
      f[2 * e] = bf16_lo(w.v[0][e]);
      f[2 * e + 1] = bf16_hi(w.v[0][e]);
    } else {
      const uint32_t two = w.v[0][e];  // (a cast of the element itself takes the first one's bits)
      const h2 h = __builtin_bit_cast(h2, two);
      f[2 * e] = (float)h[0];
      f[2 * e + 1] = (float)h[1];
    }
  }
}

// N bf16 pieces of eight values, each the operand of a matrix instruction
template <int N>
struct Split8 {
  u4 p[N];
};
template <int N>
__device__ __forceinline__ Split8<N> split8(const float (&f)[8]) {
  Split8<N> s;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a = f[2 * e], b = f[2 * e + 1];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s.p[i][e] = cvt_pk_bf16(a, b);
      a -= bf16_lo(s.p[i][e]);
      b -= bf16_hi(s.p[i][e]);
    }
  }
  return s;
}
template <int TYPE>
__device__ __forceinline__ Split8<kPieces<TYPE>> pieces8(const Raw8<TYPE> &w) {
  if constexpr (TYPE == kAdapterBf16) {
    return Split8<1>{{w.v[0]}};
  } else {
    float f[8];
    floats8<TYPE>(w, f);
    return split8<kPieces<TYPE>>(f);
  }
}

// D[4 (lane / 16) + r][lane % 16] += W[lane % 16][8 (lane / 16) + e] . X[lane % 16][the same], the
// small products first
template <int N>
__device__ __forceinline__ v4f product(const Split8<N> &w, const Split8<3> &x, v4f d) {
#pragma unroll
  for (int order = 2; order >= 0; --order)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (order - i >= 0 && order - i < 3)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(w.p[i]), as_bf8(x.p[order - i]), d, 0,
                                                    0, 0);
  return d;
}

__device__ __forceinline__ const void *job_of(const void *const (&m)[kAdapterMaxJobs], int job) {
  return job == 0 ? m[0] : job == 1 ? m[1] : m[2];
}
__device__ __forceinline__ float scale_of(const Adapters &a, int id) {
  return a.scale != nullptr ? a.scale[id] : 1.0f;
}

// The workspace: u [rows][jobs * rank] as fp32, then the rows' ids (of tiles: piece_of).
__device__ __forceinline__ float *u_of(const Adapters &a) {
  return reinterpret_cast<float *>(a.work);
}
__device__ __forceinline__ int *ids_of(const Adapters &a) {
  return reinterpret_cast<int *>(a.work + (size_t)a.seq.rows * a.njobs * a.rank * 6);
}

// ---- single tokens ----------------------------------------------------------------

// By a whole wave.
__device__ __forceinline__ int id_of_row(const Adapters &a, int r) {
  const KvRow row = kv_row_wave<false>(a.seq, r);
  if (row.i < 0) return kOutside;
  const int id = a.ids[row.i];
  return (unsigned)id < (unsigned)a.count ? id : kNone;
}

// Inputs whose products are summed in fp32; sums of more (LONG) meet in fp64.  One product is added
// after the other, and where the roundings all point one way, as those of equal products do, sums of
// 10240 inputs were up to 4.5e-6 off and of 2^20 up to 1.5e-4; both 2e-6 so.  The fp64 sums take
// registers, so kernels for fewer inputs go without.
constexpr int kSpan = 4096;

// Sums of a row's inputs times N rows of weights, by a whole wave, in all its lanes.
template <int TYPE, bool LONG, int N>
__device__ __forceinline__ void row_sums(const float *x, const void *const (&m)[N],
                                         const size_t (&first)[N], int k, float (&s)[N]) {
  double far[N] = {};
  for (int k0 = 0; k0 < k; k0 += kSpan) {
#pragma unroll
    for (int t = 0; t < N; ++t) s[t] = 0.0f;
    for (int c = k0 + 8 * (threadIdx.x & 63); c < (LONG ? min(k, k0 + kSpan) : k); c += 512) {
      const v4f x0 = *reinterpret_cast<const v4f *>(x + c);
      const v4f x1 = *reinterpret_cast<const v4f *>(x + c + 4);
      Raw8<TYPE> w[N];
#pragma unroll
      for (int t = 0; t < N; ++t) w[t] = raw8<TYPE>(m[t], first[t] + c);
#pragma unroll
      for (int t = 0; t < N; ++t) {
        float f[8];
        floats8<TYPE>(w[t], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[t] = fmaf(x0[e], f[e], s[t]);
          s[t] = fmaf(x1[e], f[e + 4], s[t]);
        }
      }
    }
    if (!LONG) break;
#pragma unroll
    for (int t = 0; t < N; ++t) {
      far[t] += (double)s[t];
      s[t] = (float)far[t];
    }
  }
#pragma unroll
  for (int t = 0; t < N; ++t) s[t] = group_sum_f32<64>(s[t]);
}

template <int TYPE, bool LONG>
__global__ __launch_bounds__(kThreads) void adapter_shrink_row_kernel(Adapters a) {
  const int all = a.njobs * a.rank, lane = threadIdx.x & 63, r = blockIdx.x;
  const int at = blockIdx.y * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int job = at / a.rank, row = at % a.rank;
  if (at >= all) return;
  const int id = id_of_row(a, r);
  if (at == 0 && lane == 0) ids_of(a)[r] = id;
  if (id < 0) return;
  const void *const m[1] = {job_of(a.a, job)};
  const size_t first[1] = {((size_t)id * a.rank + row) * a.k};
  float s[1];
  row_sums<TYPE, LONG, 1>(a.src + r * a.src_stride, m, first, a.k, s);
  if (lane == 0) u_of(a)[(size_t)r * all + at] = scale_of(a, id) * s[0];
}

// ---- tiles of rows ------------------------------------------------------------------

// Tiles of up to R rows of one sequence, and so of one adapter: those of sequence i begin at slot
// row0[i] / R + i, which leaves room for all and needs no sums over the sequences before it.  A slot
// that is left over has no rows.
__host__ __device__ inline int tile_slots(const KvBatch &b, int r) { return b.rows / r + b.batch; }
struct Tile {
  int row, rows, id;  // the first row, how many, the adapter or kNone
};
// By a whole wave; as kv_find_part looks for rows.
template <int R>
__device__ __forceinline__ Tile tile_at(const Adapters &a, int slot) {
  const KvBatch &b = a.seq;
  const int lane = threadIdx.x & 63;
  int lo = 0, n = b.batch;
  while (n > 63) {
    const int step = (n + 62) / 63, at = lo + min(lane * step, n - 1);
    const bool before = lane * step < n && kv_clamp(b.row0[at], 0, b.rows) / R + at <= slot;
    const int skip = max((int)__popcll(__ballot(before)) - 1, 0) * step;
    lo += skip;
    n = min(n - skip, step);
  }
  const int at = lo + min(lane, n);
  const int begins = kv_clamp(b.row0[at], 0, b.rows);
  const int ids = a.ids[min(at, b.batch - 1)];
  const int j = max((int)__popcll(__ballot(lane < n && begins / R + at <= slot)) - 1, 0);
  const int r0 = __builtin_amdgcn_readlane(begins, j);
  const int rows = min(__builtin_amdgcn_readlane(begins, j + 1) - r0, b.max_rows);
  const int id = __builtin_amdgcn_readlane(ids, j);
  const int first = (slot - (r0 / R + lo + j)) * R;
  return Tile{r0 + first, first < 0 ? 0 : min(rows - first, R),
              (unsigned)id < (unsigned)a.count ? id : kNone};
}

// u of tiles in the workspace: a tile of up to 16 rows has their part of [rows][3][jobs * rank]
// values, in the order in which the matrix instructions take them: [job][piece][rank / 8][rows][8].
__device__ __forceinline__ uint16_t *piece_of(const Adapters &a, int row, int rows, int job, int p) {
  const size_t first = (size_t)row * 3 * a.njobs * a.rank;
  return reinterpret_cast<uint16_t *>(a.work) + first + (size_t)(job * 3 + p) * a.rank * rows;
}

constexpr int kShrinkWaves = 8;  // that share a tile's inputs
constexpr int kShrinkStep = 64;  // inputs
constexpr int kMostT = 3;        // 16 values of u each: a workgroup's, at most

// A wave's steps.  A load whose neighbouring lanes are in different rows, as the matrix instructions
// want them, takes a cycle a lane; so rows are read by runs of 16 bytes times neighbouring lanes
// and find their lanes through LDS, the wave's own (its accesses keep their order).
template <int TYPE, int T>
struct ShrinkStep {
  static constexpr int kSize = TYPE == kAdapterF32 ? 4 : 2;
  static constexpr int kRowLanes = kShrinkStep * kSize / 16;  // of a row of A
  static constexpr int kLoads = 16 * T * kRowLanes / 64;
  static constexpr int kPitch = kShrinkStep + 16 / kSize;  // 16 rows' 16 bytes in different banks
  struct Lds {
    float x[16][kShrinkStep + 4];
    char w[16 * T][kPitch * kSize];
  };
  v4f x[4];
  u4 w[kLoads];

  __device__ __forceinline__ void load(const float *const (&src)[4], const char *const (&m)[kLoads],
                                       int k, int end) {
    const int lane = threadIdx.x & 63, kx = k + 4 * (lane & 15);
    const int kw = k + 16 / kSize * (lane % kRowLanes);
#pragma unroll
    for (int j = 0; j < 4; ++j)  // past the caches' order of use: read once, or by few workgroups
      x[j] = __builtin_nontemporal_load(
          reinterpret_cast<const v4f *>(src[j] + (kx < end ? kx : 0)));
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      w[j] = *reinterpret_cast<const u4 *>(m[j] + (size_t)(kw < end ? kw : 0) * kSize);
  }
  // into LDS, zeros behind the last input
  __device__ __forceinline__ void put(Lds &to, int k, int end) const {
    const int lane = threadIdx.x & 63;
    const bool inx = k + 4 * (lane & 15) < end;
    const bool inw = k + 16 / kSize * (lane % kRowLanes) < end;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<v4f *>(&to.x[4 * j + lane / 16][4 * (lane & 15)]) =
          inx ? x[j] : v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      *reinterpret_cast<u4 *>(
          &to.w[64 / kRowLanes * j + lane / kRowLanes][16 * (lane % kRowLanes)]) =
          inw ? w[j] : u4{0, 0, 0, 0};
  }
  __device__ __forceinline__ static void multiply(const Lds &from, v4f (&acc)[T]) {
    const int lane = threadIdx.x & 63, m = lane & 15;
#pragma unroll
    for (int h = 0; h < kShrinkStep / 32; ++h) {
      const int k0 = 32 * h + 8 * (lane / 16);
      const v4f lo = *reinterpret_cast<const v4f *>(&from.x[m][k0]);
      const v4f hi = *reinterpret_cast<const v4f *>(&from.x[m][k0 + 4]);
      const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      const Split8<3> xp = split8<3>(f);
#pragma unroll
      for (int t = 0; t < T; ++t)
        acc[t] = product(pieces8<TYPE>(raw8<TYPE>(from.w[16 * t + m], k0)), xp, acc[t]);
    }
  }
};

// u of a tile of 16 rows and 16 T of their values; each wave takes every eighth step, the partial
// sums meet in LDS.
template <int TYPE, int T, bool LONG>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(Adapters a) {
  typedef ShrinkStep<TYPE, T> Step;
  __shared__ union {
    typename Step::Lds step[kShrinkWaves];
    v4f part[kShrinkWaves][T][64];
  } sh;
  const int all = a.njobs * a.rank, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int at0 = 16 * T * blockIdx.y;
  const Tile tile = tile_at<16>(a, blockIdx.x);
  if (tile.rows <= 0 || tile.id < 0) return;
  const float *x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j] = a.src + (tile.row + min(4 * j + lane / 16, tile.rows - 1)) * a.src_stride;
  const char *m[Step::kLoads];
#pragma unroll
  for (int j = 0; j < Step::kLoads; ++j) {
    const int at = min(at0 + (64 * j + lane) / Step::kRowLanes, all - 1), job = at / a.rank;
    m[j] = reinterpret_cast<const char *>(job_of(a.a, job)) +
           ((size_t)tile.id * a.rank + (at - job * a.rank)) * a.k * Step::kSize;
  }
  v4f acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  // two steps are on their way while one is multiplied
  constexpr int kNext = kShrinkStep * kShrinkWaves;
  Step one, two;
  typename Step::Lds &mine = sh.step[wave];
  auto step = [&](Step &s, int k) {
    s.put(mine, k, a.k);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    s.load(x, m, k + 2 * kNext, a.k);
    __builtin_amdgcn_sched_barrier(0);  // asked for before the products, not where they are put
    Step::multiply(mine, acc);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  int k = kShrinkStep * wave;
  if (k < a.k) {
    one.load(x, m, k, a.k);
    two.load(x, m, k + kNext, a.k);
  }
  double far[T][4] = {};
  for (int end = kSpan; k < a.k; end += kSpan) {
    for (; k < (LONG ? min(a.k, end) : a.k); k += 2 * kNext) {
      step(one, k);
      if (k + kNext < a.k) step(two, k + kNext);
    }
    if (!LONG) break;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        far[t][e] += (double)acc[t][e];
        acc[t][e] = k < a.k ? 0.0f : (float)far[t][e];
      }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < T; ++t) sh.part[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= T) return;
  const int at = at0 + 16 * wave + 4 * (lane / 16), m16 = lane & 15;
  v4f sum = sh.part[0][wave][lane];
#pragma unroll
  for (int w = 1; w < kShrinkWaves; ++w) sum += sh.part[w][wave][lane];
  const bool has = m16 < tile.rows && at < all;
  // Pieces don't make up an infinity, nor a value that rounds to an infinite bf16; sums of such ones
  // are never finite, and are done over without pieces, one after the other.
  if (__any(has && !finite(largest(0.0f, sum)))) {
    uint64_t rows = __ballot(has && !finite(largest(0.0f, sum)));
    rows = (rows | rows >> 16 | rows >> 32 | rows >> 48) & 0xffff;
    uint64_t nan = 0;  // rows with NaN among the inputs, whose sums are what they should be
    for (; rows != 0; rows &= rows - 1) {
      const int r = __ffsll((unsigned long long)rows) - 1;
      const float *x = a.src + (tile.row + r) * a.src_stride;
      float most = 0.0f;
#pragma unroll 4
      for (int c = 4 * lane; c < a.k; c += 256)
        most = largest(most, *reinterpret_cast<const v4f *>(x + c));
      if (__any(most != most)) nan |= 1ull << r;
    }
    for (int e = 0; e < 4; ++e) {
      const float mine = e == 0 ? sum[0] : e == 1 ? sum[1] : e == 2 ? sum[2] : sum[3];
      uint64_t bad = __ballot(has && !finite(mine) && (nan >> m16 & 1) == 0);
      for (; bad != 0; bad &= bad - 1) {
        const int of = __ffsll((unsigned long long)bad) - 1;
        const int u = at0 + 16 * wave + 4 * (of / 16) + e, job = u / a.rank;
        const void *const m[1] = {job_of(a.a, job)};
        const size_t first[1] = {((size_t)tile.id * a.rank + (u - job * a.rank)) * a.k};
        float s[1];
        row_sums<TYPE, LONG, 1>(a.src + (tile.row + of % 16) * a.src_stride, m, first, a.k, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = lane == of && i == e ? s[0] : sum[i];
      }
    }
  }
  if (!has) return;
  sum *= scale_of(a, tile.id);
  const int job = at / a.rank, value = at - job * a.rank;
  // u is the sum of its pieces whatever it is: the first one of a finite value is finite, and those
  // behind the first of another are zeros
  v4f first = sum;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (finite(sum[e])) first[e] = fminf(fmaxf(sum[e], -kBf16Most), kBf16Most);
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    const v4f of = p == 0 ? first : sum;
    const u2 b = {cvt_pk_bf16(of[0], of[1]), cvt_pk_bf16(of[2], of[3])};
    *reinterpret_cast<u2 *>(piece_of(a, tile.row, tile.rows, job, p) +
                            (value / 8 * tile.rows + m16) * 8 + value % 8) = b;
    sum -= v4f{bf16_lo(b[0]), bf16_hi(b[0]), bf16_lo(b[1]), bf16_hi(b[1])};
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = finite(of[e]) ? sum[e] : 0.0f;
  }
}

constexpr int kExpandCols = 64;                // of a wave
constexpr int kExpandPitch = kExpandCols + 4;  // 16 rows' chunks of four in different banks

__host__ __device__ inline int expand_units(const int (&end)[kAdapterMaxJobs], int njobs) {
  int n = 0;
  for (int j = 0; j < njobs; ++j) {
    const int w = end[j] - (j == 0 ? 0 : end[j - 1]);
    n += (w + kExpandCols - 1) / kExpandCols;
  }
  return n;
}

// Where unit u's 64 columns lie: a job, its columns' first and how many it has, the unit's first of
// them.
struct ExpandUnit {
  int job, begin, width, c0;
};
__device__ __forceinline__ ExpandUnit expand_unit(const Adapters &a, int unit) {
  ExpandUnit u = {0, 0, a.end[0], 0};
  for (; u.job < a.njobs; ++u.job) {
    u.begin = u.job == 0 ? 0 : a.end[u.job - 1];
    u.width = a.end[u.job] - u.begin;
    const int units = (u.width + kExpandCols - 1) / kExpandCols;
    if (unit < units) break;
    unit -= units;
  }
  u.c0 = unit * kExpandCols;
  return u;
}

// dst of a row and a unit's 64 columns, by a wave; u: the row's values of the unit's job, in memory or
// LDS.  B's part is one run of memory, read 16 bytes a lane (CHUNKS a row of it at most); their
// products with u meet in LDS, where a lane has a column.
template <int TYPE, int CHUNKS>
struct ExpandRow {
  static constexpr int kSize = TYPE == kAdapterF32 ? 4 : 2, kOf = 16 / kSize;  // weights a chunk
  static constexpr int kFlight = CHUNKS < 8 ? CHUNKS : 8;                      // read together
  static constexpr int kNowhere = kExpandCols * (CHUNKS + 1), kSums = kNowhere + 1;

  u4 w[kFlight];
  float v;

  __device__ __forceinline__ void weights(const Adapters &a, const ExpandUnit &x, int id, int j0) {
    const int all = min(kExpandCols, x.width - x.c0) * (a.rank / kOf);
    const u4 *b = reinterpret_cast<const u4 *>(reinterpret_cast<const char *>(job_of(a.b, x.job)) +
                                               ((size_t)id * x.width + x.c0) * a.rank * kSize);
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const int i = (threadIdx.x & 63) + 64 * (j0 + j);
      w[j] = b[i < all ? i : 0];
    }
  }
  __device__ __forceinline__ void load(const Adapters &a, const ExpandUnit &x, int r, int id) {
    const int c = x.c0 + (threadIdx.x & 63);
    v = c < x.width ? a.base[r * a.base_stride + x.begin + c] : 0.0f;
    if (id >= 0) weights(a, x, id, 0);
  }
  __device__ __forceinline__ void finish(const Adapters &a, const ExpandUnit &x, int r, int id,
                                         const float *u, float (&sums)[kSums]) {
    const int lane = threadIdx.x & 63, c = x.c0 + lane;
    if (id >= 0) {
      const int chunks = a.rank / kOf;
      const unsigned share = (65536 + chunks - 1) / chunks;  // i / chunks is i share / 65536
      for (int j0 = 0;;) {
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
          const int i = lane + 64 * (j0 + j);
          const int col = (int)(i * share >> 16), p = i - col * chunks;
          float s = 0.0f;
          if constexpr (TYPE == kAdapterF32) {
            const v4f at = *reinterpret_cast<const v4f *>(u + kOf * p);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(at[e], __uint_as_float(w[j][e]), s);
          } else {
            float f[8];
            floats8<TYPE>(Raw8<TYPE>{{w[j]}}, f);
            const v4f lo = *reinterpret_cast<const v4f *>(u + kOf * p);
            const v4f hi = *reinterpret_cast<const v4f *>(u + kOf * p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(lo[e], f[e], s), s = fmaf(hi[e], f[e + 4], s);
          }
          // (no branch, which would take the loads with it, one after the other)
          sums[j0 + j < chunks ? col * (chunks + 1) + p : kNowhere] = s;
        }
        j0 += kFlight;
        if (j0 >= chunks) break;
        weights(a, x, id, j0);
      }
      // written and read by the same wave, whose LDS accesses keep their order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float s = 0.0f;
      for (int p = 0; p < chunks; ++p) s += sums[lane * (chunks + 1) + p];
      v += s;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (c < x.width) a.dst[r * a.dst_stride + x.begin + c] = v;
  }
};

template <int TYPE, int CHUNKS>
__global__ __launch_bounds__(kThreads) void adapter_expand_row_kernel(Adapters a) {
  typedef ExpandRow<TYPE, CHUNKS> Expand;
  __shared__ float sums[kThreads / 64][Expand::kSums];
  const int r = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const ExpandUnit x = expand_unit(a, blockIdx.y * (kThreads / 64) + wave);
  if (x.job == a.njobs) return;
  const int id = ids_of(a)[r];
  if (id == kOutside) return;
  Expand e;
  e.load(a, x, r, id);
  e.finish(a, x, r, id, u_of(a) + ((size_t)r * a.njobs + x.job) * a.rank, sums[wave]);
}

// Both products of a row by one workgroup, u in LDS: a launch less (of 3.7 us on the host), where a row
// has little to read.
constexpr int kRowWaves = 16, kRowValues = 4;  // values of u a wave has in flight
template <int TYPE, int CHUNKS, bool LONG>
__global__ __launch_bounds__(64 * kRowWaves) void adapter_row_kernel(Adapters a, int units) {
  typedef ExpandRow<TYPE, CHUNKS> Expand;
  __shared__ float u[kAdapterMaxJobs * kAdapterMaxRank];
  __shared__ float sums[kRowWaves][Expand::kSums];
  const int r = blockIdx.x, all = a.njobs * a.rank, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int id = id_of_row(a, r);
  if (id == kOutside) return;
  if (id >= 0) {
    const float *x = a.src + r * a.src_stride;
    for (int at0 = wave; at0 < all; at0 += kRowWaves * kRowValues) {
      const void *m[kRowValues];
      size_t first[kRowValues];
      float s[kRowValues];
#pragma unroll
      for (int t = 0; t < kRowValues; ++t) {
        const int at = min(at0 + t * kRowWaves, all - 1), job = at / a.rank;
        m[t] = job_of(a.a, job);
        first[t] = ((size_t)id * a.rank + (at - job * a.rank)) * a.k;
      }
      row_sums<TYPE, LONG, kRowValues>(x, m, first, a.k, s);
#pragma unroll
      for (int t = 0; t < kRowValues; ++t) {
        const int at = at0 + t * kRowWaves;
        if (lane == 0 && at < all) u[at] = scale_of(a, id) * s[t];
      }
    }
  }
  __syncthreads();
  for (int unit = wave; unit < units; unit += kRowWaves) {
    const ExpandUnit x = expand_unit(a, unit);
    Expand e;
    e.load(a, x, r, id);
    e.finish(a, x, r, id, u + x.job * a.rank, sums[wave]);
  }
}

// dst of 16 RT rows and 64 columns of a job a wave; KS: steps of 32 of the rank.  base and dst are
// read and written by whole runs of 256 bytes; the products, whose lanes have a row each, go through
// LDS.  A workgroup's four waves are WR times as many rows by 4 / WR times as many columns: 4 by 1,
// which read B once, by whole runs, and share its pieces in LDS, or, for short sequences, 1 by 4.
template <int TYPE, int KS, int RT, int WR>
__global__ __launch_bounds__(kThreads, TYPE == kAdapterF32               ? (WR > 1 ? 2 : 3)
                                       : KS == 1 && TYPE == kAdapterBf16 ? 4
                                                                         : 3)
void adapter_expand_kernel(Adapters a) {
  constexpr int kSize = TYPE == kAdapterF32 ? 4 : 2, kWaves = kThreads / 64;
  constexpr int kP = kPieces<TYPE>, kPitch = 64 * KS + 16;  // of a row of B's pieces: 16 in all banks
  constexpr int kLoads = kExpandCols * 32 * KS * kSize / 16 / kThreads;
  __shared__ float tiles[kWaves][16 * RT][kExpandPitch];
  __shared__ char shared[WR > 1 ? kP : 1][WR > 1 ? kExpandCols : 1][kPitch];
  const int lane = threadIdx.x & 63, m = lane & 15, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const ExpandUnit x = expand_unit(a, WR > 1 ? blockIdx.y : blockIdx.y * kWaves + wave);
  const int job = x.job, begin = x.begin, width = x.width, c0 = x.c0;
  if (job == a.njobs) return;
  float(&sums)[16 * RT][kExpandPitch] = tiles[wave];
  Tile tile = tile_at<16 * RT * WR>(a, blockIdx.x);
  if (tile.rows <= 0) return;
  const int k0 = 8 * quarter;
  const char *b = reinterpret_cast<const char *>(job_of(a.b, job)) +
                  ((size_t)tile.id * width + c0) * a.rank * kSize;
  const int chunks = a.rank * kSize / 16;  // of a row of B
  u4 part[kLoads];
  if (WR > 1 && tile.id >= 0) {
    const int have = min(kExpandCols, width - c0) * chunks;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = threadIdx.x + kThreads * j;
      part[j] = reinterpret_cast<const u4 *>(b)[i < have ? i : 0];
    }
  }
  if (WR > 1) {
    tile.row += 16 * RT * wave;
    tile.rows = min(tile.rows - 16 * RT * wave, 16 * RT);
  }
  const int last = max(tile.rows, 1) - 1;
  Split8<3> u[RT][KS];
  if (tile.rows > 0 && tile.id >= 0) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int rows = min(tile.rows - 16 * i, 16);  // of a tile of 16
      if (rows <= 0) {
#pragma unroll
        for (int s = 0; s < KS; ++s) u[i][s] = u[0][s];
        continue;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const int k = 32 * s + k0, at = (k < a.rank ? k : 0) / 8 * rows + min(m, rows - 1);
          u[i][s].p[p] = *reinterpret_cast<const u4 *>(
              piece_of(a, tile.row + 16 * i, rows, job, p) + at * 8);
        }
    }
  }
  // rows 4 j + quarter, four columns of them from the lane's 4 m
  const int left = width - c0 - 4 * m;
  const size_t col = begin + c0 + 4 * m;
  const bool whole = c0 + kExpandCols <= width;
  v4f old[4 * RT];
  if (tile.rows <= 0) {
    // (a wave that only waits for the others)
  } else if (whole) {
#pragma unroll
    for (int j = 0; j < 4 * RT; ++j) {
      const int row = tile.row + min(4 * j + quarter, last);
      old[j] = __builtin_nontemporal_load(  // read once
          reinterpret_cast<const v4f_any *>(a.base + row * a.base_stride + col));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4 * RT; ++j) {
      const int row = tile.row + min(4 * j + quarter, last);
      old[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) old[j][e] = a.base[row * a.base_stride + col + e];
    }
  }
  if (WR > 1) {
    if (tile.id >= 0) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = threadIdx.x + kThreads * j;
        if (i >= kExpandCols * chunks) continue;
        const int row = i / chunks, at = i - row * chunks;
        if constexpr (TYPE == kAdapterF32) {
          v4f left = __builtin_bit_cast(v4f, part[j]);
#pragma unroll
          for (int p = 0; p < kP; ++p) {
            const u2 q = {cvt_pk_bf16(left[0], left[1]), cvt_pk_bf16(left[2], left[3])};
            *reinterpret_cast<u2 *>(&shared[p][row][8 * at]) = q;
            left -= v4f{bf16_lo(q[0]), bf16_hi(q[0]), bf16_lo(q[1]), bf16_hi(q[1])};
          }
        } else {
          const Split8<kP> q = pieces8<TYPE>(Raw8<TYPE>{{part[j]}});
#pragma unroll
          for (int p = 0; p < kP; ++p) *reinterpret_cast<u4 *>(&shared[p][row][16 * at]) = q.p[p];
        }
      }
      const int pads = 4 * KS - a.rank / 8;  // of 16 bytes, behind the rank
      for (int i = threadIdx.x; i < kP * kExpandCols * pads; i += kThreads) {
        const int row = i / pads, at = a.rank / 8 + i - row * pads;
        *reinterpret_cast<u4 *>(&shared[row / kExpandCols][row % kExpandCols][16 * at]) = u4{0, 0, 0, 0};
      }
    }
    lds_barrier();
  }
  if (tile.rows <= 0) return;
  if (tile.id >= 0) {
    // values behind the rank are zeros on both sides
    constexpr int W = KS < 4 && (KS == 1 || TYPE != kAdapterF32) ? 4 : 2;  // read together
    float most = 0.0f;  // of the products' magnitudes
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (auto &v : u[i][s].p) v = 32 * s + k0 < a.rank ? v : u4{0, 0, 0, 0};
#pragma unroll
    for (int t0 = 0; t0 < 4; t0 += W) {
      Raw8<TYPE> w[W][KS];
      if (WR == 1) {
#pragma unroll
        for (int t = 0; t < W; ++t)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int c = 16 * (t0 + t) + m, k = 32 * s + k0 < a.rank ? 32 * s + k0 : 0;
            w[t][s] = raw8<TYPE>(b, (size_t)min(c, width - c0 - 1) * a.rank + k);
          }
      }
#pragma unroll
      for (int t = 0; t < W; ++t) {
        v4f d[RT] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          Split8<kP> wp;
          if (WR > 1) {
#pragma unroll
            for (int p = 0; p < kP; ++p)
              wp.p[p] = *reinterpret_cast<const u4 *>(
                  &shared[p][16 * (t0 + t) + m][64 * s + 16 * quarter]);
          } else {
            Raw8<TYPE> v = w[t][s];
#pragma unroll
            for (auto &x : v.v) x = 32 * s + k0 < a.rank ? x : u4{0, 0, 0, 0};
            wp = pieces8<TYPE>(v);
          }
#pragma unroll
          for (int i = 0; i < RT; ++i) d[i] = product(wp, u[i][s], d[i]);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          *reinterpret_cast<v4f *>(&sums[16 * i + m][16 * (t0 + t) + 4 * quarter]) = d[i];
          most = largest(most, d[i]);
        }
      }
    }
    // written and read by the same wave, whose LDS accesses keep their order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (__any(!finite(most))) {  // as in the first product; a lane a column
      uint64_t nan = 0;  // rows with NaN among u
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int rows = min(tile.rows - 16 * i, 16);
        bool some = false;
        for (int k = k0; k < a.rank && m < rows; k += 32) {
          const u4 p = *reinterpret_cast<const u4 *>(piece_of(a, tile.row + 16 * i, rows, job, 0) +
                                                     (k / 8 * rows + m) * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            some = some || bf16_lo(p[e]) != bf16_lo(p[e]) || bf16_hi(p[e]) != bf16_hi(p[e]);
        }
        const uint64_t all = __ballot(some);
        nan |= ((all | all >> 16 | all >> 32 | all >> 48) & 0xffff) << 16 * i;
      }
      for (int r = 0; r < tile.rows; ++r) {
        const bool bad = c0 + lane < width && !finite(sums[r][lane]) && (nan >> r & 1) == 0;
        if (!__any(bad)) continue;
        const int rows = min(tile.rows - r / 16 * 16, 16);
        const size_t row = (size_t)(bad ? lane : 0) * a.rank;
        float s = 0.0f;
        for (int k = 0; k < a.rank; k += 8) {
          float w[8];
          floats8<TYPE>(raw8<TYPE>(b, row + k), w);
          Split8<3> v;
#pragma unroll
          for (int p = 0; p < 3; ++p)
            v.p[p] = *reinterpret_cast<const u4 *>(
                piece_of(a, tile.row + r / 16 * 16, rows, job, p) + (k / 8 * rows + r % 16) * 8);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float x = 0.0f;
#pragma unroll
            for (int p = 2; p >= 0; --p)
              x += e % 2 ? bf16_hi(v.p[p][e / 2]) : bf16_lo(v.p[p][e / 2]);
            s = fmaf(x, w[e], s);
          }
        }
        if (bad) sums[r][lane] = s;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int j = 0; j < 4 * RT; ++j)
      old[j] += *reinterpret_cast<const v4f *>(&sums[4 * j + quarter][4 * m]);
  }
#pragma unroll
  for (int j = 0; j < 4 * RT; ++j) {
    const int r = 4 * j + quarter;
    if (r >= tile.rows) break;
    float *p = a.dst + (tile.row + r) * a.dst_stride + col;
    if (whole) {
      *reinterpret_cast<v4f_any *>(p) = old[j];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) p[e] = old[j][e];
    }
  }
}

// Up to so many rows a sequence go by the row: with more, a tile's 16 rows share what is read.
constexpr int kFewRows = 2;
// Bytes of an adapter's matrices up to which a row is one workgroup's.  The rule is for eager calls,
// where the host's launches set the time; a graph of few tokens pays for it.  us a call by two launches
// and by one, in a row of eager ones: 1 row of 80 KiB 11.0, 8.8, of 156 KiB 10.7, 8.8, of 234 KiB
// 10.4, 9.5; 32 rows 10.3, 8.3, then 10.2, 8.4, then 10.1, 10.4; 64 rows 10.1, 8.3, then 10.2, 8.3, then
// 10.0, 11.6; 200 rows 10.0, 8.4, then 11.1, 9.0, then 15.2, 12.2.  In a graph: 1 row 5.4, 6.7, then
// 5.4, 6.8, then 6.0, 9.1; 32 rows 5.6, 7.0, then 5.7, 7.1, then 6.9, 10.1; 64 rows 6.0, 7.2, then
// 6.6, 7.4, then 9.1, 11.4; 200 rows 7.7, 7.7, then 11.1, 8.9, then 15.2, 12.2.
constexpr long kRowBytes = 192 << 10;

}  // namespace

size_t adapters_work(int rows, int njobs, int rank) {
  return ((size_t)rows * (njobs * rank * 6 + 4) + 255) / 256 * 256;
}

bool adapters_one_launch(const Adapters &a) {
  const long weights = (long)a.njobs * a.rank * a.k + (long)a.end[a.njobs - 1] * a.rank;
  return a.seq.max_rows <= kFewRows && weights * (a.type == kAdapterF32 ? 4 : 2) <= kRowBytes &&
         a.seq.rows <= 1 << 21;  // (a grid has 2^32 - 1 threads at most)
}

hipError_t launch_adapters(const Adapters &a, const DeviceInfo &dev, hipStream_t stream) {
  const int rows = a.seq.rows, all = a.njobs * a.rank;
  auto by_row = [&](auto type) {
    constexpr int kSize = type() == kAdapterF32 ? 4 : 2;
    const int units = expand_units(a.end, a.njobs);
    auto go = [&](auto chunks) {
      if (adapters_one_launch(a)) {
        a.k > kSpan ? adapter_row_kernel<type(), chunks(), true>
                          <<<rows, 64 * kRowWaves, 0, stream>>>(a, units)
                    : adapter_row_kernel<type(), chunks(), false>
                          <<<rows, 64 * kRowWaves, 0, stream>>>(a, units);
      } else {
        const dim3 first(rows, (all + 3) / 4), second(rows, (units + 3) / 4);
        a.k > kSpan ? adapter_shrink_row_kernel<type(), true><<<first, kThreads, 0, stream>>>(a)
                    : adapter_shrink_row_kernel<type(), false><<<first, kThreads, 0, stream>>>(a);
        adapter_expand_row_kernel<type(), chunks()><<<second, kThreads, 0, stream>>>(a);
      }
    };
    a.rank * kSize <= 32    ? go(std::integral_constant<int, 2>())
    : a.rank * kSize <= 128 ? go(std::integral_constant<int, 8>())
                            : go(std::integral_constant<int, kAdapterMaxRank * kSize / 16>());
  };
  const int slots = tile_slots(a.seq, 16);
  auto shrink = [&](auto type, auto t) {
    const dim3 grid(slots, (all + 16 * t() - 1) / (16 * t()));
    a.k > kSpan
        ? adapter_shrink_kernel<type(), t(), true><<<grid, 64 * kShrinkWaves, 0, stream>>>(a)
        : adapter_shrink_kernel<type(), t(), false><<<grid, 64 * kShrinkWaves, 0, stream>>>(a);
  };
  auto expand = [&](auto type, auto ks, auto rt) {
    constexpr int kWaves = kThreads / 64, R = 16 * rt();
    const int units = expand_units(a.end, a.njobs);
    if (a.seq.max_rows > 2 * R)
      adapter_expand_kernel<type(), ks(), rt(), kWaves>
          <<<dim3(tile_slots(a.seq, R * kWaves), units), kThreads, 0, stream>>>(a);
    else
      adapter_expand_kernel<type(), ks(), rt(), 1>
          <<<dim3(tile_slots(a.seq, R), (units + kWaves - 1) / kWaves), kThreads, 0, stream>>>(a);
  };
  auto go = [&](auto type) {
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    if (a.seq.max_rows <= kFewRows) return by_row(type);
    // 16 values of u a workgroup until there is one for every compute unit, then more, which share x
    // (851 rows with 128 values: 16 each 13.9 us, 32 each 12.9)
    const int tiles = (all + 15) / 16;
    tiles == 1 || (long)slots * tiles <= dev.cus ? shrink(type, one)
    : tiles % kMostT != 0                            ? shrink(type, two)
                                                     : shrink(type, integral_constant<int, kMostT>());
    a.rank <= 32   ? expand(type, one, two)
    : a.rank <= 64 ? expand(type, two, two)
                   : expand(type, integral_constant<int, 4>(), one);
  };
  a.type == kAdapterF32    ? go(std::integral_constant<int, kAdapterF32>())
  : a.type == kAdapterBf16 ? go(std::integral_constant<int, kAdapterBf16>())
                           : go(std::integral_constant<int, kAdapterF16>());
  return hipGetLastError();
}

}  // namespace gh
