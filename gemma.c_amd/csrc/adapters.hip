// adapters.hip -- low-rank adapters of many requests on one batch of rows.
//
//   u = A[id] x  (rank values a job),  dst = base + scale[id] B[id] u
//
// id is that of the row's sequence; jobs are projections side by side (q, k, v; gate, up).  A launch
// for the first product, whose fp32 results lie in the workspace, and one for the second.
#include <type_traits>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kThreads = 256;

// eight neighbouring weights
template <int TYPE>
__device__ __forceinline__ void load8(const void *p, size_t at, float (&w)[8]) {
  if (TYPE == kAdapterF32) {
    const v4f a = *reinterpret_cast<const v4f *>((const float *)p + at);
    const v4f b = *reinterpret_cast<const v4f *>((const float *)p + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = a[e], w[e + 4] = b[e];
  } else if (TYPE == kAdapterBf16) {
    const u4 a = *reinterpret_cast<const u4 *>((const uint16_t *)p + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[2 * e] = bf16_lo(a[e]), w[2 * e + 1] = bf16_hi(a[e]);
  } else {
    const h8 a = *reinterpret_cast<const h8 *>((const uint16_t *)p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (float)a[e];
  }
}

// The adapter of row r, -1: none; -2: the row is in no sequence.
__device__ __forceinline__ int adapter_of(const Adapters &a, int r) {
  const KvRow row = kv_row_wave<false>(a.seq, r);
  if (row.i < 0) return -2;
  const int id = a.ids[row.i];
  return (unsigned)id < (unsigned)a.count ? id : -1;
}

// a wave for one value of u
template <int TYPE>
__global__ __launch_bounds__(kThreads) void adapter_shrink_kernel(Adapters a) {
  const int all = a.njobs * a.rank, lane = threadIdx.x & 63, r = blockIdx.x;
  const int at = blockIdx.y * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int job = at / a.rank, row = at % a.rank;
  if (at >= all) return;
  const int id = adapter_of(a, r);
  if (id < 0) return;
  const void *m = job == 0 ? a.a[0] : job == 1 ? a.a[1] : a.a[2];
  const size_t first = ((size_t)id * a.rank + row) * a.k;
  const float *x = a.src + r * a.src_stride;
  float s = 0.0f;
  for (int c = 8 * lane; c < a.k; c += 512) {
    float w[8];
    load8<TYPE>(m, first + c, w);
    const v4f x0 = *reinterpret_cast<const v4f *>(x + c);
    const v4f x1 = *reinterpret_cast<const v4f *>(x + c + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(x0[e], w[e], s), s = fmaf(x1[e], w[e + 4], s);
  }
  s = group_sum_f32<64>(s);
  if (lane == 0) reinterpret_cast<float *>(a.work)[(size_t)r * all + at] = s;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void adapter_expand_kernel(Adapters a) {
  const int n = a.end[a.njobs - 1], r = blockIdx.x;
  const int c = blockIdx.y * kThreads + threadIdx.x;
  const int id = adapter_of(a, r);
  if (id == -2 || c >= n) return;
  float v = a.base[r * a.base_stride + c];
  if (id >= 0) {
    const int job = c < a.end[0] ? 0 : a.njobs > 1 && c < a.end[1] ? 1 : a.njobs > 1 ? 2 : 0;
    const int from = job == 0 ? 0 : a.end[job - 1];
    const void *m = job == 0 ? a.b[0] : job == 1 ? a.b[1] : a.b[2];
    const size_t first = ((size_t)id * (a.end[job] - from) + (c - from)) * a.rank;
    const float *u = reinterpret_cast<const float *>(a.work) +
                     (size_t)r * a.njobs * a.rank + job * a.rank;
    float s = 0.0f;
    for (int k = 0; k < a.rank; k += 8) {
      float w[8];
      load8<TYPE>(m, first + k, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(u[k + e], w[e], s);
    }
    v += (a.scale != nullptr ? a.scale[id] : 1.0f) * s;
  }
  a.dst[r * a.dst_stride + c] = v;
}

}  // namespace

size_t adapters_work(int rows, int njobs, int rank) {
  return ((size_t)rows * njobs * rank * 4 + 255) / 256 * 256;
}

hipError_t launch_adapters(const Adapters &a, const DeviceInfo &dev, hipStream_t stream) {
  auto go = [&](auto type) {
    const dim3 first(a.seq.rows, (a.njobs * a.rank + 3) / 4);
    adapter_shrink_kernel<type()><<<first, kThreads, 0, stream>>>(a);
    const dim3 grid(a.seq.rows, (a.end[a.njobs - 1] + kThreads - 1) / kThreads);
    adapter_expand_kernel<type()><<<grid, kThreads, 0, stream>>>(a);
  };
  a.type == kAdapterF32    ? go(std::integral_constant<int, kAdapterF32>())
  : a.type == kAdapterBf16 ? go(std::integral_constant<int, kAdapterBf16>())
                           : go(std::integral_constant<int, kAdapterF16>());
  return hipGetLastError();
}

}  // namespace gh
