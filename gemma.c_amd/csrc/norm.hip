// norm.hip -- what lies between two blocks: the norm behind the one, its gate and scales, the
// residual sum, the norm in front of the other, and the codes for its first product.
//
//   z = N(y),  x' = clamp(cx x + cy g z),  h = N'(x'),  codes of h as gemma_hip_quantize makes them
//
// N(v) = (v - mean) / sqrt(var + eps) (w + offset) + b, the mean taken off or not.  Everything is
// fp64 between the roundings of x' and of h to fp32, so that h's codes are the exact ones but where
// a border between two is hit to 1e-15.
//
// A wave or a workgroup has a row, which stays in registers from its loads to its stores: each value
// is read and written once, and the bytes bound it: 4096 rows of 2560 with x, y, x' and h (168 MB) 37
// us, 4.5 TB/s (a copy 5.1); 2560 rows of 4096 the same, 1700 rows of 6144 43.
#include <type_traits>

#include "dec_common.h"
#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kNormNone = 0, kNormLayer = 2;
constexpr int kThreads = 256;  // of a workgroup whose waves have a row each

// Sum and largest over a row's NT threads.
template <int NT>
__device__ __forceinline__ double row_sum(double v, double *red) {
  return NT == 64 ? wave_sum_f64(v) : block_sum<NT>(v, red);
}
template <int NT>
__device__ __forceinline__ float row_max(float v, float *red) {
  return NT == 64 ? wave_max_dpp(v) : block_max<NT>(v, red);
}

// rows' chunks of four: NPT a thread, chunk j of thread t is t + j NT; read past the caches' order of
// use, as they are read once (4096 rows of 2560: 39 -> 37 us)
template <int NPT, int NT>
__device__ __forceinline__ void row_load(const float *p, int n4, v4f (&v)[NPT]) {
#pragma unroll
  for (int j = 0; j < NPT; ++j) {
    const int c = threadIdx.x % NT + j * NT;
    v[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (c < n4) v[j] = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(p) + c);
  }
}

// What a norm does to a value: (v - mean) * m.
struct Moments {
  double mean, m;
};
template <int NPT, int NT>
__device__ Moments moments(const v4f (&v)[NPT], const NormOf &n, int dim, double *red) {
  Moments r = {0.0, 1.0};
  if (n.kind == kNormNone) return r;
  double s = 0.0;
  if (n.kind == kNormLayer) {
#pragma unroll
    for (int j = 0; j < NPT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)v[j][e];
    r.mean = row_sum<NT>(s, red) / (double)dim;
    s = 0.0;
  }
#pragma unroll
  for (int j = 0; j < NPT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool there = 4 * (int)(threadIdx.x % NT + j * NT) < dim;
      const double d = there ? (double)v[j][e] - r.mean : 0.0;
      s = fma(d, d, s);
    }
  r.m = rms_of(row_sum<NT>(s, red), dim, n.eps);
  return r;
}

__device__ __forceinline__ v4f or_else(const float *p, int c, float other) {
  if (p == nullptr) return v4f{other, other, other, other};
  return reinterpret_cast<const v4f *>(p)[c];
}

// rounded, as the reference clamps its sums (clamp_fpx, gemma.c:2504-2506), NaN kept
__device__ __forceinline__ float clamped(double v) {
  return v > (double)FLT_MAX ? FLT_MAX : v < -(double)FLT_MAX ? -FLT_MAX : (float)v;
}

// NT threads a row: 64, a wave, without barriers, or a workgroup
template <int NPT, int NT>
__global__ __launch_bounds__(NT == 64 ? kThreads : NT) void norm_residual_kernel(NormResidual a) {
  __shared__ double red[NT / 64];
  __shared__ float redf[NT / 64];
  const int tid = threadIdx.x % NT, n4 = a.dim >> 2;
  int r = blockIdx.x;
  if (NT == 64) {
    r = r * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (r >= a.rows) return;
  }
  v4f x[NPT], y[NPT];
  row_load<NPT, NT>(a.x + r * a.x_stride, n4, x);
  if (a.y != nullptr) {
    row_load<NPT, NT>(a.y + r * a.y_stride, n4, y);
    const Moments mo = moments<NPT, NT>(y, a.after, a.dim, red);
    const bool plain = a.after.kind == kNormNone;
    const double off = a.after.w != nullptr ? (double)a.after.offset : 1.0;
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int c = tid + j * NT;
      if (c >= n4) continue;
      const v4f w = or_else(a.after.w, c, 0.0f);
      const v4f b = or_else(a.after.b, c, 0.0f);
      const v4f g = or_else(a.gate != nullptr ? a.gate + r * a.gate_stride : nullptr, c, 1.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        double z = (double)y[j][e];
        if (!plain)
          z = (z - mo.mean) * mo.m * ((double)w[e] + off) + (double)b[e];
        const double sum = (double)a.cx * (double)x[j][e] + (double)a.cy * (double)g[e] * z;
        x[j][e] = clamped(sum);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < NPT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[j][e] = a.cx != 1.0f                    ? clamped((double)a.cx * (double)x[j][e])
                  : fabsf(x[j][e]) == INFINITY ? copysignf(FLT_MAX, x[j][e])
                                               : x[j][e];
  }
  if (a.x_out != nullptr)
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (tid + j * NT < n4)
        reinterpret_cast<v4f *>(a.x_out + r * a.out_stride)[tid + j * NT] = x[j];
  if (a.h == nullptr && a.hq == nullptr) return;
  const Moments mo = moments<NPT, NT>(x, a.before, a.dim, red);
  const double off = a.before.w != nullptr ? (double)a.before.offset : 1.0;
  if (a.before.kind != kNormNone)
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int c = tid + j * NT;
      if (c >= n4) continue;
      const v4f w = or_else(a.before.w, c, 0.0f);
      const v4f b = or_else(a.before.b, c, 0.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[j][e] = (float)(((double)x[j][e] - mo.mean) * mo.m *
                              ((double)w[e] + off) +
                          (double)b[e]);
    }
  if (a.h != nullptr)
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (tid + j * NT < n4) reinterpret_cast<v4f *>(a.h + r * a.h_stride)[tid + j * NT] = x[j];
  if (a.hq == nullptr) return;
  // the bits of magnitudes order as they do, what isn't finite above all
  float amax = 0.0f;
  bool finite = true;
#pragma unroll
  for (int j = 0; j < NPT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      finite = finite && fabsf(x[j][e]) <= FLT_MAX;
      amax = fmaxf(amax, abs_daz(x[j][e]));
    }
  amax = row_max<NT>(finite ? amax : INFINITY, redf);
  finite = amax <= FLT_MAX;
  const QuantParams qp = quant_params(finite ? amax : 0.0f);
#pragma unroll
  for (int j = 0; j < NPT; ++j) {
    const int c = tid + j * NT;
    if (c < n4)
      reinterpret_cast<uint32_t *>(a.hq + r * a.hq_stride)[c] =
          finite ? pack4(quant_one(x[j][0], qp.inv), quant_one(x[j][1], qp.inv),
                         quant_one(x[j][2], qp.inv), quant_one(x[j][3], qp.inv))
                 : 0u;
  }
  if (tid == 0) a.hs[r] = finite ? qp.scale : __int_as_float(0x7fc00000);
}

}  // namespace

hipError_t launch_norm_residual(const NormResidual &a, const DeviceInfo &dev,
                                hipStream_t stream) {
  using std::integral_constant;
  const int n4 = a.dim / 4;
  auto go = [&](auto npt, auto nt) {
    constexpr int rows = nt() == 64 ? kThreads / 64 : 1;
    norm_residual_kernel<npt(), nt()>
        <<<(a.rows + rows - 1) / rows, nt() == 64 ? kThreads : nt(), 0, stream>>>(a);
  };
  auto by = [&](auto nt, auto least) {
    const int npt = (n4 + nt() - 1) / nt();
    constexpr int kLeast = least(), kMost = nt() < 256 ? 3 : 6;
    if constexpr (kLeast <= 1) {
      if (npt <= 1) return go(integral_constant<int, 1>(), nt);
    }
    if (npt <= 2) return go(integral_constant<int, 2>(), nt);
    if (npt <= 3 || kMost == 3) return go(integral_constant<int, 3>(), nt);
    if constexpr (kMost > 3)
      npt <= 4   ? go(integral_constant<int, 4>(), nt)
      : npt <= 5 ? go(integral_constant<int, 5>(), nt)
                 : go(integral_constant<int, kMost>(), nt);
  };
  // Few rows have a workgroup each, so that a row takes as little time as it can.  Of many, threads
  // have three chunks at most, which leaves room for other rows' waves, and few are without any:
  // us of 20000 rows of 256 with 64, 128 and 256 threads a row 22, 29, 43, of 8192 rows of 1152 42,
  // 34, 38, of 4096 rows of 2560 (128 and 256) 46, 37.
  const bool many = a.rows > 4 * dev.cus;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  many && n4 <= 3 * 64     ? by(integral_constant<int, 64>(), one)
  : many && n4 <= 3 * 128 ? by(integral_constant<int, 128>(), two)
  : n4 <= 6 * 256         ? by(integral_constant<int, 256>(), one)
                          : by(integral_constant<int, 1024>(), two);
  return hipGetLastError();
}

}  // namespace gh
