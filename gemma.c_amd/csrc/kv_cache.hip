// kv_cache.hip -- keys and values into the paged 8-bit cache, and back.
//
// A row of a head (hdim values) becomes hdim codes and one scale.  int8 codes
// follow gemma_hip_quantize's arithmetic (amax (1/127), x (127/amax), halves away
// from zero); e4m3 codes are x (448/amax) rounded to nearest even by the
// conversion instruction.  A row of zeros has scale 0; a row that holds a NaN or
// an infinity has codes of 0 and a NaN for its scale: whoever sees it answers
// NaN, and whoever doesn't multiplies finite codes by a weight of 0.
//
// One group of hdim / 4 lanes per row and head, 16 bytes a lane: each value is
// read once and stays in registers between the maximum and the codes.  Bound by
// memory for prompts (5 bytes and a part of a scale move per value, each way): four of up to
// 4096 rows of gemma-3-4b are written in 26 us and read in 21, 3.7 and 4.6 TB/s of the 5.1
// that a large copy reaches; by the launch for single tokens (3 us each).
#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

constexpr int kThreads = 256;

// What a group of lanes works on: one head of one row, its keys or its values.
struct KvUnit {
  int row, h;
  bool isv;
  long slot;  // -1: none
};

// Units are numbered row-major over (row, keys or values, head) of a sequence.
template <int HD>
__device__ __forceinline__ bool kv_unit(const KvCache &c, const KvBatch &b, KvUnit *u) {
  constexpr int G = HD / 4;  // lanes of a unit
  const int seq = blockIdx.y;
  const KvSeq s = kv_seq(b, seq);
  const int per = 2 * c.nkv;
  const long unit = (long)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const int i = (int)(unit / per), j = (int)(unit % per);
  if (i >= s.n) return false;
  u->row = s.r0 + i;
  u->isv = j >= c.nkv;
  u->h = u->isv ? j - c.nkv : j;
  const int pos = s.len - s.n + i;
  u->slot = pos < 0 ? -1 : kv_slot(c, b, seq, pos, u->h);
  return true;
}

template <int HD, int TYPE>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvCache c, KvBatch b, const float *k,
                                                            int k_stride, const float *v,
                                                            int v_stride) {
  constexpr int G = HD / 4;
  KvUnit u;
  if (!kv_unit<HD>(c, b, &u) || u.slot < 0) return;  // whole groups at a time
  const int lane = threadIdx.x % G;
  const float *src = u.isv ? v + (size_t)u.row * v_stride : k + (size_t)u.row * k_stride;
  const v4f x = *reinterpret_cast<const v4f *>(src + u.h * HD + 4 * lane);
  // the bits of magnitudes order as they do, what isn't finite above all
  int top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_int(x[e]) & 0x7fffffff);
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
  const bool finite = top < 0x7f800000;
  const float amax = finite ? daz(__int_as_float(top)) : 0.0f;
  uint32_t q = 0;
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
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      q = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], t, true);
    }
  }
  uint8_t *dst = u.isv ? c.v : c.k;
  *reinterpret_cast<uint32_t *>(dst + (size_t)u.slot * HD + 4 * lane) = q;
  if (lane == 0) (u.isv ? c.vs : c.ks)[u.slot] = finite ? scale : __int_as_float(0x7fc00000);
}

template <int HD, int TYPE>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvCache c, KvBatch b, float *k,
                                                           int k_stride, float *v, int v_stride) {
  constexpr int G = HD / 4;
  KvUnit u;
  if (!kv_unit<HD>(c, b, &u)) return;
  const int lane = threadIdx.x % G;
  v4f x = {};
  if (u.slot >= 0) {
    const uint32_t q =
        *reinterpret_cast<const uint32_t *>((u.isv ? c.v : c.k) + (size_t)u.slot * HD + 4 * lane);
    const float scale = (u.isv ? c.vs : c.ks)[u.slot];
    if (TYPE == kKvI8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (float)(int8_t)(q >> (8 * e)) * scale;
    } else {
      x = v4f{__builtin_amdgcn_cvt_f32_fp8(q, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(q, 1) * scale,
              __builtin_amdgcn_cvt_f32_fp8(q, 2) * scale, __builtin_amdgcn_cvt_f32_fp8(q, 3) * scale};
    }
  }
  float *dst = u.isv ? v + (size_t)u.row * v_stride : k + (size_t)u.row * k_stride;
  *reinterpret_cast<v4f *>(dst + u.h * HD + 4 * lane) = x;
}

dim3 kv_grid(const KvCache &c, const KvBatch &b) {
  const long units = (long)b.max_rows * 2 * c.nkv, per = kThreads / (c.hdim / 4);
  return dim3((unsigned)((units + per - 1) / per), b.batch);
}

}  // namespace

hipError_t launch_kv_write(const KvCache &c, const KvBatch &b, const float *k, int k_stride,
                           const float *v, int v_stride, hipStream_t stream) {
  auto go = [&](auto kernel) {
    kernel<<<kv_grid(c, b), kThreads, 0, stream>>>(c, b, k, k_stride, v, v_stride);
  };
  if (c.hdim == 256)
    c.type == kKvI8 ? go(kv_write_kernel<256, kKvI8>) : go(kv_write_kernel<256, kKvE4m3>);
  else
    c.type == kKvI8 ? go(kv_write_kernel<128, kKvI8>) : go(kv_write_kernel<128, kKvE4m3>);
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvCache &c, const KvBatch &b, float *k, int k_stride, float *v,
                          int v_stride, hipStream_t stream) {
  auto go = [&](auto kernel) {
    kernel<<<kv_grid(c, b), kThreads, 0, stream>>>(c, b, k, k_stride, v, v_stride);
  };
  if (c.hdim == 256)
    c.type == kKvI8 ? go(kv_read_kernel<256, kKvI8>) : go(kv_read_kernel<256, kKvE4m3>);
  else
    c.type == kKvI8 ? go(kv_read_kernel<128, kKvI8>) : go(kv_read_kernel<128, kKvE4m3>);
  return hipGetLastError();
}

}  // namespace gh
