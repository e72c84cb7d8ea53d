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
#include <type_traits>

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

// Units are numbered row-major over (row, keys or values, head) of a sequence; FLAT: of all
// sequences, whose row is the same for all of a wave.
template <int HD, bool FLAT>
__device__ __forceinline__ bool kv_unit(const KvCache &c, const KvBatch &b, KvUnit *u) {
  constexpr int G = HD / 4;  // lanes of a unit
  const int per = 2 * c.nkv;
  const long unit = kv_block(blockIdx.x, blockIdx.z) * (kThreads / G) + threadIdx.x / G;
  int i = (int)(unit / per);
  const int j = (int)(unit % per);
  static_assert(64 / G <= 2, "a wave's units are of one row, of which there are 2 nkv");
  const int seq = FLAT ? kv_find_wave(b, __builtin_amdgcn_readfirstlane(i)) : blockIdx.y;
  const KvSeq s = kv_seq(b, seq);
  if (FLAT) i -= s.r0;
  if (i < 0 || i >= s.n) return false;
  u->row = s.r0 + i;
  u->isv = j >= c.nkv;
  u->h = u->isv ? j - c.nkv : j;
  const int pos = s.len - s.n + i;
  u->slot = pos < 0 ? -1 : kv_slot(c, b, seq, pos, u->h);
  return true;
}

template <int HD, int TYPE, bool FLAT>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvCache c, KvBatch b, const float *k,
                                                            int k_stride, const float *v,
                                                            int v_stride) {
  constexpr int G = HD / 4;
  KvUnit u;
  if (!kv_unit<HD, FLAT>(c, b, &u) || u.slot < 0) return;  // whole groups at a time
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

template <int HD, int TYPE, bool FLAT>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvCache c, KvBatch b, float *k,
                                                           int k_stride, float *v, int v_stride) {
  constexpr int G = HD / 4;
  KvUnit u;
  if (!kv_unit<HD, FLAT>(c, b, &u)) return;
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

// By sequences times the longest one's rows, or, where most of that would be empty (prompts
// beside single tokens), by the batch's rows, at the price of a search: 2048 rows of
// gemma-3-1b beside 200 single tokens are written in 53 and 4.5 us, 8 single tokens in 2.8
// and 3.0
bool kv_flat(const KvBatch &b) { return (long)b.batch * b.max_rows > 2l * b.rows; }
dim3 kv_grid(const KvCache &c, const KvBatch &b) {
  const long units = (kv_flat(b) ? (long)b.rows : b.max_rows) * 2 * c.nkv;
  const long per = kThreads / (c.hdim / 4);
  const KvGrid g = kv_grid_of((units + per - 1) / per, kv_flat(b) ? 1 : b.batch);
  return dim3(g.x, g.y, g.z);
}

// Calls go(hdim, type, flat) with the constants that fit.
template <class F>
void kv_dispatch(const KvCache &c, const KvBatch &b, F &&go) {
  auto flat = [&](auto hd, auto type) {
    kv_flat(b) ? go(hd, type, std::true_type()) : go(hd, type, std::false_type());
  };
  auto type = [&](auto hd) {
    c.type == kKvI8 ? flat(hd, std::integral_constant<int, kKvI8>())
                    : flat(hd, std::integral_constant<int, kKvE4m3>());
  };
  c.hdim == 256 ? type(std::integral_constant<int, 256>()) : type(std::integral_constant<int, 128>());
}

}  // namespace

hipError_t launch_kv_write(const KvCache &c, const KvBatch &b, const float *k, int k_stride,
                           const float *v, int v_stride, hipStream_t stream) {
  kv_dispatch(c, b, [&](auto hd, auto type, auto flat) {
    kv_write_kernel<hd(), type(), flat()>
        <<<kv_grid(c, b), kThreads, 0, stream>>>(c, b, k, k_stride, v, v_stride);
  });
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvCache &c, const KvBatch &b, float *k, int k_stride, float *v,
                          int v_stride, hipStream_t stream) {
  kv_dispatch(c, b, [&](auto hd, auto type, auto flat) {
    kv_read_kernel<hd(), type(), flat()>
        <<<kv_grid(c, b), kThreads, 0, stream>>>(c, b, k, k_stride, v, v_stride);
  });
  return hipGetLastError();
}

}  // namespace gh
