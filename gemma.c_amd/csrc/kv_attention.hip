// kv_attention.hip -- attention over the paged 8-bit cache.
#include <float.h>
#include <math.h>

#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

// One wave per row and head, one key at a time: the running maximum and sum of a
// softmax over the keys.
template <int HD, int TYPE>
__global__ __launch_bounds__(64) void kv_attention_kernel(KvAttn a) {
  constexpr int E = HD / 64;
  const KvSeq s = kv_seq(a.b, blockIdx.y);
  const int i = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, lane = threadIdx.x;
  if (i >= s.n) return;
  const int hk = h / (a.n_heads / a.c.nkv), pos = s.len - s.n + i;
  const float *q = a.q + (size_t)(s.r0 + i) * a.q_stride + h * HD + lane * E;
  float x[E], o[E] = {}, m = -INFINITY, l = 0.0f;
  for (int e = 0; e < E; ++e) x[e] = q[e];
  const KvSpan span = kv_span(pos, s.len, a.slide, a.dense);
  auto value = [](const uint8_t *p) {
    return TYPE == kKvI8 ? (float)(int8_t)*p : __builtin_amdgcn_cvt_f32_fp8(*p, 0);
  };
  for (int key = span.lo; key <= span.hi; ++key) {
    const long slot = kv_slot(a.c, a.b, blockIdx.y, key, hk);
    if (slot < 0) continue;
    float t = 0.0f;
    for (int e = 0; e < E; ++e) t = fmaf(x[e], value(a.c.k + slot * HD + lane * E + e), t);
    for (int off = 32; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
    t = t * a.c.ks[slot] * a.asc;
    if (a.cap != 0.0f) t = a.cap * tanhf(t / a.cap);
    const float mn = fmaxf(m, t), f = expf(m - mn), p = expf(t - mn), w = p * a.c.vs[slot];
    m = mn;
    l = l * f + p;
    for (int e = 0; e < E; ++e)
      o[e] = fmaf(w, value(a.c.v + slot * HD + lane * E + e), o[e] * f);
  }
  float *out = a.out + ((size_t)(s.r0 + i) * a.n_heads + h) * HD + lane * E;
  for (int e = 0; e < E; ++e) out[e] = l != 0.0f ? o[e] / l : 0.0f;
}

}  // namespace

size_t kv_attention_work(const KvAttn &, const DeviceInfo &) { return 0; }

hipError_t launch_kv_attention(const KvAttn &a, const DeviceInfo &, hipStream_t stream) {
  const dim3 grid(a.b.max_rows * a.n_heads, a.b.batch);
  auto go = [&](auto kernel) { kernel<<<grid, 64, 0, stream>>>(a); };
  if (a.c.hdim == 256)
    a.c.type == kKvI8 ? go(kv_attention_kernel<256, kKvI8>) : go(kv_attention_kernel<256, kKvE4m3>);
  else
    a.c.type == kKvI8 ? go(kv_attention_kernel<128, kKvI8>) : go(kv_attention_kernel<128, kKvE4m3>);
  return hipGetLastError();
}

}  // namespace gh
