// sample.hip -- the next token of each row of logits: temperature, top-k, top-p
// and min-p, from a given uniform random number.
//
// The kept tokens are a prefix of the row in the order of falling logit (ties by
// rising index), and so is what each filter keeps and what lies before the token
// drawn: every step finds the first token of that order up to which a running
// count or a running weight reaches a target.  Weights exp((l - max l) / T) are
// taken in fp64 and held as whole multiples of 2^-44, so that their sums are exact
// whatever their order.
#include <float.h>
#include <limits.h>

#include "dec_common.h"
#include "gh_arith.h"
#include "gh_kernels.h"

namespace gh {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024;
constexpr int kMassBits = 44;  // of the largest weight; times 2^19 tokens: 63

// A token's place in the order: rising.  NaN and -inf have none (kNoPlace).
constexpr u64 kNoPlace = ~0ull;
__device__ __forceinline__ u64 place(float l, int index) {
  if (!(l > -INFINITY)) return kNoPlace;
  const uint32_t b = l == 0.0f ? 0u : __float_as_uint(l);
  const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)~up << 32 | (uint32_t)index;
}

struct Found {
  u64 at;            // the token's place
  u64 before, mass;  // the weights before it, and its own
};

struct Lds {
  u64 mass[256];
  uint32_t count[256];
  double tab[128];
  u64 red[kThreads / 64];
  u64 pick[3];
};

// The first token, among those at places up to `last`, up to which the running
// count (BY_COUNT) or weight reaches target >= 1; the last one where none does.
// One digit of the place at a time: eight bits of the logit, then of the index.
template <bool BY_COUNT, class W>
__device__ Found select(const float *l, int vocab, u64 last, u64 target, W &&weight, Lds &s) {
  const int tid = threadIdx.x, lane = tid & 63;
  u64 prefix = 0, before = 0;
  u64 gone = 0;  // count or weight before the prefix
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) s.mass[i] = s.count[i] = 0;
    __syncthreads();
    for (int i = tid; i < vocab; i += kThreads) {
      const u64 p = place(l[i], i);
      if (p > last || p == kNoPlace || (shift < 56 && (p >> (shift + 8)) != prefix)) continue;
      const int d = (int)(p >> shift) & 255;
      atomicAdd(&s.count[d], 1u);
      atomicAdd(&s.mass[d], weight(l[i]));
    }
    __syncthreads();
    if (tid < 64) {  // four digits a lane
      u64 c[4], m[4], sum = 0, msum = 0;
      for (int e = 0; e < 4; ++e) {
        c[e] = BY_COUNT ? s.count[4 * lane + e] : s.mass[4 * lane + e];
        m[e] = s.mass[4 * lane + e];
        sum += c[e];
        msum += m[e];
      }
      u64 at = sum, mat = msum;
      for (int off = 1; off < 64; off <<= 1) {
        const u64 t = __shfl_up(at, off, 64), mt = __shfl_up(mat, off, 64);
        if (lane >= off) {
          at += t;
          mat += mt;
        }
      }
      at += gone - sum;  // before this lane's digits
      mat += before - msum;
      // the digit in which the target is reached, or the last one that isn't empty
      int hit = -1, some = -1;
      u64 hg = 0, hb = 0, sg = 0, sb = 0;
      for (int e = 0; e < 4; ++e) {
        if (s.count[4 * lane + e] != 0) {
          some = 4 * lane + e;
          sg = at;
          sb = mat;
          if (hit < 0 && at + c[e] >= target) {
            hit = some;
            hg = at;
            hb = mat;
          }
        }
        at += c[e];
        mat += m[e];
      }
      const u64 hits = __ballot(hit >= 0), somes = __ballot(some >= 0);
      const int who = hits ? __ffsll(hits) - 1 : somes ? 63 - __clzll(somes) : 0;
      if (lane == who) {
        s.pick[0] = hits ? hit : some < 0 ? 0 : some;
        s.pick[1] = hits ? hg : sg;
        s.pick[2] = hits ? hb : sb;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | s.pick[0];
    gone = s.pick[1];
    before = s.pick[2];
    __syncthreads();
  }
  const int index = (int)(uint32_t)prefix;
  return Found{prefix, before, weight(l[index < vocab ? index : 0])};
}

__device__ u64 block_sum(u64 v, Lds &s) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < kThreads / 64; ++w) t += s.red[w];
  return t;
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample a) {
  __shared__ Lds s;
  const int row = blockIdx.x, tid = threadIdx.x;
  const float *l = a.logits + row * a.stride;
  exp_tab_load(s.tab);
  const ExpConsts ec = exp_consts();
  u64 first = kNoPlace;
  for (int i = tid; i < a.vocab; i += kThreads) first = min(first, place(l[i], i));
  for (int off = 32; off > 0; off >>= 1) first = min(first, (u64)__shfl_xor(first, off, 64));
  if ((tid & 63) == 0) s.red[tid >> 6] = first;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) first = min(first, s.red[w]);
  if (first == kNoPlace) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.probs != nullptr) a.probs[row] = 0.0f;
    }
    return;
  }
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  if (!(t > 0.0f)) {
    if (tid == 0) {
      a.tokens[row] = (int)(uint32_t)first;
      if (a.probs != nullptr) a.probs[row] = 1.0f;
    }
    return;
  }
  const float top = l[(uint32_t)first];
  auto w64 = [&](float x) {  // x has a place
    return x == top ? 1.0 : exp_tab(((double)x - (double)top) / (double)t, s.tab, ec);
  };
  auto weight = [&](float x) { return (u64)rint(ldexp(w64(x), kMassBits)); };
  const float min_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  u64 last = kNoPlace - 1;
  auto kept = [&]() {  // the weight of what is kept
    u64 sum = 0;
    for (int i = tid; i < a.vocab; i += kThreads) {
      const u64 p = place(l[i], i);
      if (p <= last && p != kNoPlace) sum += weight(l[i]);
    }
    return block_sum(sum, s);
  };
  if (k > 0 && k < a.vocab) last = select<true>(l, a.vocab, last, k, weight, s).at;
  if (top_p < 1.0f) {
    const double at_least = ceil((double)top_p * (double)kept());
    last = select<false>(l, a.vocab, last, at_least >= 1.0 ? (u64)at_least : 1, weight, s).at;
  }
  if (min_p > 0.0f) {  // the last one whose weight is large enough
    u64 most = first;
    for (int i = tid; i < a.vocab; i += kThreads) {
      const u64 p = place(l[i], i);
      if (p <= last && p != kNoPlace && w64(l[i]) >= (double)min_p) most = max(most, p);
    }
    for (int off = 32; off > 0; off >>= 1) most = max(most, (u64)__shfl_xor(most, off, 64));
    __syncthreads();
    if ((tid & 63) == 0) s.red[tid >> 6] = most;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) most = max(most, s.red[w]);
    last = most;
  }
  const u64 sum = kept();
  const float u = a.u[row];
  const double over = floor((u > 0.0f ? fmin((double)u, 1.0) : 0.0) * (double)sum);
  const Found f = select<false>(l, a.vocab, last, (u64)over + 1, weight, s);
  if (tid == 0) {
    a.tokens[row] = (int)(uint32_t)f.at;
    if (a.probs != nullptr) a.probs[row] = (float)((double)f.mass / (double)sum);
  }
}

}  // namespace

size_t sample_work(int, int) { return 0; }

hipError_t launch_sample(const Sample &a, hipStream_t stream) {
  sample_kernel<<<a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace gh
