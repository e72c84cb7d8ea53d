// kv_cache.h -- the paged 8-bit key/value cache: what its kernels and their
// launchers share.  Everything that turns the caller's device-side tables into
// addresses is here, in functions that also compile for the host.
//
// The tables (page ids, lengths, first rows) lie in device memory, where the
// host can't check them, so every value read from them is clamped or checked
// against the sizes the host has: no table, whatever it holds, leads a kernel out
// of its buffers.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define GH_HD __host__ __device__ __forceinline__
#else
#define GH_HD inline
#endif

namespace gh {

constexpr int kKvI8 = 0, kKvE4m3 = 1;  // GEMMA_HIP_CACHE_*

// k, v: codes [npages][nkv][1 << shift][hdim]; ks, vs: scales without the last axis
struct KvCache {
  uint8_t *k, *v;
  float *ks, *vs;
  int type, npages, shift, nkv, hdim;
};

// pages [batch][width], len [batch], row0 [batch + 1]; rows, max_rows and max_len
// bound what len and row0 say
struct KvBatch {
  const int *pages, *len, *row0;
  int batch, width, rows, max_rows, max_len;
};

GH_HD int kv_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Sequence b: its rows r0 .. r0 + n - 1 are its positions len - n .. len - 1.
struct KvSeq {
  int r0, n, len;
};
GH_HD KvSeq kv_seq(const KvBatch &b, int i) {
  KvSeq s;
  s.r0 = kv_clamp(b.row0[i], 0, b.rows);
  s.n = kv_clamp(b.row0[i + 1], s.r0, b.rows) - s.r0;
  if (s.n > b.max_rows) s.n = b.max_rows;
  s.len = kv_clamp(b.len[i], 0, b.max_len);
  return s;
}

// Where head h of position pos (0 <= pos < max_len) of sequence i lies: its index
// among the cache's rows of hdim codes, which is also its scale's; -1 on a page
// that isn't there.
GH_HD long kv_slot(const KvCache &c, const KvBatch &b, int i, int pos, int h) {
  const int id = b.pages[(size_t)i * b.width + (pos >> c.shift)];
  if ((unsigned)id >= (unsigned)c.npages) return -1;
  return (((long)id * c.nkv + h) << c.shift) + (pos & ((1 << c.shift) - 1));
}

// The sequence that row r belongs to, -1 for a row behind the last sequence's:
// the last i with row0[i] <= r among sequences that aren't empty.
GH_HD int kv_find(const int *row0, int batch, int r) {
  int lo = 0, hi = batch;  // row0[lo] <= r < row0[hi] once found
  if (r < row0[0] || r >= row0[batch]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row0[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The grid of a launch that needs `blocks` workgroups for each of `batch` sequences: x and z for
// the former, as a grid takes 2^32 - 1 threads a dimension at most; kv_block() is a
// workgroup's number.
constexpr long kKvMostX = 1l << 22;  // (of 256 threads)
struct KvGrid {
  unsigned x, y, z;
};
GH_HD KvGrid kv_grid_of(long blocks, int batch) {
  const long z = (blocks + kKvMostX - 1) / kKvMostX;
  return KvGrid{(unsigned)(z > 1 ? kKvMostX : blocks), (unsigned)batch, (unsigned)(z > 1 ? z : 1)};
}
GH_HD long kv_block(unsigned x, unsigned z) { return (long)z * kKvMostX + x; }

#ifdef __HIPCC__
// The sequence that row r is in if it is in one, else any; by a whole wave, for one row.
__device__ __forceinline__ int kv_find_wave(const KvBatch &b, int r) {
  const int lane = threadIdx.x & 63;
  int last = 0;
  for (int base = 0; base < b.batch; base += 64) {
    const bool from = base + lane < b.batch && b.row0[base + lane] <= r;
    const unsigned long long all = __ballot(from);
    if (all != 0) last = base + __popcll(all) - 1;
    if (all != ~0ull) break;
  }
  return __builtin_amdgcn_readfirstlane(last);
}
#endif

// Keys that a row at position pos sees: lo .. hi (hi < lo: none).
struct KvSpan {
  int lo, hi;
};
GH_HD KvSpan kv_span(int pos, int len, int slide, int dense) {
  KvSpan s;
  s.hi = pos < 0 ? -1 : dense ? len - 1 : pos;
  s.lo = !dense && slide > 0 && pos >= slide ? pos + 1 - slide : 0;
  return s;
}

}  // namespace gh
