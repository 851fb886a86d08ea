// Shared by the kernels over a paged cache: where a sequence's tokens lie, and how the
// work of attention over caches of any lengths is cut into equal pieces on the device.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "mhc_b200.h"

namespace mhc {
namespace cache {

// What the kernels need of a cache and a step (the C structs, checked and flattened).
struct View {
  void *keys, *values;
  int64_t kp, ks, kh, vp, vs, vh;  // page, slot and head strides in elements
  const int32_t *table, *lengths, *cu;
  int64_t pitch;
  int pages, size, shift;  // shift: log2(size), or -1 where size is no power of two
  int capacity;            // table_width * page_size
  int batch, T, Hk, D;
};

// New tokens [start, start + n) of sequence b, `len` tokens before them.  Within the
// step's rows whatever the offsets hold.
struct Seq {
  int start, n, len;
};
__device__ __forceinline__ Seq seq_between(const View &v, int from, int to, int len) {
  Seq s;
  s.start = min(max(from, 0), v.T);
  s.n = max(min(max(to, 0), v.T) - s.start, 0);
  s.len = len;
  return s;
}
__device__ __forceinline__ Seq seq_of(const View &v, int b) { return seq_between(v, v.cu[b], v.cu[b + 1], v.lengths[b]); }

// How many sequences end at or before row t, by a whole warp: the first that can hold it.  All offsets at once where they
// are few (a bisection is a chain of loads), else bisected.
__device__ __forceinline__ int seq_from(const View &v, int t) {
  if (v.batch <= 512) {
    int n = 0;
    for (int i = threadIdx.x & 31; i < v.batch; i += 32) n += v.cu[i + 1] <= t;
    return __reduce_add_sync(0xffffffffu, n);
  }
  int lo = 0, hi = v.batch;  // cu[lo] <= t < cu[hi + 1], if there is such
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v.cu[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int page_index(const View &v, int place) { return v.shift >= 0 ? place >> v.shift : place / v.size; }

// page and slot of a sequence's place; false where there is none
__device__ __forceinline__ bool locate(const View &v, int b, int64_t place, int &page, int &slot) {
  if (place < 0 || place >= v.capacity) return false;
  const int i = page_index(v, (int)place);
  page = v.table[b * v.pitch + i];
  slot = (int)place - i * v.size;
  return page >= 0 && page < v.pages;
}

}  // namespace cache

// Checks the structs and fills the view; MHC_OK or a status with its message set.
int cache_view(const char *who, const mhc_kv_cache *c, const mhc_cache_step *s, cache::View &v);

}  // namespace mhc
