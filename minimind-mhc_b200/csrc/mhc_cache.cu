// Moves the kept ones of a step's drafted tokens up to the places behind the context, in
// every layer of a paged cache, in place.
//
// Kept token i (row path[i] of the step) goes from place len + path[i] to len + i.  path
// ascends and path[i] >= i, so a place is written after it has been read if every column
// is moved by one thread, in order: no source of a later token lies at or below i.  A
// block takes a sequence's heads of one layer, a thread its columns of keys or of values,
// eight tokens' loads at once before their stores.  What is moved is a few hundred KB: the
// time is the launch and two dependent loads (path and page, then the row): 1.9 us for one sequence
// in 8 layers, 4.5 for 64.
#include "mhc_cache.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace keep {

constexpr int THREADS = 128;
constexpr int AT_ONCE = 8;

struct Args {
  cache::View c;
  int64_t kl, vl;  // layer strides
  const int32_t *path, *kept;
  int per_head;  // vectors of a head
};

template <typename V>
__global__ void __launch_bounds__(THREADS) keep_kernel(const Args a) {
  const int b = blockIdx.x, layer = blockIdx.y;
  const cache::Seq s = cache::seq_of(a.c, b);
  const int kept = min(a.kept[b], s.n);
  __shared__ int64_t from[2][AT_ONCE], to[2][AT_ONCE];  // offsets of keys and values; -1: not moved
  const int64_t es = sizeof(V) / (a.c.D / a.per_head);  // bytes of an element
  const int columns = a.c.Hk * a.per_head;
  for (int i0 = 1; i0 < kept; i0 += AT_ONCE) {
    __syncthreads();
    if (threadIdx.x < AT_ONCE) {
      const int i = i0 + threadIdx.x;
      int64_t src_k = -1, src_v = -1, dst_k = -1, dst_v = -1;
      if (i < kept) {
        const int p = a.path[s.start + i];
        int page, slot, page_to, slot_to;
        if (p > i && p < s.n && cache::locate(a.c, b, (int64_t)s.len + p, page, slot) &&
            cache::locate(a.c, b, (int64_t)s.len + i, page_to, slot_to)) {
          src_k = page * a.c.kp + slot * a.c.ks;
          src_v = page * a.c.vp + slot * a.c.vs;
          dst_k = page_to * a.c.kp + slot_to * a.c.ks;
          dst_v = page_to * a.c.vp + slot_to * a.c.vs;
        }
      }
      from[0][threadIdx.x] = src_k, from[1][threadIdx.x] = src_v;
      to[0][threadIdx.x] = dst_k, to[1][threadIdx.x] = dst_v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * columns; c += THREADS) {
      const int which = c >= columns, col = c - which * columns, h = col / a.per_head, x = col - h * a.per_head;
      char *base = static_cast<char *>(which ? a.c.values : a.c.keys) +
                   ((which ? layer * a.vl + h * a.c.vh : layer * a.kl + h * a.c.kh) * es + x * (int64_t)sizeof(V));
      V hold[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (from[which][i] >= 0) hold[i] = *reinterpret_cast<const V *>(base + from[which][i] * es);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
        if (from[which][i] >= 0) *reinterpret_cast<V *>(base + to[which][i] * es) = hold[i];
    }
  }
}

}  // namespace keep
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_keep_drafts(const mhc_kv_cache *cache, const mhc_cache_step *step, const int32_t *path, const int32_t *kept,
                               void *stream) {
  const char *who = "mhc_keep_drafts";
  clear_error();
  keep::Args a{};
  if (int st = cache_view(who, cache, step, a.c)) return st;
  if (step->T == 0 || step->batch == 0 || cache->layers == 0) return MHC_OK;
  if (!path || !kept) return fail(MHC_ERR_NULL, "%s: path or kept is NULL", who);
  if ((uintptr_t)path % 4 || (uintptr_t)kept % 4) return fail(MHC_ERR_ALIGN, "%s: path or kept is not 4-byte aligned", who);
  if (cache->layers > 65535) return fail(MHC_ERR_SHAPE, "%s: up to 65535 layers (got %d)", who, cache->layers);
  a.kl = cache->strides[0], a.vl = cache->strides[4];
  a.path = path, a.kept = kept;
  const int es = cache->dtype == MHC_F32 ? 4 : 2;
  bool wide = (cache->dim * es) % 16 == 0 && (uintptr_t)cache->keys % 16 == 0 && (uintptr_t)cache->values % 16 == 0;
  for (int i = 0; i < 8; ++i) wide = wide && (cache->strides[i] * es) % 16 == 0;
  const dim3 grid((unsigned)step->batch, (unsigned)cache->layers);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (wide) {
    a.per_head = cache->dim * es / 16;
    keep::keep_kernel<uint4><<<grid, keep::THREADS, 0, st>>>(a);
  } else {
    a.per_head = cache->dim;
    if (es == 4) keep::keep_kernel<uint32_t><<<grid, keep::THREADS, 0, st>>>(a);
    else keep::keep_kernel<uint16_t><<<grid, keep::THREADS, 0, st>>>(a);
  }
  return cuda_status(cudaGetLastError(), who);
}
