// Attention over a paged cache: arguments, and the cut of the work into equal pieces.
//
// The unit of work is a tile of `tile` keys for up to M rows (new tokens x heads of a
// group) of one sequence and `hw` neighbouring key heads, the item; an item counts some
// units more, for its beginning and end.  The lengths are known on the device only, so
// every block sums the units of all sequences itself (a few loads and one warp's scan) and
// takes its share of the row of all units, W / N of them and the first W % N blocks one more:
// equal work whatever the lengths.  An item that lies in one block is finished there; of one
// that is cut the blocks leave their sums, references and rows, which a second kernel joins,
// in the blocks' order.
#pragma once

#include "mhc_cache.cuh"
#include "mhc_device.cuh"

namespace mhc {
namespace cattn {

struct Args {
  cache::View c;
  const void *q;
  void *out;
  int64_t qt, qh;
  const int64_t *mask;
  int H, G;
  float c2;       // scale log2(e)
  int pieces;     // N
  int hw, tile;   // key heads and keys of a unit
  int groups;     // Hk / hw
  int whole;      // items are not cut: a block takes those that begin in its share
  int cost;       // what an item's beginning (pages, rows and queries, one after the other) and end count, in units
  int dtype;
  // what cut items leave: slot 2 c of block c's first item, 2 c + 1 of its last
  int4 *desc;       // (N): of the item that begins in block c and ends in another: parts, first new token, first row, rows + 256 key head
  float2 *part_ml;  // (2 N, hw M): reference (a score) and sum
  float *part_o;    // (2 N, hw M, DP)
  int *err_flag;    // registered host word of kernels that give up
};

struct Segment {
  cache::Seq s;
  int b, hk, row0, rows;  // key heads [hk, hk + hw), rows [row0, row0 + rows) of the sequence's n G
  int keys;               // places [0, keys) hold keys
  int k0, k1, kt;         // key tiles of this block, of the item
};

__device__ __forceinline__ int keys_of(const cache::View &v, const cache::Seq &s) {
  const int64_t l = (int64_t)s.len + s.n;
  return (int)max((int64_t)0, min(l, (int64_t)v.capacity));
}

// The step's offsets and lengths in shared memory, where they are few: every warp looks them up for every item.
constexpr int NEAR = 96;
struct Near {
  int cu[NEAR + 1], len[NEAR];
  // by all threads of the block; a barrier has to follow
  __device__ __forceinline__ void fill(const Args &a) {
    if (a.c.batch > NEAR) return;
    for (int i = threadIdx.x; i <= a.c.batch; i += blockDim.x) {
      cu[i] = a.c.cu[i];
      if (i < a.c.batch) len[i] = a.c.lengths[i];
    }
  }
  __device__ __forceinline__ cache::Seq at(const Args &a, int b) const {
    if (a.c.batch > NEAR) return cache::seq_of(a.c, b);
    return cache::seq_between(a.c, cu[b], cu[b + 1], len[b]);
  }
};

template <int M>
struct Cut {
  const Args &a;
  const Near &near;
  int first, sum, total;      // units before this lane's sequences, of them, of all
  int per;                    // sequences of a lane
  __device__ __forceinline__ Cut(const Args &args, const Near &steps) : a(args), near(steps) {
    const int lane = threadIdx.x & 31;
    per = (a.c.batch + 31) / 32;
    int64_t mine = 0;
    for (int i = 0; i < per; ++i) mine += units(lane * per + i);
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    // the host has seen to it that 32 bits hold the units of any lengths; of offsets that are none (they decrease, and
    // the sequences have more rows than there are) nothing is done
    const int64_t all = __shfl_sync(0xffffffffu, inc, 31);
    total = all > 0x7fffffff ? 0 : (int)all;
    first = (int)(inc - mine);
    sum = (int)mine;
  }
  __device__ __forceinline__ int tiles(int keys) const { return max(1, (keys + a.tile - 1) / a.tile); }
  __device__ __forceinline__ int row_tiles(int n) const { return (int)(((int64_t)n * a.G + M - 1) / M); }
  __device__ __forceinline__ int units(int b) const {
    if (b >= a.c.batch) return 0;
    const cache::Seq s = near.at(a, b);
    return s.n == 0 ? 0 : row_tiles(s.n) * a.groups * (tiles(keys_of(a.c, s)) + a.cost);
  }
  // the sequence of unit w < total, and the unit within it; whole warps
  __device__ __forceinline__ void find(int w, int &b, int &at) const {
    const int lane = threadIdx.x & 31;
    const unsigned has = __ballot_sync(0xffffffffu, w >= first && w < first + sum);
    const int owner = __ffs(has) - 1;
    int mine = lane * per;
    int left = w - first;
    if (lane == owner)
      for (int u; left >= (u = units(mine)); ++mine) left -= u;
    b = __shfl_sync(0xffffffffu, mine, owner);
    at = __shfl_sync(0xffffffffu, left, owner);
  }
};

// Runs `work(segment, slot)` over block blockIdx.x's units: slot < 0 where the item is not cut.
// Writes the block's entry of the join's table.
template <int M, typename F>
__device__ __forceinline__ void walk(const Args &a, const Near &near, F &&work) {
  const Cut<M> cut(a, near);
  const int W = cut.total, N = min(a.pieces, W), piece = blockIdx.x;
  int4 entry = make_int4(0, 0, 0, 0);
  if (piece < N) {
    const int each = W / N, more = W - each * N;
    const int w1 = each * (piece + 1) + min(piece + 1, more);
    int w = each * piece + min(piece, more), at, b;
    cut.find(w, b, at);
    while (w < w1 && b < a.c.batch) {
      Segment g;
      g.b = b;
      g.s = near.at(a, b);
      g.keys = keys_of(a.c, g.s);
      g.kt = cut.tiles(g.keys);
      const int mt = cut.row_tiles(g.s.n), span = g.kt + a.cost;
      const int all = g.s.n == 0 ? 0 : mt * a.groups * span;
      if (at >= all) {  // the next sequence that has any
        ++b;
        at = 0;
        continue;
      }
      const int item = at / span, from = at - item * span;
      // units of the item; its tiles follow the first a.cost
      const int to = a.whole ? span : min(span, from + (w1 - w));
      g.k0 = max(0, from - a.cost);
      g.k1 = a.whole && from > 0 ? g.k0 : max(0, to - a.cost);
      const int group = item / mt;
      g.hk = group * a.hw;
      g.row0 = (item - group * mt) * M;
      g.rows = (int)min((int64_t)M, (int64_t)g.s.n * a.G - g.row0);
      if (g.k1 > g.k0) {
        const bool whole = g.k0 == 0 && g.k1 == g.kt;
        if (g.k0 == 0 && !whole) {  // the last of this block, and it goes on: who else has some of it
          const int last = w - from + span - 1, longer = more * (each + 1);
          const int e = last < longer ? last / (each + 1) : more + (last - longer) / each;
          entry = make_int4(e - piece + 1, g.s.start, g.row0, g.rows + 256 * g.hk);
        }
        work(g, whole ? -1 : g.k0 == 0 ? 2 * piece + 1 : 2 * piece);
      }
      w += to - from;
      at += to - from;
    }
  }
  if (threadIdx.x == 0 && !a.whole) a.desc[piece] = entry;
}

// rows of no sequence get 0
template <typename T>
__device__ __forceinline__ void clear_rest(const Args &a) {
  const int lo = min(max(a.c.cu[0], 0), a.c.T), hi = min(max(a.c.cu[a.c.batch], 0), a.c.T);
  T *out = static_cast<T *>(a.out);
  const int64_t row = (int64_t)a.H * a.c.D, head = lo * row, tail = (int64_t)a.c.T * row;
  const int64_t step = (int64_t)gridDim.x * blockDim.x, at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = at; i < head; i += step) out[i] = T(0.f);
  for (int64_t i = hi * row + at; i < tail; i += step) out[i] = T(0.f);
}

// Whether token j of a sequence sees new token c (place len + c): c < 0 is the context.
__device__ __forceinline__ bool sees(bool masked, uint64_t bits, int j, int c) {
  return c < 0 || (masked ? c < 64 && ((bits >> c) & 1) : c <= j);
}

// what a sum with reference m is multiplied by to have reference top
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float factor(float m, float top, float c2) { return m == -INFINITY ? 0.f : ex2((m - top) * c2); }

// ---- which row of the item is which query -----------------------------------------

struct Row {
  uint64_t bits;
  int j, h;  // token of the sequence (-1 past the item's rows), head of the group
};
__device__ __forceinline__ Row row_of(const Args &a, const Segment &g, int r) {
  Row x{0, -1, 0};
  if (r < g.rows) {
    const int at = g.row0 + r;
    x.j = at / a.G;
    x.h = at - x.j * a.G;
    if (a.mask) x.bits = (uint64_t)a.mask[g.s.start + x.j];
  }
  return x;
}
// offsets of a row's elements, hk its key head
__device__ __forceinline__ int64_t q_at(const Args &a, const Segment &g, const Row &x, int hk) {
  return (int64_t)(g.s.start + x.j) * a.qt + (int64_t)(hk * a.G + x.h) * a.qh;
}
__device__ __forceinline__ int64_t out_at(const Args &a, const Segment &g, const Row &x, int hk) {
  return ((int64_t)(g.s.start + x.j) * a.H + hk * a.G + x.h) * a.c.D;
}

// The page of a key; -1: none
__device__ __forceinline__ int page_of(const Args &a, const Segment &g, int key) {
  return key < g.keys ? a.c.table[g.b * a.c.pitch + cache::page_index(a.c, key)] : -1;
}

// Launches a kernel that may begin before the one in front of it in the stream has ended (where that one allows it) and
// that waits on the device (grid_dep_wait) before it touches any memory that others write.
template <typename K, typename... A>
inline cudaError_t launch_early(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, const A &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace cattn

constexpr int CATTN_TC_ROWS = 128, CATTN_TC_KEYS = 64, CATTN_TC_BLOCKS = 2;  // rows of an item, keys of a tile, blocks of an SM
// rows of a TMA box: the greatest common divisor of a tile's keys, a power of two, and a page's
inline int cached_attn_tc_box(const mhc_kv_cache *c) {
  int rows = CATTN_TC_KEYS;
  while (c->page_size % rows) rows /= 2;
  return rows;
}
bool cached_attn_tc_eligible(const mhc_kv_cache *c);
cudaError_t launch_cached_attn_tc(const cattn::Args &a, const mhc_kv_cache *c, cudaStream_t stream);
int read_cat_error(bool clear);

}  // namespace mhc
