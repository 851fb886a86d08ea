// Attention of new tokens over a paged cache (single tokens, trees of drafted tokens,
// pieces of prompts).
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)     over the keys that a row sees
//
// Few rows share a long row of keys: the bound is reading keys and values once.  All
// query heads of a key head and all new tokens of a sequence are rows of one item (see
// the header for the cut), so a key is read once for up to 8, 16 or 32 rows; more rows go to
// mhc_cached_attn_tc.cu.
//
// A warp works alone: it takes 16 keys at a time, brings their K and V rows into a ring of
// its own with cp.async, forms the scores, keeps its own running reference and sums, and
// adds up O in registers.  The four warps of a block take neighbouring key heads of the same
// keys, whose rows lie side by side in memory, or, where there are fewer, neighbouring
// keys.  No barrier stands between the warps until an item ends; then those of one head
// join their sums through shared memory.  Page numbers are fetched one chunk ahead of the
// rows that they lead to; where pages are multiples of 16 keys a chunk has one page and a
// lane's addresses are a base and steps.
//
// 16-bit types: mma.sync m16n8k16 with the queries as the narrow operand, S^T = K Q^T and
// O^T += V^T P^T, so that 8 rows waste nothing and O takes 32 registers a lane at heads of
// 128 (with the queries as the 16 rows: twice that, two blocks an SM for four, and 123 us
// where this takes 67).  P goes from the scores' registers to the second operand's by
// movmatrix.  The matrix unit is not what bounds these few rows (16 rows of 128 need 104
// TFLOP/s at the copy rate); they are few for the 128 of tcgen05.mma.
// fp32 and what 16-byte copies cannot fetch (odd head sizes, strides, alignment): CUDA cores,
// the same structure on fp32 copies of the rows, two lanes to a key.
//
// Measured (with the join): 64 sequences of one token, 239,000 keys in all, 8 / 4 heads of
// 96, bf16: 75 us, 4.9 TB/s; one token over 200 keys 8.9 us; fp32, 16 sequences, 67,000 keys:
// 56 us, 3.7 TB/s, and with trees of 16 over 16,000 keys 73 us (instructions: 4 FMA for
// every shared-memory read of 16 bytes).  Bringing the rows by bulk copies (one a row)
// measured 4.5 TB/s at rows of 128 bytes and 1.8 at 64 against 6.2 and 5.2 by cp.async, and 6.7
// against 6.4 at 256.
//
// The reference m of a row is moved (and O and the sum rescaled) only when a score passes it
// by 2^8 (fp16: 2^4, and P is held times 2^10, so that what is 2^-34 of the largest still
// counts).  P is rounded to 16 bits for the second product; its sum is of the unrounded ones.
//
// What a row does not see: its scores are set aside before the maximum and its P is 0.  In
// the second product 0 would meet a NaN or an infinity of V there, so a chunk in which rows
// differ in what they see is searched for them, and with one the products are formed one by
// one.  Keys that do not exist (behind the last, on a page that is none) are not read: zeros.
// m starts at -inf, "nothing seen yet"; what is seen holds it at the lowest finite number
// at least, so that a row that sees only scores of -inf gives NaN, as the formula does, and
// a row that sees nothing 0.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cfloat>

#include "mhc_b200.h"
#include "mhc_cached_attn.cuh"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"
#include "mhc_sm100.cuh"

namespace mhc {
namespace cattn {

constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int CHUNK = 16;           // keys that a warp takes at a time
constexpr int KT = CHUNK * WARPS;   // keys of a tile
// Where the page table has room for so few keys, an item is one block's: nothing is cut and nothing joined.  8 / 4 heads of
// 96, bf16, every table full, us, whole items / cut ones: one new token in each of 1, 16 and 64 sequences of 256 keys
// 9.1 / 10.5, 10.9 / 13.0 and 13.0 / 18.6; of 512 keys 12.2 / 9.5, 14.0 / 11.7 and 19.3 / 20.6; of 1024 keys 17.9 / 9.9, 20.7 /
// 13.5 and 29.6 / 28.7; with 16 new tokens of 512 keys 15.4 / 13.1, 16.9 / 18.9 and 18.0 / 29.1, of 1024 22.4 / 14.9, 24.1 / 20.7
// and 27.8 / 39.8.
constexpr int WHOLE = 512;
// Rows of an item above which the tcgen05 kernel takes over, by the rows of a TMA box: small boxes are many copies for a
// tile.  16 sequences, up to 8192 keys, 8 / 4 heads of 96, trees of 16 (32 rows) and of 64 (128 rows), us, tcgen05 / warps:
// pages of 16 (boxes of 16) 38 / 60 and 38 / 145; of 100 (boxes of 4) 57 / 60 and 58 / 145; of 34 (2) 87 / 61 and 86 / 146;
// of 17 (1) 151 / 58 and 146 / 146.  Other shapes in pages of 64, with 8, 16 and 32 rows: 64 sequences up to 4096 keys, 8 / 2
// heads of 128, 42 / 41, 41 / 46 and 42 / 67; one sequence of 65,536, 8 / 4 heads of 128, 34 / 39, 34 / 43 and 35 / 55; 4 up to
// 16,384, 8 / 1 heads of 64, 14 / 17, 15 / 19 and 14 / 16.
static int tc_from(int box) { return box >= 4 ? 16 : box == 2 ? 48 : 128; }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {
  const int bytes = there ? 16 : 0;  // the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// ---- joining the warps of a block and the blocks of an item ----------------------------

// Warp w has left its sums for key head w % hw at o + w * apart (M rows of `pitch` floats), reference and sum at ml[w].
template <typename T, int M, int DP>
__device__ __forceinline__ void join_warps(const Args &a, const Segment &g, int slot, const Row *rows, const float *o, int pitch,
                                           int apart, float2 (*ml)[M], float (*fac)[M], bool vec) {
  const int hw = a.hw, all = hw * g.rows;
  for (int i = threadIdx.x; i < all; i += THREADS) {
    const int head = i / g.rows, r = i - head * g.rows;
    float top = -INFINITY, sum = 0.f;
    for (int w = head; w < WARPS; w += hw) top = fmaxf(top, ml[w][r].x);
    for (int w = head; w < WARPS; w += hw) sum = fmaf(factor(ml[w][r].x, top, a.c2), ml[w][r].y, sum);
    float scale = 1.f;
    if (slot < 0) scale = top == -INFINITY ? 0.f : 1.f / sum;
    else a.part_ml[((int64_t)slot * hw + head) * M + r] = make_float2(top, sum);
    for (int w = head; w < WARPS; w += hw) fac[w][r] = factor(ml[w][r].x, top, a.c2) * scale;
  }
  __syncthreads();
  constexpr int V = 4, PER = DP / V;
  for (int i = threadIdx.x; i < all * PER; i += THREADS) {
    const int at = i / PER, col = (i - at * PER) * V, head = at / g.rows, r = at - head * g.rows;
    if (col >= a.c.D) continue;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = head; w < WARPS; w += hw) {
      const float f = fac[w][r];
      const float4 y = *reinterpret_cast<const float4 *>(o + (int64_t)w * apart + r * pitch + col);
      x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
    }
    if (slot >= 0) {
      *reinterpret_cast<float4 *>(a.part_o + (((int64_t)slot * hw + head) * M + r) * DP + col) = x;
      continue;
    }
    T *out = static_cast<T *>(a.out) + out_at(a, g, rows[r], g.hk + head) + col;
    const float y[4] = {x.x, x.y, x.z, x.w};
    if (vec) {
      struct alignas(4 * sizeof(T)) { T e[4]; } p;
#pragma unroll
      for (int k = 0; k < 4; ++k) p.e[k] = from_f<T>(y[k]);
      *reinterpret_cast<decltype(p) *>(out) = p;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col + k < a.c.D) out[k] = from_f<T>(y[k]);
    }
  }
}

// Joins the blocks that had part of a cut item.  Every block lists the cut items (one entry for each block of the first
// kernel); a warp takes one row at a time and goes through its parts, AT_ONCE of them under way.  Where a row has more
// than a few the block's warps share them and join what they have through shared memory.
// Blocks of eight warps where rows have few parts, of sixteen where they have many (us for the whole call with blocks of 4 /
// 8 / 16 warps: 64 sequences of one token, nine parts a row, 76 / 74 / 80; trees of 64, five parts, 58 / 55 / 62; one token
// over 131,072 keys, 592 parts, - / 56 / 51).
constexpr int JOIN_PIECES = 1024;
constexpr int JOIN_ALONE = 16;  // parts that a warp goes through by itself

template <int DP>
struct Joined {
  float o[DP / 32], m = -INFINITY, l = 0.f;
  // parts begin, begin + step, ... of `count`: part i of the item of block c, row `row` of the `rows` of a slot
  template <int AT_ONCE>
  __device__ __forceinline__ void add(const Args &a, int c, int count, int64_t row, int64_t rows, int begin, int step) {
    constexpr int PER = DP / 32;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = 0.f;
    for (int i0 = begin; i0 < count; i0 += step * AT_ONCE) {
      float2 ml[AT_ONCE];
      float x[AT_ONCE][PER];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * step;
        ml[u] = make_float2(-INFINITY, 0.f);
        if (i < count) {
          // the item's first block's last slot, then the first slots of the blocks behind it
          const int64_t at = (i == 0 ? 2 * (int64_t)c + 1 : 2 * ((int64_t)c + i)) * rows + row;
          ml[u] = a.part_ml[at];
#pragma unroll
          for (int k = 0; k < PER; ++k) x[u][k] = a.part_o[at * DP + lane + 32 * k];
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (ml[u].x == -INFINITY) continue;  // nothing was seen there (or there is no such part)
        const float top = fmaxf(m, ml[u].x), f = factor(m, top, a.c2), g = factor(ml[u].x, top, a.c2);
        m = top;
        l = fmaf(l, f, ml[u].y * g);
#pragma unroll
        for (int k = 0; k < PER; ++k) o[k] = fmaf(o[k], f, x[u][k] * g);
      }
    }
  }
};

template <typename T, int M, int DP, int JOIN_THREADS>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const Args a) {
  constexpr int JOIN_WARPS = JOIN_THREADS / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int first_row[JOIN_PIECES + 1];  // rows of the cut items that begin in blocks before c
  __shared__ int parts[JOIN_PIECES];
  __shared__ int warp_rows[JOIN_WARPS];
  __shared__ float st_m[JOIN_WARPS], st_l[JOIN_WARPS];
  __shared__ float st_o[JOIN_WARPS][DP];
  constexpr int LIST = JOIN_PIECES / JOIN_THREADS;
  int mine[LIST], sum = 0, most = 0;
#pragma unroll
  for (int i = 0; i < LIST; ++i) {
    const int c = threadIdx.x * LIST + i;
    int4 d = make_int4(0, 0, 0, 0);
    if (c < a.pieces) d = a.desc[c];
    mine[i] = d.x > 0 ? (d.w & 255) * a.hw : 0;
    parts[c] = d.x;
    sum += mine[i];
    most = max(most, d.x);
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_rows[warp] = inc;
  const bool shared_out = __syncthreads_or(most > JOIN_ALONE);
  int at = inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < JOIN_WARPS; ++w) {
    if (w < warp) at += warp_rows[w];
    total += warp_rows[w];
  }
#pragma unroll
  for (int i = 0; i < LIST; ++i) {
    first_row[threadIdx.x * LIST + i] = at;
    at += mine[i];
  }
  if (threadIdx.x == 0) first_row[JOIN_PIECES] = total;
  __syncthreads();
  constexpr int PER = DP / 32;
  auto block_of = [&](int task) {  // the last block whose rows begin at or before it
    int c = 0;
#pragma unroll
    for (int step = JOIN_PIECES / 2; step; step >>= 1)
      if (first_row[c + step] <= task) c += step;
    return c;
  };
  // row and place in `out` of row `local` of the item that begins in block c
  auto row_at = [&](int c, int local, int64_t &row) -> T * {
    const int4 d = a.desc[c];
    const int n = d.w & 255, head = local / n, r = local - head * n;
    row = (int64_t)head * M + r;
    const int at = d.z + r, j = at / a.G;
    return static_cast<T *>(a.out) + ((int64_t)(d.y + j) * a.H + ((d.w >> 8) + head) * a.G + (at - j * a.G)) * a.c.D;
  };
  const int64_t rows = (int64_t)a.hw * M;
  // neighbouring rows to different blocks: the few rows of long items keep many blocks busy
  for (int base = blockIdx.x; base < total; base += gridDim.x * JOIN_WARPS) {
    const int task = base + warp * gridDim.x;
    if (task < total) {
      const int c = block_of(task);
      if (parts[c] <= JOIN_ALONE) {
        int64_t row;
        T *out = row_at(c, task - first_row[c], row);
        Joined<DP> s;
        s.template add<4>(a, c, parts[c], row, rows, 0, 1);
        const float scale = 1.f / s.l;
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (lane + 32 * k < a.c.D) out[lane + 32 * k] = from_f<T>(s.m == -INFINITY ? 0.f : s.o[k] * scale);
      }
    }
    if (!shared_out) continue;
    for (int i = 0; i < JOIN_WARPS && base + i * gridDim.x < total; ++i) {
      const int task = base + i * gridDim.x, c = block_of(task);
      if (parts[c] <= JOIN_ALONE) continue;
      int64_t row;
      T *out = row_at(c, task - first_row[c], row);
      Joined<DP> s;
      s.template add<8>(a, c, parts[c], row, rows, warp, JOIN_WARPS);
      if (lane == 0) {
        st_m[warp] = s.m;
        st_l[warp] = s.l;
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) st_o[warp][lane + 32 * k] = s.o[k];
      __syncthreads();
      if (threadIdx.x < DP && threadIdx.x < a.c.D) {
        float top = -INFINITY, l = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, st_m[w]);
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) {
          const float f = factor(st_m[w], top, a.c2);
          l = fmaf(f, st_l[w], l);
          y = fmaf(f, st_o[w][threadIdx.x], y);
        }
        out[threadIdx.x] = from_f<T>(top == -INFINITY ? 0.f : y * (1.f / l));
      }
      __syncthreads();
    }
  }
}

// ---- 16-bit types ------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
}
// infinities and NaN among the two values of a word
template <typename T>
__device__ __forceinline__ bool odd_pair(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (w & E) == E || ((w >> 16) & E) == E;
}

template <int DP, int R>
struct MmaShape {
  static constexpr int M = 8 * R;
  static constexpr int PITCH = DP * 2 + 16;  // bytes of a row: eight of them begin in different banks
  static constexpr int STAGE = 2 * CHUNK * PITCH;
  // blocks of an SM by registers (32 R and more for O), then chunks of a warp's ring by shared memory
  static constexpr int BLOCKS = R == 4 ? 2 : DP >= 128 ? 3 : 4;
  static constexpr int STAGES = BLOCKS == 2 ? (DP >= 128 ? 3 : DP >= 96 ? 4 : DP >= 64 ? 6 : 8) : DP >= 96 ? 2 : DP >= 64 ? 3 : 5;
  static constexpr int RING = STAGES * STAGE;  // of a warp
  static constexpr int SMEM = WARPS * RING;
  static constexpr int OP = DP + 4;  // floats of a row of O while the warps are joined
};

__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of an 8 x 8 matrix of 16-bit values over the warp
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int DP, int R>
__global__ void __launch_bounds__(THREADS, MmaShape<DP, R>::BLOCKS) mma_kernel(const Args a) {
  using S = MmaShape<DP, R>;
  constexpr int M = S::M, KS = DP / 16, VPR = DP / 8;
  constexpr int RPI = 32 / VPR, IT = CHUNK / RPI;  // rows that a warp's lanes copy at a time (VPR 12: 24 lanes)
  constexpr float AHEAD = std::is_same<T, __half>::value ? 4.f : 8.f, LIFT = std::is_same<T, __half>::value ? 10.f : 0.f;
  static_assert(M * S::OP * 4 <= S::RING, "O of a warp fits its ring");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int64_t off_k[WARPS][CHUNK], off_v[WARPS][CHUNK];
  __shared__ uint32_t have[WARPS][S::STAGES];  // which keys of a chunk exist
  __shared__ Near near;
  __shared__ Row rows[M];
  __shared__ float2 ml[WARPS][M];
  __shared__ float fac[WARPS][M];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3, oct = lane >> 2;
  const uint32_t ring = sm100::smem_u32(smem) + warp * S::RING;
  const int D = a.c.D;
  const int head = warp % a.hw, part = warp / a.hw;  // key head of the item; which of the tile's chunks
  const bool one_page = a.c.size % CHUNK == 0;       // a chunk never crosses a page's end
  const int fetch_row = lane / VPR, fetch_col = lane - fetch_row * VPR;
  const bool fetches = fetch_row < RPI && fetch_col * 8 < D;
  const float ahead = fminf(AHEAD / a.c2, FLT_MAX);
  if (D < DP)
    for (int i = tid; i < S::SMEM / 16; i += THREADS) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
  grid_dep_wait();
  near.fill(a);
  clear_rest<T>(a);
  __syncthreads();

  walk<M>(a, near, [&](const Segment &g, int slot) {
    const int hk = g.hk + head;
    const T *kbase = static_cast<const T *>(a.c.keys) + hk * a.c.kh, *vbase = static_cast<const T *>(a.c.values) + hk * a.c.vh;
    const int chunks = g.k1 - g.k0;
    const int key0 = g.k0 * a.tile + part * CHUNK;  // of chunk i: key0 + i * tile
    int page = page_of(a, g, one_page ? key0 : key0 + (lane & 15));
    auto fetch = [&](int i) {
      if (i < chunks) {
        const int key = key0 + i * a.tile, st = i % S::STAGES;
        const uint32_t kd = ring + st * S::STAGE + fetch_row * S::PITCH + fetch_col * 16, vd = kd + CHUNK * S::PITCH;
        if (one_page) {
          const int there = page >= 0 && page < a.c.pages ? min(max(g.keys - key, 0), CHUNK) : 0;
          if (lane == 0) have[warp][st] = (1u << there) - 1;
          const int first = key - cache::page_index(a.c, key) * a.c.size + fetch_row;
          const T *ks = kbase + fetch_col * 8, *vs = vbase + fetch_col * 8;
          if (there > 0) {
            ks += page * a.c.kp + first * a.c.ks;
            vs += page * a.c.vp + first * a.c.vs;
          }
          page = page_of(a, g, key + a.tile);
          if (fetches) {
#pragma unroll
            for (int u = 0; u < IT; ++u) {
              const bool ok = u * RPI + fetch_row < there;
              cp16(kd + u * RPI * S::PITCH, ok ? ks + (int64_t)(u * RPI) * a.c.ks : kbase, ok);
              cp16(vd + u * RPI * S::PITCH, ok ? vs + (int64_t)(u * RPI) * a.c.vs : vbase, ok);
            }
          }
        } else {
          const int mine = key + (lane & 15);
          const bool there = page >= 0 && page < a.c.pages;
          const uint32_t got = __ballot_sync(0xffffffffu, there) & 0xffffu;
          if (lane < CHUNK) {
            const int slot_at = mine - cache::page_index(a.c, mine) * a.c.size;
            off_k[warp][lane] = there ? page * a.c.kp + slot_at * a.c.ks : -1;
            off_v[warp][lane] = there ? page * a.c.vp + slot_at * a.c.vs : -1;
          }
          if (lane == 0) have[warp][st] = got;
          page = page_of(a, g, mine + a.tile);
          __syncwarp();
          if (fetches) {
#pragma unroll
            for (int u = 0; u < IT; ++u) {
              const int64_t ok = off_k[warp][u * RPI + fetch_row], ov = off_v[warp][u * RPI + fetch_row];
              cp16(kd + u * RPI * S::PITCH, kbase + (ok >= 0 ? ok + fetch_col * 8 : 0), ok >= 0);
              cp16(vd + u * RPI * S::PITCH, vbase + (ov >= 0 ? ov + fetch_col * 8 : 0), ov >= 0);
            }
          }
          __syncwarp();  // the offsets have been read
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);

    if (tid < M) rows[tid] = row_of(a, g, tid);
    __syncthreads();
    uint32_t q[R][KS][2];  // Q^T as the second operand: elements 16 k + 2 quad (+ 8) of row oct
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const Row x = rows[8 * t + oct];
      const T *src = static_cast<const T *>(a.q) + (x.j >= 0 ? q_at(a, g, x, hk) : 0);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = 16 * k + 8 * i + 2 * quad;
          q[t][k][i] = x.j >= 0 && col < D ? *reinterpret_cast<const uint32_t *>(src + col) : 0u;
        }
    }
    float o[R][KS][4];  // O^T: elements 16 k + oct (+ 8) of rows 2 quad, 2 quad + 1
    float m[R][2], l[R][2];
#pragma unroll
    for (int t = 0; t < R; ++t) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][k][i] = 0.f;
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
    for (int i = 0; i < chunks; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncwarp();  // for all lanes, and the chunk before has been read
      fetch(i + S::STAGES - 1);
      const int st = i % S::STAGES, key = key0 + i * a.tile;
      const uint32_t kt = ring + st * S::STAGE, vt = kt + CHUNK * S::PITCH;
      const uint32_t got = have[warp][st];
      if (got) {
        float s[R][4];  // S^T: keys oct and oct + 8 of rows 2 quad, 2 quad + 1
#pragma unroll
        for (int t = 0; t < R; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
        const uint32_t ka = kt + (lane & 15) * S::PITCH + (lane >> 4) * 16;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t w[4];
          ldsm4(w, ka + k * 32);
#pragma unroll
          for (int t = 0; t < R; ++t) mma16816<T>(s[t], w, q[t][k][0], q[t][k][1]);
        }
        // rows differ in what they see only from the first new token on, or where keys are missing
        const bool uneven = got != 0xffffu || key + CHUNK > g.s.len;
        uint32_t seen[R];  // bit 2 h + e: key oct + 8 h by row 2 quad + e
        bool move = false;
#pragma unroll
        for (int t = 0; t < R; ++t) {
          seen[t] = 0xfu;
          if (uneven) {
            seen[t] = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const Row x = rows[8 * t + 2 * quad + e];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int at = oct + 8 * h;
                const bool ok = ((got >> at) & 1) && x.j >= 0 && sees(a.mask != nullptr, x.bits, x.j, key + at - g.s.len);
                seen[t] |= (uint32_t)ok << (2 * h + e);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool k0 = (seen[t] >> e) & 1, k1 = (seen[t] >> (2 + e)) & 1;
            const float top = fmaxf(k0 ? fmaxf(s[t][e], -FLT_MAX) : -INFINITY, k1 ? fmaxf(s[t][2 + e], -FLT_MAX) : -INFINITY);
            move = move || top > m[t][e] + ahead;
          }
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int t = 0; t < R; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool k0 = (seen[t] >> e) & 1, k1 = (seen[t] >> (2 + e)) & 1;
              float top = fmaxf(k0 ? fmaxf(s[t][e], -FLT_MAX) : -INFINITY, k1 ? fmaxf(s[t][2 + e], -FLT_MAX) : -INFINITY);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
              top = fmaxf(top, m[t][e]);
              const float f = m[t][e] == top ? 1.f : factor(m[t][e], top, a.c2);
              m[t][e] = top;
              l[t][e] *= f;
#pragma unroll
              for (int k = 0; k < KS; ++k) {
                o[t][k][e] *= f;
                o[t][k][2 + e] *= f;
              }
            }
        }
        uint32_t p[R][2];  // P^T as the second operand: keys 2 quad, 2 quad + 1 (+ 8) of row oct
        float x[R][4];
#pragma unroll
        for (int t = 0; t < R; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[t][i] = ex2(fmaf(s[t][i] - m[t][i & 1], a.c2, LIFT));
            if (uneven && !((seen[t] >> i) & 1)) x[t][i] = 0.f;
            l[t][i & 1] += x[t][i];
          }
          p[t][0] = transposed(pack2<T>(x[t][0], x[t][1]));
          p[t][1] = transposed(pack2<T>(x[t][2], x[t][3]));
        }
        bool odd = false;
        if (uneven) {
          for (int at = lane; at < CHUNK * (DP / 2); at += 32) {
            const int r = at / (DP / 2), c = at - r * (DP / 2);
            uint32_t w;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vt + r * S::PITCH + c * 4));
            odd = odd || odd_pair<T>(w);
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
          const uint32_t va = vt + ((lane & 7) + ((lane >> 4) & 1) * 8) * S::PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t w[4];
            ldsm4t(w, va + k * 32);
#pragma unroll
            for (int t = 0; t < R; ++t) mma16816<T>(o[t][k], w, p[t][0], p[t][1]);
          }
        } else {
          // key by key: its P from the lanes that hold it (rounded, as in the product), V of this lane's elements
#pragma unroll 1
          for (int at = 0; at < CHUNK; ++at) {
            const int from = ((at & 7) << 2) | quad;
#pragma unroll
            for (int t = 0; t < R; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float w = to_f(from_f<T>(__shfl_sync(0xffffffffu, at < 8 ? x[t][e] : x[t][2 + e], from)));
                if ((__shfl_sync(0xffffffffu, seen[t], from) >> ((at < 8 ? 0 : 2) + e)) & 1) {
#pragma unroll
                  for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                      uint16_t v;
                      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(vt + at * S::PITCH + (16 * k + 8 * h + oct) * 2));
                      o[t][k][2 * h + e] = fmaf(w, to_f(*reinterpret_cast<const T *>(&v)), o[t][k][2 * h + e]);
                    }
                }
              }
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();
    float *mine = reinterpret_cast<float *>(smem + warp * S::RING);
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
        const int r = 8 * t + 2 * quad + e;
        if (oct == 0) ml[warp][r] = make_float2(m[t][e], l[t][e]);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          mine[r * S::OP + 16 * k + oct] = o[t][k][e];
          mine[r * S::OP + 16 * k + 8 + oct] = o[t][k][2 + e];
        }
      }
    __syncthreads();
    join_warps<T, M, DP>(a, g, slot, rows, reinterpret_cast<const float *>(smem), S::OP, S::RING / 4, ml, fac, true);
    __syncthreads();
    if (D < DP) {  // columns past D, where O lay, are zeros again
      for (int i = lane; i < M * S::OP / 4; i += 32) reinterpret_cast<uint4 *>(mine)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
  });
  grid_dep_launch();
}

// ---- CUDA cores ---------------------------------------------------------------------------

template <int DP>
struct CoreShape {
  static constexpr int KP = DP + 8, VP = DP;  // floats of a row of K (two lanes to a key: no conflicts) and of V
  static constexpr int STAGE = CHUNK * (KP + VP);
  static constexpr int BLOCKS = DP >= 128 ? 1 : DP >= 64 ? 2 : 3;  // of an SM
  static constexpr int STAGES = DP >= 128 ? 3 : DP >= 96 ? 2 : DP >= 64 ? 2 : 3;
  static constexpr int RING = STAGES * STAGE;  // floats of a warp
  static constexpr int OP = DP + 4;
};
template <int DP, int R>
constexpr int core_smem() {
  return 4 * (WARPS * CoreShape<DP>::RING + R * DP + WARPS * CHUNK * R);
}

// ASYNC: fp32 rows that begin at multiples of 16 bytes, copied ahead; else element by element
template <typename T, int DP, int R, bool ASYNC>
__global__ void __launch_bounds__(THREADS) core_kernel(const Args a) {
  using S = CoreShape<DP>;
  constexpr int SPLIT = DP <= 32 ? 4 : DP <= 64 ? 2 : 1;  // lanes that share four columns of O, each with every SPLIT-th key
  static_assert(R * S::OP <= S::RING, "O of a warp fits its ring");
  extern __shared__ __align__(128) float fsm[];
  float *ring = fsm + (threadIdx.x >> 5) * S::RING;
  float *qs = fsm + WARPS * S::RING;                      // (R, DP)
  // P of a chunk: (R / 4, CHUNK) times four rows; below 0: not seen
  float4 *ps = reinterpret_cast<float4 *>(qs + R * DP + (threadIdx.x >> 5) * CHUNK * R);
  __shared__ int64_t off_k[WARPS][CHUNK], off_v[WARPS][CHUNK];
  __shared__ uint32_t have[WARPS][S::STAGES];
  __shared__ Near near;
  __shared__ Row rows[R];
  __shared__ float2 ml[WARPS][R];
  __shared__ float fac[WARPS][R];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, D = a.c.D;
  const float ahead = fminf(8.f / a.c2, FLT_MAX);
  for (int i = tid; i < WARPS * S::RING; i += THREADS) fsm[i] = 0.f;
  grid_dep_wait();
  near.fill(a);
  clear_rest<T>(a);
  __syncthreads();

  walk<R>(a, near, [&](const Segment &g, int slot) {
    for (int r = tid; r < R; r += THREADS) rows[r] = row_of(a, g, r);
    __syncthreads();
    for (int i = tid; i < R * DP; i += THREADS) {
      const int r = i / DP, x = i - r * DP;
      qs[i] = rows[r].j >= 0 && x < D ? to_f(static_cast<const T *>(a.q)[q_at(a, g, rows[r], g.hk) + x]) : 0.f;
    }
    const T *kbase = static_cast<const T *>(a.c.keys) + g.hk * a.c.kh, *vbase = static_cast<const T *>(a.c.values) + g.hk * a.c.vh;
    const int chunks = g.k1 - g.k0, key0 = g.k0 * KT + warp * CHUNK;  // hw is 1 here, a tile KT keys
    int page = page_of(a, g, key0 + (lane & 15));
    auto fetch = [&](int i) {
      if (i < chunks) {
        const int key = key0 + i * KT + (lane & 15), st = i % S::STAGES;
        const bool there = page >= 0 && page < a.c.pages;
        const uint32_t got = __ballot_sync(0xffffffffu, there) & 0xffffu;
        if (lane < CHUNK) {
          const int slot_at = key - cache::page_index(a.c, key) * a.c.size;
          off_k[warp][lane] = there ? page * a.c.kp + slot_at * a.c.ks : -1;
          off_v[warp][lane] = there ? page * a.c.vp + slot_at * a.c.vs : -1;
        }
        if (lane == 0) have[warp][st] = got;
        page = page_of(a, g, key + KT);
        __syncwarp();
        float *kt = ring + st * S::STAGE, *vt = kt + CHUNK * S::KP;
        if constexpr (ASYNC) {
          for (int at = lane; at < CHUNK * (DP / 4); at += 32) {
            const int r = at / (DP / 4), x = (at - r * (DP / 4)) * 4;
            if (x < D) {
              const int64_t ok = off_k[warp][r], ov = off_v[warp][r];
              cp16(sm100::smem_u32(kt + r * S::KP + x), kbase + (ok >= 0 ? ok + x : 0), ok >= 0);
              cp16(sm100::smem_u32(vt + r * S::VP + x), vbase + (ov >= 0 ? ov + x : 0), ov >= 0);
            }
          }
        } else {
          for (int r = 0; r < CHUNK; ++r) {
            const int64_t ok = off_k[warp][r], ov = off_v[warp][r];
            for (int x = lane; x < D; x += 32) {
              kt[r * S::KP + x] = ok >= 0 ? to_f(kbase[ok + x]) : 0.f;
              vt[r * S::VP + x] = ov >= 0 ? to_f(vbase[ov + x]) : 0.f;
            }
          }
        }
        __syncwarp();  // the offsets have been read
      }
      cp_commit();
    };
    for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);
    __syncthreads();  // qs
    float o[R][4], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    const int mykey = lane >> 1, part = lane & 1;
    const int col = SPLIT == 1 ? lane * 4 : (lane % (32 / SPLIT)) * 4, share = SPLIT == 1 ? 0 : lane / (32 / SPLIT);
    for (int i = 0; i < chunks; ++i) {
      cp_wait<S::STAGES - 2>();
      __syncwarp();  // for all lanes, and the chunk before has been read
      fetch(i + S::STAGES - 1);
      const int st = i % S::STAGES, key = key0 + i * KT;
      const float *kt = ring + st * S::STAGE, *vt = kt + CHUNK * S::KP;
      const uint32_t got = have[warp][st];
      if (got) {
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = 0.f;
#pragma unroll 4
        for (int x = 0; x < DP / 8; ++x) {
          const float4 k = *reinterpret_cast<const float4 *>(kt + mykey * S::KP + (2 * x + part) * 4);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 q = *reinterpret_cast<const float4 *>(qs + r * DP + (2 * x + part) * 4);
            s[r] = fmaf(q.x, k.x, s[r]);
            s[r] = fmaf(q.y, k.y, s[r]);
            s[r] = fmaf(q.z, k.z, s[r]);
            s[r] = fmaf(q.w, k.w, s[r]);
          }
        }
        const bool uneven = got != 0xffffu || key + CHUNK > g.s.len;
        uint32_t seen = 0;
        bool move = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
          bool ok = true;
          if (uneven)
            ok = ((got >> mykey) & 1) && rows[r].j >= 0 && sees(a.mask != nullptr, rows[r].bits, rows[r].j, key + mykey - g.s.len);
          seen |= (uint32_t)ok << r;
          move = move || (ok && fmaxf(s[r], -FLT_MAX) > m[r] + ahead);
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float top = (seen >> r) & 1 ? fmaxf(s[r], -FLT_MAX) : -INFINITY;
#pragma unroll
            for (int w = 2; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            top = fmaxf(top, m[r]);
            const float f = m[r] == top ? 1.f : factor(m[r], top, a.c2);
            m[r] = top;
            l[r] *= f;
            o[r][0] *= f, o[r][1] *= f, o[r][2] *= f, o[r][3] *= f;
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool ok = (seen >> r) & 1;
          s[r] = ok ? ex2((s[r] - m[r]) * a.c2) : -1.f;
          if (part == 0 && ok) l[r] += s[r];
        }
#pragma unroll
        for (int r = 0; r < R / 4; ++r)  // a key's two lanes write half of its rows each
          if (part == (2 * r) / (R / 4 + R / 4 % 2)) ps[r * CHUNK + mykey] = make_float4(s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]);
        __syncwarp();
        if (col < DP) {
          if (!uneven) {
#pragma unroll 4
            for (int at = share; at < CHUNK; at += SPLIT) {
              const float4 v = *reinterpret_cast<const float4 *>(vt + at * S::VP + col);
#pragma unroll
              for (int r4 = 0; r4 < R / 4; ++r4) {
                const float4 p4 = ps[r4 * CHUNK + at];
                const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  float(&y)[4] = o[4 * r4 + k];
                  y[0] = fmaf(p[k], v.x, y[0]);
                  y[1] = fmaf(p[k], v.y, y[1]);
                  y[2] = fmaf(p[k], v.z, y[2]);
                  y[3] = fmaf(p[k], v.w, y[3]);
                }
              }
            }
          } else {
#pragma unroll 1
            for (int at = share; at < CHUNK; at += SPLIT) {
              const float4 v = *reinterpret_cast<const float4 *>(vt + at * S::VP + col);
              const float *p = reinterpret_cast<const float *>(ps + at);
#pragma unroll
              for (int r = 0; r < R; ++r) {
                const float x = p[(r / 4) * CHUNK * 4 + r % 4];
                if (x < 0.f) continue;
                o[r][0] = fmaf(x, v.x, o[r][0]);
                o[r][1] = fmaf(x, v.y, o[r][1]);
                o[r][2] = fmaf(x, v.z, o[r][2]);
                o[r][3] = fmaf(x, v.w, o[r][3]);
              }
            }
          }
        }
      }
      __syncwarp();  // P has been read
    }
    cp_wait<0>();
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int w = 2; w < 32; w <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
      if (lane == 0) ml[warp][r] = make_float2(m[r], l[r]);
#pragma unroll
      for (int w = 32 / SPLIT; w < 32; w <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[r][k] += __shfl_xor_sync(0xffffffffu, o[r][k], w);
      if (share == 0 && col < DP) *reinterpret_cast<float4 *>(ring + r * S::OP + col) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
    }
    __syncthreads();
    join_warps<T, R, DP>(a, g, slot, rows, fsm, S::OP, S::RING, ml, fac, a.c.D % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0);
    __syncthreads();
    if (D < DP)  // columns past D, where O lay, are zeros again
      for (int i = lane; i < R * S::OP; i += 32) ring[i] = 0.f;
    __syncwarp();
  });
  grid_dep_launch();
}

// ---- choice and launch ---------------------------------------------------------------------

// Which kernel, for how many rows, on how many blocks.  The lengths of the sequences' new tokens are on the device; on
// average there are T / batch of them.
enum Kind { CORE, MMA, TC };
struct Choice {
  Kind kind;
  int m, dp, hw, pieces, cost;
  bool whole;
  size_t desc, ml, o, total;  // bytes of the workspace
};
static Choice choose(const mhc_kv_cache *c, const mhc_cache_step *s, int H, Kind most) {
  Choice x{};
  const int G = H / c->kv_heads, sms = device_sm_count() > 0 ? device_sm_count() : 148;
  const int64_t rows = (s->T + s->batch - 1) / s->batch * G;
  x.kind = most == TC && rows <= tc_from(cached_attn_tc_box(c)) ? MMA : most;
  x.dp = (c->dim + 31) / 32 * 32;
  x.hw = 1;
  x.cost = 2;
  x.whole = (int64_t)s->table_width * c->page_size <= WHOLE;
  if (x.kind == TC) {
    x.m = CATTN_TC_ROWS;
    x.pieces = sms * CATTN_TC_BLOCKS;
    x.cost = 8;
  } else if (x.kind == MMA) {
    x.m = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    // the warps of a block take neighbouring key heads of the same keys, which lie side by side in memory
    if (!x.whole) x.hw = c->kv_heads % 4 == 0 ? 4 : c->kv_heads % 2 == 0 ? 2 : 1;
    x.pieces = sms * (x.m == 32 ? 2 : x.dp >= 128 ? 3 : 4);
  } else {
    x.m = rows <= 4 ? 4 : 16;
    x.pieces = sms * (x.dp >= 128 ? 1 : x.dp >= 64 ? 2 : 3);
  }
  if (x.pieces > JOIN_PIECES) x.pieces = JOIN_PIECES;
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const size_t rows_kept = (size_t)x.pieces * 2 * x.hw * x.m;
  x.desc = up((size_t)x.pieces * sizeof(int4));
  x.ml = up(rows_kept * sizeof(float2));
  x.o = up(rows_kept * x.dp * sizeof(float));
  x.total = x.desc + x.ml + x.o;
  return x;
}

template <typename K>
static cudaError_t start(K kernel, const Args &a, int blocks, int smem, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e != cudaSuccess ? e : launch_early(kernel, dim3((unsigned)blocks), THREADS, smem, st, a);
}

// the join begins while the last blocks of the first kernel still run, and waits for them on the device
template <typename T, int M, int DP>
static cudaError_t join(const Args &a, cudaStream_t st) {
  if (a.whole) return cudaSuccess;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  const int64_t rows = (int64_t)a.c.T * a.H;
  const int64_t items = (int64_t)a.c.batch * a.groups;  // one tile of rows each, at least
  if (a.pieces > JOIN_ALONE * items) return launch_early(join_kernel<T, M, DP, 512>, dim3((unsigned)(rows < 2 * sms ? rows : 2 * sms)), 512, 0, st, a);
  return launch_early(join_kernel<T, M, DP, 256>, dim3((unsigned)(rows < 4 * sms ? rows : 4 * sms)), 256, 0, st, a);
}

template <typename F>
static cudaError_t with_dp(int dp, F &&f) {
  switch (dp) {
    case 32: return f(IC<32>{});
    case 64: return f(IC<64>{});
    case 96: return f(IC<96>{});
    default: return f(IC<128>{});
  }
}

static cudaError_t launch(const Args &a, const Choice &x, const mhc_kv_cache *cache, bool async, cudaStream_t st) {
  return with_dp(x.dp, [&](auto dp) -> cudaError_t {
    constexpr int DP = decltype(dp)::value;
    if (x.kind == TC) {
      const cudaError_t e = launch_cached_attn_tc(a, cache, st);
      if (e != cudaSuccess) return e;
      return a.dtype == MHC_BF16 ? join<__nv_bfloat16, CATTN_TC_ROWS, DP>(a, st) : join<__half, CATTN_TC_ROWS, DP>(a, st);
    }
    if (x.kind == MMA) {
      auto go = [&](auto tag, auto r) -> cudaError_t {
        using T = decltype(tag);
        constexpr int R = decltype(r)::value;
        cudaError_t e = start(mma_kernel<T, DP, R>, a, x.pieces, MmaShape<DP, R>::SMEM, st);
        return e != cudaSuccess ? e : join<T, 8 * R, DP>(a, st);
      };
      auto by_rows = [&](auto tag) -> cudaError_t {
        return x.m == 8 ? go(tag, IC<1>{}) : x.m == 16 ? go(tag, IC<2>{}) : go(tag, IC<4>{});
      };
      return a.dtype == MHC_BF16 ? by_rows(__nv_bfloat16{}) : by_rows(__half{});
    }
    return with_dtype(a.dtype, [&](auto tag) -> cudaError_t {
      using T = decltype(tag);
      auto go = [&](auto r) -> cudaError_t {
        constexpr int R = decltype(r)::value;
        cudaError_t e;
        if constexpr (std::is_same<T, float>::value)
          e = async ? start(core_kernel<T, DP, R, true>, a, x.pieces, core_smem<DP, R>(), st)
                    : start(core_kernel<T, DP, R, false>, a, x.pieces, core_smem<DP, R>(), st);
        else
          e = start(core_kernel<T, DP, R, false>, a, x.pieces, core_smem<DP, R>(), st);
        return e != cudaSuccess ? e : join<T, R, DP>(a, st);
      };
      return x.m == 4 ? go(IC<4>{}) : go(IC<16>{});
    });
  });
}

// rows of the cache (and, for the tensor cores, of q) that 16-byte copies can fetch
static bool rows_aligned(const mhc_kv_cache *c) {
  const int es = c->dtype == MHC_F32 ? 4 : 2;
  bool ok = (c->dim * es) % 16 == 0 && (uintptr_t)c->keys % 16 == 0 && (uintptr_t)c->values % 16 == 0;
  for (int i : {1, 2, 3, 5, 6, 7}) ok = ok && (c->strides[i] * es) % 16 == 0;
  return ok;
}

}  // namespace cattn
}  // namespace mhc

using namespace mhc;

extern "C" {

size_t mhc_cached_attn_workspace(const mhc_kv_cache *cache, const mhc_cache_step *step, int H) {
  if (!cache || !step || step->batch < 1 || cache->kv_heads < 1 || H < 1 || H % cache->kv_heads || cache->dim < 1 || cache->dim > 128) return 0;
  size_t most = 0;  // for any of the kernels: which one runs depends on the pointers too
  for (cattn::Kind k : {cattn::CORE, cattn::MMA, cattn::TC}) {
    const size_t need = cattn::choose(cache, step, H, k).total;
    most = need > most ? need : most;
  }
  return most;
}

int mhc_cached_attn(const mhc_kv_cache *cache, const mhc_cache_step *step, const void *q, int H, const int64_t *q_strides,
                    const int64_t *mask, float scale, void *out, void *workspace, size_t workspace_bytes, void *stream) {
  const char *who = "mhc_cached_attn";
  clear_error();
  cattn::Args a{};
  if (int st = cache_view(who, cache, step, a.c)) return st;
  if (cache->dim > 128) return fail(MHC_ERR_SHAPE, "%s: head sizes up to 128 are supported (got %d)", who, cache->dim);
  if (H < 1 || H % cache->kv_heads) return fail(MHC_ERR_SHAPE, "%s: %d query heads cannot share %d key heads", who, H, cache->kv_heads);
  // a sequence's rows (new tokens x heads of a group) are counted in 32 bits
  if (step->T * (H / cache->kv_heads) > 0x7fffffff - 4096)
    return fail(MHC_ERR_SHAPE, "%s: %lld tokens of %d heads for a key head are more rows than one call takes", who, (long long)step->T,
                H / cache->kv_heads);
  a.c2 = (float)((double)scale * 1.4426950408889634);
  if (!(scale > 0.f) || !(a.c2 < INFINITY)) return fail(MHC_ERR_SHAPE, "%s: scale must be positive and finite (got %g)", who, scale);
  if (step->T == 0) return MHC_OK;
  if (!q || !out || !q_strides) return fail(MHC_ERR_NULL, "%s: required pointer is NULL", who);
  const size_t es = cache->dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)q % es || (uintptr_t)out % es || (uintptr_t)mask % 8) return fail(MHC_ERR_ALIGN, "%s: a pointer is not aligned to its elements", who);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (step->batch == 0 || cache->pages == 0)  // nothing is seen
    return cuda_status(cudaMemsetAsync(out, 0, (size_t)step->T * H * cache->dim * es, st), who);
  const size_t need = mhc_cached_attn_workspace(cache, step, H);
  if (!workspace || workspace_bytes < need) return fail(MHC_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
  if ((uintptr_t)workspace % 256) return fail(MHC_ERR_ALIGN, "%s: workspace must be 256-byte aligned", who);
  const bool async = cattn::rows_aligned(cache);
  const bool mma = async && cache->dtype != MHC_F32 && (uintptr_t)q % 16 == 0 && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0 &&
                   (uintptr_t)out % 16 == 0 && !generic_forced();
  const cattn::Choice x = cattn::choose(cache, step, H, !mma ? cattn::CORE : cached_attn_tc_eligible(cache) ? cattn::TC : cattn::MMA);
  a.q = q, a.out = out, a.qt = q_strides[0], a.qh = q_strides[1];
  a.mask = mask, a.H = H, a.G = H / cache->kv_heads;
  a.pieces = x.pieces, a.hw = x.hw, a.groups = a.c.Hk / x.hw, a.cost = x.cost, a.whole = x.whole, a.dtype = cache->dtype;
  a.tile = x.kind == cattn::TC ? CATTN_TC_KEYS : cattn::KT / x.hw;
  a.err_flag = host_error_flag();
  // an upper bound of the units of all sequences
  const double units = ((double)step->T * a.G / x.m + step->batch) * a.groups * ((double)a.c.capacity / a.tile + 1 + x.cost);
  if (units > 2e9) return fail(MHC_ERR_SHAPE, "%s: %lld tokens over up to %d keys are more than one call takes", who, (long long)step->T, a.c.capacity);
  char *ws = static_cast<char *>(workspace);
  a.desc = reinterpret_cast<int4 *>(ws);
  a.part_ml = reinterpret_cast<float2 *>(ws + x.desc);
  a.part_o = reinterpret_cast<float *>(ws + x.desc + x.ml);
  return cuda_status(cattn::launch(a, x, cache, async, st), who);
}

}  // extern "C"
