// Causal attention over packed sequences, forward and backward, on CUDA cores:
// every type, every head size up to 128, any token and head strides.
//
//   O_i  = sum_j P_ij V_j,   P_ij = exp(scale q_i . k_j - L_i),   start(i) <= j <= i
//   D_i  = dO_i . O_i,       dS_ij = P_ij (dO_i . V_j - D_i)
//   dQ_i = scale sum_j dS_ij K_j
//   dK_j = scale sum_{h in group, i} dS_ij Q_i,   dV_j = sum_{h in group, i} P_ij dO_i
//
// fp32 throughout.  A block owns 64 rows (32 where that leaves SMs with less than four
// blocks: it is the loads' latency that other blocks then cover) and walks tiles of 64
// columns; a thread, 16 for every 4 rows, holds a 4 x 4 piece of the scores and 4 rows
// x D / 16 columns of the result in registers, the operands are staged as fp32 in
// shared memory and multiplied two at a time (fma.rn.f32x2).  A value that a lane
// reads from shared memory costs a wavefront of the SM, a pair of products half a
// cycle: 4 rows of a thread rather than 2 (and 256 threads) in blocks of 32 rows took
// 2 x 512 tokens, 8 heads of 64, from 212 to 171 us, forward and backward.  8 rows of a
// thread (half the warps) take 222 there and 2.63 ms against 2.38 at 4 x 2048; loading
// the next operands by hand while these are multiplied changes nothing at 2 x 512 and
// takes 2.62 ms at 4 x 2048.
// Forward: one pass with the running maximum and sum.  Backward: the scores again
// from the saved L, in two kernels of the same form (a block owns 64 queries and
// sums dQ, or 64 keys and sums dK and dV over the heads that share them), so
// every gradient is a sum in a fixed order.  The shared-memory operands bound it (71 to
// 78 % of the wavefronts an SM can have, 28 to 34 % of the FFMA pipe, 4 x 2048 tokens).
// Not tried: each fp32 operand as three bf16 parts, six products on the tensor cores.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <mutex>

#include "mhc_attn_redo.cuh"
#include "mhc_attn_tc.cuh"
#include "mhc_b200.h"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace attn {

constexpr int TILE = 64;  // columns
constexpr int R = 4;      // rows of a thread
constexpr int threads_of(int rows) { return rows / R * 16; }
constexpr int PP = TILE + 4;  // pitch of a score tile

// ROWS rows of one head as fp32 into shared memory, zero outside of the packed range
// and past column D
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void load_tile(float *dst, const T *src, int64_t ts, int row0, int D, Span range) {
#pragma unroll 8
  for (int e = threadIdx.x; e < ROWS * DP; e += THREADS) {
    const int r = e / DP, c = e - r * DP;
    const int t = row0 + r;
    dst[r * (DP + 4) + c] = t >= range.start && t < range.end && c < D ? to_f(src[(int64_t)t * ts + c]) : 0.f;
  }
}

// The same for fp32 rows at multiples of 16 bytes, as asynchronous copies: the next
// tile is on its way while this one is worked on.
template <int DP, int ROWS, int THREADS>
__device__ __forceinline__ void copy_tile(float *dst, const float *src, int64_t ts, int row0, int D, Span range) {
#pragma unroll 8
  for (int e = threadIdx.x; e < ROWS * DP / 4; e += THREADS) {
    const int r = e / (DP / 4), c = (e - r * (DP / 4)) * 4;
    const int t = row0 + r;
    const bool in = t >= range.start && t < range.end && c < D;
    const float *from = in ? src + (int64_t)t * ts + c : src;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst + r * (DP + 4) + c)), "l"(from),
                 "r"(in ? 16 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void copy_word(float *dst, const float *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// s[i][j] = sum_d A[ty*R+i][d] B[tx+16j][d], even and odd d apart until the end
template <int DP>
__device__ __forceinline__ void scores(const float *A, const float *B, int ty, int tx, float (&s)[R][4]) {
  uint64_t acc[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0ull;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    ulonglong2 x[R], y[4];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const ulonglong2 *>(A + (ty * R + i) * (DP + 4) + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const ulonglong2 *>(B + (tx + 16 * j) * (DP + 4) + d);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = sm100::f2_fma(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = sm100::f2_fma(x[i].y, y[j].y, acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo, hi;
      sm100::f2_unpack(acc[i][j], lo, hi);
      s[i][j] = lo + hi;
    }
}

// acc[i][c] += sum_kk W[ty*R+i][kk] B[kk][2 tx + 32 c, + 1], columns in pairs
template <int DP>
__device__ __forceinline__ void accumulate(const float *W, const float *B, int ty, int tx, uint64_t (&acc)[R][DP / 32]) {
#pragma unroll 2
  for (int kk = 0; kk < TILE; kk += 4) {
    float4 w[R];
#pragma unroll
    for (int i = 0; i < R; ++i) w[i] = *reinterpret_cast<const float4 *>(W + (ty * R + i) * PP + kk);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint64_t b[DP / 32];
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) b[c] = *reinterpret_cast<const uint64_t *>(B + (kk + u) * (DP + 4) + 2 * tx + 32 * c);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float wi = u == 0 ? w[i].x : (u == 1 ? w[i].y : (u == 2 ? w[i].z : w[i].w));
        const uint64_t w2 = sm100::f2_pack(wi, wi);
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) acc[i][c] = sm100::f2_fma(w2, b[c], acc[i][c]);
      }
    }
  }
}

// lo != null: what the rounding to T left over, itself in T.  Whether there was a NaN.
template <typename T, int DP>
__device__ __forceinline__ bool store_rows(T *dst, T *lo, int64_t ts, int row0, int64_t T_, int D, int ty, int tx,
                                           const uint64_t (&acc)[R][DP / 32], const float (&mul)[R]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int t = row0 + ty * R + i;
    if (t >= T_) continue;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int col = 2 * tx + 32 * (c / 2) + (c & 1);
      if (col < D) {
        float v, w;
        sm100::f2_unpack(acc[i][c / 2], v, w);
        v = (c & 1 ? w : v) * mul[i];
        bad |= isnan(v);
        const T r = from_f<T>(v);
        dst[(int64_t)t * ts + col] = r;
        if (lo) lo[(int64_t)t * ts + col] = from_f<T>(v - to_f(r));
      }
    }
  }
  return bad;
}

// Which rows of which head a block has.  The blocks go out in the order of their work,
// longest first; where all of them are resident at once, a second one on each SM, the
// second ones go out the other way around, so that a long one shares its SM with a
// short one.  Against rows in order, fp32, forward / dQ / dK and dV: 1024 tokens, 8 / 4
// heads of 96 123 -> 84 / 163 -> 110 / 262 -> 271 us (128 blocks: no order), 4 x 2048, 8
// of 64 641 -> 503 / 938 -> 821 / 1230 -> 1115 us, 2 x 512 42 -> 39 / 55 -> 52 / 70 ->
// 67 us for 3 us of sorting in each direction.
struct Work {
  const int *order;  // tiles of TM rows by their work; null: with an SM for every block it does not matter
  int heads;
  int total;  // blocks with work
  int fold;   // 0, or the SMs: blocks behind that many take the ranks backwards
};
struct Rows {
  int row0, head;  // row0 < 0: none
};
template <int ROWS, bool LATE>  // LATE: later rows of a tile have more work
__device__ __forceinline__ Rows rows_of(const Work &w, int64_t T) {
  constexpr int SUB = TM / ROWS;
  const int block = (int)blockIdx.x, rank = w.fold && block >= w.fold ? 3 * w.fold - 1 - block : block;
  if (rank >= w.total) return {-1, 0};
  const int at = rank / w.heads, sub = at % SUB, tile = at / SUB;
  const int64_t row0 = (int64_t)(w.order ? w.order[tile] : tile) * TM + (LATE ? SUB - 1 - sub : sub) * ROWS;
  return {row0 < T ? (int)row0 : -1, rank % w.heads};
}

template <typename T, int DP, int ROWS, bool ASYNC>
__global__ void __launch_bounds__(threads_of(ROWS)) attn_fwd_generic_kernel(const __grid_constant__ Args a, const Work work) {
  constexpr int THREADS = threads_of(ROWS);
  extern __shared__ float sm[];
  constexpr int TS = TILE * (DP + 4);
  float *Q = sm, *P = Q + ROWS * (DP + 4), *KV = P + ROWS * PP;  // ASYNC: two pairs of tiles
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const Rows own = rows_of<ROWS, true>(work, a.T);
  if (own.row0 < 0) return;
  const int q0 = own.row0, h = own.head, hk = h / (a.H / a.Hk);
  const Span range = packed_range(a);
  int start[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int t = q0 + ty * R + i;
    start[i] = t < a.T ? span_of(a, t).start : t + 1;
  }
  load_tile<T, DP, ROWS, THREADS>(Q, static_cast<const T *>(a.q) + h * a.qh, a.qt, q0, a.D, range);
  uint64_t acc[R][DP / 32] = {};
  float mx[R], sum[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    mx[i] = -INFINITY;
    sum[i] = 0.f;
  }
  const int first = span_of(a, q0).start, last = min((int64_t)q0 + ROWS, a.T);
  auto fetch = [&](int k0, int buf) {
    const T *kp = static_cast<const T *>(a.k) + hk * a.kh, *vp = static_cast<const T *>(a.v) + hk * a.vh;
    if constexpr (ASYNC) {
      copy_tile<DP, TILE, THREADS>(KV + 2 * buf * TS, kp, a.kt, k0, a.D, range);
      copy_tile<DP, TILE, THREADS>(KV + (2 * buf + 1) * TS, vp, a.vt, k0, a.D, range);
    } else {
      load_tile<T, DP, TILE, THREADS>(KV, kp, a.kt, k0, a.D, range);
      load_tile<T, DP, TILE, THREADS>(KV + TS, vp, a.vt, k0, a.D, range);
    }
  };
  if (ASYNC) {
    if (first < last) fetch(first, 0);
    copies_done();
  }
  int buf = 0;
  for (int k0 = first; k0 < last; k0 += TILE) {
    __syncthreads();  // the tile before last is done with
    if (ASYNC) {
      if (k0 + TILE < last) fetch(k0 + TILE, buf ^ 1);
      copies_done();
      copies_wait<1>();
    } else {
      fetch(k0, 0);
    }
    __syncthreads();
    const float *K = KV + 2 * buf * TS, *V = K + TS;
    if (ASYNC) buf ^= 1;
    float s[R][4];
    scores<DP>(Q, K, ty, tx, s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = q0 + ty * R + i;
      float m = mx[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx + 16 * j;
        s[i][j] = key >= start[i] && key <= t ? s[i][j] * a.scale_log2 : -INFINITY;
        m = fmaxf(m, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float base = m == -INFINITY ? 0.f : m;  // nothing visible yet
      const float fix = exp2f(mx[i] - base);
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(s[i][j] - base);
        part += p;
        P[(ty * R + i) * PP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      sum[i] = sum[i] * fix + part;
      mx[i] = m;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) acc[i][c] = sm100::f2_mul(acc[i][c], sm100::f2_pack(fix, fix));
    }
    __syncwarp();  // a row of P is written and read by the same 16 lanes
    accumulate<DP>(P, V, ty, tx, acc);
  }
  float inv[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int t = q0 + ty * R + i;
    inv[i] = sum[i] == 0.f ? 0.f : 1.f / sum[i];
    if (tx == 0 && t < a.T) a.lse[(int64_t)h * a.Tp + t] = sum[i] == 0.f ? INFINITY : mx[i] + log2f(sum[i]);
  }
  T *lo = a.o_lo ? static_cast<T *>(a.o_lo) + (int64_t)h * a.D : nullptr;
  T *out = static_cast<T *>(a.o) + (int64_t)h * a.D;
  if (__syncthreads_or(store_rows<T, DP>(out, lo, (int64_t)a.H * a.D, q0, a.T, a.D, ty, tx, acc, inv)))
    redo_out_rows<T>(a, h, q0, ROWS, tid >> 5, THREADS / 32, tid & 31);
}

// DKV = false: a block owns 64 queries of one head, sums dQ over their keys.
// DKV = true: a block owns 64 keys of one key head, sums dK and dV over the queries
// that see them, of every head of the group or, with splits, of its share of them.
template <typename T, int DP, int ROWS, bool DKV, bool ASYNC>
__global__ void __launch_bounds__(threads_of(ROWS)) attn_bwd_generic_kernel(const __grid_constant__ Args a, const Work work) {
  constexpr int THREADS = threads_of(ROWS);
  extern __shared__ float sm[];
  constexpr int TS = TILE * (DP + 4), RS = ROWS * (DP + 4);
  constexpr int STAGE = 2 * TS + 2 * TILE;  // two tiles, lse and D; ASYNC: two stages
  float *R1 = sm, *R2 = R1 + RS, *W = R2 + RS, *CS = W + ROWS * PP;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const Rows own = rows_of<ROWS, !DKV>(work, a.T);
  if (own.row0 < 0) return;
  const int G = a.H / a.Hk, splits = DKV ? a.splits : 1, per = G / splits;
  const int r0 = own.row0, rh = own.head / splits, part = own.head % splits;
  const Span range = packed_range(a);
  const T *q = static_cast<const T *>(a.q), *k = static_cast<const T *>(a.k), *v = static_cast<const T *>(a.v);
  const T *dout = static_cast<const T *>(a.dout);
  const int64_t ot = (int64_t)a.H * a.D;
  int bound[R];  // DKV: the end of the key's sequence; else the start of the query's
  int alone[R];  // the column whose dS is 0: a sequence's first token, as a query, sees itself only; none: -1
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int t = r0 + ty * R + i;
    const Span s = t < a.T ? span_of(a, t) : Span{t + 1, t};
    bound[i] = DKV ? s.end : s.start;
    alone[i] = s.start == t ? t : -1;
  }
  if (DKV) {
    load_tile<T, DP, ROWS, THREADS>(R1, k + rh * a.kh, a.kt, r0, a.D, range);
    load_tile<T, DP, ROWS, THREADS>(R2, v + rh * a.vh, a.vt, r0, a.D, range);
  } else {
    load_tile<T, DP, ROWS, THREADS>(R1, q + rh * a.qh, a.qt, r0, a.D, range);
    load_tile<T, DP, ROWS, THREADS>(R2, dout + (int64_t)rh * a.D, ot, r0, a.D, range);
  }
  uint64_t acc1[R][DP / 32] = {}, acc2[DKV ? R : 1][DP / 32] = {};
  const int64_t end_rows = min((int64_t)r0 + ROWS, a.T);
  const int first = DKV ? r0 : span_of(a, r0).start;
  const int last = DKV ? span_of(a, (int)end_rows - 1).end : (int)end_rows;
  const int tiles = last > first ? (last - first + TILE - 1) / TILE : 0, n = tiles * (DKV ? per : 1);
  auto fetch = [&](int it, int buf) {
    const int h = DKV ? rh * G + part * per + it / tiles : rh, c0 = first + it % tiles * TILE;
    float *c1 = CS + buf * STAGE, *c2 = c1 + TS, *l = c2 + TS, *d = l + TILE;
    const T *s1 = DKV ? q + h * a.qh : k + (rh / G) * a.kh, *s2 = DKV ? dout + (int64_t)h * a.D : v + (rh / G) * a.vh;
    const int64_t t1 = DKV ? a.qt : a.kt, t2 = DKV ? ot : a.vt;
    if constexpr (ASYNC) {
      copy_tile<DP, TILE, THREADS>(c1, s1, t1, c0, a.D, range);
      copy_tile<DP, TILE, THREADS>(c2, s2, t2, c0, a.D, range);
    } else {
      load_tile<T, DP, TILE, THREADS>(c1, s1, t1, c0, a.D, range);
      load_tile<T, DP, TILE, THREADS>(c2, s2, t2, c0, a.D, range);
    }
    if (tid < TILE) {  // lse and D of the tile's columns, or of the block's rows
      const int64_t t = (DKV ? c0 : r0) + tid;
      const bool in = t < a.T;
      const int64_t at = (int64_t)h * a.Tp + (in ? t : 0);
      if (ASYNC) {
        copy_word(l + tid, a.lse + at, in);
        copy_word(d + tid, a.delta + at, in);
      } else {
        l[tid] = in ? a.lse[at] : 0.f;
        d[tid] = in ? a.delta[at] : 0.f;
      }
    }
  };
  if (ASYNC) {
    if (n > 0) fetch(0, 0);
    copies_done();
  }
  {
    int buf = 0;
    for (int it = 0; it < n; ++it) {
      const int c0 = first + it % tiles * TILE;
      __syncthreads();  // the tile before last is done with
      if (ASYNC) {
        if (it + 1 < n) fetch(it + 1, buf ^ 1);
        copies_done();
        copies_wait<1>();
      } else {
        fetch(it, 0);
      }
      __syncthreads();
      const float *C1 = CS + buf * STAGE, *C2 = C1 + TS, *L = C2 + TS, *Dl = L + TILE;
      if (ASYNC) buf ^= 1;
      float p[R][4], ds[R][4];
      scores<DP>(R1, C1, ty, tx, p);
      scores<DP>(R2, C2, ty, tx, ds);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = r0 + ty * R + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = c0 + tx + 16 * j;
          const bool seen = DKV ? c >= r && c < bound[i] : c <= r && c >= bound[i];
          const int n = DKV ? tx + 16 * j : ty * R + i;
          p[i][j] = seen ? exp2f(fmaf(p[i][j], a.scale_log2, -L[n])) : 0.f;
          ds[i][j] = seen ? (c == alone[i] ? 0.f : p[i][j]) * (ds[i][j] - Dl[n]) : 0.f;
        }
      }
      if constexpr (DKV) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) W[(ty * R + i) * PP + tx + 16 * j] = p[i][j];
        __syncwarp();
        accumulate<DP>(W, C2, ty, tx, acc2);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) W[(ty * R + i) * PP + tx + 16 * j] = ds[i][j];
      __syncwarp();
      accumulate<DP>(W, C1, ty, tx, acc1);
    }
  }
  float sc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) sc[i] = a.scale;
  if constexpr (DKV) {
    float one[R];
#pragma unroll
    for (int i = 0; i < R; ++i) one[i] = 1.f;
    const int64_t kt = (int64_t)a.Hk * a.D;
    auto store = [&](auto *dk, auto *dv) {
      using U = std::remove_pointer_t<decltype(dk)>;
      bool bad = store_rows<U, DP>(dk + (int64_t)rh * a.D, static_cast<U *>(nullptr), kt, r0, a.T, a.D, ty, tx, acc1, sc);
      bad |= store_rows<U, DP>(dv + (int64_t)rh * a.D, static_cast<U *>(nullptr), kt, r0, a.T, a.D, ty, tx, acc2, one);
      if (__syncthreads_or(bad)) redo_dkv_rows<T, U>(a, rh, r0, ROWS, rh * G + part * per, per, dk, dv, tid >> 5, THREADS / 32, tid & 31);
    };
    if (splits > 1)
      store(a.parts + 2 * part * a.T * kt, a.parts + (2 * part + 1) * a.T * kt);
    else
      store(static_cast<T *>(a.dk), static_cast<T *>(a.dv));
  } else {
    T *dq = static_cast<T *>(a.dq) + (int64_t)rh * a.D;
    if (__syncthreads_or(store_rows<T, DP>(dq, static_cast<T *>(nullptr), ot, r0, a.T, a.D, ty, tx, acc1, sc)))
      redo_dq_rows<T>(a, rh, r0, ROWS, tid >> 5, THREADS / 32, tid & 31);
  }
}

// dK and dV from the parts of the blocks that share their keys, in order
template <typename T>
__global__ void __launch_bounds__(256) attn_join_any_kernel(const Args a) {
  const int64_t n = a.T * a.Hk * a.D;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < 2 * n; e += (int64_t)gridDim.x * 256) {
    const int second = e >= n;
    const int64_t at = e - second * n;
    float s = 0.f;
    for (int p = 0; p < a.splits; ++p) s += __ldcs(a.parts + (int64_t)(p * 2 + second) * n + at);
    static_cast<T *>(second ? a.dv : a.dk)[at] = from_f<T>(s);
  }
}

// D_i = dO_i . O_i.  O is its rounded value plus what the rounding left over: D is
// subtracted from dO . V, of which it is the mean, so with few keys the rounding of
// O alone would show in dS as an error of its own size.  Four lanes a row, the rows
// of all heads as they lie; it reads O, its rest and dO once, and a lane asks for all
// of its part before it adds (16 lanes a row, 4 rows in turn: 22 us at 16384 tokens, 8
// heads of 96; so: 11.6).  fp16: also the largest finite |dO| and |V| of every
// sequence, kept at its first token.
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

template <typename T, int VEC>
__global__ void __launch_bounds__(256) attn_delta_kernel(const Args a, uint32_t *amax) {
  const int l = threadIdx.x & 3;
  const T *o = static_cast<const T *>(a.out), *lo = static_cast<const T *>(a.out_lo), *d = static_cast<const T *>(a.dout);
  const int64_t row = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2), rows = a.T * a.H;
  constexpr int MOST = VEC == 8 ? 4 : 1;  // pieces of a row of 128 that a lane has at once
  float s = 0.f, most_o = 0.f, most_v = 0.f;
  if (row < rows) {
    for (int c0 = l * VEC; c0 < a.D; c0 += MOST * 4 * VEC) {
      T ov[MOST][VEC], lv[MOST][VEC], dv[MOST][VEC];
#pragma unroll
      for (int u = 0; u < MOST; ++u) {
        const int c = c0 + u * 4 * VEC;
        if (c >= a.D) continue;
        const int64_t at = row * a.D + c;
        if constexpr (VEC == 8) {
          *reinterpret_cast<uint4 *>(ov[u]) = ldg_stream(o + at);
          *reinterpret_cast<uint4 *>(dv[u]) = *reinterpret_cast<const uint4 *>(d + at);
          if (lo) *reinterpret_cast<uint4 *>(lv[u]) = ldg_stream(lo + at);
        } else {
          ov[u][0] = o[at];
          dv[u][0] = d[at];
          if (lo) lv[u][0] = lo[at];
        }
      }
#pragma unroll
      for (int u = 0; u < MOST; ++u) {
        if (c0 + u * 4 * VEC >= a.D) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s = fmaf(to_f(ov[u][e]) + (lo ? to_f(lv[u][e]) : 0.f), to_f(dv[u][e]), s);
          if (amax) most_o = fmaxf(most_o, finite_abs(to_f(dv[u][e])));
        }
      }
    }
  }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  // the rest of the last tile, which the kernels load with it
  const int64_t pad = a.Tp - a.T;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pad * a.H; i += (int64_t)gridDim.x * 256)
    a.delta[i / pad * a.Tp + a.T + i % pad] = 0.f;
  const int64_t t = row / a.H, h = row - t * a.H;
  const Span range = packed_range(a);
  // outside of the sequences dO may hold anything; there D must not make a NaN of P = 0 times dP - D
  if (row < rows && l == 0) a.delta[h * a.Tp + t] = t >= range.start && t < range.end ? s : 0.f;
  if (amax) {
    if (row >= rows || t < range.start || t >= range.end)
      most_o = 0.f;
    else if (h < a.Hk)
      for (int c = l; c < a.D; c += 4) most_v = fmaxf(most_v, finite_abs(to_f(static_cast<const T *>(a.v)[t * a.vt + h * a.vh + c])));
    // a row's sequence by its first token; rows outside of all go with the warp's first
    const bool in = row < rows && t >= range.start && t < range.end;
    int start = in ? span_of(a, (int)t).start : -1;
    const unsigned have = __ballot_sync(0xffffffffu, in);
    if (have) {
      const int one = __shfl_sync(0xffffffffu, start, __ffs((int)have) - 1);
      start = in ? start : one;
      const bool whole = __all_sync(0xffffffffu, start == one);
      for (int x = whole ? 16 : 2; x; x >>= 1) {
        most_o = fmaxf(most_o, __shfl_xor_sync(0xffffffffu, most_o, x));
        most_v = fmaxf(most_v, __shfl_xor_sync(0xffffffffu, most_v, x));
      }
      if ((threadIdx.x & (whole ? 31 : 3)) == 0) {  // of non-negative floats the bits are in order: a maximum in any order
        atomicMax(amax + 2 * (int64_t)start, __float_as_uint(most_o));
        atomicMax(amax + 2 * (int64_t)start + 1, __float_as_uint(most_v));
      }
    }
  }
}

template <typename F>
static cudaError_t with_dim(int D, F &&f) {
  if (D <= 32) return f(IC<32>{});
  if (D <= 64) return f(IC<64>{});
  if (D <= 96) return f(IC<96>{});
  return f(IC<128>{});
}

// opt-in shared memory of a kernel, set once per device
template <auto KERN>
static cudaError_t allow_smem(size_t bytes) {
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return e;
}

// whether blocks of 32 rows: with 64 an SM would have less than four
static bool short_rows(int64_t T, int heads) {
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  return (T + TILE - 1) / TILE * heads < 4 * (int64_t)sms;
}

// whether every row of the tensors the kernels walk begins at a multiple of 16 bytes
static bool fp32_rows(const Args &a, bool backward) {
  const uintptr_t ps = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (backward ? (uintptr_t)a.dout : 0);
  return a.dtype == MHC_F32 && !(ps & 15) && !((a.qt | a.qh | a.kt | a.kh | a.vt | a.vh | a.D) & 3);
}

// The grid; order: where the tiles' order stands, or will once it is needed.
template <int ROWS>
static cudaError_t plan(const Args &a, int heads, size_t smem, const int *order, Work &w, unsigned &grid) {
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  const int64_t tiles = (a.T + TM - 1) / TM, total = tiles * (TM / ROWS) * heads;
  if (total > 0x7fffffff) return cudaErrorInvalidValue;
  const bool two = 2 * (smem + 1024) <= 228 * 1024;  // blocks of an SM
  w = {total > sms ? order : nullptr, heads, (int)total, two && total > sms && total <= 2 * sms ? sms : 0};
  grid = (unsigned)(w.fold ? 2 * sms : total);
  return cudaSuccess;
}

template <typename T, int DP, int ROWS, bool ASYNC>
static cudaError_t run_fwd(const Args &a, int *order, cudaStream_t stream) {
  constexpr size_t smem = (size_t)((ROWS + (ASYNC ? 4 : 2) * TILE) * (DP + 4) + ROWS * PP) * 4;
  static_assert(smem <= 232448, "shared memory of a block");
  cudaError_t e = allow_smem<attn_fwd_generic_kernel<T, DP, ROWS, ASYNC>>(smem);
  if (e != cudaSuccess) return e;
  Work w;
  unsigned grid;
  e = plan<ROWS>(a, a.H, smem, order, w, grid);
  if (e == cudaSuccess && w.order) e = launch_attn_orders(a, order, nullptr, stream);
  if (e != cudaSuccess) return e;
  attn_fwd_generic_kernel<T, DP, ROWS, ASYNC><<<grid, threads_of(ROWS), smem, stream>>>(a, w);
  return cudaGetLastError();
}

template <typename T, int DP, int ROWS, bool DKV, bool ASYNC>
static cudaError_t run_bwd(const Args &a, const int *order, cudaStream_t stream) {
  constexpr size_t smem = (size_t)(2 * ROWS * (DP + 4) + ROWS * PP + (ASYNC ? 2 : 1) * 2 * TILE * (DP + 5)) * 4;
  static_assert(smem <= 232448, "shared memory of a block");
  cudaError_t e = allow_smem<attn_bwd_generic_kernel<T, DP, ROWS, DKV, ASYNC>>(smem);
  if (e != cudaSuccess) return e;
  Work w;
  unsigned grid;
  e = plan<ROWS>(a, DKV ? a.Hk * a.splits : a.H, smem, order, w, grid);
  if (e != cudaSuccess) return e;
  attn_bwd_generic_kernel<T, DP, ROWS, DKV, ASYNC><<<grid, threads_of(ROWS), smem, stream>>>(a, w);
  return cudaGetLastError();
}

// blocks of 32 or 64 rows, copied or loaded tiles.  Two stages of D = 128 with 64 rows
// do not fit: those stay with 32.
template <typename T, int DP>
static cudaError_t pick_fwd(const Args &a, int *order, cudaStream_t stream) {
  if constexpr (std::is_same<T, float>::value) {
    if (fp32_rows(a, false))
      return short_rows(a.T, a.H) ? run_fwd<T, DP, 32, true>(a, order, stream) : run_fwd<T, DP, 64, true>(a, order, stream);
  }
  return short_rows(a.T, a.H) ? run_fwd<T, DP, 32, false>(a, order, stream) : run_fwd<T, DP, 64, false>(a, order, stream);
}
template <typename T, int DP, bool DKV>
static cudaError_t pick_bwd(const Args &a, const int *order, cudaStream_t stream) {
  const bool few = short_rows(a.T, DKV ? a.Hk * a.splits : a.H);
  if constexpr (std::is_same<T, float>::value) {
    if (fp32_rows(a, true)) {
      if constexpr (DP <= 96)
        if (!few) return run_bwd<T, DP, 64, DKV, true>(a, order, stream);
      return run_bwd<T, DP, 32, DKV, true>(a, order, stream);
    }
  }
  return few ? run_bwd<T, DP, 32, DKV, false>(a, order, stream) : run_bwd<T, DP, 64, DKV, false>(a, order, stream);
}

}  // namespace attn

cudaError_t launch_attn_fwd_generic(const attn::Args &a, int *order, cudaStream_t stream) {
  return with_dtype(a.dtype, [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    return attn::with_dim(a.D, [&](auto d) -> cudaError_t { return attn::pick_fwd<T, decltype(d)::value>(a, order, stream); });
  });
}

cudaError_t launch_attn_delta(const attn::Args &a, uint32_t *amax, cudaStream_t stream) {
  const int64_t blocks = (a.T * a.H + 63) / 64;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks);
  const bool vec = a.D % 8 == 0 && !(((uintptr_t)a.out | (uintptr_t)a.out_lo | (uintptr_t)a.dout) & 15);
  return with_dtype(a.dtype, [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if constexpr (sizeof(T) == 2) {
      if (vec) {
        attn::attn_delta_kernel<T, 8><<<grid, 256, 0, stream>>>(a, amax);
        return cudaGetLastError();
      }
    }
    attn::attn_delta_kernel<T, 1><<<grid, 256, 0, stream>>>(a, amax);
    return cudaGetLastError();
  });
}

cudaError_t launch_attn_bwd_generic(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream) {
  return with_dtype(a.dtype, [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    return attn::with_dim(a.D, [&](auto d) -> cudaError_t {
      constexpr int DP = decltype(d)::value;
      const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
      cudaError_t e = cudaSuccess;  // one direction's blocks of 32 rows could be more than the SMs
      if ((a.T + attn::TM - 1) / attn::TM * 4 * a.H > sms) e = launch_attn_orders(a, order_q, order_k, stream);
      if (e == cudaSuccess && a.dq) e = attn::pick_bwd<T, DP, false>(a, order_q, stream);
      if (e == cudaSuccess && a.dk) e = attn::pick_bwd<T, DP, true>(a, order_k, stream);
      if (e == cudaSuccess && a.dk && a.splits > 1) {
        attn::attn_join_any_kernel<T><<<grid_for(2 * a.T * a.Hk * a.D, 256, sms, 8), 256, 0, stream>>>(a);
        e = cudaGetLastError();
      }
      return e;
    });
  });
}

}  // namespace mhc

using namespace mhc;

static int check_attn(const char *who, attn::Args &a, const int64_t *strides, float scale) {
  if (a.T < 0 || a.T > 2147483647LL - 512) return fail(MHC_ERR_SHAPE, "%s: T = %lld", who, (long long)a.T);
  if (a.H < 1 || a.Hk < 1 || a.H > 65535 || a.H % a.Hk)
    return fail(MHC_ERR_SHAPE, "%s: %d query heads cannot share %d key heads", who, a.H, a.Hk);
  if (a.D < 1 || a.D > 128) return fail(MHC_ERR_SHAPE, "%s: head sizes up to 128 are supported (got %d)", who, a.D);
  if (a.dtype != MHC_F32 && a.dtype != MHC_BF16 && a.dtype != MHC_F16) return fail(MHC_ERR_DTYPE, "%s: bad dtype code %d", who, a.dtype);
  if (!(scale > 0.f) || scale > 3e38f) return fail(MHC_ERR_SHAPE, "%s: scale must be positive and finite", who);
  if (a.cu) {
    if (a.batch < 1) return fail(MHC_ERR_SHAPE, "%s: cu_seqlens of %d sequences", who, a.batch);
    if ((uintptr_t)a.cu & 3) return fail(MHC_ERR_ALIGN, "%s: cu_seqlens is misaligned", who);
  } else if (a.T > 0 && (a.seqlen < 1 || a.T % a.seqlen)) {
    return fail(MHC_ERR_SHAPE, "%s: %lld tokens are not sequences of %lld", who, (long long)a.T, (long long)a.seqlen);
  }
  if (!strides) return fail(MHC_ERR_NULL, "%s: strides is NULL", who);
  for (int i = 0; i < 6; ++i)
    if (strides[i] < 0) return fail(MHC_ERR_SHAPE, "%s: negative stride", who);
  a.qt = strides[0]; a.qh = strides[1]; a.kt = strides[2]; a.kh = strides[3]; a.vt = strides[4]; a.vh = strides[5];
  a.scale = scale;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.err_flag = host_error_flag();
  return MHC_OK;
}

static bool misaligned(size_t es, std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if ((uintptr_t)p % es) return true;
  return false;
}

extern "C" {

size_t mhc_attn_fwd_workspace(int64_t T) { return T < 1 ? 256 : attn_order_bytes(T) + 256; }

int mhc_attn_fwd(const void *q, const void *k, const void *v, int dtype, int64_t T, int H, int Hk, int D,
                 const int64_t *strides, const int32_t *cu_seqlens, int batch, int64_t seqlen, float scale, void *out,
                 void *out_lo, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  attn::Args a{};
  a.q = q; a.k = k; a.v = v; a.o = out; a.o_lo = out_lo; a.lse = lse;
  a.T = T; a.Tp = mhc_attn_lse_pitch(T); a.H = H; a.Hk = Hk; a.D = D; a.dtype = dtype;
  a.cu = cu_seqlens; a.batch = batch; a.seqlen = seqlen;
  if (int st = check_attn("mhc_attn_fwd", a, strides, scale)) return st;
  if (T == 0) return MHC_OK;
  if (!q || !k || !v || !out || !lse) return fail(MHC_ERR_NULL, "mhc_attn_fwd: required pointer is NULL");
  if (misaligned(dtype == MHC_F32 ? 4 : 2, {q, k, v, out, out_lo}) || ((uintptr_t)lse & 3))
    return fail(MHC_ERR_ALIGN, "mhc_attn_fwd: a pointer is not aligned to its elements");
  if (!workspace || workspace_bytes < mhc_attn_fwd_workspace(T))
    return fail(MHC_ERR_WORKSPACE, "mhc_attn_fwd: workspace %zu < %zu bytes", workspace_bytes, mhc_attn_fwd_workspace(T));
  if ((uintptr_t)workspace & 15) return fail(MHC_ERR_ALIGN, "mhc_attn_fwd: workspace is not 16-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!generic_forced() && attn_tc_eligible(a)) {
    const cudaError_t e = launch_attn_fwd_tc(a, static_cast<int *>(workspace), st);
    if (e != cudaErrorNotSupported) return cuda_status(e, "mhc_attn_fwd");
    cudaGetLastError();
  }
  return cuda_status(launch_attn_fwd_generic(a, static_cast<int *>(workspace), st), "mhc_attn_fwd");
}

int64_t mhc_attn_lse_pitch(int64_t T) { return T < 1 ? 0 : (T + 127) / 128 * 128; }

// delta, the two orders of the work, the maxima of fp16, the parts of dK and dV
size_t mhc_attn_bwd_workspace(int64_t T, int H, int Hk, int D) {
  if (T < 1 || H < 1 || Hk < 1 || H % Hk || D < 1 || D > 128) return 256;
  const int splits = attn_bwd_splits(T, H, Hk);
  const size_t parts = splits > 1 ? (size_t)splits * 2 * T * Hk * D * 4 : 0;
  return (size_t)mhc_attn_lse_pitch(T) * (4 * (size_t)H + 8) + 2 * attn_order_bytes(T) + 256 + parts;
}

int mhc_attn_bwd(const void *q, const void *k, const void *v, const void *out, const void *out_lo, const void *dout,
                 const float *lse, int dtype, int64_t T, int H, int Hk, int D, const int64_t *strides, const int32_t *cu_seqlens,
                 int batch, int64_t seqlen, float scale, void *dq, void *dk, void *dv, void *workspace,
                 size_t workspace_bytes, void *stream) {
  clear_error();
  attn::Args a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.out_lo = out_lo; a.dout = dout; a.lse = const_cast<float *>(lse);
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.T = T; a.Tp = mhc_attn_lse_pitch(T); a.H = H; a.Hk = Hk; a.D = D; a.dtype = dtype;
  a.cu = cu_seqlens; a.batch = batch; a.seqlen = seqlen;
  if (int st = check_attn("mhc_attn_bwd", a, strides, scale)) return st;
  if (T == 0) return MHC_OK;
  // dq, or dk and dv together, may be left out
  if (!q || !k || !v || !out || !dout || !lse || !dk != !dv || (!dq && !dk))
    return fail(MHC_ERR_NULL, "mhc_attn_bwd: required pointer is NULL");
  if (misaligned(dtype == MHC_F32 ? 4 : 2, {q, k, v, out, out_lo, dout, dq, dk, dv}) || ((uintptr_t)lse & 3))
    return fail(MHC_ERR_ALIGN, "mhc_attn_bwd: a pointer is not aligned to its elements");
  if (!workspace || workspace_bytes < mhc_attn_bwd_workspace(T, H, Hk, D))
    return fail(MHC_ERR_WORKSPACE, "mhc_attn_bwd: workspace %zu < %zu bytes", workspace_bytes, mhc_attn_bwd_workspace(T, H, Hk, D));
  if ((uintptr_t)workspace & 15) return fail(MHC_ERR_ALIGN, "mhc_attn_bwd: workspace is not 16-byte aligned");
  a.delta = static_cast<float *>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool tc = !generic_forced() && attn_tc_bwd_eligible(a);
  int *order = reinterpret_cast<int *>(a.delta + a.Tp * H);
  const size_t on = attn_order_bytes(T) / 4;
  uint32_t *amax = nullptr;
  cudaError_t e = cudaSuccess;
  if (tc && dtype == MHC_F16) {
    amax = reinterpret_cast<uint32_t *>(order + 2 * on);
    a.amax = amax;
    e = cudaMemsetAsync(amax, 0, (size_t)a.Tp * 8, st);
  }
  if (e == cudaSuccess) e = launch_attn_delta(a, amax, st);
  a.splits = attn_bwd_splits(T, H, Hk);
  const uintptr_t at = (reinterpret_cast<uintptr_t>(order + 2 * on) + (uintptr_t)a.Tp * 8 + 15) & ~(uintptr_t)15;
  a.parts = a.splits > 1 ? reinterpret_cast<float *>(at) : nullptr;
  if (e == cudaSuccess && tc) {
    e = launch_attn_bwd_tc(a, order, order + on, st);
    if (e != cudaErrorNotSupported) return cuda_status(e, "mhc_attn_bwd");
    cudaGetLastError();
    e = cudaSuccess;
  }
  if (e == cudaSuccess) e = launch_attn_bwd_generic(a, order, order + on, st);
  return cuda_status(e, "mhc_attn_bwd");
}

}  // extern "C"
