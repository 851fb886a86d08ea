// Rows of the attention that a masked value has reached.
//
// The products run over whole tiles: the weight of a pair that a row does not see is
// exactly 0, and 0 times an infinity or a NaN that lies there is a NaN.  It cannot hide:
// a row that took one in has a NaN in its result.  So a block that meets a NaN in what
// it writes does those rows again from the formula, over the visible pairs only, one
// warp a row, in fp32; a row that is a NaN by the formula comes out as one again.  No
// other row pays for it (the tests of the results take no measurable time), and a row
// of nothing but NaN ends after its first 32 pairs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_attn.cuh"
#include "mhc_device.cuh"

namespace mhc {
namespace attn {

constexpr int LANE_D = 4;  // values of a row of up to 128 that a lane has: lane + 32 u

template <typename T>
__device__ __forceinline__ bool row_has_nan(const T *row, int D, int lane) {
  bool bad = false;
  for (int d = lane; d < D; d += 32) bad |= isnan(to_f(row[d]));
  return __any_sync(0xffffffffu, bad);
}
// a row as the lanes hold it, zero past D
template <typename T>
__device__ __forceinline__ void lane_row(const void *p, int64_t at, int D, int lane, float (&x)[LANE_D]) {
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) x[u] = lane + 32 * u < D ? to_f(static_cast<const T *>(p)[at + lane + 32 * u]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void lane_store(T *p, int D, int lane, const float (&x)[LANE_D]) {
#pragma unroll
  for (int u = 0; u < LANE_D; ++u)
    if (lane + 32 * u < D) p[lane + 32 * u] = from_f<T>(x[u]);
}
__device__ __forceinline__ float lane_dot(const float (&x)[LANE_D], const float (&y)[LANE_D]) {
  float s = 0.f;
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) s = fmaf(x[u], y[u], s);
  return warp_sum(s);
}
__device__ __forceinline__ bool lane_all_nan(const float (&x)[LANE_D], int D, int lane) {
  bool all = true;
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) all &= lane + 32 * u >= D || isnan(x[u]);
  return __all_sync(0xffffffffu, all);
}

// out (and out_lo) of token i, head h
template <typename T>
__device__ __noinline__ void redo_out(const Args &a, int h, int i, int lane) {
  const int hk = h / (a.H / a.Hk);
  float q[LANE_D], o[LANE_D] = {}, m = -INFINITY, sum = 0.f;
  lane_row<T>(a.q, (int64_t)i * a.qt + h * a.qh, a.D, lane, q);
  const int start = span_of(a, i).start;
  for (int j = start; j <= i; ++j) {
    float k[LANE_D], v[LANE_D];
    lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
    lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
    const float s = lane_dot(q, k) * a.scale_log2, top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float fix = exp2f(m - base), p = exp2f(s - base);
    sum = sum * fix + p;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) o[u] = o[u] * fix + p * v[u];
    m = top;
    if (((j - start) & 31) == 31 && (isnan(sum) || lane_all_nan(o, a.D, lane))) break;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float lo[LANE_D];
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) {
    o[u] *= inv;
    lo[u] = o[u] - to_f(from_f<T>(o[u]));
  }
  const int64_t at = ((int64_t)i * a.H + h) * a.D;
  lane_store(static_cast<T *>(a.o) + at, a.D, lane, o);
  if (a.o_lo) lane_store(static_cast<T *>(a.o_lo) + at, a.D, lane, lo);
}

// dq of token i, head h
template <typename T>
__device__ __noinline__ void redo_dq(const Args &a, int h, int i, int lane) {
  const int hk = h / (a.H / a.Hk);
  const int64_t at = ((int64_t)i * a.H + h) * a.D, stat = (int64_t)h * a.Tp + i;
  float q[LANE_D], g[LANE_D], dq[LANE_D] = {};
  lane_row<T>(a.q, (int64_t)i * a.qt + h * a.qh, a.D, lane, q);
  lane_row<T>(a.dout, at, a.D, lane, g);
  const float lse = a.lse[stat], mean = a.delta[stat];
  const int start = span_of(a, i).start;
  for (int j = start; j <= i; ++j) {
    float k[LANE_D], v[LANE_D];
    lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
    lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
    const float ds = exp2f(fmaf(lane_dot(q, k), a.scale_log2, -lse)) * (lane_dot(g, v) - mean);
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) dq[u] = fmaf(ds, k[u], dq[u]);
    if (((j - start) & 31) == 31 && lane_all_nan(dq, a.D, lane)) break;
  }
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) dq[u] *= a.scale;
  lane_store(static_cast<T *>(a.dq) + at, a.D, lane, dq);
}

// dk and dv of token j, key head hk, over `heads` query heads from h0 on
template <typename T, typename U>
__device__ __noinline__ void redo_dkv(const Args &a, int hk, int j, int h0, int heads, U *dk_row, U *dv_row, int lane) {
  float k[LANE_D], v[LANE_D], dk[LANE_D] = {}, dv[LANE_D] = {};
  lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
  lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
  const int end = span_of(a, j).end;
  bool dead = false;
  for (int h = h0; h < h0 + heads && !dead; ++h)
    for (int i = j; i < end && !dead; ++i) {
      float q[LANE_D], g[LANE_D];
      lane_row<T>(a.q, (int64_t)i * a.qt + h * a.qh, a.D, lane, q);
      lane_row<T>(a.dout, ((int64_t)i * a.H + h) * a.D, a.D, lane, g);
      const int64_t stat = (int64_t)h * a.Tp + i;
      const float p = exp2f(fmaf(lane_dot(k, q), a.scale_log2, -a.lse[stat])), ds = p * (lane_dot(v, g) - a.delta[stat]);
#pragma unroll
      for (int u = 0; u < LANE_D; ++u) {
        dk[u] = fmaf(ds, q[u], dk[u]);
        dv[u] = fmaf(p, g[u], dv[u]);
      }
      dead = ((i - j) & 31) == 31 && lane_all_nan(dk, a.D, lane) && lane_all_nan(dv, a.D, lane);
    }
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) dk[u] *= a.scale;
  lane_store(dk_row, a.D, lane, dk);
  lane_store(dv_row, a.D, lane, dv);
}

// The same where one of the two rows has a NaN: rows of dk and dv, or of a block's part of them
template <typename T, typename U>
__device__ __forceinline__ void redo_dkv_rows(const Args &a, int hk, int row0, int rows, int h0, int heads, U *dk, U *dv, int warp,
                                              int warps, int lane) {
  for (int r = warp; r < rows && row0 + r < a.T; r += warps) {
    const int64_t at = ((int64_t)(row0 + r) * a.Hk + hk) * a.D;
    const bool bad = row_has_nan(dk + at, a.D, lane) || row_has_nan(dv + at, a.D, lane);
    if (bad) redo_dkv<T, U>(a, hk, row0 + r, h0, heads, dk + at, dv + at, lane);
  }
}

}  // namespace attn
}  // namespace mhc
