// Rows of the attention that a masked value has reached.
//
// The products run over whole tiles: the weight of a pair that a row does not see is
// exactly 0, and 0 times an infinity or a NaN that lies there is a NaN.  It cannot hide:
// a row that took one in has a NaN in its result.  So a block that meets a NaN in what
// it writes looks its rows through, one warp a row:
//   - A NaN that the formula gives is left alone: a NaN among the row's own statistics
//     (lse, and D in the backward, both of visible pairs only), or in the column that is
//     summed, at a token that the row sees.
//   - Any other row is done again from the formula, over the visible pairs only, in fp32.
// Without a NaN in its rows a block pays for the tests of its results alone, which do not
// show in its time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_attn.cuh"
#include "mhc_device.cuh"

namespace mhc {
namespace attn {

constexpr int LANE_D = 4;            // values of a row of up to 128 that a lane has: lane + 32 u
constexpr int NOWHERE = 0x7fffffff;  // after every token

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

// The lane's columns of rows [lo, hi) of x (`stride` apart): the first row whose value is not finite, NOWHERE if none
template <typename T>
__device__ __noinline__ void first_not_finite(const T *x, int64_t stride, int lo, int hi, int D, int lane, int (&at)[LANE_D]) {
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) at[u] = NOWHERE;
  for (int j0 = lo; j0 < hi; j0 += 8) {
    bool open = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v[LANE_D];
      lane_row<T>(x, (int64_t)min(j0 + e, hi - 1) * stride, D, lane, v);
#pragma unroll
      for (int u = 0; u < LANE_D; ++u)
        if (at[u] == NOWHERE && !isfinite(v[u])) at[u] = min(j0 + e, hi - 1);
    }
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) open |= at[u] == NOWHERE && lane + 32 * u < D;
    if (!__any_sync(0xffffffffu, open)) break;
  }
}

// out (and out_lo) of token i, head h
template <typename T>
__device__ __noinline__ void redo_out(const Args &a, int h, int i, int lane) {
  const int hk = h / (a.H / a.Hk);
  float q[LANE_D], o[LANE_D] = {}, m = -INFINITY, sum = 0.f;
  lane_row<T>(a.q, (int64_t)i * a.qt + h * a.qh, a.D, lane, q);
#pragma unroll 4
  for (int j = span_of(a, i).start; j <= i; ++j) {
    float k[LANE_D], v[LANE_D];
    lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
    lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
    const float s = lane_dot(q, k) * a.scale_log2, top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float fix = exp2f(m - base), p = exp2f(s - base);
    sum = sum * fix + p;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) o[u] = o[u] * fix + p * v[u];
    m = top;
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

// Rows [row0, row0 + rows) of head h of out; each warp of the block calls it
template <typename T>
__device__ __noinline__ void redo_out_rows(const Args &a, int h, int row0, int rows, int warp, int warps, int lane) {
  const int hk = h / (a.H / a.Hk), last = (int)min((int64_t)row0 + rows, a.T);
  int start = -1, at[LANE_D];
  for (int i = row0 + warp; i < last; i += warps) {
    float o[LANE_D];
    lane_row<T>(a.o, ((int64_t)i * a.H + h) * a.D, a.D, lane, o);
    bool bad = false;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) bad |= isnan(o[u]);
    if (!__any_sync(0xffffffffu, bad) || isnan(a.lse[(int64_t)h * a.Tp + i])) continue;
    const Span s = span_of(a, i);
    if (s.start != start) {  // for the rows of this sequence
      start = s.start;
      first_not_finite(static_cast<const T *>(a.v) + hk * a.vh, a.vt, start, min(s.end, last), a.D, lane, at);
    }
    bad = false;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) bad |= isnan(o[u]) && at[u] > i;
    if (__any_sync(0xffffffffu, bad)) redo_out<T>(a, h, i, lane);
  }
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
#pragma unroll 4
  for (int j = start; j <= i; ++j) {
    float k[LANE_D], v[LANE_D];
    lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
    lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
    const float p = exp2f(fmaf(lane_dot(q, k), a.scale_log2, -lse));
    const float ds = (start == i ? 0.f : p) * (lane_dot(g, v) - mean);  // alone: 0 but for rounding
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) dq[u] = fmaf(ds, k[u], dq[u]);
  }
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) dq[u] *= a.scale;
  lane_store(static_cast<T *>(a.dq) + at, a.D, lane, dq);
}

// Rows of head h of dq.  A D that is not finite leaves no dS of its row finite.
template <typename T>
__device__ __noinline__ void redo_dq_rows(const Args &a, int h, int row0, int rows, int warp, int warps, int lane) {
  for (int i = row0 + warp; i < row0 + rows && i < a.T; i += warps) {
    const int64_t stat = (int64_t)h * a.Tp + i;
    if (isnan(a.lse[stat]) || !isfinite(a.delta[stat])) continue;
    float x[LANE_D];
    lane_row<T>(a.dq, ((int64_t)i * a.H + h) * a.D, a.D, lane, x);
    bool bad = false;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) bad |= isnan(x[u]);
    if (__any_sync(0xffffffffu, bad)) redo_dq<T>(a, h, i, lane);
  }
}

// dk and dv of token j, key head hk, over `heads` query heads from h0 on
template <typename T, typename U>
__device__ __noinline__ void redo_dkv(const Args &a, int hk, int j, int h0, int heads, U *dk_row, U *dv_row, int lane) {
  float k[LANE_D], v[LANE_D], dk[LANE_D] = {}, dv[LANE_D] = {};
  lane_row<T>(a.k, (int64_t)j * a.kt + hk * a.kh, a.D, lane, k);
  lane_row<T>(a.v, (int64_t)j * a.vt + hk * a.vh, a.D, lane, v);
  const int start = span_of(a, j).start, end = span_of(a, j).end;
  for (int h = h0; h < h0 + heads; ++h)
#pragma unroll 4
    for (int i = j; i < end; ++i) {
      float q[LANE_D], g[LANE_D];
      lane_row<T>(a.q, (int64_t)i * a.qt + h * a.qh, a.D, lane, q);
      lane_row<T>(a.dout, ((int64_t)i * a.H + h) * a.D, a.D, lane, g);
      const int64_t stat = (int64_t)h * a.Tp + i;
      const float p = exp2f(fmaf(lane_dot(k, q), a.scale_log2, -a.lse[stat]));
      const float ds = (start == i ? 0.f : p) * (lane_dot(v, g) - a.delta[stat]);
#pragma unroll
      for (int u = 0; u < LANE_D; ++u) {
        dk[u] = fmaf(ds, q[u], dk[u]);
        dv[u] = fmaf(p, g[u], dv[u]);
      }
    }
#pragma unroll
  for (int u = 0; u < LANE_D; ++u) dk[u] *= a.scale;
  lane_store(dk_row, a.D, lane, dk);
  lane_store(dv_row, a.D, lane, dv);
}

// Rows of key head hk of dk and dv, or of a block's part of them.  Every column of dk has to do with all of dS; a
// column of dv only with that column of dO.
template <typename T, typename U>
__device__ __noinline__ void redo_dkv_rows(const Args &a, int hk, int row0, int rows, int h0, int heads, U *dk, U *dv, int warp,
                                              int warps, int lane) {
  // the rows backwards, so that what a row adds to the queries of the last one is looked at once
  const int last = (int)min((int64_t)row0 + rows, a.T) - 1;
  int end = -1, from = 0;  // seen so far: queries [from, end)
  bool nan_p = false, bad_d = false, known[LANE_D];  // among them: a NaN of lse, a D that is not finite, columns of dO
  for (int j = last - warp; j >= row0; j -= warps) {
    const int64_t row = ((int64_t)j * a.Hk + hk) * a.D;
    float x[LANE_D], y[LANE_D];
    lane_row<U>(dk, row, a.D, lane, x);
    lane_row<U>(dv, row, a.D, lane, y);
    bool bad_k = false, bad_v = false;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) {
      bad_k |= isnan(x[u]);
      bad_v |= isnan(y[u]);
    }
    bad_k = __any_sync(0xffffffffu, bad_k);
    bad_v = __any_sync(0xffffffffu, bad_v);
    if (!bad_k && !bad_v) continue;
    const Span s = span_of(a, j);
    if (s.end != end) {
      end = from = s.end;
      nan_p = bad_d = false;
#pragma unroll
      for (int u = 0; u < LANE_D; ++u) known[u] = false;
    }
    for (int h = h0; h < h0 + heads; ++h) {
      for (int i = j + lane; i < from; i += 32) {
        nan_p |= isnan(a.lse[(int64_t)h * a.Tp + i]);
        bad_d |= !isfinite(a.delta[(int64_t)h * a.Tp + i]);
      }
      int at[LANE_D];
      first_not_finite(static_cast<const T *>(a.dout) + (int64_t)h * a.D, (int64_t)a.H * a.D, j, from, a.D, lane, at);
#pragma unroll
      for (int u = 0; u < LANE_D; ++u) known[u] |= at[u] != NOWHERE;
    }
    from = j;
    nan_p = __any_sync(0xffffffffu, nan_p);
    bad_d = __any_sync(0xffffffffu, bad_d);
    if (nan_p) continue;
    bool redo = bad_k && !bad_d;
#pragma unroll
    for (int u = 0; u < LANE_D; ++u) redo |= isnan(y[u]) && !known[u];
    if (__any_sync(0xffffffffu, redo)) redo_dkv<T, U>(a, hk, j, h0, heads, dk + row, dv + row, lane);
  }
}

}  // namespace attn
}  // namespace mhc
