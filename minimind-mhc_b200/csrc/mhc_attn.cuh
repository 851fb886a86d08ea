// Shared by the attention kernels: the arguments and which keys a token sees.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mhc {
namespace attn {

// q (T, H, D), k / v (T, Hk, D) with token and head strides in elements and
// contiguous rows; out, dout, dq and dk / dv are contiguous; lse and delta are
// (H, Tp) fp32; o_lo / out_lo hold what the rounding of out left over, or are null.  lse is in base 2: log2 of the sum of exp2(score * scale_log2).
struct Args {
  const void *q, *k, *v, *out, *out_lo, *dout;
  void *o, *o_lo, *dq, *dk, *dv;
  float *lse, *delta;
  const uint32_t *amax;  // fp16 backward: at a sequence's start s, 2 s and 2 s + 1: the bits of its largest finite |dO| and |V|
  int64_t T, Tp;         // Tp: T up to whole tiles of 128, the pitch of lse and delta
  int H, Hk, D, dtype;
  int64_t qt, qh, kt, kh, vt, vh;
  const int32_t *cu;  // (batch + 1) offsets of the packed sequences, or null: sequences of seqlen tokens
  int batch;
  int64_t seqlen;
  float scale, scale_log2;
  int splits;    // blocks that share a tile of keys in the backward, each with some of the group's heads
  float *parts;  // their dK and dV: (splits, 2, T, Hk, D) fp32, where there are more than one
  int *err_flag;
};

// The sequence [start, end) of token i.  A token outside of every sequence
// (before cu[0], from cu[batch] on) has start = i + 1, end = i: it sees nothing and
// nothing sees it.  Both are monotone in i, and within [0, T] whatever cu holds.
struct Span {
  int start, end;
};
__device__ __forceinline__ Span span_of(const Args &a, int i) {
  Span s;
  if (a.cu == nullptr) {
    const int l = (int)a.seqlen;
    s.start = i / l * l;
    s.end = s.start + l;
    return s;
  }
  if (i < a.cu[0] || i >= a.cu[a.batch]) {
    s.start = i + 1;
    s.end = i;
    return s;
  }
  int lo = 0, hi = a.batch;  // cu[lo] <= i < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= i) lo = mid; else hi = mid;
  }
  s.start = max(0, min(a.cu[lo], i));
  s.end = max(i + 1, (int)min((int64_t)a.cu[lo + 1], a.T));
  return s;
}
// tokens inside some sequence: [first, last)
__device__ __forceinline__ Span packed_range(const Args &a) {
  Span s;
  s.start = a.cu ? max(0, a.cu[0]) : 0;
  s.end = a.cu ? (int)min((int64_t)max(0, a.cu[a.batch]), a.T) : (int)a.T;
  return s;
}

}  // namespace attn

cudaError_t launch_attn_fwd_generic(const attn::Args &a, int *order, cudaStream_t stream);
cudaError_t launch_attn_bwd_generic(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream);
cudaError_t launch_attn_delta(const attn::Args &a, uint32_t *amax, cudaStream_t stream);

}  // namespace mhc
