// AdamW over many tensors in one launch, moments in fp32 or in 8 bits.
//
//   g' = g * clip                     clip = min(1, max_norm / (||g|| + 1e-6)), or 1
//   m' = b1 m + (1 - b1) g'           v' = b2 v + ((1 - b2) g') g'
//   p' = p (1 - lr wd) - (lr / (1 - b1^t)) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Every value is touched once, so the kernel is bound by HBM: 28 bytes a value
// with fp32 parameters, gradients and moments, 16 with 8-bit moments.  The
// tensors' table travels as a kernel argument (up to 31 KB), so a step needs no
// copy to the device, no table kept between calls and one launch for up to
// MAX_TENSORS tensors.
//
// 8-bit moments: 256 consecutive values share one fp32 scale, the largest
// magnitude among them.  m = (c / 127)^2 * sign * scale with c = round(127
// sqrt(|m| / scale)): the squared spacing keeps small momenta (down to 6e-5 of
// the largest) apart.  v = (c / 255)^4 * scale with c = round(255 (v /
// scale)^(1/4)): a step divides by sqrt(v), whose spacing is then quadratic, and
// a code of zero is kept for v = 0 (anything above it takes at least 1), since a
// v rounded to zero would divide by eps.  The step itself uses the fp32 m' and
// v'; only what is stored is rounded.  A block with a non-finite moment gets the
// non-finite scale and so reads back as NaN, as fp32 moments would.
// What decides a code uses single IEEE operations (no contraction, no approximate
// division or root): a value next to the edge between two codes then falls on the
// same side wherever the formula is evaluated in fp32.
//
// A warp owns one block of 256 values at a time, a lane 4 + 4 of them (16-byte
// accesses in fp32, 8-byte in 16-bit types, 4-byte for codes), so the block's
// largest magnitude is one warp reduction.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "mhc_b200.h"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace adamw {

constexpr int QB = 256;             // values per 8-bit block, per warp step
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CHUNK = QB * WARPS * 2;  // values of one tensor a block takes at a time
constexpr int MAX_TENSORS = 440;    // 72 bytes each: the largest table a launch's 32,764 bytes of arguments carry
// The smaller table of the two: 1.7 KB of arguments where a launch of the large one moves 31 KB.  A step's call, 14
// tensors of 10,000 values: 10.9 us with the small table, 12.5 with the large one (16.4 and 20.1 with the norm's launch);
// 24 tensors: 12.9 and 14.6.  A third one in between would gain 2 us of 23 at 60 tensors.
constexpr int FEW_TENSORS = 24;

struct Entry {
  void *p;
  const void *g;
  void *m, *v;
  float *ms, *vs;
  int64_t n;
  int first_chunk;
  uint8_t pdt, gdt, vec, pad;
  float rbc2, step_size;  // 1 / sqrt(1 - b2^t), lr / (1 - b1^t) at the tensor's own step t
};
static_assert(sizeof(Entry) == 72, "table entry");

template <int N>
struct Table {
  Entry t[N];
  int count, chunks;
};

struct Scalars {
  float b1, c1, b2, c2, eps, keep;  // c = 1 - b, keep = 1 - lr wd
  float max_norm;
  const double *partials;  // squared-norm partials, or null: no clipping
  int npartials;
  float *norm_out;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The values a lane holds of its warp's block: value index base + lane_value(e),
// e < 8; two runs of four.
__device__ __forceinline__ int lane_value(int lane, int e) { return (e >> 2) * 128 + lane * 4 + (e & 3); }

// A lane's 8 values of a runtime-typed tensor as they lie in memory.  Loading and
// converting are apart, so that a lane asks for everything before it waits for the
// first of it (bf16 parameters converted as they came: 1.40 ms for the 321 M values
// of the MoE decoder, against 1.14 ms).
struct Raw {
  uint4 a, b;  // 16-bit types: the lower halves
};
template <bool KEEP = false>  // for another pass over the same values
__device__ __forceinline__ Raw load_raw(const void *p, int dt, int64_t base, int lane) {
  Raw r;
  if (dt == MHC_F32) {
    const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + base + lane * 4);
    r.a = KEEP ? __ldg(q) : __ldcs(q);
    r.b = KEEP ? __ldg(q + 32) : __ldcs(q + 32);
  } else {
    const uint2 *q = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + base + lane * 4);
    const uint2 x = KEEP ? __ldg(q) : __ldcs(q), y = KEEP ? __ldg(q + 32) : __ldcs(q + 32);
    r.a.x = x.x; r.a.y = x.y;
    r.b.x = y.x; r.b.y = y.y;
  }
  return r;
}
__device__ __forceinline__ void convert4(const uint4 &r, int dt, float *o) {
  if (dt == MHC_F32) {
    o[0] = __uint_as_float(r.x); o[1] = __uint_as_float(r.y); o[2] = __uint_as_float(r.z); o[3] = __uint_as_float(r.w);
  } else if (dt == MHC_BF16) {
    o[0] = __uint_as_float(r.x << 16); o[1] = __uint_as_float(r.x & 0xffff0000u);
    o[2] = __uint_as_float(r.y << 16); o[3] = __uint_as_float(r.y & 0xffff0000u);
  } else {
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&r.x));
    const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
    o[0] = x.x; o[1] = x.y; o[2] = y.x; o[3] = y.y;
  }
}
__device__ __forceinline__ void convert8(const Raw &r, int dt, float (&o)[8]) {
  convert4(r.a, dt, o);
  convert4(r.b, dt, o + 4);
}
__device__ __forceinline__ void store4(void *p, int dt, int64_t i, const float *v) {
  if (dt == MHC_F32) {
    __stcs(reinterpret_cast<float4 *>(static_cast<float *>(p) + i), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint2 r;
    if (dt == MHC_BF16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      r.x = *reinterpret_cast<const uint32_t *>(&a);
      r.y = *reinterpret_cast<const uint32_t *>(&b);
    } else {
      const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
      r.x = *reinterpret_cast<const uint32_t *>(&a);
      r.y = *reinterpret_cast<const uint32_t *>(&b);
    }
    __stcs(reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i), r);
  }
}
// value by value, for blocks that end early or lie at odd addresses
__device__ __forceinline__ void load_each(const void *p, int dt, int64_t base, int64_t n, int lane, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t i = base + lane_value(lane, e);
    o[e] = i < n ? load_dyn(p, dt, i) : 0.f;
  }
}
__device__ __forceinline__ void store8(void *p, int dt, int64_t base, int64_t n, bool whole, int lane, const float (&v)[8]) {
  if (whole) {
    store4(p, dt, base + lane * 4, v);
    store4(p, dt, base + 128 + lane * 4, v + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = base + lane_value(lane, e);
      if (i < n) store_dyn(p, dt, i, v[e]);
    }
  }
}

// 8-bit codes of a lane, four to a word, and as numbers (signed for m, unsigned for v)
__device__ __forceinline__ uint2 load_codes(const void *p, int64_t base, int64_t n, bool whole, int lane) {
  const uint8_t *q = static_cast<const uint8_t *>(p);
  if (whole)
    return make_uint2(__ldcs(reinterpret_cast<const uint32_t *>(q + base + lane * 4)),
                      __ldcs(reinterpret_cast<const uint32_t *>(q + base + 128 + lane * 4)));
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t i = base + lane_value(lane, e);
    if (i < n) w[e >> 2] |= (uint32_t)q[i] << (8 * (e & 3));
  }
  return make_uint2(w[0], w[1]);
}
// through the low bits of 2^23 (byte 0x4B, then the code): the integer conversions and
// rounding instructions run at the special function unit's rate, which the roots need
template <bool SIGNED>
__device__ __forceinline__ float code_value(const uint2 &w, int e) {
  const uint32_t word = SIGNED ? (e < 4 ? w.x : w.y) ^ 0x80808080u : (e < 4 ? w.x : w.y);
  const float f = __uint_as_float(__byte_perm(word, 0x4B000000u, 0x7650u | (e & 3)));
  return f - (SIGNED ? 8388736.f : 8388608.f);
}
// codes in the low bytes of eight words
__device__ __forceinline__ void store_codes(void *p, int64_t base, int64_t n, bool whole, int lane, const uint32_t (&c)[8]) {
  uint8_t *q = static_cast<uint8_t *>(p);
  if (whole) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __byte_perm(c[h * 4], c[h * 4 + 1], 0x0040), hi = __byte_perm(c[h * 4 + 2], c[h * 4 + 3], 0x0040);
      __stcs(reinterpret_cast<uint32_t *>(q + base + h * 128 + lane * 4), __byte_perm(lo, hi, 0x5410));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t i = base + lane_value(lane, e);
      if (i < n) q[i] = (uint8_t)c[e];
    }
  }
}

__device__ __forceinline__ float unpack_m(float c, float scale) {
  return __fmul_rn(__fmul_rn(c * fabsf(c), scale), (float)(1.0 / 16129.0));
}
__device__ __forceinline__ float unpack_v(float c, float scale) {
  const float cc = c * c;  // an integer up to 65025: exact
  return __fmul_rn(__fmul_rn(__fmul_rn(__fmul_rn(cc, scale), (float)(1.0 / 65025.0)), cc), (float)(1.0 / 65025.0));
}
__device__ __forceinline__ int pack_m(float m, float safe) {
  const float r = rintf(__fmul_rn(__fsqrt_rn(__fdiv_rn(fabsf(m), safe)), 127.f));
  return __float2int_rn(m < 0.f ? -r : r);  // NaN converts to 0
}
__device__ __forceinline__ int pack_v(float v, float safe) {
  const int c = __float2int_rn(__fmul_rn(__fsqrt_rn(__fsqrt_rn(__fdiv_rn(v, safe))), 255.f));
  return v > 0.f && c < 1 ? 1 : c;
}

__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The same codes, mostly without the IEEE division and roots (three long sequences
// a value: with them the 8-bit step took 2.02 ms for 321 M values, against 1.40 ms).
// y = 127 sqrt(|m| / safe), or 255 (v / safe)^(1/4), from a reciprocal and
// approximate roots is off by at most 4 and 5 units of 2^-23 of itself (roundings of
// the reciprocal, two or three products, a root of 2^-23 each), 6.1e-5 and 1.6e-4 at
// the largest code.  Only where y is nearer than EDGE to the middle between two codes
// can the exact value round to the other; there the lane's codes are done again
// exactly.  `inv` = 1 / safe; scales too small for it to be a normal number are
// passed with inv = 0 and are all done exactly.  A code is the low byte of y + 1.5 *
// 2^23, where the addition rounds to the nearest integer (in two's complement).
template <bool SIGNED>
__device__ __forceinline__ void pack_codes(const float (&x)[8], float safe, float inv, uint32_t (&c)[8]) {
  constexpr float EDGE = SIGNED ? 1e-4f : 2.5e-4f;
  constexpr float kMagic = 12582912.f;
  bool near = inv == 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = fabsf(x[e]) * inv;
    float y;
    if (SIGNED)
      y = copysignf(sqrt_approx(q) * 127.f, x[e]);
    else
      y = fmaxf(sqrt_approx(sqrt_approx(q)) * 255.f, x[e] > 0.f ? 1.f : 0.f);  // above zero stays above zero
    const float t = y + kMagic;
    near |= !(fabsf(y - (t - kMagic)) < 0.5f - EDGE);  // NaN too
    if (!SIGNED) near |= q != q;                       // which fmaxf drops
    c[e] = __float_as_uint(t);
  }
  if (near) {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      float v = x[0];
#pragma unroll
      for (int u = 1; u < 8; ++u) v = e == u ? x[u] : v;
      const uint32_t k = (uint32_t)(SIGNED ? pack_m(v, safe) : pack_v(v, safe));
#pragma unroll
      for (int u = 0; u < 8; ++u) c[u] = e == u ? k : c[u];
    }
  }
}

// table entry of a chunk: the last one whose first chunk is not above it
template <int N>
__device__ __forceinline__ int entry_of(const Table<N> &tab, int chunk) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].first_chunk <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// Clip factor from the partial sums, each block for itself: the same sum in the
// same order everywhere.
__device__ __forceinline__ float clip_factor(const Scalars &s) {
  __shared__ double sh[WARPS];
  double a = 0.0;
  for (int i = threadIdx.x; i < s.npartials; i += THREADS) a += s.partials[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) t += sh[w];
  const float norm = (float)sqrt(t);
  if (blockIdx.x == 0 && threadIdx.x == 0 && s.norm_out) *s.norm_out = norm;
  const float f = __fdiv_rn(s.max_norm, __fadd_rn(norm, 1e-6f));
  return f < 1.f ? f : (f >= 1.f ? 1.f : f);  // NaN stays NaN
}

template <int N, bool Q8>
__global__ void __launch_bounds__(THREADS, 4) adamw_kernel(const __grid_constant__ Table<N> tab, const Scalars s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float clip = 1.f;
  if (s.partials) clip = clip_factor(s);
  for (int c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    // behind the norm's pass the last gradients are the ones still in L2 (58 M fp32 values: 323 -> 317 us with the norm)
    const int chunk = s.partials ? tab.chunks - 1 - c : c;
    const int ei = entry_of(tab, chunk);
    const Entry &t = tab.t[ei];
    const int64_t first = (int64_t)(chunk - t.first_chunk) * CHUNK;
#pragma unroll 1
    for (int it = 0; it < CHUNK / (QB * WARPS); ++it) {
      const int64_t base = first + (int64_t)(it * WARPS + warp) * QB;
      if (base >= t.n) break;
      const bool whole = t.vec && base + QB <= t.n;
      float p[8], g[8], m[8], v[8];
      if constexpr (Q8) {
        const float sm = t.ms[base / QB], sv = t.vs[base / QB];
        const uint2 cm = load_codes(t.m, base, t.n, whole, lane), cv = load_codes(t.v, base, t.n, whole, lane);
        if (whole) {
          const Raw rp = load_raw(t.p, t.pdt, base, lane), rg = load_raw(t.g, t.gdt, base, lane);
          convert8(rp, t.pdt, p);
          convert8(rg, t.gdt, g);
        } else {
          load_each(t.p, t.pdt, base, t.n, lane, p);
          load_each(t.g, t.gdt, base, t.n, lane, g);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[e] = unpack_m(code_value<true>(cm, e), sm);
          v[e] = unpack_v(code_value<false>(cv, e), sv);
        }
      } else if (whole) {
        const Raw rm = load_raw(t.m, MHC_F32, base, lane), rv = load_raw(t.v, MHC_F32, base, lane);
        const Raw rp = load_raw(t.p, t.pdt, base, lane), rg = load_raw(t.g, t.gdt, base, lane);
        convert8(rp, t.pdt, p);
        convert8(rg, t.gdt, g);
        convert8(rm, MHC_F32, m);
        convert8(rv, MHC_F32, v);
      } else {
        load_each(t.p, t.pdt, base, t.n, lane, p);
        load_each(t.g, t.gdt, base, t.n, lane, g);
        load_each(t.m, MHC_F32, base, t.n, lane, m);
        load_each(t.v, MHC_F32, base, t.n, lane, v);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float gr = s.partials ? __fmul_rn(g[e], clip) : g[e];
        m[e] = __fadd_rn(__fmul_rn(m[e], s.b1), __fmul_rn(gr, s.c1));
        v[e] = __fadd_rn(__fmul_rn(v[e], s.b2), __fmul_rn(__fmul_rn(gr, s.c2), gr));
        const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v[e]), t.rbc2), s.eps);
        p[e] = __fsub_rn(__fmul_rn(p[e], s.keep), __fmul_rn(__fdiv_rn(m[e], denom), t.step_size));
      }
      store8(t.p, t.pdt, base, t.n, whole, lane, p);
      if constexpr (Q8) {
        float am = 0.f, av = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          am = max_nan(am, fabsf(m[e]));
          av = max_nan(av, v[e]);
        }
        am = warp_max_nan(am);
        av = warp_max_nan(av);
        if (lane == 0) {
          t.ms[base / QB] = am;
          t.vs[base / QB] = av;
        }
        // an empty block divides by one; every code is then zero
        const float dm = am > 0.f ? am : 1.f, dv = av > 0.f ? av : 1.f;
        uint32_t c[8];
        pack_codes<true>(m, dm, dm > 1e-30f ? __fdiv_rn(1.f, dm) : 0.f, c);
        store_codes(t.m, base, t.n, whole, lane, c);
        pack_codes<false>(v, dv, dv > 1e-30f ? __fdiv_rn(1.f, dv) : 0.f, c);
        store_codes(t.v, base, t.n, whole, lane, c);
      } else {
        store8(t.m, MHC_F32, base, t.n, whole, lane, m);
        store8(t.v, MHC_F32, base, t.n, whole, lane, v);
      }
    }
  }
}

// Squared norm of all gradients: one partial a block, summed in a fixed order by
// whoever reads them.  fp32 within a lane's few values, fp64 from there on.
template <int N>
__global__ void __launch_bounds__(THREADS) grad_norm_kernel(const __grid_constant__ Table<N> tab, double *partials,
                                                            int accumulate) {
  __shared__ double sh[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double total = 0.0;
  for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    const int ei = entry_of(tab, chunk);
    const Entry &t = tab.t[ei];
    const int64_t first = (int64_t)(chunk - t.first_chunk) * CHUNK;
    float a = 0.f;
#pragma unroll
    for (int it = 0; it < CHUNK / (QB * WARPS); ++it) {
      const int64_t base = first + (int64_t)(it * WARPS + warp) * QB;
      if (base >= t.n) break;
      float g[8];
      if (t.vec && base + QB <= t.n)
        convert8(load_raw<true>(t.g, t.gdt, base, lane), t.gdt, g);
      else
        load_each(t.g, t.gdt, base, t.n, lane, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) a = fmaf(g[e], g[e], a);
    }
    total += (double)a;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) sh[warp] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    double r = accumulate ? partials[blockIdx.x] : 0.0;
    for (int w = 0; w < WARPS; ++w) r += sh[w];
    partials[blockIdx.x] = r;
  }
}

// The values 8-bit moments stand for.
template <bool SIGNED>
__global__ void __launch_bounds__(THREADS) unpack_kernel(const uint8_t *codes, const float *scales, float *out,
                                                         int64_t n, int vec) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t blocks = (n + QB - 1) / QB;
  for (int64_t b = (int64_t)blockIdx.x * WARPS + warp; b < blocks; b += (int64_t)gridDim.x * WARPS) {
    const int64_t base = b * QB;
    const bool whole = vec && base + QB <= n;
    const float s = scales[b];
    const uint2 w = load_codes(codes, base, n, whole, lane);
    float c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = SIGNED ? unpack_m(code_value<true>(w, e), s) : unpack_v(code_value<false>(w, e), s);
    store8(out, MHC_F32, base, n, whole, lane, c);
  }
}

// Blocks of the norm for an SM: each leaves a partial that every block of the step reads.  58 M fp32 values, norm and
// step, over the step alone: 2: 75 us, 4: 40, 8: 41.
constexpr int NORM_BLOCKS_PER_SM = 4;

// Fills tables of up to N tensors and launches each of them: launch(table, first).
template <int N, typename F>
static cudaError_t for_tables(const mhc_adamw_tensor *ts, int count, int state_bits, double lr, double beta1,
                              double beta2, F &&launch) {
  bool first = true;
  int64_t step = 0;
  float rbc2 = 0.f, step_size = 0.f;
  for (int at = 0; at < count;) {
    Table<N> tab;
    tab.count = 0;
    int64_t chunks = 0;
    while (at < count && tab.count < N) {
      const mhc_adamw_tensor &t = ts[at];
      const int64_t c = (t.n + CHUNK - 1) / CHUNK;
      if (chunks + c > (int64_t)1 << 30) break;  // never the table's first: n is at most 2^40
      ++at;
      if (t.n == 0) continue;
      if (t.step != step) {
        step = t.step;
        rbc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
        step_size = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
      }
      Entry &e = tab.t[tab.count++];
      e.p = t.param;
      e.g = t.grad;
      e.m = t.exp_avg;
      e.v = t.exp_avg_sq;
      e.ms = t.exp_avg_scale;
      e.vs = t.exp_avg_sq_scale;
      e.n = t.n;
      e.first_chunk = (int)chunks;
      e.pdt = (uint8_t)t.param_dtype;
      e.gdt = (uint8_t)t.grad_dtype;
      // whether blocks of 4 values may be read and written at once
      const uintptr_t pa = t.param_dtype == MHC_F32 ? 15 : 7, ga = t.grad_dtype == MHC_F32 ? 15 : 7;
      const uintptr_t sa = state_bits == 8 ? 3 : 15;
      e.vec = !((uintptr_t)t.param & pa) && !((uintptr_t)t.grad & ga) && !((uintptr_t)t.exp_avg & sa) &&
              !((uintptr_t)t.exp_avg_sq & sa);
      e.pad = 0;
      e.rbc2 = rbc2;
      e.step_size = step_size;
      chunks += c;
    }
    if (tab.count == 0) continue;
    tab.chunks = (int)chunks;
    launch(tab, first);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    first = false;
  }
  return cudaSuccess;
}

template <int N>
static cudaError_t run_norm(const mhc_adamw_tensor *ts, int count, int accumulate, double *partials, int grid,
                            cudaStream_t stream) {
  return for_tables<N>(ts, count, 32, 0.0, 0.0, 0.0, [&](const Table<N> &tab, bool first) {
    // every block writes its partial, so the grid does not shrink with the work
    grad_norm_kernel<N><<<grid, THREADS, 0, stream>>>(tab, partials, first ? accumulate : 1);
  });
}

template <int N, bool Q8>
static cudaError_t run_step(const mhc_adamw_tensor *ts, int count, double lr, double beta1, double beta2, const Scalars &s,
                            int sms, cudaStream_t stream) {
  return for_tables<N>(ts, count, Q8 ? 8 : 32, lr, beta1, beta2, [&](const Table<N> &tab, bool) {
    // twice what is resident: 282 us at 58 M fp32 values, 921 at 236 M with 8-bit moments, 4 for an SM: 284, 969
    const int cap = sms * 8;
    adamw_kernel<N, Q8><<<tab.chunks < cap ? tab.chunks : cap, THREADS, 0, stream>>>(tab, s);
  });
}

static int sm_count_or_default() {
  const int v = device_sm_count();
  return v > 0 ? v : 148;
}

}  // namespace adamw
}  // namespace mhc

using namespace mhc;

// tensors with values; < 0: a status code
static int64_t check_tensors(const char *who, const mhc_adamw_tensor *ts, int count, int state_bits, bool grads_only) {
  if (count < 0) return fail(MHC_ERR_SHAPE, "%s: count %d", who, count);
  if (count > 0 && !ts) return fail(MHC_ERR_NULL, "%s: tensors is NULL", who);
  const bool q8 = state_bits == 8;
  int64_t live = 0;
  for (int i = 0; i < count; ++i) {
    const mhc_adamw_tensor &t = ts[i];
    if (t.n < 0 || t.n > (int64_t)1 << 40) return fail(MHC_ERR_SHAPE, "%s: tensor %d has %lld values", who, i, (long long)t.n);
    if (t.n == 0) continue;
    ++live;
    const bool types = (grads_only || t.param_dtype == MHC_F32 || t.param_dtype == MHC_BF16 || t.param_dtype == MHC_F16) &&
                       (t.grad_dtype == MHC_F32 || t.grad_dtype == MHC_BF16 || t.grad_dtype == MHC_F16);
    if (!types) return fail(MHC_ERR_DTYPE, "%s: tensor %d: bad dtype code", who, i);
    const uintptr_t ga = t.grad_dtype == MHC_F32 ? 3 : 1;
    if (!t.grad) return fail(MHC_ERR_NULL, "%s: tensor %d: grad is NULL", who, i);
    if ((uintptr_t)t.grad & ga) return fail(MHC_ERR_ALIGN, "%s: tensor %d is not aligned to its elements", who, i);
    if (grads_only) continue;
    if (t.step < 1) return fail(MHC_ERR_SHAPE, "%s: tensor %d: steps count from 1 (got %lld)", who, i, (long long)t.step);
    if (!t.param || !t.exp_avg || !t.exp_avg_sq || (q8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return fail(MHC_ERR_NULL, "%s: tensor %d: required pointer is NULL", who, i);
    const uintptr_t pa = t.param_dtype == MHC_F32 ? 3 : 1, sa = q8 ? 0 : 3;
    if (((uintptr_t)t.param & pa) || (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & sa) ||
        (q8 && (((uintptr_t)t.exp_avg_scale | (uintptr_t)t.exp_avg_sq_scale) & 3)))
      return fail(MHC_ERR_ALIGN, "%s: tensor %d is not aligned to its elements", who, i);
  }
  return live;
}

// mhc_adamw_step's arguments: tensors with values, or a status code < 0
static int64_t check_step(const char *who, const mhc_adamw_tensor *ts, int count, int state_bits, double lr, double beta1,
                          double beta2, double eps, double weight_decay) {
  if (state_bits != 8 && state_bits != 32)
    return fail(MHC_ERR_UNSUPPORTED, "%s: state_bits must be 8 or 32 (got %d)", who, state_bits);
  if (!(lr >= 0.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) ||
      !(beta2 >= 0.0 && beta2 < 1.0))
    return fail(MHC_ERR_SHAPE, "%s: lr, eps, weight_decay >= 0 and betas in [0, 1) are wanted", who);
  return check_tensors(who, ts, count, state_bits, false);
}

extern "C" {

size_t mhc_grad_norm_workspace(void) {
  return (size_t)adamw::sm_count_or_default() * adamw::NORM_BLOCKS_PER_SM * sizeof(double);
}

int mhc_grad_norm(const mhc_adamw_tensor *tensors, int count, int accumulate, void *workspace, size_t workspace_bytes,
                  void *stream) {
  clear_error();
  const int64_t live = check_tensors("mhc_grad_norm", tensors, count, 32, true);
  if (live < 0) return (int)live;
  const size_t need = mhc_grad_norm_workspace();
  if (!workspace || workspace_bytes < need)
    return fail(MHC_ERR_WORKSPACE, "mhc_grad_norm: workspace %zu < %zu bytes", workspace_bytes, need);
  if ((uintptr_t)workspace & 7) return fail(MHC_ERR_ALIGN, "mhc_grad_norm: workspace is not 8-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (live == 0)
    return accumulate ? MHC_OK : cuda_status(cudaMemsetAsync(workspace, 0, need, st), "mhc_grad_norm");
  const int grid = adamw::sm_count_or_default() * adamw::NORM_BLOCKS_PER_SM;
  double *pw = static_cast<double *>(workspace);
  return cuda_status(live <= adamw::FEW_TENSORS
                         ? adamw::run_norm<adamw::FEW_TENSORS>(tensors, count, accumulate, pw, grid, st)
                         : adamw::run_norm<adamw::MAX_TENSORS>(tensors, count, accumulate, pw, grid, st),
                     "mhc_grad_norm");
}

int mhc_adamw_check(const mhc_adamw_tensor *tensors, int count, int state_bits, double lr, double beta1, double beta2,
                    double eps, double weight_decay) {
  clear_error();
  const int64_t live = check_step("mhc_adamw_check", tensors, count, state_bits, lr, beta1, beta2, eps, weight_decay);
  return live < 0 ? (int)live : MHC_OK;
}

int mhc_adamw_step(const mhc_adamw_tensor *tensors, int count, int state_bits, double lr, double beta1, double beta2,
                   double eps, double weight_decay, double max_norm, const void *norm_workspace, float *norm_out,
                   void *stream) {
  clear_error();
  const int64_t live = check_step("mhc_adamw_step", tensors, count, state_bits, lr, beta1, beta2, eps, weight_decay);
  if (live < 0) return (int)live;
  if (max_norm > 0.0 && (!norm_workspace || ((uintptr_t)norm_workspace & 7)))
    return fail(MHC_ERR_WORKSPACE, "mhc_adamw_step: clipping needs the workspace that mhc_grad_norm filled");
  if (live == 0) return MHC_OK;
  const int sms = adamw::sm_count_or_default();
  adamw::Scalars s;
  s.b1 = (float)beta1;
  s.c1 = (float)(1.0 - beta1);
  s.b2 = (float)beta2;
  s.c2 = (float)(1.0 - beta2);
  s.eps = (float)eps;
  s.keep = (float)(1.0 - lr * weight_decay);
  s.max_norm = (float)max_norm;
  s.partials = max_norm > 0.0 ? static_cast<const double *>(norm_workspace) : nullptr;
  s.npartials = sms * adamw::NORM_BLOCKS_PER_SM;
  s.norm_out = s.partials ? norm_out : nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  constexpr int F = adamw::FEW_TENSORS, M = adamw::MAX_TENSORS;
  cudaError_t e;
  if (live <= F)
    e = state_bits == 8 ? adamw::run_step<F, true>(tensors, count, lr, beta1, beta2, s, sms, st)
                        : adamw::run_step<F, false>(tensors, count, lr, beta1, beta2, s, sms, st);
  else
    e = state_bits == 8 ? adamw::run_step<M, true>(tensors, count, lr, beta1, beta2, s, sms, st)
                        : adamw::run_step<M, false>(tensors, count, lr, beta1, beta2, s, sms, st);
  return cuda_status(e, "mhc_adamw_step");
}

int mhc_adamw_unpack(const void *codes, int is_signed, const float *scales, float *out, int64_t n, void *stream) {
  clear_error();
  if (n < 0 || n > (int64_t)1 << 40) return fail(MHC_ERR_SHAPE, "mhc_adamw_unpack: %lld values", (long long)n);
  if (n == 0) return MHC_OK;
  if (!codes || !scales || !out) return fail(MHC_ERR_NULL, "mhc_adamw_unpack: required pointer is NULL");
  if (((uintptr_t)scales & 3) || ((uintptr_t)out & 3)) return fail(MHC_ERR_ALIGN, "mhc_adamw_unpack: scales / out misaligned");
  const int vec = !((uintptr_t)codes & 3) && !((uintptr_t)out & 15);
  const int64_t blocks = (n + adamw::QB - 1) / adamw::QB;
  const unsigned grid = grid_for(blocks, adamw::WARPS, device_sm_count(), 8);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t *c = static_cast<const uint8_t *>(codes);
  if (is_signed)
    adamw::unpack_kernel<true><<<grid, adamw::THREADS, 0, st>>>(c, scales, out, n, vec);
  else
    adamw::unpack_kernel<false><<<grid, adamw::THREADS, 0, st>>>(c, scales, out, n, vec);
  return cuda_status(cudaGetLastError(), "mhc_adamw_unpack");
}

}  // extern "C"
