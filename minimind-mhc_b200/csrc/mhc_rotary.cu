// Rotary positions, alone and on the way into a paged cache.
//
//   angle = position * w_i                    pair i of a head's first `part` elements
//   (a, b) -> gain (a cos - b sin, b cos + a sin)
//
// The gradient is the same rotation by the negative angle.
//
// The angle of a far position needs more bits than an fp32 product has (position 10^6
// leaves 2^-4 of a radian).  Here w_i is a fraction of a turn in 64 bits of fixed point
// and the product is one integer multiplication whose overflow is the whole turns: exact
// modulo a turn to 2^-65 position.  Its top two bits, rounded, are the quarter turn; the
// rest, within an eighth of a turn, becomes a float and goes into two short Taylor series
// (sincospif, which reduces its argument again, took a third of the kernel's instructions).
//
// Every element is read and written once; what bounds it besides is instructions.  A block takes
// a few tokens: the angles of a token are computed once for all its heads and kept in
// shared memory, in the order in which threads read them; then a thread keeps its place
// in a head (two vectors that hold VEC pairs, or one that is only copied) and walks over
// rows, two heads of one token at a time, so that they share the angles' way out of shared
// memory.  v moves into a cache with the others, without a rotation.
//
// Neighbouring threads take neighbouring places and heads: with a token's angles in the
// registers of a thread that walks over its heads the instructions are a third, but a
// warp's accesses lie 1.5 KB apart, and 16384 tokens of 12 heads of 96 took 27 us for 15.
// Measured: those 14.7 us (75 MB, 5.1 TB/s), 8191 tokens of 10 heads of 128 in fp32 14.4 us
// (84 MB, 5.8 TB/s); into a cache 24 prompts, 17,900 tokens, 24 us (110 MB, 4.5 TB/s; fp32 40 us, 5.4), one token of
// each of 16 sequences 3.3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_cache.cuh"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace rotary {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 16;  // of a block
constexpr int MAX_D = 256;  // a head's items fit a block even as scalars

struct Args {
  const void *q, *k, *v;
  void *qo, *ko;  // contiguous; ko unused with a cache
  int64_t qt, qh, kt, kh, vt, vh;
  int64_t T, period;
  int H, Hk, Hv, D, part, half, tokens;  // Hv: 0, or Hk with a cache; tokens of a block
  int pair_items, items, rows_at_once;   // of a head: vectors of pairs, and all; rows that a block takes at a time
  int twos;                              // rows of a token: head h < twos together with head h + twos
  uint64_t by_twos;                      // 2^32 over it, rounded up: divides the rows of a block
  const uint64_t *turns;
  const void *pos;
  int pos_bytes;
  float gain, sign;
  cache::View c;
};

struct Cs {
  float c, s;
};
// sin and cos of y, |y| <= pi / 4 (and a little): their Taylor series up to y^9 and y^10, whose next terms are 2e-9 and
// 2e-10 there
__device__ __forceinline__ Cs near_zero(float y) {
  const float z = y * y;
  const float s = fmaf(y * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), y);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  return {c, s};
}
__device__ __forceinline__ Cs angle(uint64_t turn, int64_t pos, float gain, float sign) {
  const uint64_t f = turn * (uint64_t)pos;
  // the upper half will do from here on: 2^-32 of a turn
  const uint32_t top = (uint32_t)(f >> 32), quarter = (top + (1u << 29)) >> 30;
  const int32_t rest = (int32_t)(top - (quarter << 30));  // in [-2^29, 2^29): within an eighth of a turn
  const Cs w = near_zero((float)rest * (6.283185307179586f * 0x1p-32f));
  float c = (quarter & 1) ? -w.s : w.c, s = (quarter & 1) ? w.c : w.s;
  if (quarter & 2) {
    c = -c;
    s = -s;
  }
  return {c * gain, s * (gain * sign)};
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T x[VEC];
};

// A word of two 16-bit values and back.
template <typename T>
__device__ __forceinline__ float2 two(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t word(float x, float y) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}

// The pairs of two vectors turned; pair i's cos and sin at cs[i * apart].
template <typename T, int VEC, bool ILV>
__device__ __forceinline__ void turn(Pack<T, VEC> &x, Pack<T, VEC> &y, const Cs *cs, int apart) {
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    uint32_t *a = reinterpret_cast<uint32_t *>(&x), *b = reinterpret_cast<uint32_t *>(&y);
    if constexpr (ILV) {  // a word is a pair
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        uint32_t &w = i < VEC / 2 ? a[i % (VEC / 2)] : b[i % (VEC / 2)];
        const Cs k = cs[i * apart];
        const float2 p = two<T>(w);
        w = word<T>(p.x * k.c - p.y * k.s, p.y * k.c + p.x * k.s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const Cs k = cs[2 * i * apart], l = cs[(2 * i + 1) * apart];
        const float2 p = two<T>(a[i]), q = two<T>(b[i]);
        a[i] = word<T>(p.x * k.c - q.x * k.s, p.y * l.c - q.y * l.s);
        b[i] = word<T>(q.x * k.c + p.x * k.s, q.y * l.c + p.y * l.s);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      T &first = !ILV ? x.x[i] : 2 * i < VEC ? x.x[(2 * i) % VEC] : y.x[(2 * i) % VEC];
      T &second = !ILV ? y.x[i] : 2 * i + 1 < VEC ? x.x[(2 * i + 1) % VEC] : y.x[(2 * i + 1) % VEC];
      const float p = to_f(first), q = to_f(second);
      const Cs k = cs[i * apart];
      first = from_f<T>(p * k.c - q * k.s);
      second = from_f<T>(q * k.c + p * k.s);
    }
  }
}

template <typename T, int VEC, bool ILV, bool CACHE>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const Args a) {
  extern __shared__ Cs table[];  // of token t: pair i of place p at t half + i (half / VEC) + p
  __shared__ int64_t at_k[MAX_TOKENS], at_v[MAX_TOKENS], at_pos[MAX_TOKENS];
  grid_dep_launch();  // the attention behind an append sets itself up meanwhile
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.T - t0);
  if (tid < 32) {  // at most as many tokens
    const int64_t t = t0 + tid;
    int b = CACHE ? cache::seq_from(a.c, (int)t0) : 0;
    if (tid < tokens) {
      int64_t pos = a.period > 0 ? (int64_t)((uint32_t)t % (uint32_t)a.period) : t;
      if (a.pos) pos = a.pos_bytes == 8 ? static_cast<const int64_t *>(a.pos)[pos] : static_cast<const int32_t *>(a.pos)[pos];
      if (CACHE) {
        while (b < a.c.batch && a.c.cu[b + 1] <= t) ++b;
        int page = 0, slot = 0;
        const bool known = b < a.c.batch && a.c.cu[b] <= t;
        bool there = false;
        if (known) {
          const int64_t place = (int64_t)a.c.lengths[b] + (t - a.c.cu[b]);
          there = cache::locate(a.c, b, place, page, slot);
          if (!a.pos) pos = place;
        }
        at_k[tid] = there ? page * a.c.kp + slot * a.c.ks : -1;
        // -2: of no sequence, its rotated query is 0
        at_v[tid] = there ? page * a.c.vp + slot * a.c.vs : (known ? -1 : -2);
      }
      at_pos[tid] = pos;
    }
  }
  __syncthreads();
  for (int i = tid; i < tokens * a.half; i += blockDim.x) {
    const int t = i / a.half, p = i - t * a.half, place = p / VEC;
    table[t * a.half + (p - place * VEC) * a.pair_items + place] = angle(a.turns[p], at_pos[t], a.gain, a.sign);
  }
  __syncthreads();
  const int item = tid % a.items, lane_row = tid / a.items;
  if (lane_row >= a.rows_at_once) return;
  const bool pair = item < a.pair_items;
  // first element of the item's vector (the second vector of a pair item lies at `hop` behind it)
  const int col = pair ? item * VEC * (ILV ? 2 : 1) : a.part + (item - a.pair_items) * VEC;
  const int hop = ILV ? VEC : a.half;
  const int heads = a.H + a.Hk + a.Hv;
  using P = Pack<T, VEC>;
  for (int r = lane_row; r < tokens * a.twos; r += a.rows_at_once) {
    const int tl = (int)(((uint64_t)r * a.by_twos) >> 32), h0 = r - tl * a.twos;
    const int64_t t = t0 + tl;
    P x[2], y[2];
    T *dst[2];
    bool live[2], turns[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      int h = h0 + u * a.twos;
      live[u] = h < heads;
      turns[u] = pair && h < a.H + a.Hk;
      const T *src = nullptr;
      dst[u] = nullptr;
      if (h < a.H) {
        src = static_cast<const T *>(a.q) + t * a.qt + h * a.qh + col;
        dst[u] = static_cast<T *>(a.qo) + (t * a.H + h) * (int64_t)a.D + col;
      } else if ((h -= a.H) < a.Hk) {
        src = static_cast<const T *>(a.k) + t * a.kt + h * a.kh + col;
        if (CACHE) {
          live[u] = live[u] && at_k[tl] >= 0;
          dst[u] = static_cast<T *>(a.c.keys) + at_k[tl] + h * a.c.kh + col;
        } else {
          dst[u] = static_cast<T *>(a.ko) + (t * a.Hk + h) * (int64_t)a.D + col;
        }
      } else if (CACHE) {
        h -= a.Hk;
        live[u] = live[u] && at_k[tl] >= 0;
        src = static_cast<const T *>(a.v) + t * a.vt + h * a.vh + col;
        dst[u] = static_cast<T *>(a.c.values) + at_v[tl] + h * a.c.vh + col;
      }
      if (live[u]) {
        x[u] = *reinterpret_cast<const P *>(src);
        if (pair) y[u] = *reinterpret_cast<const P *>(src + hop);
      }
    }
    const Cs *cs = table + tl * a.half + item;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!live[u]) continue;
      if (turns[u]) turn<T, VEC, ILV>(x[u], y[u], cs, a.pair_items);
      if (CACHE && h0 + u * a.twos < a.H && at_v[tl] == -2) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u].x[i] = y[u].x[i] = from_f<T>(0.f);
      }
      *reinterpret_cast<P *>(dst[u]) = x[u];
      if (pair) *reinterpret_cast<P *>(dst[u] + hop) = y[u];
    }
  }
}

// whether every row of a tensor begins at a multiple of `bytes`
static bool fits(const void *p, int64_t st, int64_t sh, size_t es, size_t bytes) {
  return (uintptr_t)p % bytes == 0 && (st * (int64_t)es) % (int64_t)bytes == 0 && (sh * (int64_t)es) % (int64_t)bytes == 0;
}

static cudaError_t launch(Args a, int dtype, bool ilv, bool with_cache, cudaStream_t st) {
  const size_t es = dtype == MHC_F32 ? 4 : 2;
  // the widest vectors that every row and both parts of a head allow
  auto usable = [&](int vec) {
    const size_t bytes = vec * es;
    bool ok = a.half % vec == 0 && (a.D - a.part) % vec == 0 && a.D % vec == 0;
    if (a.H) ok = ok && fits(a.q, a.qt, a.qh, es, bytes) && fits(a.qo, 0, 0, es, bytes);
    if (a.Hk) ok = ok && fits(a.k, a.kt, a.kh, es, bytes);
    if (!with_cache) return ok && (!a.Hk || fits(a.ko, 0, 0, es, bytes));
    return ok && fits(a.v, a.vt, a.vh, es, bytes) && fits(a.c.keys, a.c.ks, a.c.kh, es, bytes) && fits(a.c.keys, a.c.kp, 0, es, bytes) &&
           fits(a.c.values, a.c.vs, a.c.vh, es, bytes) && fits(a.c.values, a.c.vp, 0, es, bytes);
  };
  const int wide = (int)(16 / es);
  const int vec = usable(wide) ? wide : usable(wide / 2) ? wide / 2 : 1;
  a.pair_items = a.half / vec;
  a.items = a.pair_items + (a.D - a.part) / vec;
  // half blocks where a few tokens fit them: the last ones end nearer together (16384 tokens of 12 heads of 96, both
  // directions: 30.5 us with whole ones, 29.4 with half; 8191 of 10 heads of 128, fp32: 15.2, 14.4)
  const int threads = a.items <= THREADS / 4 ? THREADS / 2 : THREADS;
  a.rows_at_once = threads / a.items;
  if (a.rows_at_once < 1) return cudaErrorInvalidValue;
  const int heads = a.H + a.Hk + a.Hv;
  a.twos = (heads + 1) / 2;
  a.by_twos = (((uint64_t)1 << 32) + a.twos - 1) / a.twos;
  // a thread takes about two pairs of heads, fewer where that would leave SMs without a block
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  int64_t tokens = (2 * a.rows_at_once) / a.twos;
  tokens = tokens > MAX_TOKENS ? MAX_TOKENS : tokens;
  const int64_t spread = (a.T + sms - 1) / sms;
  tokens = tokens > spread ? spread : tokens;
  a.tokens = tokens < 1 ? 1 : (int)tokens;
  const int64_t blocks = (a.T + a.tokens - 1) / a.tokens;
  const size_t smem = sizeof(Cs) * a.tokens * a.half;
  return with_dtype(dtype, [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    constexpr int W = 16 / (int)sizeof(T);
    auto go = [&](auto v, auto i, auto c) -> cudaError_t {
      rotary_kernel<T, decltype(v)::value, decltype(i)::value != 0, decltype(c)::value != 0><<<(unsigned)blocks, threads, smem, st>>>(a);
      return cudaGetLastError();
    };
    auto by_vec = [&](auto i, auto c) -> cudaError_t {
      if (vec == W) return go(IC<W>{}, i, c);
      if (vec == W / 2) return go(IC<W / 2>{}, i, c);
      return go(IC<1>{}, i, c);
    };
    if (ilv) return with_cache ? by_vec(IC<1>{}, IC<1>{}) : by_vec(IC<1>{}, IC<0>{});
    return with_cache ? by_vec(IC<0>{}, IC<1>{}) : by_vec(IC<0>{}, IC<0>{});
  });
}

static int check_rotary(const char *who, const mhc_rotary *r, int D) {
  if (r->part < 2 || r->part % 2 || r->part > D)
    return fail(MHC_ERR_SHAPE, "%s: an even part of 2 to %d elements is wanted (got %d)", who, D, r->part);
  if (!r->turns) return fail(MHC_ERR_NULL, "%s: turns is NULL", who);
  if ((uintptr_t)r->turns % 8) return fail(MHC_ERR_ALIGN, "%s: turns is not 8-byte aligned", who);
  return MHC_OK;
}
static int check_positions(const char *who, const void *p, int bytes) {
  if (!p) return MHC_OK;
  if (bytes != 4 && bytes != 8) return fail(MHC_ERR_DTYPE, "%s: positions of 4 or 8 bytes are wanted (got %d)", who, bytes);
  if ((uintptr_t)p % bytes) return fail(MHC_ERR_ALIGN, "%s: positions are not aligned to their elements", who);
  return MHC_OK;
}

}  // namespace rotary

int cache_view(const char *who, const mhc_kv_cache *c, const mhc_cache_step *s, cache::View &v) {
  if (!c || !s) return fail(MHC_ERR_NULL, "%s: cache or step is NULL", who);
  if (c->dtype != MHC_F32 && c->dtype != MHC_BF16 && c->dtype != MHC_F16) return fail(MHC_ERR_DTYPE, "%s: bad dtype code %d", who, c->dtype);
  if (c->pages < 0 || c->pages > 0x7fffffff || c->page_size < 1 || c->kv_heads < 1 || c->kv_heads > 16384 || c->dim < 1 ||
      c->dim > rotary::MAX_D || c->layers < 0)
    return fail(MHC_ERR_SHAPE, "%s: bad cache: %lld pages of %d, %d heads of %d, %d layers", who, (long long)c->pages, c->page_size,
                c->kv_heads, c->dim, c->layers);
  if (s->T < 0 || s->T > 0x7fffffff - 4096 || s->batch < 0 || s->batch > 1 << 30 || s->table_width < 0 || (int64_t)s->table_width * c->page_size > 0x7fffffff - 4096)
    return fail(MHC_ERR_SHAPE, "%s: bad step: %lld rows, %d sequences, a table of %d pages of %d", who, (long long)s->T, s->batch,
                s->table_width, c->page_size);
  if (s->batch > 0 && (!s->lengths || !s->cu_tokens || (s->table_width > 0 && !s->page_table)))
    return fail(MHC_ERR_NULL, "%s: a pointer of the step is NULL", who);
  if (c->pages > 0 && (!c->keys || !c->values)) return fail(MHC_ERR_NULL, "%s: keys or values is NULL", who);
  if ((uintptr_t)s->page_table % 4 || (uintptr_t)s->lengths % 4 || (uintptr_t)s->cu_tokens % 4)
    return fail(MHC_ERR_ALIGN, "%s: a pointer of the step is not aligned to its elements", who);
  const size_t es = c->dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)c->keys % es || (uintptr_t)c->values % es) return fail(MHC_ERR_ALIGN, "%s: keys or values is not aligned to its elements", who);
  v.keys = c->keys;
  v.values = c->values;
  v.kp = c->strides[1], v.ks = c->strides[2], v.kh = c->strides[3];
  v.vp = c->strides[5], v.vs = c->strides[6], v.vh = c->strides[7];
  v.table = s->page_table;
  v.lengths = s->lengths;
  v.cu = s->cu_tokens;
  v.pitch = s->table_pitch;
  v.pages = (int)c->pages;
  v.size = c->page_size;
  v.shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c->page_size == 1 << i) v.shift = i;
  v.capacity = s->table_width * c->page_size;
  v.batch = s->batch;
  v.T = (int)s->T;
  v.Hk = c->kv_heads;
  v.D = c->dim;
  return MHC_OK;
}

}  // namespace mhc

using namespace mhc;

extern "C" {

int mhc_rotate(const mhc_rotary *r, const void *q, void *q_out, int H, const void *k, void *k_out, int Hk, int dtype, int64_t T,
               int D, const int64_t *strides, const void *positions, int position_bytes, int64_t period, int inverse, void *stream) {
  const char *who = "mhc_rotate";
  clear_error();
  if (!r || !strides) return fail(MHC_ERR_NULL, "%s: rotary or strides is NULL", who);
  if (dtype != MHC_F32 && dtype != MHC_BF16 && dtype != MHC_F16) return fail(MHC_ERR_DTYPE, "%s: bad dtype code %d", who, dtype);
  if (T < 0 || T > 0x7fffffff || H < 0 || Hk < 0 || H + Hk < 1 || H > 16384 || Hk > 16384 || D < 2 || D > rotary::MAX_D || period < 0 || period > 0x7fffffff)
    return fail(MHC_ERR_SHAPE, "%s: T = %lld, %d and %d heads of %d (up to %d), period %lld", who, (long long)T, H, Hk, D, rotary::MAX_D,
                (long long)period);
  if (int st = rotary::check_rotary(who, r, D)) return st;
  if (int st = rotary::check_positions(who, positions, position_bytes)) return st;
  if (T == 0) return MHC_OK;
  if ((H && (!q || !q_out)) || (Hk && (!k || !k_out))) return fail(MHC_ERR_NULL, "%s: required pointer is NULL", who);
  const size_t es = dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)q % es || (uintptr_t)q_out % es || (uintptr_t)k % es || (uintptr_t)k_out % es)
    return fail(MHC_ERR_ALIGN, "%s: a pointer is not aligned to its elements", who);
  rotary::Args a{};
  a.q = q, a.qo = q_out, a.H = H;
  a.k = k, a.ko = k_out, a.Hk = Hk;
  a.qt = strides[0], a.qh = strides[1], a.kt = strides[2], a.kh = strides[3];
  a.T = T, a.period = period, a.D = D, a.part = r->part, a.half = r->part / 2;
  a.turns = r->turns, a.pos = positions, a.pos_bytes = position_bytes;
  a.gain = r->gain, a.sign = inverse ? -1.f : 1.f;
  return cuda_status(rotary::launch(a, dtype, r->interleaved != 0, false, reinterpret_cast<cudaStream_t>(stream)), who);
}

int mhc_append_kv(const mhc_kv_cache *cache, const mhc_cache_step *step, const void *k, const void *v, const void *q, void *q_out,
                  int H, const int64_t *strides, const mhc_rotary *r, const void *positions, int position_bytes, void *stream) {
  const char *who = "mhc_append_kv";
  clear_error();
  rotary::Args a{};
  if (int st = cache_view(who, cache, step, a.c)) return st;
  if (!strides) return fail(MHC_ERR_NULL, "%s: strides is NULL", who);
  const int D = cache->dim;
  if (H < 0 || H > 16384) return fail(MHC_ERR_SHAPE, "%s: %d query heads", who, H);
  if (r) {
    if (int st = rotary::check_rotary(who, r, D)) return st;
  } else {
    H = 0;
  }
  if (int st = rotary::check_positions(who, positions, position_bytes)) return st;
  if (step->T == 0) return MHC_OK;
  if (!k || !v || (H && (!q || !q_out))) return fail(MHC_ERR_NULL, "%s: required pointer is NULL", who);
  const size_t es = cache->dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)q % es || (uintptr_t)q_out % es || (uintptr_t)k % es || (uintptr_t)v % es)
    return fail(MHC_ERR_ALIGN, "%s: a pointer is not aligned to its elements", who);
  if (step->batch == 0 && H == 0) return MHC_OK;
  if (step->batch == 0)  // rows of no sequence
    return cuda_status(cudaMemsetAsync(q_out, 0, (size_t)step->T * H * D * es, reinterpret_cast<cudaStream_t>(stream)), who);
  a.q = q, a.qo = q_out, a.H = H;
  a.k = k, a.v = v, a.Hk = a.Hv = cache->kv_heads;
  a.qt = strides[0], a.qh = strides[1], a.kt = strides[2], a.kh = strides[3], a.vt = strides[4], a.vh = strides[5];
  a.T = step->T, a.period = 0, a.D = D;
  a.pos = positions, a.pos_bytes = position_bytes;
  a.sign = 1.f;
  if (r) {
    a.part = r->part, a.half = r->part / 2, a.turns = r->turns, a.gain = r->gain;
  }
  return cuda_status(rotary::launch(a, cache->dtype, r && r->interleaved, true, reinterpret_cast<cudaStream_t>(stream)), who);
}

}  // extern "C"
