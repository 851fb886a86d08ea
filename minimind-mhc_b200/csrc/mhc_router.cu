// Top-k router with its balance loss.
//
//   p[t,:]    = softmax(z[t,:])                       over E experts
//   idx[t,:]  = the k largest z[t,:], the lower index first among equals
//   w[t,j]    = p[t,idx_j] / S,  S = sum_j p[t,idx_j] + 1e-20
//   counts[e] = how often e was chosen
//   loss      = coef * E * sum_e (counts[e] / T) * (1/T) sum_t p[t,e]
//
// and for upstream gradients dw (T, k) and dloss (the counts are constants):
//
//   dp[t,e] = dloss coef E / T * counts[e] / T + [e = idx_j] (dw_j - <dw, w>) / S
//   dz[t,e] = p[t,e] (dp[t,e] - <p, dp>)
//
// One pass over the logits in each direction: a group of G lanes owns a token, a
// lane V neighbouring experts of it (G V >= E; 16 bytes of 16-bit logits), so the
// softmax, the choice and the products stay in registers.  A choice is the
// maximum of keys that hold the value's order and, below it, the index reversed:
// one comparison settles both.  16-bit logits and an index fit one 32-bit key,
// fp32 logits take 64 bits.  A lane's experts stay the same for all its tokens,
// so the column sums of p and the counts are registers too, joined per block and
// then over the blocks in a fixed order: no atomics, the same bits every time.
//
// A row of -inf only has p = 0 and w = 0 (and the experts of lowest index);
// a NaN counts as the largest logit and makes the row's weights and the loss NaN.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_b200.h"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"

namespace mhc {
namespace router {

constexpr int THREADS = 256;
constexpr int MAX_E = 512;

// Order-preserving keys: larger value, then lower expert index, is the larger key; 0
// is below every key of a real logit.  The logit can be read back from its key.
template <typename T>
struct KeyOf {  // 16-bit logits: the order of their own bits above the reversed index
  using type = uint32_t;
  static __device__ __forceinline__ uint32_t make(T x, int e) {
    const uint32_t low = 0xffffu - (uint32_t)e;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // bf16 is the upper half of an fp32
      const float v = to_f(x) + 0.f;                        // -0 and 0 are equal
      const uint32_t b = __float_as_uint(v);
      const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
      return ((v == v ? o : 0xffffffffu) & 0xffff0000u) | low;
    } else {
      uint32_t b = (uint32_t)*reinterpret_cast<const uint16_t *>(&x);
      if (b == 0x8000u) b = 0;
      uint32_t o = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
      if (to_f(x) != to_f(x)) o = 0xffffu;
      return (o << 16) | low;
    }
  }
  static __device__ __forceinline__ int expert(uint32_t k) { return (int)(0xffffu - (k & 0xffffu)); }
  static __device__ __forceinline__ float value(uint32_t k) {
    const uint32_t o = k >> 16;
    const uint16_t b = (uint16_t)((o & 0x8000u) ? (o & 0x7fffu) : ~o);
    return to_f(*reinterpret_cast<const T *>(&b));
  }
};
template <>
struct KeyOf<float> {
  using type = unsigned long long;
  static __device__ __forceinline__ unsigned long long make(float x, int e) {
    const uint32_t b = __float_as_uint(x + 0.f);
    const uint32_t o = x != x ? 0xffffffffu : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
    return ((unsigned long long)o << 32) | (0xffffffffu - (uint32_t)e);
  }
  static __device__ __forceinline__ int expert(unsigned long long k) { return (int)(0xffffffffu - (uint32_t)k); }
  static __device__ __forceinline__ float value(unsigned long long k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
  }
};

// largest first: bitonic network
template <int V, typename K>
__device__ __forceinline__ void sort_down(K (&k)[V]) {
#pragma unroll
  for (int size = 2; size <= V; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d; d >>= 1)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = i ^ d;
        if (j > i) {
          const bool down = (i & size) == 0;
          const K hi = max(k[i], k[j]), lo = min(k[i], k[j]);
          k[i] = down ? hi : lo;
          k[j] = down ? lo : hi;
        }
      }
}

// Over the G lanes of a group.  Whole warps run these (a group past the last token
// repeats it): with a mask for each group the groups of a warp would take turns.
template <int G, typename K>
__device__ __forceinline__ K group_max(K v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) {
    const K w = __shfl_xor_sync(0xffffffffu, v, o);
    v = max(v, w);
  }
  return v;
}
template <int G>
__device__ __forceinline__ float group_maxf(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// a lane's V logits of one row
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T *row, int e0, int E, bool vec, T (&x)[V]) {
  constexpr int PER = 16 / (int)sizeof(T);
  if (vec && V % PER == 0 && e0 + V <= E) {
#pragma unroll
    for (int q = 0; q < V / PER; ++q) {
      const uint4 r = *reinterpret_cast<const uint4 *>(row + e0 + q * PER);
      const T *s = reinterpret_cast<const T *>(&r);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[(q * PER + i) % V] = s[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = e0 + i < E ? row[e0 + i] : from_f<T>(0.f);
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float LOG2E = 1.44269504088896340736f;

// exp(z - top) for a logit of a row whose largest is `top`: the special function's
// 2^x (2 ulp) in place of expf's 9 instructions.  The difference is taken before it is
// scaled: it is never above zero, so the largest logit gives exactly 1 and a row's sum
// is at least 1 however large the logits are (scaled first, the rounding of top log2(e)
// would be an exponent of hundreds from 1e10 on).  +inf - inf is NaN, as the quotient
// would be.
__device__ __forceinline__ float exp_below(float z, float top) { return exp2_approx((z - top) * LOG2E); }

// softmax of the group's row; lanes past E hold p = 0.  An all -inf row gives 0.
// p = exp_below(z, top) * scale for any logit z of the row.
template <typename T, int G, int V>
__device__ __forceinline__ void softmax_row(const T (&x)[V], int e0, int E, float (&p)[V], float &top, float &scale) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = e0 + i < E ? to_f(x[i]) : -INFINITY;
    mx = fmaxf(mx, p[i]);
  }
  mx = group_maxf<G>(mx);
  top = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = exp_below(p[i], top);
    sum += p[i];
  }
  sum = group_sum<G>(sum);
  scale = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] *= scale;
}

struct Args {
  const void *z;
  int64_t T, row_stride;
  int E, k, vec;
  float scale;  // coef * E
};

// the block's (or, with one block, everybody's) loss from column sums and counts
__device__ __forceinline__ void write_loss(const float *sums, const int64_t *cnt, const Args &a, int64_t *counts,
                                           float *loss) {
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) counts[e] = cnt[e];
  if (threadIdx.x < 32) {
    double s = 0.0;
    const double it = 1.0 / (double)a.T;
    for (int e = threadIdx.x; e < a.E; e += 32) s += (double)cnt[e] * it * ((double)sums[e] * it);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *loss = (float)(s * (double)a.scale);
  }
}

template <typename T, int G, int V, int SL>
__global__ void __launch_bounds__(THREADS, 4) route_fwd_kernel(Args a, float *w, int64_t *idx, int64_t *counts, float *loss,
                                                            float *part_sum, int *part_cnt) {
  using Key = KeyOf<T>;
  using K = typename Key::type;
  constexpr int ROWS = THREADS / G;  // tokens a block takes at a time
  __shared__ float sh_sum[G * V];
  __shared__ float stage_sum[THREADS / 32][G * V];
  __shared__ int stage_cnt[THREADS / 32][G * V];
  __shared__ int64_t sh_cnt[G * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G, e0 = gl * V;
  float col[V];
  int cnt[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    col[i] = 0.f;
    cnt[i] = 0;
  }
  const T *z = static_cast<const T *>(a.z);
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  T next[V];
  auto fetch = [&](int64_t t) { load_logits<T, V>(z + (t < a.T ? t : a.T - 1) * a.row_stride, e0, a.E, a.vec, next); };
  fetch((int64_t)blockIdx.x * ROWS + threadIdx.x / G);
  for (int64_t tb = (int64_t)blockIdx.x * ROWS; tb < a.T; tb += stride) {
    const int64_t t = tb + threadIdx.x / G;
    const bool live = t < a.T;
    T x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = next[i];
    if (tb + stride < a.T) fetch(t + stride);
    float p[V], largest, scale;
    softmax_row<T, G, V>(x, e0, a.E, p, largest, scale);
    K key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = e0 + i < a.E ? Key::make(x[i], e0 + i) : (K)0;
    }
    // a lane's keys in order, so that only its first can be the next choice.  The j-th choice is kept by lane j % G of
    // the group, in slot j / G of SL.
    sort_down<V, K>(key);
    K top[SL];
    unsigned chosen = 0;
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      top[s] = 0;
      for (int r = 0; r < G && s * G + r < a.k; ++r) {
        const K best = group_max<G, K>(key[0]);
        if (key[0] == best) {
          chosen |= 1u << (Key::expert(best) - e0);
#pragma unroll
          for (int i = 0; i + 1 < V; ++i) key[i] = key[i + 1];
          key[V - 1] = 0;
        }
        if (gl == r) top[s] = best;
      }
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        col[i] += p[i];
        cnt[i] += (chosen >> i) & 1u;
      }
    }
    float pe[SL], total = 0.f;
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      pe[s] = 0.f;
      if (s * G + gl < a.k) pe[s] = exp_below(Key::value(top[s]), largest) * scale;
      total += pe[s];
    }
    total = group_sum<G>(total) + 1e-20f;
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      const int j = s * G + gl;
      if (live && j < a.k) {
        w[t * a.k + j] = pe[s] / total;  // k = 1: exactly 1
        idx[t * a.k + j] = Key::expert(top[s]);
      }
    }
  }
  // lanes of a warp that own the same experts, then the block's warps
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) {
      col[i] += __shfl_xor_sync(0xffffffffu, col[i], o);
      cnt[i] += __shfl_xor_sync(0xffffffffu, cnt[i], o);
    }
    if (lane < G) {
      stage_sum[warp][e0 + i] = col[i];
      stage_cnt[warp][e0 + i] = cnt[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += THREADS) {
    float s = 0.f;
    int c = 0;
    for (int q = 0; q < THREADS / 32; ++q) {
      s += stage_sum[q][e];
      c += stage_cnt[q][e];
    }
    if (gridDim.x == 1) {
      sh_sum[e] = s;
      sh_cnt[e] = c;
    } else {
      part_sum[(int64_t)blockIdx.x * a.E + e] = s;
      part_cnt[(int64_t)blockIdx.x * a.E + e] = c;
    }
  }
  if (gridDim.x == 1) {
    __syncthreads();
    write_loss(sh_sum, sh_cnt, a, counts, loss);
  }
}

// Joins the blocks' partial sums in a fixed order: `lanes` threads of each block of a
// cluster share an expert, the first block adds the others' sums to its own and forms
// the loss.  It is the reading that counts, one SM has too few loads under way: 592
// blocks, 64 / 512 experts: one block 8.4 / 45 us, a cluster of eight 4.5 / 10.
constexpr int JOIN = 8;
__global__ void __cluster_dims__(JOIN, 1, 1) __launch_bounds__(1024) route_join_kernel(Args a, const float *part_sum, const int *part_cnt, int blocks,
                                                          int64_t *counts, float *loss) {
  __shared__ float sh_sum[MAX_E];
  __shared__ int64_t sh_cnt[MAX_E];
  __shared__ float st_sum[1024];
  __shared__ int64_t st_cnt[1024];
  const int rank = (int)blockIdx.x;  // one cluster
  int pad = 1;
  while (pad < a.E) pad <<= 1;
  const int lanes = 1024 / pad, e = threadIdx.x % pad, l = threadIdx.x / pad;
  float s = 0.f;
  int64_t c = 0;
  if (e < a.E) {
    constexpr int AT_ONCE = 8;  // in flight; summed in order
    for (int b0 = rank + JOIN * l; b0 < blocks; b0 += JOIN * lanes * AT_ONCE) {
      float vs[AT_ONCE];
      int vc[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int b = b0 + u * JOIN * lanes;
        vs[u] = b < blocks ? part_sum[(int64_t)b * a.E + e] : 0.f;
        vc[u] = b < blocks ? part_cnt[(int64_t)b * a.E + e] : 0;
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        s += vs[u];
        c += vc[u];
      }
    }
  }
  st_sum[threadIdx.x] = s;
  st_cnt[threadIdx.x] = c;
  __syncthreads();
  if (threadIdx.x < a.E) {
    float ts = 0.f;
    int64_t tc = 0;
    for (int q = 0; q < lanes; ++q) {
      ts += st_sum[q * pad + threadIdx.x];
      tc += st_cnt[q * pad + threadIdx.x];
    }
    sh_sum[threadIdx.x] = ts;
    sh_cnt[threadIdx.x] = tc;
  }
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  cluster.sync();
  if (rank == 0 && threadIdx.x < a.E) {  // the own thread's values: the others read nothing of this block
    float ts = sh_sum[threadIdx.x];
    int64_t tc = sh_cnt[threadIdx.x];
    for (int r = 1; r < JOIN; ++r) {
      ts += cluster.map_shared_rank(sh_sum, r)[threadIdx.x];
      tc += cluster.map_shared_rank(sh_cnt, r)[threadIdx.x];
    }
    sh_sum[threadIdx.x] = ts;
    sh_cnt[threadIdx.x] = tc;
  }
  cluster.sync();  // the others' memory has been read
  if (rank == 0) write_loss(sh_sum, sh_cnt, a, counts, loss);
}

template <typename T, int G, int V, int SL>
__global__ void __launch_bounds__(THREADS, 4) route_bwd_kernel(Args a, const float *w, const int64_t *idx,
                                                            const int64_t *counts, const float *dw, const float *dloss,
                                                            T *dz) {
  constexpr int ROWS = THREADS / G;
  const int lane = threadIdx.x & 31;
  const int gl = lane % G, e0 = gl * V;
  float load[V];
  const double f = dloss ? (double)*dloss * (double)a.scale / ((double)a.T * (double)a.T) : 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) load[i] = dloss && e0 + i < a.E ? (float)(f * (double)counts[e0 + i]) : 0.f;
  __shared__ __align__(16) float scatter[THREADS * V];
  float *stripe = scatter + threadIdx.x / G * (G * V);
#pragma unroll
  for (int i = 0; i < V; i += 4) *reinterpret_cast<float4 *>(stripe + e0 + i) = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncwarp();
  const T *z = static_cast<const T *>(a.z);
  for (int64_t tb = (int64_t)blockIdx.x * ROWS; tb < a.T; tb += (int64_t)gridDim.x * ROWS) {
    const bool live = tb + threadIdx.x / G < a.T;
    const int64_t t = live ? tb + threadIdx.x / G : a.T - 1;
    T x[V];
    load_logits<T, V>(z + t * a.row_stride, e0, a.E, a.vec, x);
    float p[V], dp[V], largest, scale;
    softmax_row<T, G, V>(x, e0, a.E, p, largest, scale);
#pragma unroll
    for (int i = 0; i < V; ++i) dp[i] = load[i];
    if (dw) {
      // Lane j % G has the j-th choice: its gradient, its weight and the probability of its expert.  What comes of it
      // goes to the lane that owns the expert through the row's stripe of shared memory, all zeros in between.
      int es[SL];
      float ds[SL], dot = 0.f, total = 0.f;
#pragma unroll
      for (int s = 0; s < SL; ++s) {
        const int j = s * G + gl;
        es[s] = -1;
        ds[s] = 0.f;
        if (j < a.k) {
          es[s] = (int)idx[t * a.k + j];
          ds[s] = dw[t * a.k + j];
          dot = fmaf(ds[s], w[t * a.k + j], dot);
          total += exp_below(to_f(z[t * a.row_stride + es[s]]), largest) * scale;
        }
      }
      dot = group_sum<G>(dot);
      const float inv = 1.f / (group_sum<G>(total) + 1e-20f);
#pragma unroll
      for (int s = 0; s < SL; ++s)
        if (es[s] >= 0) stripe[es[s]] = (ds[s] - dot) * inv;
      __syncwarp();
      // An expert's lane also clears its word: the barrier then stands between every access of one lane and the next
      // access of another, the next token's write included (the shuffles in between order no memory).
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        float4 *mine = reinterpret_cast<float4 *>(stripe + e0 + i);
        const float4 d = *mine;
        *mine = make_float4(0.f, 0.f, 0.f, 0.f);
        dp[i] += d.x; dp[i + 1] += d.y; dp[i + 2] += d.z; dp[i + 3] += d.w;
      }
      __syncwarp();
    }
    float pd = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) pd = fmaf(p[i], dp[i], pd);
    pd = group_sum<G>(pd);
    if (!live) continue;  // the last round
    T *out = dz + t * a.E + e0;
    constexpr int PER = 16 / (int)sizeof(T);
    T o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = from_f<T>(p[i] * (dp[i] - pd));
    if (V % PER == 0 && e0 + V <= a.E && a.E % PER == 0) {
#pragma unroll
      for (int q = 0; q < V / PER; ++q) {
        uint4 r;
        T *d = reinterpret_cast<T *>(&r);
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] = o[(q * PER + i) % V];
        *reinterpret_cast<uint4 *>(out + q * PER) = r;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e0 + i < a.E) out[i] = o[i];
    }
  }
}

// f(IC<G>, IC<V>, IC<SL>) of the smallest group that covers E experts, and of the
// slots a lane needs for k choices: one where the group has a lane for each, else
// two, else the most there can be (k <= E <= G V)
template <typename F>
static cudaError_t with_group(int E, int k, F &&f) {
  auto slots = [&](auto g, auto v) -> cudaError_t {
    constexpr int G = decltype(g)::value, V = decltype(v)::value;
    if (k <= G) return f(g, v, IC<1>{});
    if (k <= 2 * G) return f(g, v, IC<2>{});
    return f(g, v, IC<V>{});
  };
  if (E <= 8) return slots(IC<1>{}, IC<8>{});
  if (E <= 16) return slots(IC<2>{}, IC<8>{});
  if (E <= 32) return slots(IC<4>{}, IC<8>{});
  if (E <= 64) return slots(IC<8>{}, IC<8>{});
  if (E <= 128) return slots(IC<16>{}, IC<8>{});
  if (E <= 256) return slots(IC<32>{}, IC<8>{});
  return slots(IC<32>{}, IC<16>{});
}
static int group_of(int E) {
  int g = 1;
  while (g * 8 < E && g < 32) g <<= 1;
  return g;
}
// Four blocks an SM, as many as are resident: more partial sums to join buy nothing (262,144 x 64, top 6, bf16, forward:
// 2: 69 us, 4: 58, 8: 58; 65,536 x 256: 85, 71, 75).
static int blocks_for(int64_t T, int E, int sms) {
  const int rows = THREADS / group_of(E);
  const int64_t b = (T + rows - 1) / rows;
  const int64_t cap = (int64_t)(sms > 0 ? sms : 148) * 4;
  return (int)(b < cap ? b : cap);
}

}  // namespace router
}  // namespace mhc

using namespace mhc;

static int check_router(const char *who, int64_t T, int E, int k, int dtype, int64_t row_stride) {
  if (T < 0 || T > (int64_t)1 << 40) return fail(MHC_ERR_SHAPE, "%s: T = %lld", who, (long long)T);
  if (E < 1 || E > router::MAX_E) return fail(MHC_ERR_SHAPE, "%s: 1 to %d experts are supported (got %d)", who, router::MAX_E, E);
  if (k < 1 || k > E) return fail(MHC_ERR_SHAPE, "%s: k must be in [1, %d] (got %d)", who, E, k);
  if (dtype != MHC_F32 && dtype != MHC_BF16 && dtype != MHC_F16) return fail(MHC_ERR_DTYPE, "%s: bad dtype code %d", who, dtype);
  if (row_stride < E) return fail(MHC_ERR_SHAPE, "%s: row stride %lld < %d experts", who, (long long)row_stride, E);
  return MHC_OK;
}

extern "C" {

size_t mhc_route_fwd_workspace(int64_t T, int E) {
  if (T < 1 || E < 1 || E > router::MAX_E) return 0;
  const int blocks = router::blocks_for(T, E, device_sm_count());
  return blocks > 1 ? (size_t)blocks * (size_t)E * 8 : 0;  // one block keeps its sums to itself
}

int mhc_route_fwd(const void *logits, int dtype, int64_t T, int E, int64_t row_stride, int k, float coef, float *weights,
                  int64_t *experts, int64_t *counts, float *loss, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  if (int st = check_router("mhc_route_fwd", T, E, k, dtype, row_stride)) return st;
  if (!counts || !loss || (T > 0 && (!logits || !weights || !experts)))
    return fail(MHC_ERR_NULL, "mhc_route_fwd: required pointer is NULL");
  const size_t es = dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)logits % es || (uintptr_t)weights % 4 || (uintptr_t)experts % 8 || (uintptr_t)counts % 8 || (uintptr_t)loss % 4)
    return fail(MHC_ERR_ALIGN, "mhc_route_fwd: a pointer is not aligned to its elements");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (T == 0) {  // no token: no expert chosen, no loss
    cudaError_t e = cudaMemsetAsync(counts, 0, (size_t)E * 8, st);
    if (e == cudaSuccess) e = cudaMemsetAsync(loss, 0, 4, st);
    return cuda_status(e, "mhc_route_fwd");
  }
  const int blocks = router::blocks_for(T, E, device_sm_count());
  if (blocks > 1 && (!workspace || workspace_bytes < mhc_route_fwd_workspace(T, E)))
    return fail(MHC_ERR_WORKSPACE, "mhc_route_fwd: workspace %zu < %zu bytes", workspace_bytes, mhc_route_fwd_workspace(T, E));
  if ((uintptr_t)workspace % 4) return fail(MHC_ERR_ALIGN, "mhc_route_fwd: workspace is not 4-byte aligned");
  router::Args a{logits, T, row_stride, E, k, ((uintptr_t)logits % 16 == 0 && (row_stride * es) % 16 == 0) ? 1 : 0,
                 coef * (float)E};
  float *ps = static_cast<float *>(workspace);
  int *pc = reinterpret_cast<int *>(ps + (size_t)blocks * E);
  cudaError_t e = with_dtype(dtype, [&](auto tag) -> cudaError_t {
    using T_ = decltype(tag);
    return router::with_group(E, k, [&](auto g, auto v, auto sl) -> cudaError_t {
      router::route_fwd_kernel<T_, decltype(g)::value, decltype(v)::value, decltype(sl)::value>
          <<<blocks, router::THREADS, 0, st>>>(a, weights, experts, counts, loss, ps, pc);
      return cudaGetLastError();
    });
  });
  if (e == cudaSuccess && blocks > 1) {
    router::route_join_kernel<<<router::JOIN, 1024, 0, st>>>(a, ps, pc, blocks, counts, loss);
    e = cudaGetLastError();
  }
  return cuda_status(e, "mhc_route_fwd");
}

int mhc_route_bwd(const void *logits, int dtype, int64_t T, int E, int64_t row_stride, int k, float coef,
                  const float *weights, const int64_t *experts, const int64_t *counts, const float *dweights,
                  const float *dloss, void *dlogits, void *stream) {
  clear_error();
  if (int st = check_router("mhc_route_bwd", T, E, k, dtype, row_stride)) return st;
  if (T == 0) return MHC_OK;
  if (!logits || !weights || !experts || !counts || !dlogits)
    return fail(MHC_ERR_NULL, "mhc_route_bwd: required pointer is NULL");
  const size_t es = dtype == MHC_F32 ? 4 : 2;
  if ((uintptr_t)logits % es || (uintptr_t)weights % 4 || (uintptr_t)experts % 8 || (uintptr_t)counts % 8 ||
      (uintptr_t)dweights % 4 || (uintptr_t)dloss % 4 || (uintptr_t)dlogits % 16)
    return fail(MHC_ERR_ALIGN, "mhc_route_bwd: a pointer is not aligned (dlogits: 16 bytes, others: their elements)");
  router::Args a{logits, T, row_stride, E, k, ((uintptr_t)logits % 16 == 0 && (row_stride * es) % 16 == 0) ? 1 : 0,
                 coef * (float)E};
  const int rows = router::THREADS / router::group_of(E);
  // nothing to join here: 4 to 8 blocks an SM are alike (50 to 54 us at 262,144 x 64 with autograd's part), 16 take 58
  const int64_t want = (T + rows - 1) / rows, cap = (int64_t)(device_sm_count() > 0 ? device_sm_count() : 148) * 8;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = with_dtype(dtype, [&](auto tag) -> cudaError_t {
    using T_ = decltype(tag);
    return router::with_group(E, k, [&](auto g, auto v, auto sl) -> cudaError_t {
      router::route_bwd_kernel<T_, decltype(g)::value, decltype(v)::value, decltype(sl)::value>
          <<<grid, router::THREADS, 0, st>>>(a, weights, experts, counts, dweights, dloss, static_cast<T_ *>(dlogits));
      return cudaGetLastError();
    });
  });
  return cuda_status(e, "mhc_route_bwd");
}

}  // extern "C"
