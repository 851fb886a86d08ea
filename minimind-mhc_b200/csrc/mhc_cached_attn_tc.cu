// Attention over a paged cache on the 5th-generation tensor cores, for items of more rows
// than the warp-wide products of mhc_cached_attn.cu take at once (bf16 / fp16; pages that
// divide a tile of 128 keys or are made of such tiles).
//
//   S = Q K^T    tcgen05.mma, M = N = 128, K = D, both operands in shared memory
//   P = exp2((S - m) c)                         c = scale log2(e), one thread per row
//   O += P V     A = P from TMEM (it replaces S there), B = V as it lies in memory
//
// The rows are those of one item, up to 128 new tokens x heads of a group.  A step (S,
// softmax, O) is a chain of waits; two of them run side by side: the key tiles of an item
// go in turn to two sets of four softmax warps with scores, sums and O of their own, over
// the same queries, and the tensor core serves one while the other's softmax runs.  In the
// end the two O lie in TMEM in the same lanes, so each set joins half of the columns of
// both without moving them; only references and sums cross through shared memory.
//
// K and V come by TMA, one box for each page and 64 columns of a tile, the lanes of a
// warp one page each, two or more tiles ahead, across the ends of items too.  V rows that do
// not exist are zeroed in shared memory (a P of 0 times a NaN would be NaN), and so are
// infinities and NaN of new tokens' V, which some rows of the item do not see: the rows
// that see one add it in the end.
//
// Warps 0-3 and 4-7: the two softmax sets; 8: TMA; 9: MMA issue.  Every wait is bounded; a
// block whose wait runs out writes NaN over its share.
#include <cfloat>
#include <mutex>

#include "mhc_attn_tc.cuh"
#include "mhc_cached_attn.cuh"

namespace mhc {

__device__ int g_cat_error = 0;

namespace cattn {

namespace {

using namespace sm100;
using attn::BLK;
using attn::TM;
using attn::Tile;
using attn::idesc_of;
using attn::mma_rows;
using attn::mma_sum;
using attn::pack2;
using attn::wait_warp_parity;

constexpr int NTHREADS = 320;
constexpr int W_TMA = 8, W_MMA = 9;
constexpr int TMEM_COLS = 512;
constexpr uint32_t S_COL = 0, O_COL = 256;  // two score tiles, two results, 128 columns each
enum { ERR_TMA = 61, ERR_MMA = 62, ERR_SOFTMAX = 63 };
constexpr int ODD = 8;  // items whose odd values are remembered: more than the TMA warp can be ahead

template <int DP>
struct Cfg {
  using L = Tile<DP, false>;
  static constexpr uint32_t TILE = L::BYTES;
  static constexpr int ST = DP <= 64 ? 6 : 3;  // stages of K and of V
  static constexpr size_t SMEM = TILE + 2 * ST * TILE + 1024;
};

constexpr int B_QF = 0, B_LAND = 1, B_SF = 2, B_PF = 4, B_OF = 6, B_DRAIN = 8, B_KF = 9;
// then ST each: KF, KE, VF, VE

// Tensor maps of keys and values: (D, slots and heads by their strides, pages) in boxes of one page's rows (128 at most) x 64
// columns; head_first: the second axis is the head.
struct Maps {
  CUtensorMap k, v;
  int k_head_first, v_head_first;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *tmap, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void give_up(int code, volatile int *abort_flag, int *err_flag) {
  *abort_flag = 1;
  report_give_up(&g_cat_error, err_flag, code);
}
// the softmax threads only
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ bool finite16(uint16_t w) {
  constexpr uint16_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7f80 : 0x7c00;
  return (w & E) != E;
}

// the 32 columns from `base` on that a row sees: keys that exist, of the context or among its new tokens
__device__ __forceinline__ uint32_t seen_columns(const Args &a, const Segment &g, const Row &x, int base) {
  const uint32_t there = attn::bits_between(0, g.keys - base), context = attn::bits_between(0, g.s.len - base);
  uint32_t fresh;
  if (a.mask) {
    const int c = base - g.s.len;  // the first column's new token
    fresh = c >= 64 ? 0u : c >= 0 ? (uint32_t)(x.bits >> c) : c > -32 ? (uint32_t)(x.bits << -c) : 0u;
  } else {
    fresh = attn::bits_between(g.s.len - base, g.s.len + x.j + 1 - base);
  }
  return there & (context | fresh);
}

template <typename T, int DP>
__global__ void __launch_bounds__(NTHREADS, 1) cached_attn_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a) {
  using C = Cfg<DP>;
  using L = typename C::L;
  constexpr int ST = C::ST, M = CATTN_TC_ROWS;
  constexpr int B_KE = B_KF + ST, B_VF = B_KE + ST, B_VE = B_VF + ST, NBARS = B_VE + ST;
  constexpr float LAZY = std::is_same<T, __half>::value ? 4.f : 8.f, LIFT = std::is_same<T, __half>::value ? 10.f : 0.f;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ volatile int odd_item[ODD];  // item i + 1 where item i has odd values among its new tokens' V
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - raw);
  // references and sums of both sets, where the queries lie: their last product is done by then
  float2(*sums)[TM] = reinterpret_cast<float2(*)[TM]>(gen);
  const uint32_t qs = base, ks = qs + C::TILE, vs = ks + ST * C::TILE;
  volatile int *abort_flag = &abort_word;
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  if (tid == 0) {
    abort_word = 0;
    for (int i = 0; i < ODD; ++i) odd_item[i] = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_SF + i), 1);
      mbar_init(BAR(B_PF + i), 128);
      mbar_init(BAR(B_OF + i), 1);
    }
    mbar_init(BAR(B_QF), 256);
    mbar_init(BAR(B_LAND), 1);
    mbar_init(BAR(B_DRAIN), 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(BAR(B_KF + i), 1);
      mbar_init(BAR(B_KE + i), 1);
      mbar_init(BAR(B_VF + i), 1);
      mbar_init(BAR(B_VE + i), 1);
    }
    fence_mbar_init_cluster();
  }
  if (warp == W_MMA) {
    tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  clear_rest<T>(a);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);

  if (warp == W_TMA) {
    // ---------------- TMA: a lane for each page of a tile ----------------
    bool ok = true;
    int t = 0, nk = 0, nv = 0, lands = 0, items = 0;  // key tiles, K and V tiles asked for, V tiles looked through, items so far
    const int rows = min(a.c.size, TM), boxes = TM / rows;  // of a box, in a tile
    walk<M>(a, [&](const Segment &g, int) {
      const int item = items++;
      if (!ok) return;
      for (int j = g.k0; j < g.k1; ++j, ++t) {
        const int s = t % ST, key = j * TM + lane * rows;
        const uint32_t free_par = ((uint32_t)(t / ST) & 1u) ^ 1u;
        int page = lane < boxes ? page_of(a, g, key) : -1;
        if (page >= a.c.pages) page = -1;
        const int slot = page >= 0 ? key - cache::page_index(a.c, key) * a.c.size : 0;
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t bytes = (uint32_t)(__popc(there) * rows * 128) * L::FULL;
        auto load = [&](uint32_t dst, const CUtensorMap &map, int head_first, uint32_t bar) {
          if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
          __syncwarp();
          if (page >= 0)
#pragma unroll
            for (int b = 0; b < L::FULL; ++b)
              tma_load_4d(dst + b * BLK + lane * rows * 128, &map, b * 64, head_first ? g.hk : slot, head_first ? slot : g.hk, page, bar);
        };
        if (!wait_warp_parity(BAR(B_KE + s), free_par, abort_flag)) { ok = false; break; }
        load(ks + s * C::TILE, maps.k, maps.k_head_first, BAR(B_KF + s));
        nk = t + 1;
        if (!wait_warp_parity(BAR(B_VE + s), free_par, abort_flag)) { ok = false; break; }
        const int end = (j + 1) * TM;
        const bool gaps = g.keys < end || there != (boxes == 32 ? 0xffffffffu : (1u << boxes) - 1), fresh = (g.s.n > 1 || a.mask) && g.s.len < end;
        load(vs + s * C::TILE, maps.v, maps.v_head_first, BAR(gaps || fresh ? B_LAND : B_VF + s));
        nv = t + 1;
        if (gaps || fresh) {
          if (!wait_warp_parity(BAR(B_LAND), (uint32_t)lands & 1u, abort_flag)) ok = false;
          ++lands;
          uint8_t *tile = gen + (vs - base) + s * C::TILE;
          bool odd = false;
          for (int i = lane; i < TM * L::FULL * 8; i += 32) {  // 16 bytes at a time; neighbouring lanes in one row
            const int r = i / (L::FULL * 8), c = i - r * (L::FULL * 8), at = j * TM + r;
            uint4 *p = reinterpret_cast<uint4 *>(tile + (c >> 3) * BLK + r * 128 + (c & 7) * 16);
            if (at >= g.keys || !((there >> (r / rows)) & 1)) {
              *p = make_uint4(0u, 0u, 0u, 0u);
            } else if (fresh && at >= g.s.len) {
              uint4 x = *p;
              uint16_t *e = reinterpret_cast<uint16_t *>(&x);
              bool bad = false;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (!finite16<T>(e[k])) {
                  e[k] = 0;
                  bad = true;
                }
              if (bad) *p = x;
              odd = odd || bad;
            }
          }
          fence_proxy_async_smem();
          if (__any_sync(0xffffffffu, odd) && lane == 0) odd_item[item % ODD] = item + 1;
          __threadfence_block();
          __syncwarp();
          if (lane == 0) mbar_arrive(BAR(B_VF + s));
          if (!ok) break;
        }
      }
    });
    if (!ok && lane == 0) give_up(ERR_TMA, abort_flag, a.err_flag);
    // copies in flight land before the block may exit
    for (int p = nk > ST ? nk - ST : 0; p < nk; ++p) wait_parity<false>(BAR(B_KF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
    for (int p = nv > ST ? nv - ST : 0; p < nv; ++p) wait_parity<false>(BAR(B_VF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
  } else if (warp == W_MMA) {
    // ---------------- MMA issue: the warp runs it, one lane issues ----------------
    constexpr uint32_t id_s = idesc_of<T>(128, 0), id_o = idesc_of<T>(L::N_FULL, 1);
    bool ok = true;
    int t0 = 0, qn = 0, pf[2] = {0, 0};
    auto wait_warp = [&](uint32_t bar, uint32_t par) {
      if (!wait_warp_parity(bar, par, abort_flag)) ok = false;
      return ok;
    };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) umma_commit(bar);
    };
    walk<M>(a, [&](const Segment &g, int) {
      if (!ok) return;
      const int n = g.k1 - g.k0;
      auto scores = [&](int j) {
        const int t = t0 + j;
        if (!wait_warp(BAR(B_KF + t % ST), (uint32_t)(t / ST) & 1u)) return;
        tc_fence_after();
        mma_rows<L>(tmem + S_COL + (j & 1) * 128u, qs, ks + (t % ST) * C::TILE, id_s);
        commit(BAR(B_SF + (j & 1)));
        commit(BAR(B_KE + t % ST));
      };
      if (!wait_warp(BAR(B_QF), (uint32_t)qn & 1u)) return;
      ++qn;
      tc_fence_after();
      scores(0);
      if (ok && n > 1) scores(1);
      for (int j = 0; j < n && ok; ++j) {
        const int t = t0 + j, s = j & 1;
        if (!wait_warp(BAR(B_VF + t % ST), (uint32_t)(t / ST) & 1u)) return;
        if (!wait_warp(BAR(B_PF + s), (uint32_t)pf[s] & 1u)) return;
        ++pf[s];
        tc_fence_after();
        mma_sum<L>(tmem + O_COL + s * 128u, tmem + S_COL + s * 128u, 16u, vs + (t % ST) * C::TILE, id_o, 0u, j < 2);
        commit(BAR(B_OF + s));
        commit(BAR(B_VE + t % ST));
        // S of the step after next may follow P V of this one at once: the tensor core runs them in order
        if (j + 2 < n) scores(j + 2);
      }
      t0 += n;
    });
    if (!ok && lane == 0) give_up(ERR_MMA, abort_flag, a.err_flag);
    commit(BAR(B_DRAIN));
    __syncwarp();
  } else {
    // ---------------- softmax: thread = row, set t every other key tile ----------------
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL + t * 128u, o_addr = tmem + lanes + O_COL;
    const uint64_t c2 = f2_pack(a.c2, a.c2), lift2 = f2_pack(LIFT, LIFT);
    bool ok = true;
    int sf = 0, of = 0, items = 0;
    walk<M>(a, [&](const Segment &g, int slot) {
      // after a wait of any role has run out the items are walked through all the same: every thread meets the barriers
      const int item = items++;
      const Row x = row_of(a, g, r);
      if (ok) {  // this set's half of the row's queries; the last products on the tile are done
        constexpr int VEC = L::FULL * 8, HALF = VEC / 2;  // 16-byte vectors
        const T *src = static_cast<const T *>(a.q) + (x.j >= 0 ? q_at(a, g, x, g.hk) : 0);
        uint4 v[HALF];
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          const int c = t * HALF + i;
          v[i] = x.j >= 0 && c * 8 < a.c.D ? *reinterpret_cast<const uint4 *>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
          const int c = t * HALF + i;
          *reinterpret_cast<uint4 *>(gen + (c >> 3) * BLK + r * 128 + (((c & 7) ^ (r & 7)) * 16)) = v[i];
        }
        fence_proxy_async_smem();
        mbar_arrive(BAR(B_QF));
      }
      const bool any_rows = (warp & 3) * 32 < g.rows;
      const int psize = min(a.c.size, TM), boxes = TM / psize;
      float ref = -INFINITY, sum = 0.f;
      int steps = 0;
      for (int j = g.k0 + t; ok && j < g.k1; j += 2, ++steps) {
        const int k0 = j * TM;
        // which of the tile's pages there are
        int page = lane < boxes ? page_of(a, g, k0 + lane * psize) : 0;
        const unsigned missing = __ballot_sync(0xffffffffu, lane < boxes && k0 + lane * psize < g.keys && (page < 0 || page >= a.c.pages));
        if (!wait_warp_parity(BAR(B_SF + t), (uint32_t)sf & 1u, abort_flag)) { ok = false; break; }
        ++sf;
        tc_fence_after();
        if (any_rows) {
          uint32_t w[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32_nowait(s_addr + q * 32, w[q]);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(w[q][e]));  // not read before the wait
          bool some = true;
          if (missing || k0 + TM > g.s.len || k0 + TM > g.keys) {
            some = false;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t seen = x.j >= 0 ? seen_columns(a, g, x, k0 + q * 32) : 0u;
              if (missing) {
#pragma unroll 1
                for (int e = 0; e < 32; ++e)
                  if ((missing >> ((q * 32 + e) / psize)) & 1) seen &= ~(1u << e);
              }
              some = some || seen;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen & (1u << e))) w[q][e] = 0xff800000u;
            }
          }
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; ++e)
#pragma unroll
            for (int q = 0; q < 4; ++q) m[q] = fmaxf(m[q], __uint_as_float(w[q][e]));
          const float top = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), some ? -FLT_MAX : -INFINITY);
          const bool grow = (top - ref) * a.c2 > LAZY;  // both -inf: NaN, no
          if (__any_sync(0xffffffffu, grow)) {
            const float next = grow ? top : ref;
            const float fix = grow ? factor(ref, next, a.c2) : 1.f;  // 0 for the first visible keys
            ref = next;
            sum *= fix;
            if (steps > 0) {  // O holds the earlier tiles' sum, once their product is done
              if (!wait_warp_parity(BAR(B_OF + t), (uint32_t)(of - 1) & 1u, abort_flag)) { ok = false; break; }
              tc_fence_after();
#pragma unroll
              for (int d = 0; d < DP; d += 16) {  // in pieces that leave the scores in their registers
                uint32_t o[16];
                tmem_ld16u(o_addr + t * 128u + d, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
                tmem_st16(o_addr + t * 128u + d, o);
              }
              tmem_wait_st();
            }
          }
          const float off = ref == -INFINITY ? 0.f : -ref;
          const uint64_t off2 = f2_pack(off, off);
          uint64_t acc[2] = {0ull, 0ull};
          uint32_t p[2][32];
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float y, z;
              f2_unpack(f2_fma(f2_add(f2_pack(__uint_as_float(w[q][e]), __uint_as_float(w[q][e + 1])), off2), c2, lift2), y, z);
              y = ex2(y);
              z = ex2(z);
              acc[(e >> 1) & 1] = f2_add(acc[(e >> 1) & 1], f2_pack(y, z));
              p[q >> 1][(q & 1) * 16 + (e >> 1)] = pack2<T>(y, z);
            }
          tmem_st32(s_addr, p[0]);
          tmem_st32(s_addr + 32, p[1]);
          tmem_wait_st();
          float y, z;
          f2_unpack(f2_add(acc[0], acc[1]), y, z);
          sum += y + z;
        }
        tc_fence_before();
        mbar_arrive(BAR(B_PF + t));
        ++of;
      }
      if (ok && steps > 0 && !wait_warp_parity(BAR(B_OF + t), (uint32_t)(of - 1) & 1u, abort_flag)) ok = false;
      tc_fence_after();
      if (steps > 0) sums[t][r] = make_float2(ref, sum);
      tc_fence_before();
      softmax_sync();
      tc_fence_after();
      if (any_rows && !*abort_flag) {
        const bool both = g.k1 - g.k0 > 1;
        const float2 s0 = sums[0][r], s1 = both ? sums[1][r] : make_float2(-INFINITY, 0.f);
        const float top = fmaxf(s0.x, s1.x);
        const float f0 = factor(s0.x, top, a.c2), f1 = factor(s1.x, top, a.c2);
        const float all = fmaf(f0, s0.y, f1 * s1.y);
        float scale = 1.f;
        if (slot < 0) scale = top == -INFINITY ? 0.f : 1.f / all;
        else if (t == 0 && x.j >= 0) a.part_ml[(int64_t)slot * M + r] = make_float2(top, all);
        const float w0 = f0 * scale, w1 = f1 * scale;
        const bool odd = odd_item[item % ODD] == item + 1;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const int d = t * (DP / 2) + i * 16;
          uint32_t o0[16], o1[16];
          tmem_ld16u(o_addr + d, o0);
          float y[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(o0[e]) * w0;
          if (both) {
            tmem_ld16u(o_addr + 128u + d, o1);
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = fmaf(__uint_as_float(o1[e]), w1, y[e]);
          }
          if (odd && x.j >= 0) {  // infinities and NaN that the row sees, of the new tokens in this block's tiles
#pragma unroll 1
            for (int key = max(g.s.len, g.k0 * TM); key < min(g.keys, g.k1 * TM); ++key) {
              const int c = key - g.s.len;
              if (a.mask ? c >= 64 || !((x.bits >> c) & 1) : c > x.j) continue;
              const int page = page_of(a, g, key);
              if (page < 0 || page >= a.c.pages) continue;
              const T *v = static_cast<const T *>(a.c.values) + page * a.c.vp +
                           (key - cache::page_index(a.c, key) * a.c.size) * a.c.vs + g.hk * a.c.vh;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (d + e < a.c.D && !finite16<T>(*reinterpret_cast<const uint16_t *>(v + d + e))) y[e] += to_f(v[d + e]);
            }
          }
          if (x.j < 0) continue;
          if (slot >= 0) {
            float *dst = a.part_o + ((int64_t)slot * M + r) * DP + d;
#pragma unroll
            for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4 *>(dst + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
          } else {
            T *dst = static_cast<T *>(a.out) + out_at(a, g, x, g.hk) + d;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (d + h * 8 < a.c.D)  // D is a multiple of 8
                *reinterpret_cast<uint4 *>(dst + h * 8) = make_uint4(pack2<T>(y[h * 8], y[h * 8 + 1]), pack2<T>(y[h * 8 + 2], y[h * 8 + 3]),
                                                                    pack2<T>(y[h * 8 + 4], y[h * 8 + 5]), pack2<T>(y[h * 8 + 6], y[h * 8 + 7]));
          }
        }
      }
      tc_fence_before();
      softmax_sync();
      tc_fence_after();
    });
    if (!ok && lane == 0) give_up(ERR_SOFTMAX, abort_flag, a.err_flag);
  }

  // ---------------- teardown ----------------
  __syncthreads();
  if (warp == W_MMA) {
    wait_parity<false>(BAR(B_DRAIN), 0u, nullptr);
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  if (*abort_flag) {
    // a wait gave up: this block's share becomes NaN instead of partly written
    const T bad = from_f<T>(__int_as_float(0x7fc00000));
    walk<M>(a, [&](const Segment &g, int slot) {
      for (int i = tid; i < g.rows * a.c.D; i += NTHREADS) {
        const int r = i / a.c.D;
        if (slot < 0) static_cast<T *>(a.out)[out_at(a, g, row_of(a, g, r), g.hk) + i % a.c.D] = bad;
        else a.part_ml[(int64_t)slot * M + r] = make_float2(0.f, __int_as_float(0x7fc00000));
      }
    });
  }
  grid_dep_launch();
#undef BAR
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// strides of one tensor for its map: of an axis of one element any will do
struct Axes {
  int64_t slot, head, page;
  bool head_first;
};
Axes axes_of(const mhc_kv_cache *c, const int64_t *s) {
  Axes x{s[2], s[3], s[1], false};
  if (c->page_size == 1) x.slot = c->dim;
  if (c->kv_heads == 1) x.head = x.slot * c->page_size;
  x.head_first = x.head < x.slot;
  if (c->pages == 1) x.page = (x.slot > x.head ? x.slot : x.head);
  return x;
}
bool axes_ok(const mhc_kv_cache *c, const Axes &x) {
  const int64_t most = (int64_t)1 << 38;
  return x.slot % 8 == 0 && x.head % 8 == 0 && x.page % 8 == 0 && x.slot >= c->dim && x.head >= c->dim && x.page >= x.slot && x.page >= x.head &&
         x.page < most;
}
bool make_map(CUtensorMap *map, const mhc_kv_cache *c, void *p, const Axes &x) {
  auto enc = encode_fn();
  if (!enc) return false;
  const cuuint32_t rows = c->page_size < TM ? c->page_size : TM;
  const cuuint64_t dims[4] = {(cuuint64_t)c->dim, (cuuint64_t)(x.head_first ? c->kv_heads : c->page_size),
                              (cuuint64_t)(x.head_first ? c->page_size : c->kv_heads), (cuuint64_t)c->pages};
  const cuuint64_t strides[3] = {(cuuint64_t)(x.head_first ? x.head : x.slot) * 2, (cuuint64_t)(x.head_first ? x.slot : x.head) * 2,
                                 (cuuint64_t)x.page * 2};
  const cuuint32_t box[4] = {64u, x.head_first ? 1u : rows, x.head_first ? rows : 1u, 1u}, ones[4] = {1, 1, 1, 1};
  return enc(map, c->dtype == MHC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, p, dims, strides, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
cudaError_t run(const Args &a, const Maps &maps, cudaStream_t stream) {
  using C = Cfg<DP>;
  auto kern = cached_attn_tc_kernel<T, DP>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
  if (e != cudaSuccess) return e;
  kern<<<a.pieces, NTHREADS, C::SMEM, stream>>>(maps, a);
  return cudaGetLastError();
}

}  // namespace
}  // namespace cattn

// What TMA asks of the cache: rows of 16-byte multiples that do not overlap, in pages of which a tile of 128 keys has a
// whole number, or the other way round.
bool cached_attn_tc_eligible(const mhc_kv_cache *c) {
  if (c->dtype == MHC_F32 || c->dim % 8 || c->page_size % 8 || (attn::TM % c->page_size && c->page_size % attn::TM)) return false;
  if ((uintptr_t)c->keys % 16 || (uintptr_t)c->values % 16) return false;
  return cattn::axes_ok(c, cattn::axes_of(c, c->strides)) && cattn::axes_ok(c, cattn::axes_of(c, c->strides + 4));
}

cudaError_t launch_cached_attn_tc(const cattn::Args &a, const mhc_kv_cache *c, cudaStream_t stream) {
  cattn::Maps maps;
  const cattn::Axes k = cattn::axes_of(c, c->strides), v = cattn::axes_of(c, c->strides + 4);
  if (!cattn::make_map(&maps.k, c, c->keys, k) || !cattn::make_map(&maps.v, c, c->values, v)) return cudaErrorNotSupported;
  maps.k_head_first = k.head_first;
  maps.v_head_first = v.head_first;
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if (a.c.D <= 32) return cattn::run<T, 32>(a, maps, stream);
    if (a.c.D <= 64) return cattn::run<T, 64>(a, maps, stream);
    if (a.c.D <= 96) return cattn::run<T, 96>(a, maps, stream);
    return cattn::run<T, 128>(a, maps, stream);
  };
  return a.dtype == MHC_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

int read_cat_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_cat_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_cat_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mhc
