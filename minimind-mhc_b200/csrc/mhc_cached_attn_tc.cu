// Attention over a paged cache on the 5th-generation tensor cores, for items of more rows
// than the warp-wide products of mhc_cached_attn.cu take at once (bf16 / fp16).
//
//   S = Q K^T    tcgen05.mma, M = 128, N = 64, K = D, both operands in shared memory
//   P = exp2((S - m) c)                         c = scale log2(e), one thread per row
//   O += P V     A = P from TMEM (it replaces S there), B = V as it lies in memory
//
// The rows are those of one item, up to 128 new tokens x heads of a group.  A step (scores,
// softmax, product) is a chain of waits, an item begins with three loads one after another
// (lengths, pages and rows; queries), and ends with O's way out: two blocks run on an SM, each
// with half of TMEM and of shared memory, so that one works while the other waits.  (One
// block with tiles of 128 keys and two sets of softmax warps, the key tiles in turn, took
// 1.5 us a tile and 14 us for an item's two ends.)  Scores are formed one tile ahead, into the
// other of two buffers.
//
// K and V come by TMA, a box for the rows that lie in one page wherever a tile begins (of 64
// keys and pages of 48, 16; of pages of 17, each by itself) and 64 columns, the lanes of a
// warp one or two boxes each, across the ends of items too.  V rows that do
// not exist are zeroed in shared memory (a P of 0 times a NaN would be NaN), and so are
// infinities and NaN of those new tokens' V that some rows of the item do not see: the rows
// that see one add it in the end.  (Without a mask those are the item's own tokens but the
// first and what lies behind them, with one the sequence's first 64: however long a piece
// of a prompt, a row looks through 128 keys at most.)  The softmax threads do that, half a row
// of V each, before they hand over P.
//
// What bounds it: a tile takes a block 1.0 to 1.2 us (two of them an SM: 32 KB of K and V each,
// at 128 rows the softmax's chain and 2^x, at 32 rows HBM: 1.5 us a tile is the copy rate); an item's
// two ends about 10 us, half of it instructions that have not run before.  Measured (with the
// join): 16 sequences with trees of up to 64, 127,000 keys in all, 8 / 2 heads of 128, 256 rows:
// 55 us; 16 tokens over 131,072 keys, 8 / 4 heads of 128: 57 us, 4.7 TB/s.
//
// Warps 0-3: softmax, a row each; 4: TMA; 5: MMA issue.  Every wait is bounded; a block whose
// wait runs out writes NaN over its share.
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
using attn::idesc_of;
using attn::pack2;
using attn::wait_warp_parity;

constexpr int TN = CATTN_TC_KEYS;
constexpr uint32_t KBLK = TN * 128;  // 64 keys x 64 values of 16 bits, 128-byte swizzle
constexpr int NTHREADS = 192;
constexpr int W_TMA = 4, W_MMA = 5;
constexpr int TMEM_COLS = 256;
constexpr uint32_t S_COL = 0, O_COL = 128;  // two score tiles of 64 columns; the result
enum { ERR_TMA = 61, ERR_MMA = 62, ERR_SOFTMAX = 63 };

template <int DP>
struct Cfg {
  static constexpr int FULL = (DP + 63) / 64;  // blocks of 64 columns, filled up with zeros
  static constexpr uint32_t Q = FULL * BLK, TILE = FULL * KBLK;
  static constexpr int ST = DP <= 64 ? 5 : 2;  // stages of K and of V
  static constexpr size_t SMEM = Q + 2 * ST * TILE + 1024;
};

constexpr int B_QF = 0, B_DRAIN = 1, B_SF = 2, B_PF = 4, B_OF = 6, B_KF = 8;
// then ST each: KF, KE, VF, VE

// S [128 x 64] = Q K^T over DP columns
template <int DP>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t idesc) {
  const uint64_t ad = umma_desc_sw128(q), bd = umma_desc_sw128(k);
  if (elect_one()) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      umma_bf16(d, ad + ((uint64_t)((kk >> 2) * (int)BLK + (kk & 3) * 32) >> 4), bd + ((uint64_t)((kk >> 2) * (int)KBLK + (kk & 3) * 32) >> 4),
                idesc, kk > 0);
  }
}
// O [128 x DP] (+)= P V: P in TMEM, 32 keys in 16 columns; V's rows are the summed index
__device__ __forceinline__ void mma_product(uint32_t d, uint32_t p, uint32_t v, uint32_t idesc, bool begin) {
  const uint64_t bd = umma_desc(v, KBLK, 1024, 2);
  if (elect_one()) {
#pragma unroll
    for (int kk = 0; kk < TN / 16; ++kk) umma_f16_ts(d, p + kk * 8u, bd + kk * (2048 >> 4), idesc, !begin || kk > 0);
  }
}

// Tensor maps of keys and values: (D, slots and heads by their strides, pages) in boxes of the rows that pages and tiles have in common x 64
// columns; head_first: the second axis is the head.
struct Maps {
  CUtensorMap k, v;
  int k_head_first, v_head_first;
  int rows;  // of a box: they lie in one page wherever a tile begins
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
template <typename T>
__device__ __forceinline__ bool finite16(uint16_t w) {
  constexpr uint16_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7f80 : 0x7c00;
  return (w & E) != E;
}

// two values with zeros in the place of infinities and NaN
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  if ((w & E) == E) w &= 0xffff0000u;
  if ((w & (E << 16)) == (E << 16)) w &= 0xffffu;
  return w;
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
__global__ void __launch_bounds__(NTHREADS, CATTN_TC_BLOCKS)
cached_attn_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a) {
  using C = Cfg<DP>;
  constexpr int ST = C::ST, M = CATTN_TC_ROWS;
  constexpr int B_KE = B_KF + ST, B_VF = B_KE + ST, B_VE = B_VF + ST, NBARS = B_VE + ST;
  constexpr float LAZY = std::is_same<T, __half>::value ? 4.f : 8.f, LIFT = std::is_same<T, __half>::value ? 10.f : 0.f;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ volatile int odd_item;  // the block's last item that had infinities or NaN among its new tokens' V
  __shared__ Near near;
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - raw);
  const uint32_t qs = base, ks = qs + C::Q, vs = ks + ST * C::TILE;
  volatile int *abort_flag = &abort_word;
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  if (tid == 0) {
    abort_word = odd_item = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_SF + i), 1);
      mbar_init(BAR(B_PF + i), 128);
      mbar_init(BAR(B_OF + i), 1);
    }
    mbar_init(BAR(B_QF), 128);
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
  grid_dep_wait();
  near.fill(a);
  clear_rest<T>(a);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);

  if (warp == W_TMA) {
    // ---------------- TMA: the lanes have a box or two of a tile each ----------------
    bool ok = true;
    int t = 0, nk = 0, nv = 0;  // key tiles, K and V tiles asked for so far
    const int rows = maps.rows, boxes = TN / rows;  // of a box, in a tile
    walk<M>(a, near, [&](const Segment &g, int) {
      if (!ok) return;
      for (int j = g.k0; j < g.k1; ++j, ++t) {
        const int s = t % ST;
        const uint32_t free_par = ((uint32_t)(t / ST) & 1u) ^ 1u;
        int page[2], slot[2], count = 0;  // a lane's boxes
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int box = lane + 32 * u, key = j * TN + box * rows;
          page[u] = box < boxes ? page_of(a, g, key) : -1;
          if (page[u] >= a.c.pages) page[u] = -1;
          slot[u] = page[u] >= 0 ? key - cache::page_index(a.c, key) * a.c.size : 0;
          count += __popc(__ballot_sync(0xffffffffu, page[u] >= 0));
        }
        auto load = [&](uint32_t dst, const CUtensorMap &map, int head_first, uint32_t bar) {
          if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(count * rows * 128) * C::FULL);
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (page[u] >= 0)
#pragma unroll
              for (int b = 0; b < C::FULL; ++b)
                tma_load_4d(dst + b * KBLK + (lane + 32 * u) * rows * 128, &map, b * 64, head_first ? g.hk : slot[u],
                            head_first ? slot[u] : g.hk, page[u], bar);
        };
        if (!wait_warp_parity(BAR(B_KE + s), free_par, abort_flag)) { ok = false; break; }
        load(ks + s * C::TILE, maps.k, maps.k_head_first, BAR(B_KF + s));
        nk = t + 1;
        if (!wait_warp_parity(BAR(B_VE + s), free_par, abort_flag)) { ok = false; break; }
        load(vs + s * C::TILE, maps.v, maps.v_head_first, BAR(B_VF + s));
        nv = t + 1;
      }
    });
    if (!ok && lane == 0) give_up(ERR_TMA, abort_flag, a.err_flag);
    // copies in flight land before the block may exit
    for (int p = nk > ST ? nk - ST : 0; p < nk; ++p) wait_parity<false>(BAR(B_KF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
    for (int p = nv > ST ? nv - ST : 0; p < nv; ++p) wait_parity<false>(BAR(B_VF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
  } else if (warp == W_MMA) {
    // ---------------- MMA issue: the warp runs it, one lane issues ----------------
    constexpr uint32_t id_s = idesc_of<T>(TN, 0), id_o = idesc_of<T>(DP, 1);
    bool ok = true;
    int t0 = 0, qn = 0, pf[2] = {0, 0};
    auto wait_warp = [&](uint32_t bar, uint32_t par) {
      if (!wait_warp_parity(bar, par, abort_flag)) ok = false;
      return ok;
    };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) umma_commit(bar);
    };
    walk<M>(a, near, [&](const Segment &g, int) {
      if (!ok) return;
      const int n = g.k1 - g.k0;
      auto scores = [&](int j) {
        const int t = t0 + j;
        if (!wait_warp(BAR(B_KF + t % ST), (uint32_t)(t / ST) & 1u)) return;
        tc_fence_after();
        mma_scores<DP>(tmem + S_COL + (j & 1) * 64u, qs, ks + (t % ST) * C::TILE, id_s);
        commit(BAR(B_SF + (j & 1)));
        commit(BAR(B_KE + t % ST));
      };
      if (!wait_warp(BAR(B_QF), (uint32_t)qn & 1u)) return;
      ++qn;
      tc_fence_after();
      scores(0);
      for (int j = 0; j < n && ok; ++j) {
        const int t = t0 + j, s = j & 1;
        // beside the softmax of this tile; the buffer's last P has been read by then, the tensor core goes in order
        if (j + 1 < n) scores(j + 1);
        if (!ok || !wait_warp(BAR(B_VF + t % ST), (uint32_t)(t / ST) & 1u)) return;
        if (!wait_warp(BAR(B_PF + s), (uint32_t)pf[s] & 1u)) return;
        ++pf[s];
        tc_fence_after();
        mma_product(tmem + O_COL, tmem + S_COL + s * 64u, vs + (t % ST) * C::TILE, id_o, j == 0);
        commit(BAR(B_OF + s));
        commit(BAR(B_VE + t % ST));
      }
      t0 += n;
    });
    if (!ok && lane == 0) give_up(ERR_MMA, abort_flag, a.err_flag);
    commit(BAR(B_DRAIN));
    __syncwarp();
  } else {
    // ---------------- softmax: thread = row ----------------
    const int r = tid;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL, o_addr = tmem + lanes + O_COL;
    const uint64_t c2 = f2_pack(a.c2, a.c2), lift2 = f2_pack(LIFT, LIFT);
    const int rows = maps.rows, boxes = TN / rows;
    bool ok = true;
    int sf[2] = {0, 0}, of[2] = {0, 0}, tile0 = 0, items = 0;  // score tiles taken from and products asked of each buffer; key tiles of earlier items
    walk<M>(a, near, [&](const Segment &g, int slot) {
      if (!ok) return;
      ++items;
      const Row x = row_of(a, g, r);
      {  // the warp's rows of queries, neighbouring lanes along a row; the last products on the tile are done
        constexpr int VEC = C::FULL * 8, AT = 32 / VEC;  // 16-byte vectors of a row, rows at a time
        const int64_t mine = x.j >= 0 ? q_at(a, g, x, g.hk) : -1;
        const int c = lane % VEC;
#pragma unroll 1
        for (int i0 = 0; i0 < VEC; i0 += 8) {
          uint4 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int64_t at = __shfl_sync(0xffffffffu, mine, (i0 + i) * AT + lane / VEC);
            v[i] = at >= 0 && c * 8 < a.c.D ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + at + c * 8) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = warp * 32 + (i0 + i) * AT + lane / VEC;
            *reinterpret_cast<uint4 *>(gen + (c >> 3) * BLK + row * 128 + (((c & 7) ^ (row & 7)) * 16)) = v[i];
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(BAR(B_QF));
      }
      const bool any_rows = warp * 32 < g.rows;
      const int n = g.k1 - g.k0;
      const int shared = a.mask ? 0 : g.row0 / a.G + 1;  // new tokens that every row sees
      float ref = -INFINITY, sum = 0.f;
      for (int i = 0; i < n; ++i) {
        const int k0 = (g.k0 + i) * TN, s = i & 1;
        // which of the tile's pages there are
        uint64_t missing = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int box = lane + 32 * u, key = k0 + box * rows, page = box < boxes ? page_of(a, g, key) : 0;
          missing |= (uint64_t)__ballot_sync(0xffffffffu, box < boxes && key < g.keys && (page < 0 || page >= a.c.pages)) << (32 * u);
        }
        if (!wait_warp_parity(BAR(B_SF + s), (uint32_t)sf[s] & 1u, abort_flag)) { ok = false; break; }
        ++sf[s];
        tc_fence_after();
        if (any_rows) {
          uint32_t w[2][32];
          tmem_ld32_nowait(s_addr + s * 64u, w[0]);
          tmem_ld32_nowait(s_addr + s * 64u + 32u, w[1]);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(w[q][e]));  // not read before the wait
          bool some = true;
          if (missing || k0 + TN > g.s.len || k0 + TN > g.keys) {
            some = false;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t seen = x.j >= 0 ? seen_columns(a, g, x, k0 + q * 32) : 0u;
              if (missing) {
#pragma unroll 1
                for (int e = 0; e < 32; ++e)
                  if ((missing >> ((q * 32 + e) / rows)) & 1) seen &= ~(1u << e);
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
            for (int q = 0; q < 2; ++q) m[2 * q + (e & 1)] = fmaxf(m[2 * q + (e & 1)], __uint_as_float(w[q][e]));
          const float top = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), some ? -FLT_MAX : -INFINITY);
          const bool grow = (top - ref) * a.c2 > LAZY;  // both -inf: NaN, no
          if (__any_sync(0xffffffffu, grow)) {
            const float next = grow ? top : ref;
            const float fix = grow ? factor(ref, next, a.c2) : 1.f;  // 0 for the first visible keys
            ref = next;
            sum *= fix;
            if (i > 0) {  // O holds the earlier tiles' sum, once their product is done
              if (!wait_warp_parity(BAR(B_OF + (s ^ 1)), (uint32_t)(of[s ^ 1] - 1) & 1u, abort_flag)) { ok = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int d = 0; d < DP; d += 16) {  // in pieces that leave the scores in their registers
                uint32_t o[16];
                tmem_ld16u(o_addr + d, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
                tmem_st16(o_addr + d, o);
              }
              tmem_wait_st();
            }
          }
          const float off = ref == -INFINITY ? 0.f : -ref;
          const uint64_t off2 = f2_pack(off, off);
          uint64_t acc[2] = {0ull, 0ull};
          uint32_t p[32];
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float y, z;
              f2_unpack(f2_fma(f2_add(f2_pack(__uint_as_float(w[q][e]), __uint_as_float(w[q][e + 1])), off2), c2, lift2), y, z);
              y = ex2(y);
              z = ex2(z);
              acc[q] = f2_add(acc[q], f2_pack(y, z));
              p[q * 16 + (e >> 1)] = pack2<T>(y, z);
            }
          tmem_st32(s_addr + s * 64u, p);
          tmem_wait_st();
          float y, z;
          f2_unpack(f2_add(acc[0], acc[1]), y, z);
          sum += y + z;
        }
        const bool fresh = k0 + TN - g.s.len > shared;  // V that not every row sees
        if (missing || fresh || k0 + TN > g.keys) {  // thread r looks after half of V's row r / 2
          const int tile = tile0 + i, st = tile % ST, vr = r >> 1, at = k0 + vr;
          if (!wait_warp_parity(BAR(B_VF + st), (uint32_t)(tile / ST) & 1u, abort_flag)) { ok = false; break; }
          const bool gone = at >= g.keys || ((missing >> (vr / rows)) & 1);
          if (gone || (fresh && at - g.s.len >= shared)) {
            uint8_t *row = gen + (vs - base) + st * C::TILE + vr * 128;
#pragma unroll
            for (int c = 0; c < C::FULL * 4; ++c) {
              uint4 *v = reinterpret_cast<uint4 *>(row + (c >> 2) * KBLK + ((((c & 3) * 2 + (r & 1)) + (lane & ~1)) & 7) * 16);
              const uint4 y = *v;
              const uint4 z = gone ? make_uint4(0u, 0u, 0u, 0u)
                                   : make_uint4(finite_pair<T>(y.x), finite_pair<T>(y.y), finite_pair<T>(y.z), finite_pair<T>(y.w));
              if (z.x != y.x || z.y != y.y || z.z != y.z || z.w != y.w) {
                *v = z;
                if (!gone) odd_item = items;
              }
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        mbar_arrive(BAR(B_PF + s));
        ++of[s];
      }
      if (!ok) return;
      tile0 += n;
      const int last = (n - 1) & 1;
      if (!wait_warp_parity(BAR(B_OF + last), (uint32_t)(of[last] - 1) & 1u, abort_flag)) { ok = false; return; }
      tc_fence_after();
      if (any_rows) {
        float scale = 1.f;
        if (slot < 0) scale = ref == -INFINITY ? 0.f : 1.f / sum;
        else if (x.j >= 0) a.part_ml[(int64_t)slot * M + r] = make_float2(ref, sum);
        // 32 columns at a time through the place of the warp's queries, so that neighbouring lanes write along a row
        const int64_t mine = x.j < 0 ? -1 : slot >= 0 ? ((int64_t)slot * M + r) * DP : out_at(a, g, x, g.hk);
        float4 *hold = reinterpret_cast<float4 *>(gen + warp * 4096);
#pragma unroll 1
        for (int d = 0; d < DP; d += 32) {  // (what runs once for an item is kept short: its instructions come from far)
          uint32_t o[32];
          tmem_ld32u(o_addr + d, o);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            hold[lane * 8 + (e ^ (lane & 7))] = make_float4(__uint_as_float(o[4 * e]) * scale, __uint_as_float(o[4 * e + 1]) * scale,
                                                            __uint_as_float(o[4 * e + 2]) * scale, __uint_as_float(o[4 * e + 3]) * scale);
          __syncwarp();
#pragma unroll 2
          for (int i = 0; i < 8; ++i) {
            const int row = 4 * i + (lane >> 3), e = lane & 7;
            const int64_t at = __shfl_sync(0xffffffffu, mine, row);
            const float4 y = hold[row * 8 + (e ^ (row & 7))];
            if (at < 0 || d + 4 * e >= a.c.D) continue;
            if (slot >= 0) *reinterpret_cast<float4 *>(a.part_o + at + d + 4 * e) = y;
            else *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + at + d + 4 * e) = make_uint2(pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      // (the next item's is set only after all have come to its queries)
      if (odd_item == items && x.j >= 0) {  // a row adds what it sees of the infinities and NaN that were taken out of V
        const int first = max(g.s.len + shared, g.k0 * TN), end = min(min(g.keys, g.k1 * TN), g.s.len + (a.mask ? 64 : x.j + 1));
        for (int key = first; key < end; ++key) {
          const int page = page_of(a, g, key);
          if (!sees(a.mask != nullptr, x.bits, x.j, key - g.s.len) || page < 0 || page >= a.c.pages) continue;
          const T *v = static_cast<const T *>(a.c.values) + page * a.c.vp + (key - cache::page_index(a.c, key) * a.c.size) * a.c.vs +
                       g.hk * a.c.vh;
          for (int d = 0; d < a.c.D; d += 8) {
            const uint4 y = *reinterpret_cast<const uint4 *>(v + d);
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint16_t bits = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
              if (finite16<T>(bits)) continue;
              const float add = to_f(*reinterpret_cast<const T *>(&bits));
              if (slot >= 0) {
                a.part_o[((int64_t)slot * M + r) * DP + d + e] += add;
              } else {
                T *out = static_cast<T *>(a.out) + out_at(a, g, x, g.hk) + d + e;
                *out = from_f<T>(to_f(*out) + add);
              }
            }
          }
        }
      }
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
    walk<M>(a, near, [&](const Segment &g, int slot) {
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
bool make_map(CUtensorMap *map, const mhc_kv_cache *c, void *p, const Axes &x, cuuint32_t rows) {
  auto enc = encode_fn();
  if (!enc) return false;
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
  return launch_early(kern, dim3((unsigned)a.pieces), NTHREADS, C::SMEM, stream, maps, a);
}

}  // namespace
}  // namespace cattn

// What TMA asks of the cache: rows of 16-byte multiples that do not overlap.
bool cached_attn_tc_eligible(const mhc_kv_cache *c) {
  if (c->dtype == MHC_F32 || c->dim % 8 || (uintptr_t)c->keys % 16 || (uintptr_t)c->values % 16) return false;
  return cattn::axes_ok(c, cattn::axes_of(c, c->strides)) && cattn::axes_ok(c, cattn::axes_of(c, c->strides + 4));
}

cudaError_t launch_cached_attn_tc(const cattn::Args &a, const mhc_kv_cache *c, cudaStream_t stream) {
  cattn::Maps maps;
  const cattn::Axes k = cattn::axes_of(c, c->strides), v = cattn::axes_of(c, c->strides + 4);
  maps.rows = cached_attn_tc_box(c);
  if (!cattn::make_map(&maps.k, c, c->keys, k, maps.rows) || !cattn::make_map(&maps.v, c, c->values, v, maps.rows)) return cudaErrorNotSupported;
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
