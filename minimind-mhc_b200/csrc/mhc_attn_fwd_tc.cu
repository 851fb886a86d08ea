// Forward of causal attention over packed sequences on the 5th-generation tensor
// cores (bf16 / fp16, head sizes that are multiples of 8 up to 128).
//
// A block works on two tiles of 128 queries at once: two heads that share their
// keys where a group has an even number of heads, else two neighbouring tiles of
// one head.  Both read the same 128-key tiles of K and V, streamed by TMA, and take
// turns: while one tile's scores go through the softmax, the tensor core forms the
// other's products.
//
//   S = Q K^T       tcgen05.mma, M = N = 128, K = D, both operands in shared memory
//   P = exp2(S c - m)                      c = scale log2(e), one thread per row
//   O += P V        A = P from TMEM (it replaces S there), B = V as it lies in memory
//                   (its rows are the summed index: an MN-major operand)
//
// m is a row's reference, not its exact running maximum: it is moved, and O and the
// row's sum rescaled, only when the maximum has grown past it by more than 2^8.
// That is rare after the first tiles, exact in the end (the reference cancels), and
// keeps O in TMEM from start to end.  The row sum is of the fp32 P.  m is kept as a
// score, before its scaling: P = exp2(fma(S, c, -round(m c))) leaves the rounding of m c
// in every P of the row, where it cancels, but it is an exponent that grows with m.
// Rows with |m c| above 2^10 (a part in 2^14 there) are subtracted first and scaled
// then, one more addition a score.
//
// Which keys a row sees is decided per row (its sequence's start, itself), so one
// tile may hold many short sequences: the number of tiles depends on T only, and
// the lengths stay on the device.  Only tiles that cross a start or the diagonal
// compare indices.
//
// The grid is one block per SM and walks the tiles in the order of their work
// (attn_order_kernel), forwards and backwards in turn.  Warps 0-3 and 4-7: the two
// tiles' softmax and epilogue; 8: TMA; 9: MMA issue.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "mhc_attn_redo.cuh"
#include "mhc_attn_tc.cuh"

namespace mhc {

__device__ int g_atf_error = 0;

namespace attn {

namespace {

constexpr int NTHREADS = 320;
constexpr int W_TMA = 8, W_MMA = 9;
constexpr int TMEM_COLS = 512;
constexpr uint32_t S_COL = 0, O_COL = 256;  // two score tiles, two results, 128 columns each
constexpr float LAZY = 8.f;                 // a row's reference may lag its maximum by 2^8
constexpr float FAR = 1024.f;               // scaled references beyond it are subtracted before the scaling

enum { ERR_TMA = 41, ERR_MMA = 42, ERR_SOFTMAX = 43 };

// one piece of work, published by the TMA warp
struct Item {
  int q0[2], head[2];  // q0 < 0: no such tile
  int k0;              // first key of the first tile
  int first[2], last[2];  // each tile's steps [first, last) of the n
  int n;
  int kv_head;
  int done;
};

template <int DP>
struct Cfg {
  using L = Tile<DP, false>;
  static constexpr uint32_t TILE = L::BYTES;
  static constexpr int ST = DP <= 64 ? 4 : 2;  // stages of K and of V
};

constexpr int B_ITEM_F = 0, B_ITEM_E = 2, B_QF = 4, B_QE = 5, B_LAND = 6, B_SF = 7, B_PF = 9, B_OF = 11, B_DRAIN = 13,
              B_KF = 14;
// then ST each: KF, KE, VF, VE

struct Sched {
  const int *order;  // null: last tile first
  int tiles, pairs, by_head, items;
};

__device__ __forceinline__ void give_up(int code, volatile int *abort_flag, int *err_flag) {
  *abort_flag = 1;
  report_give_up(&g_atf_error, err_flag, code);
}

__device__ __forceinline__ bool item_of(const Args &a, const Sched &s, int64_t rank, Item &it) {
  if (rank >= s.items) {
    it.done = 1;
    return false;
  }
  it.done = 0;
  const int at = (int)(rank / s.pairs), p = (int)(rank % s.pairs);
  const int G = a.H / a.Hk;
  if (s.by_head) {
    const int tile = s.order ? s.order[at] : s.tiles - 1 - at;
    it.q0[0] = it.q0[1] = tile * TM;
    it.head[0] = 2 * p;
    it.head[1] = 2 * p + 1;
  } else {
    const int n2 = (s.tiles + 1) / 2;
    const int tile = 2 * (s.order ? s.order[at] : n2 - 1 - at);
    it.q0[0] = tile * TM;
    it.q0[1] = tile + 1 < s.tiles ? (tile + 1) * TM : -1;
    it.head[0] = it.head[1] = p;
  }
  it.kv_head = it.head[0] / G;
  it.k0 = 0;
  int lo[2], hi[2];
  int k_lo = 0x7fffffff, k_hi = 0;
  for (int t = 0; t < 2; ++t) {
    lo[t] = hi[t] = 0;
    if (it.q0[t] < 0) continue;
    const int first = span_of(a, it.q0[t]).start, end = (int)min((int64_t)it.q0[t] + TM, a.T);
    if (first >= end) continue;
    lo[t] = first / TM;
    hi[t] = it.q0[t] / TM + 1;
    k_lo = min(k_lo, lo[t]);
    k_hi = max(k_hi, hi[t]);
  }
  it.n = k_hi > k_lo ? k_hi - k_lo : 0;
  if (it.n == 0) k_lo = 0;
  it.k0 = k_lo * TM;
  for (int t = 0; t < 2; ++t) {
    it.first[t] = hi[t] > lo[t] ? lo[t] - k_lo : 0;
    it.last[t] = hi[t] > lo[t] ? hi[t] - k_lo : 0;
  }
  return true;
}

template <typename T, int DP>
__global__ void __launch_bounds__(NTHREADS, 1)
attn_fwd_tc_kernel(const __grid_constant__ Map qmap, const __grid_constant__ Map kmap, const __grid_constant__ Map vmap,
                   const __grid_constant__ Args a, const Sched sched) {
  using C = Cfg<DP>;
  using L = typename C::L;
  constexpr int ST = C::ST;
  constexpr int B_KE = B_KF + ST, B_VF = B_KE + ST, B_VE = B_VF + ST, NBARS = B_VE + ST;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Item items[2];
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, redo_word;  // redo: a NaN has been written
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - raw);
  const uint32_t qs = base, ks = qs + 2 * C::TILE, vs = ks + ST * C::TILE;
  volatile int *abort_flag = &abort_word;
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  if (tid == 0) {
    abort_word = redo_word = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_ITEM_F + i), 1);
      mbar_init(BAR(B_ITEM_E + i), 257);  // the softmax threads and the MMA thread have read it
      mbar_init(BAR(B_SF + i), 1);
      mbar_init(BAR(B_PF + i), 128);
      mbar_init(BAR(B_OF + i), 1);
    }
    mbar_init(BAR(B_QF), 1);
    mbar_init(BAR(B_QE), 1);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);
  grid_dep_launch();
  grid_dep_wait();

  if (warp == W_TMA) {
    // ---------------- TMA: whole warp, lane 0 issues ----------------
    const Span range = packed_range(a);
    bool ok = true;
    int g = 0, lands = 0, qn = 0;  // key tiles, tiles cleaned, query pairs loaded so far
    for (int i = 0; ok; ++i) {
      Item it;
      const bool live = item_of(a, sched, snake(i, blockIdx.x, gridDim.x), it);
      if (!wait_warp_parity(BAR(B_ITEM_E + (i & 1)), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
      if (lane == 0) {
        items[i & 1] = it;
        mbar_arrive(BAR(B_ITEM_F + (i & 1)));
      }
      __syncwarp();
      if (!live) break;
      if (it.n == 0) continue;
      if (!wait_warp_parity(BAR(B_QE), ((uint32_t)qn & 1u) ^ 1u, abort_flag)) { ok = false; break; }
      ++qn;
      if (lane == 0) {
        mbar_arrive_expect_tx(BAR(B_QF), 2 * C::TILE);
        load_rows<L>(qs, qmap, it.head[0], it.q0[0], BAR(B_QF));
        // without a second tile the first is loaded twice: the products of its copy are not used
        load_rows<L>(qs + C::TILE, qmap, it.head[1], it.q0[1] < 0 ? it.q0[0] : it.q0[1], BAR(B_QF));
      }
      for (int j = 0; j < it.n && ok; ++j, ++g) {
        const int s = g % ST;
        const uint32_t free_par = ((uint32_t)(g / ST) & 1u) ^ 1u;
        const int row = it.k0 + j * TM;
        if (!wait_warp_parity(BAR(B_KE + s), free_par, abort_flag)) { ok = false; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(BAR(B_KF + s), C::TILE);
          load_rows<L>(ks + s * C::TILE, kmap, it.kv_head, row, BAR(B_KF + s));
        }
        if (!wait_warp_parity(BAR(B_VE + s), free_par, abort_flag)) { ok = false; break; }
        const bool clean = row < range.start || min((int64_t)row + TM, a.T) > range.end;
        if (lane == 0) {
          mbar_arrive_expect_tx(BAR(clean ? B_LAND : B_VF + s), C::TILE);
          load_rows<L>(vs + s * C::TILE, vmap, it.kv_head, row, BAR(clean ? B_LAND : B_VF + s));
        }
        __syncwarp();
        if (clean) {
          if (!wait_warp_parity(BAR(B_LAND), (uint32_t)lands & 1u, abort_flag)) ok = false;
          ++lands;
          zero_outside<L>(gen + (vs - base) + s * C::TILE, row, range, lane);
          if (lane == 0) mbar_arrive(BAR(B_VF + s));
        }
      }
    }
    if (!ok && lane == 0) give_up(ERR_TMA, abort_flag, a.err_flag);
    // copies in flight land before the block may exit
    for (int p = g > ST ? g - ST : 0; p < g; ++p) {
      wait_parity<false>(BAR(B_KF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
      wait_parity<false>(BAR(B_VF + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
    }
    if (qn > 0) wait_parity<false>(BAR(B_QF), (uint32_t)(qn - 1) & 1u, nullptr);
  } else if (warp == W_MMA) {
    // ---------------- MMA issue: the warp runs it, one lane issues ----------------
    {
      constexpr uint32_t id_s = idesc_of<T>(128, 0), id_o = idesc_of<T>(L::N_FULL, 1), id_t = idesc_of<T>(32, 1);
      bool ok = true;
      auto wait_warp = [&](uint32_t bar, uint32_t par) { return wait_warp_parity(bar, par, abort_flag); };
      auto commit = [&](uint32_t bar) {
        if (elect_one()) umma_commit(bar);
      };
      int i = 0, qn = 0, gk = 0, pf[2] = {0, 0};
      struct Step {
        int j, n, first[2], last[2], g;
      } cur, nxt;
      // the next step after (j, n) of the current item, or of the next item that has any
      auto advance = [&](Step &s) -> bool {
        if (s.j + 1 < s.n) {
          ++s.j;
        } else {
          while (true) {
            if (!wait_warp(BAR(B_ITEM_F + (i & 1)), (uint32_t)(i >> 1) & 1u)) { ok = false; return false; }
            const Item &it = items[i & 1];
            const bool done = uniform(it.done);
            s.j = 0;
            s.n = uniform(it.n);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              s.first[t] = uniform(it.first[t]);
              s.last[t] = uniform(it.last[t]);
            }
            if (elect_one()) mbar_arrive(BAR(B_ITEM_E + (i & 1)));
            ++i;
            if (done) return false;
            if (s.n > 0) break;
          }
          if (!wait_warp(BAR(B_QF), (uint32_t)qn & 1u)) { ok = false; return false; }
          ++qn;
        }
        s.g = gk++;
        return true;
      };
      auto scores = [&](const Step &s, int t) {
        if (s.j < s.first[t] || s.j >= s.last[t]) return;
        mma_rows<L>(tmem + S_COL + t * 128u, qs + t * C::TILE, ks + (s.g % ST) * C::TILE, id_s);
        commit(BAR(B_SF + t));
      };
      auto after_scores = [&](const Step &s) {
        commit(BAR(B_KE + s.g % ST));
        if (s.j == s.n - 1) commit(BAR(B_QE));
      };
      auto wait_k = [&](const Step &s) {
        if (!wait_warp(BAR(B_KF + s.g % ST), (uint32_t)(s.g / ST) & 1u)) ok = false;
        tc_fence_after();
      };
      cur.j = cur.n = 0;
      bool have = advance(cur);
      if (have && ok) {
        wait_k(cur);
        if (ok) {
          scores(cur, 0);
          scores(cur, 1);
          after_scores(cur);
        }
      }
      auto product = [&](const Step &s, int t) {
        if (s.j < s.first[t] || s.j >= s.last[t]) return;
        if (!wait_warp(BAR(B_PF + t), (uint32_t)pf[t] & 1u)) { ok = false; return; }
        ++pf[t];
        tc_fence_after();
        mma_sum<L>(tmem + O_COL + t * 128u, tmem + S_COL + t * 128u, 16u, vs + (s.g % ST) * C::TILE, id_o, id_t, s.j == s.first[t]);
        commit(BAR(B_OF + t));
      };
      // tile 0's product, its next scores, then the same for tile 1: each tile's softmax runs beside the other's
      // products.  S of the next step may follow P V of this one at once: the tensor core runs them in order.
      while (have && ok) {
        nxt = cur;
        const bool same_item = cur.j + 1 < cur.n;
        bool more = same_item && advance(nxt);
        if (!wait_warp(BAR(B_VF + cur.g % ST), (uint32_t)(cur.g / ST) & 1u)) { ok = false; break; }
        if (more) wait_k(nxt);
        if (!ok) break;
        product(cur, 0);
        if (!ok) break;
        if (more) scores(nxt, 0);
        product(cur, 1);
        if (!ok) break;
        commit(BAR(B_VE + cur.g % ST));
        if (!same_item) {  // the next item's queries may still be on their way
          more = advance(nxt);
          if (!ok) break;
          if (more) wait_k(nxt);
          if (!ok) break;
          if (more) scores(nxt, 0);
        }
        if (more) {
          scores(nxt, 1);
          after_scores(nxt);
        }
        cur = nxt;
        have = more;
      }
      if (!ok && lane == 0) give_up(ERR_MMA, abort_flag, a.err_flag);
      commit(BAR(B_DRAIN));
    }
    __syncwarp();
  } else {
    // ---------------- softmax: thread = row of tile t ----------------
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL + t * 128u, o_addr = tmem + lanes + O_COL + t * 128u;
    const int row = (warp & 3) * 32 + lane;
    const float c = a.scale_log2;
    const uint64_t c2 = f2_pack(c, c);
    bool ok = true;
    int sf = 0, of = 0;
    for (int i = 0; ok; ++i) {
      if (!wait_warp_parity(BAR(B_ITEM_F + (i & 1)), (uint32_t)(i >> 1) & 1u, abort_flag)) { ok = false; break; }
      const int q0 = items[i & 1].q0[t], head = items[i & 1].head[t], first = items[i & 1].first[t], last = items[i & 1].last[t];
      const int k00 = items[i & 1].k0, done = items[i & 1].done;
      mbar_arrive(BAR(B_ITEM_E + (i & 1)));
      if (done) break;
      if (q0 < 0) continue;
      const int tok = q0 + row;
      const int start = tok < a.T ? span_of(a, tok).start : tok + 1;
      float ref = -INFINITY, sum = 0.f;
      for (int j = first; j < last; ++j) {
        const int k0 = k00 + j * TM;
        if (!wait_warp_parity(BAR(B_SF + t), (uint32_t)sf & 1u, abort_flag)) { ok = false; break; }
        ++sf;
        tc_fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32_nowait(s_addr + q * 32, r[q]);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(r[q][e]));  // not read before the wait
        if (__any_sync(0xffffffffu, k0 < start || k0 + TM - 1 > tok)) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t seen = bits_between(start - k0 - q * 32, tok + 1 - k0 - q * 32);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen & (1u << e))) r[q][e] = 0xff800000u;
          }
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; ++e)
#pragma unroll
          for (int q = 0; q < 4; ++q) m[q] = fmaxf(m[q], __uint_as_float(r[q][e]));
        const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        const bool grow = (top - ref) * c > LAZY;  // both -inf or both inf: NaN, no
        if (__any_sync(0xffffffffu, grow)) {
          const float next = grow ? top : ref;
          const float fix = grow ? exp2_approx((ref - next) * c) : 1.f;  // 0 for the first visible keys
          ref = next;
          sum *= fix;
          if (j > first) {  // O holds the earlier tiles' sum, once their product is done
            if (!wait_warp_parity(BAR(B_OF + t), (uint32_t)(of - 1) & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
            // in pieces that leave the scores in their registers
#pragma unroll
            for (int d = 0; d < DP; d += 16) {
              uint32_t o[16];
              tmem_ld16u(o_addr + d, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
              tmem_st16(o_addr + d, o);
            }
            tmem_wait_st();
          }
        }
        float neg = ref == -INFINITY ? 0.f : -ref * c;
        const bool far = fabsf(neg) > FAR;
        if (__any_sync(0xffffffffu, far)) {
          const float off = far ? ref : 0.f;
          neg = far ? 0.f : neg;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 32; ++e) r[q][e] = __float_as_uint(__uint_as_float(r[q][e]) - off);
        }
        const uint64_t n2 = f2_pack(neg, neg);
        uint64_t acc[2] = {0ull, 0ull};
        uint32_t p[2][32];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x, y;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(r[q][e]), __uint_as_float(r[q][e + 1])), c2, n2), x, y);
            x = exp2_approx(x);
            y = exp2_approx(y);
            acc[(e >> 1) & 1] = f2_add(acc[(e >> 1) & 1], f2_pack(x, y));
            p[q >> 1][(q & 1) * 16 + (e >> 1)] = pack2<T>(x, y);
          }
        tmem_st32(s_addr, p[0]);
        tmem_st32(s_addr + 32, p[1]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(BAR(B_PF + t));
        ++of;
        float x, y;
        f2_unpack(f2_add(acc[0], acc[1]), x, y);
        sum += x + y;
      }
      if (!ok) break;
      const bool seen = last > first;
      if (seen) {
        if (!wait_warp_parity(BAR(B_OF + t), (uint32_t)(of - 1) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (tok < a.T) a.lse[(int64_t)head * a.Tp + tok] = sum == 0.f ? INFINITY : ref * c + log2f(sum);
      bool bad = false;
      const int64_t at = ((int64_t)tok * a.H + head) * a.D;
      T *out = static_cast<T *>(a.o) + at, *lo = a.o_lo ? static_cast<T *>(a.o_lo) + at : nullptr;
#pragma unroll
      for (int d = 0; d < DP; d += 16) {
        uint32_t o[16];
        if (seen) {
          tmem_ld16u(o_addr + d, o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0u;
        }
        uint32_t w[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __uint_as_float(o[2 * e]) * inv, y = __uint_as_float(o[2 * e + 1]) * inv;
          bad |= isnan(x) || isnan(y);
          w[e] = pack2<T>(x, y);
          const float2 back = unpack2<T>(w[e]);
          l[e] = pack2<T>(x - back.x, y - back.y);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (tok < a.T && d + h * 8 < a.D) {  // D is a multiple of 8
            *reinterpret_cast<uint4 *>(out + d + h * 8) = make_uint4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3]);
            if (lo) *reinterpret_cast<uint4 *>(lo + d + h * 8) = make_uint4(l[h * 4], l[h * 4 + 1], l[h * 4 + 2], l[h * 4 + 3]);
          }
      }
      if (bad && tok < a.T) redo_word = 1;
      tc_fence_before();
    }
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
    for (int i = 0;; ++i) {
      Item it;
      if (!item_of(a, sched, snake(i, blockIdx.x, gridDim.x), it)) break;
      for (int t = 0; t < 2; ++t)
        for (int e = tid; it.q0[t] >= 0 && e < TM * a.D; e += NTHREADS) {
          const int64_t tok = it.q0[t] + e / a.D;
          if (tok < a.T) static_cast<T *>(a.o)[(tok * a.H + it.head[t]) * a.D + e % a.D] = bad;
        }
    }
  } else if (redo_word) {
    for (int i = 0;; ++i) {
      Item it;
      if (!item_of(a, sched, snake(i, blockIdx.x, gridDim.x), it)) break;
      for (int t = 0; t < 2; ++t)
        if (it.q0[t] >= 0) redo_out_rows<T>(a, it.head[t], it.q0[t], TM, warp, NTHREADS / 32, lane);
    }
  }
#undef BAR
}

template <typename T, int DP>
cudaError_t run(const Args &a, const Map &q, const Map &k, const Map &v, const Sched &s, int grid, cudaStream_t stream) {
  using C = Cfg<DP>;
  constexpr size_t smem = 2 * C::TILE + 2 * C::ST * C::TILE + 1024;
  auto kern = attn_fwd_tc_kernel<T, DP>;
  static std::mutex mu;
  static bool done[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !done[dev]) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess) return e;
      if (dev < 64) done[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(NTHREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  e = cudaLaunchKernelEx(&cfg, kern, q, k, v, a, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Counting sort of the tiles by work, largest first, one block each for queries (by
// the keys they see) and keys (by the queries that see them).  Equal bins come
// out in any order: the order decides who computes a tile, not what comes out.
constexpr int BINS = 1024;
__global__ void __launch_bounds__(BINS) attn_order_kernel(const Args a, int step, int tiles, int *order_q, int *order_k) {
  const int keys = blockIdx.x;  // 0: tiles of queries, 1: of keys
  int *order = keys ? order_k : order_q;
  __shared__ int hist[BINS], warps[32], most;
  const int tid = threadIdx.x;
  hist[tid] = 0;
  if (tid == 0) most = 0;
  __syncthreads();
  const int last_token = (int)a.T - 1;
  auto work = [&](int i) {
    const int r0 = i * step * TM, r1 = min(r0 + step * TM - 1, last_token);
    const int w = keys ? span_of(a, r1).end - r0 : r1 + 1 - span_of(a, r0).start;
    return max(0, w + TM - 1) / TM;
  };
  int mine = 0;
  for (int i = tid; i < tiles; i += BINS) mine = max(mine, work(i));
  atomicMax(&most, mine);
  __syncthreads();
  const int top = max(1, most);
  auto bin = [&](int i) { return BINS - 1 - (int)((int64_t)work(i) * (BINS - 1) / top); };  // largest first
  for (int i = tid; i < tiles; i += BINS) atomicAdd(&hist[bin(i)], 1);
  __syncthreads();
  const int mycount = hist[tid];
  int x = mycount;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if ((tid & 31) >= o) x += y;
  }
  if ((tid & 31) == 31) warps[tid >> 5] = x;
  __syncthreads();
  if (tid < 32) {
    int w = warps[tid];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (tid >= o) w += y;
    }
    warps[tid] = w;
  }
  __syncthreads();
  hist[tid] = x - mycount + (tid >= 32 ? warps[(tid >> 5) - 1] : 0);
  __syncthreads();
  for (int i = tid; i < tiles; i += BINS) order[atomicAdd(&hist[bin(i)], 1)] = i;
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

}  // namespace

bool map_eligible(const void *p, int D, int heads, int64_t T, int64_t ts, int64_t hs) {
  if (((uintptr_t)p & 15) || D % 8 || ts % 8 || hs % 8) return false;
  if ((T > 1 && ts < D) || (heads > 1 && hs < D)) return false;  // rows that overlap (broadcast heads or tokens)
  return ts < ((int64_t)1 << 38) && hs < ((int64_t)1 << 38);
}

bool make_map(Map &map, const void *p, int dtype, int64_t T, int heads, int D, int64_t ts, int64_t hs) {
  auto enc = encode_fn();
  if (!enc || !map_eligible(p, D, heads, T, ts, hs)) return false;
  if (T == 1 && ts < D) ts = D;  // an axis of one element may come with any stride
  if (heads == 1 && hs < D) hs = D;
  map.token_first = heads > 1 && hs > ts;
  const bool f = map.token_first != 0;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)(f ? T : heads), (cuuint64_t)(f ? heads : T)};
  const cuuint64_t strides[2] = {(cuuint64_t)(f ? ts : hs) * 2, (cuuint64_t)(f ? hs : ts) * 2};
  const cuuint32_t estr[3] = {1, 1, 1};
  for (int tail = 0; tail < 2; ++tail) {
    const cuuint32_t box[3] = {tail ? 32u : 64u, (cuuint32_t)(f ? TM : 1), (cuuint32_t)(f ? 1 : TM)};
    if (enc(tail ? &map.t : &map.m, dtype == MHC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void *>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            tail ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

}  // namespace attn

size_t attn_order_bytes(int64_t T) { return (size_t)((T + attn::TM - 1) / attn::TM) * 4; }

cudaError_t launch_attn_orders(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream) {
  const int tiles = (int)((a.T + attn::TM - 1) / attn::TM);
  attn::attn_order_kernel<<<order_k ? 2 : 1, attn::BINS, 0, stream>>>(a, 1, tiles, order_q, order_k);
  return cudaGetLastError();
}

bool attn_tc_eligible(const attn::Args &a) {
  if (a.dtype != MHC_BF16 && a.dtype != MHC_F16) return false;
  if (((uintptr_t)a.o | (uintptr_t)a.o_lo) & 15) return false;
  return attn::map_eligible(a.q, a.D, a.H, a.T, a.qt, a.qh) && attn::map_eligible(a.k, a.D, a.Hk, a.T, a.kt, a.kh) &&
         attn::map_eligible(a.v, a.D, a.Hk, a.T, a.vt, a.vh);
}

bool attn_tc_bwd_eligible(const attn::Args &a) {
  if (((uintptr_t)a.dout | (uintptr_t)a.dq | (uintptr_t)a.dk | (uintptr_t)a.dv | (uintptr_t)a.lse) & 15) return false;
  return attn_tc_eligible(a);
}

cudaError_t launch_attn_fwd_tc(const attn::Args &a, int *order, cudaStream_t stream) {
  attn::Map q, k, v;
  if (!attn::make_map(q, a.q, a.dtype, a.T, a.H, a.D, a.qt, a.qh) || !attn::make_map(k, a.k, a.dtype, a.T, a.Hk, a.D, a.kt, a.kh) ||
      !attn::make_map(v, a.v, a.dtype, a.T, a.Hk, a.D, a.vt, a.vh))
    return cudaErrorNotSupported;
  attn::Sched s;
  s.tiles = (int)((a.T + attn::TM - 1) / attn::TM);
  s.by_head = (a.H / a.Hk) % 2 == 0;
  s.pairs = s.by_head ? a.H / 2 : a.H;
  const int rows = s.by_head ? s.tiles : (s.tiles + 1) / 2;
  if ((int64_t)rows * s.pairs > 0x7fffffff) return cudaErrorNotSupported;
  s.items = rows * s.pairs;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  s.order = nullptr;
  // with a block for every piece of work their order does not matter
  if (s.items > sms && order) {
    attn::attn_order_kernel<<<1, attn::BINS, 0, stream>>>(a, s.by_head ? 1 : 2, rows, order, nullptr);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    s.order = order;
  }
  const int grid = s.items < sms ? s.items : sms;
  auto go = [&](auto tag) -> cudaError_t {
    using T = decltype(tag);
    if (a.D <= 32) return attn::run<T, 32>(a, q, k, v, s, grid, stream);
    if (a.D <= 64) return attn::run<T, 64>(a, q, k, v, s, grid, stream);
    if (a.D <= 96) return attn::run<T, 96>(a, q, k, v, s, grid, stream);
    return attn::run<T, 128>(a, q, k, v, s, grid, stream);
  };
  return a.dtype == MHC_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

int read_atf_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_atf_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_atf_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mhc
