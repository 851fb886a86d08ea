// Backward of causal attention over packed sequences on the 5th-generation tensor
// cores (bf16 / fp16, head sizes that are multiples of 8 up to 128).
//
// Two kernels of one form, each of which owns the rows of what it sums, so no two
// blocks add to the same gradient and every sum has a fixed order:
//
//   DKV: a block owns 128 keys of one key head and walks the queries that see them,
//        of every head of the group:       rows R1 = K, R2 = V, columns C1 = Q, C2 = dO
//          S = R1 C1^T, P = exp2(S c - lse_col);       dV += P C2
//          dP = R2 C2^T, dS = P (dP - D_col);          dK += dS C1
//   DQ:  a block owns 128 queries of one head and walks their keys:
//                                          rows R1 = Q, R2 = dO, columns C1 = K, C2 = V
//          S, P, dP, dS as above with lse and D of the row;   dQ += dS C1
//
// A sequence's first token sees itself only: its P is 1 whatever the score, and its dS
// is made the 0 that dP - D is but for the order of two sums.
//
// (seven products of 128 x 128 x D a tile where five would do if dQ were added up
// over blocks: two more on the tensor core instead of atomics in an order that
// changes).  P and dS never leave TMEM: a thread reads a quarter of a row of S, writes
// P as 16-bit values, which is the A operand of the next product, and dS over dP the
// same way; the column operands serve S and dP as they are (K-major) and the
// gradients as they lie (their rows are the summed index: MN-major).
//
// What bounds it is the chain of a step, not the tensor core (43 % busy) nor the 2^x
// (30 %): scores, their reading, 2^x, dS, each handed on through an mbarrier at 150 to
// 250 cycles.  So the tensor core is given S(j+1) as soon as S(j) has been read, where
// P has columns of its own, and dP(j+1) behind dK(j); and 16 warps, not 8, share the
// softmax, as a warp mostly waits on itself.  At 16384 tokens, D = 96, 8 over 4 heads:
// 8 warps 1.55 ms, 16 warps 1.38 ms, scores ahead and a third stage of tiles 1.30 to
// 1.37 ms (750 to 800 TFLOP/s, 0.46 to 0.49 of the measured peak); two halves of 64
// columns with barriers of their own, which overlap better on paper, 2.19 ms, since
// they double the hand-offs.
//
// fp16 has no room for small dS or P: P is held times 2^10, and dS times a power of
// two from the largest finite |dO| and |V| of its sequence that no dS can overflow
// (|dS| <= 2 D max|dO| max|V|); both come off in fp32 at the end.  bf16 needs
// neither.
//
// Grid, order of the work, masks and tokens outside of the sequences: as in the
// forward kernel.  Warps 0-15: softmax (four to each quarter of the rows, 32 columns
// each) and epilogue; 16: TMA; 17: MMA issue.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "mhc_attn_redo.cuh"
#include "mhc_attn_tc.cuh"

namespace mhc {

__device__ int g_atb_error = 0;

namespace attn {

namespace {

constexpr int NSOFT = 16;             // softmax warps: four to each quarter of the rows
constexpr int W_TMA = NSOFT, W_MMA = NSOFT + 1;
constexpr int NTHREADS = (NSOFT + 2) * 32;
constexpr int TMEM_COLS = 512;
// columns of TMEM: S; dP (two of them for DQ); the results; P
constexpr uint32_t S_COL = 0, DP_COL = 128, A1_COL = 256;
constexpr float P_SHIFT = 10.f;  // fp16: P times 2^10

enum { ERR_TMA = 51, ERR_MMA = 52, ERR_SOFTMAX = 53 };

struct Item {
  int r0, head;   // first row, row head (DKV: key head)
  int c_head;     // first column head
  int part;       // DKV: which of the blocks that share the keys
  int c0, cols;   // first column tile's first token, column tiles
  int n;          // steps: cols, times the group's heads for DKV
  int done;
};

template <int DP>
struct Cfg {
  using L = Tile<DP, true>;
  static constexpr uint32_t TILE = L::BYTES;
  static constexpr int ST = DP <= 64 ? 4 : (DP <= 96 ? 3 : 2);  // stages of C1 and of C2
  static constexpr uint32_t VEC = 2 * TM * 4;       // a stage's lse and D of its columns
  static constexpr uint32_t A2_COL = A1_COL + DP;   // dV
  static constexpr bool OWN_P = DP <= 96;           // P has 64 columns of its own; else it replaces S
  static constexpr uint32_t P_COL = OWN_P ? 448 : S_COL;
};

constexpr int B_ITEM_F = 0, B_ITEM_E = 2, B_RF = 4, B_RE = 5, B_LAND = 6, B_SF = 7, B_SE = 8, B_PF = 9, B_DPF = 10,
              B_DSF = 12, B_ACC_F = 14, B_DRAIN = 15, B_1F = 16;  // dP and dS: one for even steps, one for odd
// then ST each: 1F, 1E, 2F, 2E

struct Sched {
  const int *order;  // null: tile 0 first for keys, the last first for queries
  int tiles, heads, items;
};

__device__ __forceinline__ void give_up(int code, volatile int *abort_flag, int *err_flag) {
  *abort_flag = 1;
  report_give_up(&g_atb_error, err_flag, code);
}

template <bool DKV>
__device__ __forceinline__ bool item_of(const Args &a, const Sched &s, int64_t rank, Item &it) {
  if (rank >= s.items) {
    it.done = 1;
    it.n = 0;
    return false;
  }
  it.done = 0;
  const int at = (int)(rank / s.heads);
  const int p = (int)(rank % s.heads), G = a.H / a.Hk, per = DKV ? G / a.splits : 1;
  it.head = DKV ? p / a.splits : p;
  it.part = DKV ? p % a.splits : 0;
  it.c_head = DKV ? it.head * G + it.part * per : p / G;
  const int tile = s.order ? s.order[at] : (DKV ? at : s.tiles - 1 - at);
  it.r0 = tile * TM;
  const int r1 = (int)min((int64_t)it.r0 + TM, a.T) - 1;
  int lo, hi;  // column tiles
  if (DKV) {
    const int end = span_of(a, r1).end;
    lo = tile;
    hi = end > it.r0 ? (end - 1) / TM + 1 : tile;
  } else {
    const int first = span_of(a, it.r0).start;
    lo = first / TM;
    hi = first <= r1 ? tile + 1 : lo;
  }
  it.c0 = lo * TM;
  it.cols = hi - lo;
  it.n = it.cols * per;
  return true;
}

// fp16: the power of two that a token's row of dS is held times, from max|dO| and max|V| of its sequence
__device__ __forceinline__ float ds_factor(const Args &a, int tok, int start) {
  if (start > tok) return 1.f;  // outside of every sequence
  const float b = 2.f * (float)a.D * __uint_as_float(a.amax[2 * (int64_t)start]) * __uint_as_float(a.amax[2 * (int64_t)start + 1]);
  if (!(b > 0.f)) return 1.f;
  const int e = 15 - (ilogbf(b) + 1);  // b 2^e < 2^15
  return ldexpf(1.f, max(-60, min(60, e)));
}

// where the dP of the g-th column tile lies
template <bool DKV>
__device__ __forceinline__ uint32_t dp_col(int g) { return DKV || (g & 1) == 0 ? DP_COL : DP_COL + 256u; }

template <typename T, int DP, bool DKV>
__global__ void __launch_bounds__(NTHREADS, 1)
attn_bwd_tc_kernel(const __grid_constant__ Map r1map, const __grid_constant__ Map r2map, const __grid_constant__ Map c1map,
                   const __grid_constant__ Map c2map, const __grid_constant__ Args a, const Sched sched) {
  using C = Cfg<DP>;
  using L = typename C::L;
  constexpr int ST = C::ST;
  constexpr int B_1E = B_1F + ST, B_2F = B_1E + ST, B_2E = B_2F + ST, NBARS = B_2E + ST;
  constexpr bool F16 = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Item items[2];
  __shared__ __align__(8) uint64_t bars[NBARS];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, redo_word;  // redo: a NaN has been written
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - raw);
  const uint32_t rs = base, c1s = rs + 2 * C::TILE, c2s = c1s + ST * C::TILE, vecs = c2s + ST * C::TILE;
  volatile int *abort_flag = &abort_word;
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
#define WAIT_WARP(bar, par) (wait_warp_parity((bar), (par), abort_flag))
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

  if (tid == 0) {
    abort_word = redo_word = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_ITEM_F + i), 1);
      mbar_init(BAR(B_ITEM_E + i), NSOFT + 1);  // the softmax warps and the MMA warp have read it
    }
    mbar_init(BAR(B_RF), 1);
    mbar_init(BAR(B_RE), 1);
    mbar_init(BAR(B_LAND), 1);
    mbar_init(BAR(B_SF), 1);
    mbar_init(BAR(B_SE), NSOFT);
    mbar_init(BAR(B_PF), NSOFT);
    for (int i = 0; i < 2; ++i) {
      mbar_init(BAR(B_DPF + i), 1);
      mbar_init(BAR(B_DSF + i), NSOFT);
    }
    mbar_init(BAR(B_ACC_F), 1);
    mbar_init(BAR(B_DRAIN), 1);
    for (int i = 0; i < 4 * ST; ++i) mbar_init(BAR(B_1F + i), 1);
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
    int g = 0, lands = 0, rn = 0;  // g: column tiles so far
    // a column tile: rows outside of the sequences are zeroed, since as B operands of the gradients they
    // meet P = dS = 0, which a NaN would survive
    auto column = [&](uint32_t dst, const Map &map, int head, int row, int full, bool vec, int h) {
      const bool clean = row < range.start || min((int64_t)row + TM, a.T) > range.end;
      const uint32_t bar = clean ? BAR(B_LAND) : BAR(full);
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, C::TILE + (vec ? C::VEC : 0u));
        load_rows<L>(dst, map, head, row, bar);
        if (vec) {
          const uint32_t v = vecs + (uint32_t)(g % ST) * C::VEC;
          bulk_load(v, a.lse + (int64_t)h * a.Tp + row, TM * 4, bar);
          bulk_load(v + TM * 4, a.delta + (int64_t)h * a.Tp + row, TM * 4, bar);
        }
      }
      __syncwarp();
      if (clean) {
        if (!WAIT_WARP(BAR(B_LAND), (uint32_t)lands & 1u)) ok = false;
        ++lands;
        zero_outside<L>(gen + (dst - base), row, range, lane);
        if (lane == 0) mbar_arrive(BAR(full));
      }
    };
    for (int i = 0; ok; ++i) {
      Item it;
      const bool live = item_of<DKV>(a, sched, snake(i, blockIdx.x, gridDim.x), it);
      if (!WAIT_WARP(BAR(B_ITEM_E + (i & 1)), ((uint32_t)(i >> 1) & 1u) ^ 1u)) { ok = false; break; }
      if (lane == 0) {
        items[i & 1] = it;
        mbar_arrive(BAR(B_ITEM_F + (i & 1)));
      }
      __syncwarp();
      if (!live) break;
      if (it.n == 0) continue;
      if (!WAIT_WARP(BAR(B_RE), ((uint32_t)rn & 1u) ^ 1u)) { ok = false; break; }
      ++rn;
      // rows of tokens outside of the sequences are zeroed as well: P = 0 is not enough where dP could be a NaN
      const bool clean = it.r0 < range.start || min((int64_t)it.r0 + TM, a.T) > range.end;
      if (lane == 0) {
        const uint32_t bar = BAR(clean ? B_LAND : B_RF);
        mbar_arrive_expect_tx(bar, 2 * C::TILE);
        load_rows<L>(rs, r1map, it.head, it.r0, bar);
        load_rows<L>(rs + C::TILE, r2map, it.head, it.r0, bar);
      }
      __syncwarp();
      if (clean) {
        if (!WAIT_WARP(BAR(B_LAND), (uint32_t)lands & 1u)) { ok = false; break; }
        ++lands;
        zero_outside<L>(gen, it.r0, range, lane);
        zero_outside<L>(gen + C::TILE, it.r0, range, lane);
        if (lane == 0) mbar_arrive(BAR(B_RF));
      }
      for (int j = 0; j < it.n && ok; ++j, ++g) {
        const int s = g % ST;
        const uint32_t free_par = ((uint32_t)(g / ST) & 1u) ^ 1u;
        const int row = it.c0 + (j % it.cols) * TM;
        const int head = it.c_head + j / it.cols;
        if (!WAIT_WARP(BAR(B_1E + s), free_par)) { ok = false; break; }
        column(c1s + s * C::TILE, c1map, head, row, B_1F + s, DKV, head);
        if (!WAIT_WARP(BAR(B_2E + s), free_par)) { ok = false; break; }
        column(c2s + s * C::TILE, c2map, head, row, B_2F + s, false, head);
      }
    }
    if (!ok && lane == 0) give_up(ERR_TMA, abort_flag, a.err_flag);
    // copies in flight land before the block may exit
    for (int p = g > ST ? g - ST : 0; p < g; ++p) {
      wait_parity<false>(BAR(B_1F + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
      wait_parity<false>(BAR(B_2F + p % ST), (uint32_t)(p / ST) & 1u, nullptr);
    }
    if (rn > 0) wait_parity<false>(BAR(B_RF), (uint32_t)(rn - 1) & 1u, nullptr);
  } else if (warp == W_MMA) {
    // ---------------- MMA issue: the warp runs it, one lane issues ----------------
    {
      constexpr uint32_t id_s = idesc_of<T>(128, 0), id_g = idesc_of<T>(L::N_FULL, 1), id_t = idesc_of<T>(32, 1);
      bool ok = true;
      auto wait_warp = [&](uint32_t bar, uint32_t par) { return wait_warp_parity(bar, par, abort_flag); };
      auto commit = [&](uint32_t bar) {
        if (elect_one()) umma_commit(bar);
      };
      int i = 0, rn = 0, gk = 0;
      struct Step {
        int j, n, g;
      } cur, nxt;
      bool rows_due = false;  // an item's steps are known, its rows not yet here
      // The next step, of this item or of the next one that has any: 1, or 0 past the last, or (block = false) -1
      // while it is not known or its rows are still on their way.
      auto advance = [&](Step &s, bool block) -> int {
        if (!rows_due) {
          if (s.j + 1 < s.n) {
            ++s.j;
            s.g = gk++;
            return 1;
          }
          while (true) {
            const uint32_t bar = BAR(B_ITEM_F + (i & 1)), par = (uint32_t)(i >> 1) & 1u;
            if (!block && !__all_sync(0xffffffffu, mbar_test_wait(bar, par))) return -1;
            if (!wait_warp(bar, par)) { ok = false; return 0; }
            const bool done = uniform(items[i & 1].done);
            s.j = 0;
            s.n = uniform(items[i & 1].n);
            __syncwarp();
            if (elect_one()) mbar_arrive(BAR(B_ITEM_E + (i & 1)));
            ++i;
            if (done) return 0;
            if (s.n > 0) break;
          }
          rows_due = true;
        }
        if (!block && !__all_sync(0xffffffffu, mbar_test_wait(BAR(B_RF), (uint32_t)rn & 1u))) return -1;
        if (!wait_warp(BAR(B_RF), (uint32_t)rn & 1u)) { ok = false; return 0; }
        rows_due = false;
        ++rn;
        s.g = gk++;
        return 1;
      };
      auto arrived = [&](int bar, const Step &s) {
        if (!wait_warp(BAR(bar + s.g % ST), (uint32_t)(s.g / ST) & 1u)) ok = false;
      };
      auto is_here = [&](int bar, const Step &s) {
        return __all_sync(0xffffffffu, mbar_test_wait(BAR(bar + s.g % ST), (uint32_t)(s.g / ST) & 1u)) != 0;
      };
      auto scores = [&](const Step &s) {
        tc_fence_after();
        mma_rows<L>(tmem + S_COL, rs, c1s + (s.g % ST) * C::TILE, id_s);
        commit(BAR(B_SF));
      };
      auto dprob = [&](const Step &s) {
        tc_fence_after();
        mma_rows<L>(tmem + dp_col<DKV>(s.g), rs + C::TILE, c2s + (s.g % ST) * C::TILE, id_s);
        commit(BAR(B_DPF + (s.g & 1)));
        if (!DKV) commit(BAR(B_2E + s.g % ST));
        if (s.j == s.n - 1) commit(BAR(B_RE));
      };
      // The order of a step: S(j+1) goes out as soon as S(j) has been read (P with columns of its own, or DQ) or
      // behind dV(j) (P in its place); dP(j+1) with it where dP has two places (DQ), else behind dK(j).  What has not
      // arrived by then goes out at the end of the step.  The next step may be another item's.
      cur.j = cur.n = 0;
      int have = advance(cur, true);
      if (have == 1 && ok) {
        arrived(B_1F, cur);
        if (ok) scores(cur);
        if (ok) arrived(B_2F, cur);
        if (ok) dprob(cur);
      }
      while (have == 1 && ok) {
        const bool last = cur.j == cur.n - 1;
        nxt = cur;
        have = advance(nxt, false);
        if (!ok) break;
        bool s_due = have != 0, d_due = s_due;
        if (!DKV || C::OWN_P) {
          if (!wait_warp(BAR(B_SE), (uint32_t)cur.g & 1u)) { ok = false; break; }
          // DQ has nothing else to issue until dS: with three stages the next tile is as good as here
          const bool sure = !DKV && ST >= 3 && !last;
          if (sure) {
            arrived(B_1F, nxt);
            arrived(B_2F, nxt);
            if (!ok) break;
          }
          if (have == 1 && (sure || is_here(B_1F, nxt))) {
            scores(nxt);
            s_due = false;
            if (!DKV && (sure || is_here(B_2F, nxt))) {
              dprob(nxt);
              d_due = false;
            }
          }
        }
        if (DKV) {
          if (!wait_warp(BAR(B_PF), (uint32_t)cur.g & 1u)) { ok = false; break; }
          tc_fence_after();
          mma_sum<L>(tmem + C::A2_COL, tmem + C::P_COL, C::OWN_P ? 16u : 32u, c2s + (cur.g % ST) * C::TILE, id_g, id_t, cur.j == 0);
          commit(BAR(B_2E + cur.g % ST));
          if (s_due && have == 1 && is_here(B_1F, nxt)) {
            scores(nxt);
            s_due = false;
          }
        }
        if (!wait_warp(BAR(B_DSF + (cur.g & 1)), (uint32_t)(cur.g >> 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        mma_sum<L>(tmem + A1_COL, tmem + dp_col<DKV>(cur.g), 32u, c1s + (cur.g % ST) * C::TILE, id_g, id_t, cur.j == 0);
        commit(BAR(B_1E + cur.g % ST));
        if (last) commit(BAR(B_ACC_F));
        if (have == -1) have = advance(nxt, true);
        if (have != 1 || !ok) break;
        if (s_due) {
          arrived(B_1F, nxt);
          if (!ok) break;
          scores(nxt);
        }
        if (d_due) {
          arrived(B_2F, nxt);
          if (!ok) break;
          dprob(nxt);
        }
        cur = nxt;
      }
      if (!ok && lane == 0) give_up(ERR_MMA, abort_flag, a.err_flag);
      commit(BAR(B_DRAIN));
    }
    __syncwarp();
  } else {
    // ---------------- softmax: thread = a quarter of a row ----------------
    const int part = warp >> 2;  // its columns: 32 from 32 part
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL + part * 32u;
    const uint32_t p_addr = tmem + lanes + C::P_COL + part * (C::OWN_P ? 16u : 32u);
    const int row = (warp & 3) * 32 + lane;
    const float c = a.scale_log2;
    const uint64_t c2 = f2_pack(c, c);
    const float shift = F16 ? P_SHIFT : 0.f;
    const float out2 = F16 ? exp2f(-P_SHIFT) : 1.f;
    bool ok = true;
    int step = 0, nacc = 0;
    auto arrive = [&](int bar) {  // the warp's TMEM accesses are complete
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(bar));
    };
    for (int i = 0; ok; ++i) {
      if (!WAIT_WARP(BAR(B_ITEM_F + (i & 1)), (uint32_t)(i >> 1) & 1u)) { ok = false; break; }
      const int r0 = items[i & 1].r0, head = items[i & 1].head, c00 = items[i & 1].c0, cols = items[i & 1].cols;
      const int n = items[i & 1].n, done = items[i & 1].done, split = items[i & 1].part;
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(B_ITEM_E + (i & 1)));
      if (done) break;
      const int tok = r0 + row;
      Span sp{tok + 1, tok};
      if (tok < a.T) sp = span_of(a, tok);
      const float held = F16 ? ds_factor(a, tok, sp.start) : 1.f;
      const float dsf = F16 ? held * out2 : 1.f;  // what dS is held times, P's own factor off
      const float out1 = a.scale / held;
      float row_lse = 0.f, row_d = 0.f;
      if (!DKV) {
        row_lse = shift - a.lse[(int64_t)head * a.Tp + tok];  // padded to whole tiles
        row_d = -a.delta[(int64_t)head * a.Tp + tok];
      }
      int ct = 0;
      for (int j = 0; j < n; ++j, ++step) {
        const int col0 = c00 + ct * TM + part * 32;
        ct = ct + 1 == cols ? 0 : ct + 1;
        const float *vec = reinterpret_cast<const float *>(gen + (vecs - base) + (step % ST) * C::VEC) + part * 32;
        if (!WAIT_WARP(BAR(B_SF), (uint32_t)step & 1u)) { ok = false; break; }
        tc_fence_after();
        uint32_t r[32];
        tmem_ld32u(s_addr, r);
        if (!DKV || C::OWN_P) arrive(B_SE);  // S may be overwritten
        if (DKV) {
          // the columns' lse and D came with C1: its barrier orders them (its phase is complete, S was formed from it)
          if (!WAIT_WARP(BAR(B_1F + step % ST), (uint32_t)(step / ST) & 1u)) { ok = false; break; }
        }
        // columns of this part that the row sees: [lo, hi)
        // (dS of a sequence's first token, which sees itself only, is 0: DQ takes it as a row that sees nothing)
        const int lo = (DKV ? tok : sp.start) - col0, hi = (DKV ? sp.end : sp.start == tok ? tok : tok + 1) - col0;
        const bool cut = __any_sync(0xffffffffu, lo > 0 || hi < 32);
        float p[32];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float n0 = row_lse, n1 = row_lse, n2 = row_lse, n3 = row_lse;
          if (DKV) {
            const float4 l = *reinterpret_cast<const float4 *>(vec + e);
            n0 = shift - l.x; n1 = shift - l.y; n2 = shift - l.z; n3 = shift - l.w;
          }
          float x0, x1, x2, x3;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), c2, f2_pack(n0, n1)), x0, x1);
          f2_unpack(f2_fma(f2_pack(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), c2, f2_pack(n2, n3)), x2, x3);
          p[e] = exp2_approx(x0);
          p[e + 1] = exp2_approx(x1);
          p[e + 2] = exp2_approx(x2);
          p[e + 3] = exp2_approx(x3);
        }
        if (cut) {
          const uint32_t seen = bits_between(lo, hi);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen & (1u << e))) p[e] = 0.f;
        }
        if (DKV) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack2<T>(p[2 * e], p[2 * e + 1]);
          if (C::OWN_P && step > 0) {  // the last P has been used: its dV released the stage of its C2
            if (!WAIT_WARP(BAR(B_2E + (step - 1) % ST), (uint32_t)((step - 1) / ST) & 1u)) { ok = false; break; }
            tc_fence_after();
          }
          tmem_st16(p_addr, w);
          tmem_wait_st();
          arrive(B_PF);
          // behind P, which dV needs: the first token's dS with itself
          const uint32_t self = sp.start == tok && lo >= 0 && lo < 32 ? 1u << lo : 0u;
          if (cut && __any_sync(0xffffffffu, self != 0u)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (self & (1u << e)) p[e] = 0.f;
          }
        }
        if (!WAIT_WARP(BAR(B_DPF + (step & 1)), (uint32_t)(step >> 1) & 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_addr = tmem + lanes + dp_col<DKV>(step) + part * 32u;
        tmem_ld32u(d_addr, r);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float m0 = row_d, m1 = row_d, m2 = row_d, m3 = row_d;
          if (DKV) {
            const float4 d = *reinterpret_cast<const float4 *>(vec + TM + e);
            m0 = -d.x; m1 = -d.y; m2 = -d.z; m3 = -d.w;
          }
          const uint64_t u = f2_mul(f2_pack(p[e], p[e + 1]),
                                    f2_add(f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), f2_pack(m0, m1)));
          const uint64_t v = f2_mul(f2_pack(p[e + 2], p[e + 3]),
                                    f2_add(f2_pack(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), f2_pack(m2, m3)));
          float x0, x1, x2, x3;
          f2_unpack(u, x0, x1);
          f2_unpack(v, x2, x3);
          if (F16) {
            x0 *= dsf; x1 *= dsf; x2 *= dsf; x3 *= dsf;
          }
          w[e >> 1] = pack2<T>(x0, x1);
          w[(e >> 1) + 1] = pack2<T>(x2, x3);
        }
        tmem_st16(d_addr, w);
        tmem_wait_st();
        arrive(B_DSF + (step & 1));
      }
      if (!ok) break;
      if (n > 0) {
        if (!WAIT_WARP(BAR(B_ACC_F), (uint32_t)nacc & 1u)) { ok = false; break; }
        ++nacc;
        tc_fence_after();
      }
      // epilogue: every fourth 16 columns of the row's results
      const int64_t at = ((int64_t)tok * (DKV ? a.Hk : a.H) + head) * a.D;
      constexpr int PIECES = DP / 16;
      bool bad = false;
#pragma unroll 1
      for (int q = part; q < (DKV ? 2 : 1) * PIECES; q += 4) {
        const bool second = DKV && q >= PIECES;
        const int d = (second ? q - PIECES : q) * 16;
        T *dst = static_cast<T *>(DKV ? (second ? a.dv : a.dk) : a.dq) + at;
        const float mul = second ? out2 : out1;
        uint32_t o[16];
        if (n > 0) {
          tmem_ld16u(tmem + lanes + (second ? C::A2_COL : A1_COL) + d, o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) bad |= isnan(__uint_as_float(o[e]));
        if (DKV && a.splits > 1) {
          float *pd = a.parts + ((int64_t)(split * 2 + second) * a.T * a.Hk * a.D) + at + d;
#pragma unroll
          for (int h = 0; h < 4; ++h)
            if (tok < a.T && d + h * 4 < a.D)
              *reinterpret_cast<float4 *>(pd + h * 4) = make_float4(__uint_as_float(o[4 * h]) * mul, __uint_as_float(o[4 * h + 1]) * mul,
                                                                    __uint_as_float(o[4 * h + 2]) * mul, __uint_as_float(o[4 * h + 3]) * mul);
          continue;
        }
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = pack2<T>(__uint_as_float(o[2 * e]) * mul, __uint_as_float(o[2 * e + 1]) * mul);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (tok < a.T && d + h * 8 < a.D)
            *reinterpret_cast<uint4 *>(dst + d + h * 8) = make_uint4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3]);
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
      if (!item_of<DKV>(a, sched, snake(i, blockIdx.x, gridDim.x), it)) break;
      for (int e = tid; e < TM * a.D; e += NTHREADS) {
        const int64_t tok = it.r0 + e / a.D;
        if (tok >= a.T) continue;
        const int64_t at = (tok * (DKV ? a.Hk : a.H) + it.head) * a.D + e % a.D;
        if (DKV && a.splits > 1) {
          for (int w = 0; w < 2; ++w) a.parts[(int64_t)(it.part * 2 + w) * a.T * a.Hk * a.D + at] = __int_as_float(0x7fc00000);
        } else if (DKV) {
          static_cast<T *>(a.dk)[at] = bad;
          static_cast<T *>(a.dv)[at] = bad;
        } else {
          static_cast<T *>(a.dq)[at] = bad;
        }
      }
    }
  } else if (redo_word) {
    constexpr int WARPS = NTHREADS / 32;
    for (int i = 0;; ++i) {
      Item it;
      if (!item_of<DKV>(a, sched, snake(i, blockIdx.x, gridDim.x), it)) break;
      if constexpr (DKV) {
        const int64_t n = a.T * a.Hk * a.D;
        const int per = a.H / a.Hk / a.splits;
        if (a.splits > 1)
          redo_dkv_rows<T, float>(a, it.head, it.r0, TM, it.c_head, per, a.parts + 2 * it.part * n, a.parts + (2 * it.part + 1) * n, warp,
                                  WARPS, lane);
        else
          redo_dkv_rows<T, T>(a, it.head, it.r0, TM, it.c_head, per, static_cast<T *>(a.dk), static_cast<T *>(a.dv), warp, WARPS, lane);
      } else {
        redo_dq_rows<T>(a, it.head, it.r0, TM, warp, WARPS, lane);
      }
    }
  }
#undef WAIT_WARP
#undef BAR
}

// dK and dV from the parts of the blocks that share their keys, in order
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const Args a) {
  const int64_t n = a.T * a.Hk * a.D, quads = n / 4;  // D is a multiple of 8
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < 2 * quads; q += (int64_t)gridDim.x * 256) {
    const int second = q >= quads;
    const int64_t at = (q - second * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < a.splits; ++p) {
      const float4 v = __ldcs(reinterpret_cast<const float4 *>(a.parts + (int64_t)(p * 2 + second) * n + at));
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<uint2 *>(static_cast<T *>(second ? a.dv : a.dk) + at) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
  }
}

template <typename T, int DP, bool DKV>
cudaError_t run(const Args &a, const Map &r1, const Map &r2, const Map &c1, const Map &c2, const int *order, int sms,
                cudaStream_t stream) {
  using C = Cfg<DP>;
  constexpr size_t smem = 2 * C::TILE + C::ST * (2 * C::TILE + C::VEC) + 1024;
  static_assert(smem <= 232448 - 1024, "shared memory of a block");
  auto kern = attn_bwd_tc_kernel<T, DP, DKV>;
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
  Sched s;
  s.tiles = (int)((a.T + TM - 1) / TM);
  s.heads = DKV ? a.Hk * a.splits : a.H;
  if ((int64_t)s.tiles * s.heads > 0x7fffffff) return cudaErrorNotSupported;
  s.items = s.tiles * s.heads;
  s.order = s.items > sms ? order : nullptr;  // with a block for every piece of work their order does not matter
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(s.items < sms ? s.items : sms), 1, 1);
  cfg.blockDim = dim3(NTHREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  e = cudaLaunchKernelEx(&cfg, kern, r1, r2, c1, c2, a, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace
}  // namespace attn

// Into how many the heads of a group are shared out where keys alone make too few
// pieces of work: two for every SM or all heads apart.  (13 sequences, 8191 tokens, 8
// heads over 2, D = 64: dK and dV in 166 us with 128 pieces, 66 us with 512 (52 since the masks are
// bits) and 7 us to join them.  On CUDA cores, 1024 tokens, 8 / 4 heads of 96, fp32:
// 274 us without, 136 and 5 with.)
int attn_bwd_splits(int64_t T, int H, int Hk) {
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148, G = H / Hk;
  const int64_t tiles = (T + attn::TM - 1) / attn::TM;
  int s = 1;
  while (s < G && (tiles * Hk * s < 2 * (int64_t)sms || G % s)) ++s;
  return s;
}

cudaError_t launch_attn_bwd_tc(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream) {
  attn::Map q, k, v, d;
  const int64_t ot = (int64_t)a.H * a.D;
  if (!attn::make_map(q, a.q, a.dtype, a.T, a.H, a.D, a.qt, a.qh) || !attn::make_map(k, a.k, a.dtype, a.T, a.Hk, a.D, a.kt, a.kh) ||
      !attn::make_map(v, a.v, a.dtype, a.T, a.Hk, a.D, a.vt, a.vh) || !attn::make_map(d, a.dout, a.dtype, a.T, a.H, a.D, ot, a.D))
    return cudaErrorNotSupported;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  auto both = [&](auto tag, auto dim) -> cudaError_t {
    using T = decltype(tag);
    constexpr int DP = decltype(dim)::value;
    cudaError_t e = cudaSuccess;
    // DQ has at least as many pieces of work as DKV
    if ((a.T + attn::TM - 1) / attn::TM * a.H > sms) e = launch_attn_orders(a, order_q, order_k, stream);
    if (e == cudaSuccess && a.dk) e = attn::run<T, DP, true>(a, k, v, q, d, order_k, sms, stream);
    if (e == cudaSuccess && a.dq) e = attn::run<T, DP, false>(a, q, d, k, v, order_q, sms, stream);
    if (e == cudaSuccess && a.dk && a.splits > 1) {
      attn::attn_join_kernel<T><<<grid_for(2 * a.T * a.Hk * a.D / 4, 256, sms, 8), 256, 0, stream>>>(a);
      e = cudaGetLastError();
    }
    return e;
  };
  auto go = [&](auto tag) -> cudaError_t {
    if (a.D <= 32) return both(tag, IC<32>{});
    if (a.D <= 64) return both(tag, IC<64>{});
    if (a.D <= 96) return both(tag, IC<96>{});
    return both(tag, IC<128>{});
  };
  return a.dtype == MHC_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

int read_atb_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_atb_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_atb_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace mhc
