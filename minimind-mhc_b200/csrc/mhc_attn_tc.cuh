// What the tensor-core attention kernels (sm_100a) share: tiles, tensor maps, the
// operand descriptors and the order of the work.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mhc_attn.cuh"
#include "mhc_device.cuh"
#include "mhc_dispatch.cuh"
#include "mhc_kernels.h"
#include "mhc_sm100.cuh"

namespace mhc {
namespace attn {

using namespace sm100;

constexpr int TM = 128;               // rows of a tile, queries or keys
constexpr uint32_t BLK = TM * 128;    // 128 rows x 64 values of 16 bits, 128-byte swizzle

// A tile of 128 rows x DP values in shared memory: blocks of 64 columns in the
// 128-byte swizzle.  Where DP is no multiple of 64 the last block is 32 columns in the
// 64-byte swizzle (SPLIT: D = 96 takes 24 KB, and a third stage of the streamed tiles
// fits), or a whole one filled up with zeros (the products are one instruction wider
// instead of two: forward at 16384 tokens, D = 96: 411 us against 444).
template <int DP, bool SPLIT>
struct Tile {
  static constexpr int TAIL = SPLIT ? DP % 64 : 0, FULL = SPLIT ? DP / 64 : (DP + 63) / 64;
  static_assert(TAIL == 0 || TAIL == 32, "head sizes are rounded up to multiples of 32");
  static constexpr uint32_t TAIL_AT = FULL * BLK;
  static constexpr uint32_t BYTES = TAIL_AT + (TAIL ? BLK / 2 : 0);
  static constexpr int N_FULL = TAIL ? FULL * 64 : DP;  // columns of a product on the full blocks
  static constexpr int K_FULL = N_FULL / 16;            // its steps where they are the summed index
};

// D fp32, A and B of type T (bf16: format 1, fp16: format 0), M = 128
template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int N, int b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(TM >> 4) << 24);
}

// D [128 x 128] = A B^T, both K-major tiles of DP columns.  One lane issues.
template <typename L>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  const uint64_t ad = umma_desc_sw128(a), bd = umma_desc_sw128(b);
  const uint64_t at = umma_desc_sw64(a + L::TAIL_AT), bt = umma_desc_sw64(b + L::TAIL_AT);
  if (elect_one()) {
#pragma unroll
    for (int kk = 0; kk < L::K_FULL; ++kk) {
      const uint64_t step = (uint64_t)((kk >> 2) * (int)BLK + (kk & 3) * 32) >> 4;  // addresses in 16-byte units
      umma_bf16(d, ad + step, bd + step, idesc, kk > 0);
    }
#pragma unroll
    for (int kk = 0; kk < L::TAIL / 16; ++kk) umma_bf16(d, at + kk * 2, bt + kk * 2, idesc, L::FULL > 0 || kk > 0);
  }
}

// D [128 x DP] (+)= A B, of two widths (id_full, id_tail): A [128 x 128] 16-bit in TMEM, 32 of its columns in 16 TMEM
// columns, `pitch` apart; B a tile whose rows are the summed index (MN-major).
template <typename L>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t a, uint32_t pitch, uint32_t b, uint32_t id_full, uint32_t id_tail,
                                        bool begin) {
  const uint64_t bd = umma_desc(b, BLK, 1024, 2), bt = umma_desc(b + L::TAIL_AT, 16, 512, 4);
  if (elect_one()) {
    if constexpr (L::FULL > 0) {
#pragma unroll
      for (int kk = 0; kk < TM / 16; ++kk)
        umma_f16_ts(d, a + (kk >> 1) * pitch + (kk & 1) * 8u, bd + kk * (2048 >> 4), id_full, !begin || kk > 0);
    }
    if constexpr (L::TAIL > 0) {
#pragma unroll
      for (int kk = 0; kk < TM / 16; ++kk)
        umma_f16_ts(d + L::FULL * 64, a + (kk >> 1) * pitch + (kk & 1) * 8u, bt + kk * (1024 >> 4), id_tail, !begin || kk > 0);
    }
  }
}

// Tensor maps of (T, heads, D) in boxes of 128 rows x 64 columns (m) and x 32 columns
// (t), and whether the second axis is the token (heads farther apart than tokens).
struct Map {
  CUtensorMap m, t;
  int token_first;
};
template <typename L>
__device__ __forceinline__ void load_rows(uint32_t dst, const Map &map, int head, int row, uint32_t bar) {
  const int y = map.token_first ? row : head, z = map.token_first ? head : row;
#pragma unroll
  for (int b = 0; b < L::FULL; ++b) tma_load_3d(dst + b * BLK, &map.m, b * 64, y, z, bar);
  if constexpr (L::TAIL > 0) tma_load_3d(dst + L::TAIL_AT, &map.t, L::FULL * 64, y, z, bar);
}

// false where TMA cannot read the tensor
bool make_map(Map &map, const void *p, int dtype, int64_t T, int heads, int D, int64_t ts, int64_t hs);
// the same test without building the map
bool map_eligible(const void *p, int D, int heads, int64_t T, int64_t ts, int64_t hs);

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// two fp32 rounded to a pair of T, a in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// A whole warp's wait.  Most phases are complete when they are asked for: one probe
// without the clock reads of the bounded wait first.
__device__ __forceinline__ bool wait_warp_parity(uint32_t bar, uint32_t parity, const volatile int *abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_parity<false>(bar, parity, abort_flag)) != 0;
}

// Zeroes the rows of a landed tile that lie outside of [range.start, range.end): a
// masked score of exactly 0 times a NaN there would still be NaN.  One warp; the
// caller signals the tile afterwards.
template <typename L>
__device__ __forceinline__ void zero_outside(uint8_t *tile, int row0, Span range, int lane) {
  for (int r = 0; r < TM; ++r) {
    if (row0 + r >= range.start && row0 + r < range.end) continue;
    if (lane < L::FULL * 8) *reinterpret_cast<uint4 *>(tile + (lane >> 3) * BLK + r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    if (L::TAIL > 0 && lane >= 28) *reinterpret_cast<uint4 *>(tile + L::TAIL_AT + r * 64 + (lane - 28) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Bits [lo, hi) of 32: which of a row's columns it sees.  Tested one constant bit at a
// time they turn into predicates several at once, where comparing each column's index
// with both ends took three instructions a column.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  const uint32_t below = hi <= 0 ? 0u : (hi >= 32 ? 0xffffffffu : (1u << hi) - 1u);
  return lo <= 0 ? below : (lo >= 32 ? 0u : below & (0xffffffffu << lo));
}

// rank of the i-th piece of work of a block among pieces sorted by size: forwards and
// backwards in turn, so that every block's pieces sum to nearly the same
__device__ __forceinline__ int64_t snake(int i, int block, int blocks) {
  return (int64_t)i * blocks + ((i & 1) ? blocks - 1 - block : block);
}

}  // namespace attn

int attn_bwd_splits(int64_t T, int H, int Hk);
bool attn_tc_eligible(const attn::Args &a);      // what both directions ask of q, k, v, out
bool attn_tc_bwd_eligible(const attn::Args &a);
size_t attn_order_bytes(int64_t T);
cudaError_t launch_attn_fwd_tc(const attn::Args &a, int *order, cudaStream_t stream);
// the order of the tiles of queries and, where order_k is not null, of keys, in one launch
cudaError_t launch_attn_orders(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream);
cudaError_t launch_attn_bwd_tc(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream);

}  // namespace mhc
