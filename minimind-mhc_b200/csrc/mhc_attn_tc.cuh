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
constexpr uint32_t HALF = BLK / 2;    // 64 rows of them

// blocks of 64 columns that a head of D <= DP values takes
__host__ __device__ constexpr int nblk(int DP) { return (DP + 63) / 64; }

// D fp32, A and B of type T (bf16: format 1, fp16: format 0), M = 128
template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int N, int b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(TM >> 4) << 24);
}

// What a descriptor's start address (16-byte units) moves by for the kk-th 16 values
// of the summed index: along a row of a K-major tile, or 16 rows of an MN-major one.
// `block`: from 64 columns to the next 64.
__host__ __device__ constexpr uint64_t k_step(int kk, uint32_t block) { return (uint64_t)((kk >> 2) * (int)block + (kk & 3) * 32) >> 4; }
__host__ __device__ constexpr uint64_t mn_step(int kk) { return (uint64_t)(kk * 2048) >> 4; }

// A tensor map of (T, heads, D) in boxes of 64 rows x 64 columns, and whether its
// second axis is the token (heads farther apart than tokens).
struct Map {
  CUtensorMap m;
  int token_first;
};
__device__ __forceinline__ void load_box(uint32_t dst, const Map &map, int col, int head, int row, uint32_t bar) {
  tma_load_3d(dst, &map.m, col, map.token_first ? row : head, map.token_first ? head : row, bar);
}
// 64 rows, blocks of 64 columns HALF bytes apart
__device__ __forceinline__ void load_half(uint32_t dst, const Map &map, int nb, int head, int row, uint32_t bar) {
  for (int b = 0; b < nb; ++b) load_box(dst + b * HALF, map, b * 64, head, row, bar);
}
// 128 rows, blocks of 64 columns BLK bytes apart
__device__ __forceinline__ void load_rows(uint32_t dst, const Map &map, int nb, int head, int row, uint32_t bar) {
  for (int b = 0; b < nb; ++b) {
    load_box(dst + b * BLK, map, b * 64, head, row, bar);
    load_box(dst + b * BLK + HALF, map, b * 64, head, row + 64, bar);
  }
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

// Zeroes the rows of landed blocks of `rows` rows x 64 columns, `pitch` bytes apart,
// that lie outside of [range.start, range.end): a masked score of exactly 0 times a
// NaN there would still be NaN.  One warp; the caller signals the tile afterwards.
__device__ __forceinline__ void zero_outside(uint8_t *tile, int nb, uint32_t pitch, int rows, int row0, Span range, int lane) {
  for (int r = 0; r < rows; ++r) {
    if (row0 + r >= range.start && row0 + r < range.end) continue;
    for (int b = lane; b < nb * 8; b += 32)
      *reinterpret_cast<uint4 *>(tile + (b >> 3) * pitch + r * 128 + (b & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// rank of the i-th piece of work of a block among pieces sorted by size: forwards and
// backwards in turn, so that every block's pieces sum to nearly the same
__device__ __forceinline__ int64_t snake(int i, int block, int blocks) {
  return (int64_t)i * blocks + ((i & 1) ? blocks - 1 - block : block);
}

}  // namespace attn

// tiles of 128 tokens in the order of their work, largest first: order[rank] = tile.
// keys != 0: the work of a tile of keys (the queries that see it)
cudaError_t launch_attn_order(const attn::Args &a, int keys, int *order, cudaStream_t stream);

bool attn_tc_eligible(const attn::Args &a);      // what both directions ask of q, k, v, out
bool attn_tc_bwd_eligible(const attn::Args &a);
size_t attn_order_bytes(int64_t T);
cudaError_t launch_attn_fwd_tc(const attn::Args &a, int *order, cudaStream_t stream);
cudaError_t launch_attn_bwd_tc(const attn::Args &a, int *order_q, int *order_k, cudaStream_t stream);

}  // namespace mhc
