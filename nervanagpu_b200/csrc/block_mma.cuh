// Pieces of the 4-bit products: bulk copies and tcgen05 with scales in tensor memory.
#pragma once
#include "blocks.cuh"
#include "common.cuh"

namespace ngb {

// upper word of the descriptor of a K-major operand in rows of 128 bytes: 8 rows 1024 bytes apart, version 1, 128-byte swizzle
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem) {
  return (static_cast<uint64_t>(kDescHi) << 32) | (1u << 16) | (smem >> 4);
}
// Instruction descriptor: E2M1 operands, N >> 3, scales E4M3 or E8M0, M >> 4.
__host__ __device__ constexpr uint32_t block_idesc(int m, int n, bool nv) {
  return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((nv ? 0u : 1u) << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// 32 rows of 16 bytes in shared memory to 4 columns of tensor memory, the same in each of the four groups of 32 lanes.
// kPair: both CTAs of a pair, each from its own shared memory.
template <bool kPair>
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint32_t smem) {
  const uint64_t desc = (static_cast<uint64_t>((128u >> 4) | (1u << 14)) << 32) | (1u << 16) | (smem >> 4);
  if (kPair) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

#define NG_BLOCK_MMA(group, vec)                                                                                           \
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n tcgen05.mma.cta_group::" group                                 \
               ".kind::mxf4nvf4.block_scale.scale_vec::" vec " [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d), "l"(a),    \
               "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                                       \
               : "memory")
template <bool kNv, bool kPair>
__device__ __forceinline__ void tc_mma_blocks(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                              uint32_t accumulate) {
  if (kNv && kPair) NG_BLOCK_MMA("2", "4X");
  else if (kNv) NG_BLOCK_MMA("1", "4X");
  else if (kPair) NG_BLOCK_MMA("2", "2X");
  else NG_BLOCK_MMA("1", "2X");
}
#undef NG_BLOCK_MMA

// One k-block of 256 numbers: its scales to tensor memory (A's tiles at ta, B's behind them, kRowTiles x 4 columns per
// tile), then four MMAs of 64. a, b, sa, sb: shared memory; B's scale tiles of 128 columns are kScales bytes apart.
template <bool kNv, bool kPair, int kRowTiles>
__device__ __forceinline__ void mma_kblock(uint32_t d, uint32_t a, uint32_t b, uint32_t sa, uint32_t sb, uint32_t ta, uint32_t idesc,
                                           bool first) {
  constexpr int kTiles = kNv ? 4 : 2;
  constexpr uint32_t kScales = kTiles * kScaleTile;
  const uint32_t tb = ta + kTiles * 4;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    tc_copy_scales<kPair>(ta + t * 4, sa + t * kScaleTile);
#pragma unroll
    for (int c = 0; c < kRowTiles; ++c) tc_copy_scales<kPair>(tb + (t * kRowTiles + c) * 4, sb + c * kScales + t * kScaleTile);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int t = kNv ? j : j / 2;
    const uint32_t id = kNv ? 0u : (j & 1) * 2u;       // which of the tile's four scales are this MMA's first
    tc_mma_blocks<kNv, kPair>(d, operand_desc(a + 32u * j), operand_desc(b + 32u * j), idesc | (id << 4) | (id << 29), ta + t * 4,
                              tb + t * kRowTiles * 4, !(first && j == 0));
  }
}

}  // namespace ngb
