// Output stage of the persistent products on matrices in blocks: a warp takes 32 rows x kCols columns of an
// accumulator from tensor memory through a staged box of [32 rows][128 bytes] (128-byte swizzle) to C.
#pragma once
#include "common.cuh"
#include "epilogue.cuh"

namespace ngb {

struct OutParams {
  int M, N;
  void* C;
  long long ldc;
  int out_f32;
  int store;              // 1: TMA can address C's rows, whole; 0: one number per lane and access
  EpiArgs ea;
};

// fp16, rounded to nearest, nothing added: all columns to registers first, then `release` gives the accumulator back.
template <int kCols, typename F>
__device__ __forceinline__ void out_lean(const OutParams& p, const CUtensorMap* mapC, uint32_t taddr, uint32_t stage, uint8_t* stage_gen,
                                         int m0, int n0, F release) {
  const int lane = threadIdx.x & 31;
  const bool as_is = p.ea.alpha == 1.0f && !p.ea.relu;
  uint32_t w[kCols / 2];
#pragma unroll
  for (int c = 0; c < kCols; c += 32) {
    uint32_t r[32];
    tc_ld_32x32(taddr + c, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a = __uint_as_float(r[2 * i]), b = __uint_as_float(r[2 * i + 1]);
      if (!as_is) {
        a = epi_scale(p.ea, a);
        b = epi_scale(p.ea, b);
      }
      const __half2 h = __floats2half2_rn(a, b);
      w[c / 2 + i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  tc_fence_before();
  __syncwarp();
  release();
  if (m0 >= p.M) return;
#pragma unroll
  for (int c = 0; c < kCols; c += 64) {
    if (n0 + c >= p.N) break;
    if (lane == 0) tma_store_wait_read<0>();       // (the box before must have left)
    __syncwarp();
#pragma unroll
    for (int g = 0; g < 8; ++g)
      *reinterpret_cast<uint4*>(stage_gen + lane * 128 + ((g ^ (lane & 7)) << 4)) =
          make_uint4(w[c / 2 + 4 * g], w[c / 2 + 4 * g + 1], w[c / 2 + 4 * g + 2], w[c / 2 + 4 * g + 3]);
    if (p.store) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_5d(mapC, stage, n0 + c, m0, 0, 0, 0);
        tma_store_commit();
      }
    } else {
      // rows at any address: a row at a time, two numbers per lane
      __syncwarp();
      __half* out = static_cast<__half*>(p.C) + m0 * p.ldc + n0 + c + lane;
      const int rows = min(32, p.M - m0), cols = p.N - n0 - c - lane;
#pragma unroll 8
      for (int i = 0; i < rows; ++i, out += p.ldc) {
        const uint8_t* src = stage_gen + i * 128 + ((lane * 2) & 15);
        if (cols > 0) out[0] = *reinterpret_cast<const __half*>(src + (((lane >> 3) ^ (i & 7)) << 4));
        if (cols > 32) out[32] = *reinterpret_cast<const __half*>(src + (((4 + (lane >> 3)) ^ (i & 7)) << 4));
      }
      __syncwarp();
    }
  }
}

// Everything else: fp32, C added, stochastic rounding.
template <int kCols, typename F>
__device__ __forceinline__ void out_any(const OutParams& p, const CUtensorMap* mapC, uint32_t taddr, uint32_t stage, uint8_t* stage_gen,
                                        int m0, int n0, F release) {
  const int lane = threadIdx.x & 31;
  const long long row = m0 + lane;
  const bool f32 = p.out_f32;
  const int esz = f32 ? 4 : 2;
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    uint32_t r[32];
    tc_ld_32x32(taddr + c, r);
    tc_wait_ld();
    if (c + 32 >= kCols) {     // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      release();
    }
    if (m0 >= p.M || n0 + c >= p.N) continue;
    // into this lane's row of the staged box: 32 columns are 64 bytes of fp16 (half a row) or 128 of fp32
    const int at = f32 ? 0 : (c & 32) * 2;
    if (at == 0) {             // (the box before must have left)
      if (lane == 0) tma_store_wait_read<0>();
      __syncwarp();
    }
    uint8_t* dst = stage_gen + lane * 128;
    const uint32_t sw = (lane & 7) << 4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[8 * g + i]);
      uint4 lo, hi;
      const int col = n0 + c + 8 * g;
      const int nvalid = row < p.M ? max(0, min(8, p.N - col)) : 0;
      const unsigned long long lin = static_cast<unsigned long long>(row) * p.N + col;
      const void* oldp = nvalid > 0 ? static_cast<const uint8_t*>(p.C) + (row * p.ldc + col) * esz : nullptr;
      if (f32) epi_pack8<true>(p.ea, v, oldp, lin, lo, hi, max(nvalid, 1));
      else epi_pack8<false>(p.ea, v, oldp, lin, lo, hi, max(nvalid, 1));
      if (f32) {
        *reinterpret_cast<uint4*>(dst + ((32 * g) ^ sw)) = lo;
        *reinterpret_cast<uint4*>(dst + ((32 * g + 16) ^ sw)) = hi;
      } else {
        *reinterpret_cast<uint4*>(dst + ((at + 16 * g) ^ sw)) = lo;
      }
    }
    if (!f32 && at == 0 && n0 + c + 32 < p.N) continue;    // the other half of the box comes next
    const int col0 = n0 + (f32 ? c : c & ~63);
    if (p.store) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_5d(mapC, stage, col0, m0, 0, 0, 0);
        tma_store_commit();
      }
    } else {
      __syncwarp();
      const int rows = min(32, p.M - m0), cols = min(128 / esz, p.N - col0);
      for (int i = 0; i < rows; ++i) {
        uint8_t* out = static_cast<uint8_t*>(p.C) + ((m0 + i) * p.ldc + col0) * esz;
        for (int j = lane; j < cols; j += 32) {
          const uint8_t* src = stage_gen + i * 128 + (((j * esz) & 112) ^ ((i & 7) << 4)) + ((j * esz) & 15);
          if (f32) reinterpret_cast<float*>(out)[j] = *reinterpret_cast<const float*>(src);
          else reinterpret_cast<__half*>(out)[j] = *reinterpret_cast<const __half*>(src);
        }
      }
      __syncwarp();
    }
  }
}

}  // namespace ngb
