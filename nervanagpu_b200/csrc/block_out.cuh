// Output stage of the persistent products on matrices in blocks: a warp takes 32 rows x kCols columns of an
// accumulator from tensor memory through a staged box of [32 rows][128 bytes] (128-byte swizzle) to C.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "epilogue.cuh"

namespace ngb {

struct OutParams {
  int M, N;
  void* C;
  long long ldc;
  int out_f32;
  int store;              // 1: C's rows are whole aligned vectors, which TMA can address; 0: any address
  EpiArgs ea;
};

// What C held, loaded as bits and converted when used: a load with its conversion under one condition becomes a branch, and
// waits for the one before.
template <typename E>
using OldBits = std::conditional_t<sizeof(E) == 2, unsigned short, float>;
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(unsigned short x) { return __half2float(__ushort_as_half(x)); }
__device__ __forceinline__ void epi_put(float c, float* out) { *out = c; }
__device__ __forceinline__ void epi_put(float c, __half* out) { *out = f2h_rn(c); }
// One output, rounded to nearest.
template <typename E>
__device__ __forceinline__ void epi_store_nearest(const EpiArgs& e, float acc, float old, E* out) {
  float c = epi_scale(e, acc);
  if (e.beta != 0.0f) c = fmaf(e.beta, old, c);
  epi_put(c, out);
}

__device__ __forceinline__ void tc_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// fp16, rounded to nearest, nothing added: all columns to registers first, then `release` gives the accumulator back.
template <int kCols, typename F>
__device__ __forceinline__ void out_lean(const OutParams& p, const CUtensorMap* mapC, uint32_t taddr, uint32_t stage, uint8_t* stage_gen,
                                         int m0, int n0, F release) {
  const int lane = threadIdx.x & 31;
  const bool as_is = p.ea.alpha == 1.0f && !p.ea.relu;
  uint32_t w[kCols / 2];
#pragma unroll
  for (int c = 0; c < kCols; c += 16) {      // (by 32 columns the registers did not suffice in tiles of 256)
    uint32_t r[16];
    tc_ld_32x16(taddr + c, r);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
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
#pragma unroll 1
      for (int i0 = 0; i0 < rows; i0 += 16) {
        __half x[16], y[16];   // (all of them first: no load passes a store)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint8_t* src = stage_gen + (i0 + i) * 128 + ((lane * 2) & 15);
          x[i] = *reinterpret_cast<const __half*>(src + (((lane >> 3) ^ (i & 7)) << 4));
          y[i] = *reinterpret_cast<const __half*>(src + (((4 + (lane >> 3)) ^ (i & 7)) << 4));
        }
#pragma unroll
        for (int i = 0; i < 16; ++i, out += p.ldc) {
          if (i0 + i < rows && cols > 0) out[0] = x[i];
          if (i0 + i < rows && cols > 32) out[32] = y[i];
        }
      }
      __syncwarp();
    }
  }
}

// Everything else: fp32, C added, stochastic rounding. 32 columns at a time go through the staged box in fp32, so that
// neighbouring lanes read and write neighbours of C, and what C held in 16 or 32 rows is on its way together. (With a row per lane
// each access touched 32 sectors, and the loads of one chunk waited for the stores of the last: with C added, 5664 x 546 x 1698
// 28.5 -> 15.4 us and 4096 x 9216 x 128 160 -> 45, against 8.4 and 20 without.) First, rows of C at any address: a number per lane.
template <int kCols, typename E, typename F>
__device__ __forceinline__ void out_odd(const OutParams& p, uint32_t taddr, uint8_t* stage_gen, int m0, int n0, F release) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    const int rows = min(32, p.M - m0), col = n0 + c + lane;
    E* out = static_cast<E*>(p.C) + m0 * p.ldc + col;
    uint32_t r[32];
    tc_ld_32x32(taddr + c, r);
    tc_wait_ld();
    if (c + 32 >= kCols) {     // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      release();
    }
    if (m0 >= p.M || n0 + c >= p.N) continue;
#pragma unroll
    for (int g = 0; g < 8; ++g)
      *reinterpret_cast<uint4*>(stage_gen + lane * 128 + ((g ^ (lane & 7)) << 4)) = make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
    __syncwarp();
    auto at = [&](int i) {
      return *reinterpret_cast<const float*>(stage_gen + i * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4);
    };
    if (sizeof(E) == 2 && p.ea.sr_bits) {
      // eight neighbours at a time, which share their random bits
      const int first = n0 + c + (lane & 3) * 8;
#pragma unroll 1
      for (int i = lane >> 2; i < rows && first < p.N; i += 8) {
        const uint8_t* src = stage_gen + i * 128;
        const float4 x = *reinterpret_cast<const float4*>(src + (((lane & 3) * 2 ^ (i & 7)) << 4));
        const float4 y = *reinterpret_cast<const float4*>(src + (((lane & 3) * 2 + 1 ^ (i & 7)) << 4));
        E* row = static_cast<E*>(p.C) + (m0 + i) * p.ldc;
        epi_store8_call<false>(p.ea, x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, row, row, first,
                               static_cast<unsigned long long>(m0 + i) * p.N + first, min(8, p.N - first), false);
      }
    } else if (col < p.N) {
      // (fp32: with 32 rows at a time the registers did not suffice, 1001 x 4097 x 125 17.6 us for 13.0; fp16 with 16: 20.4 for 15.1)
      constexpr int kRows = sizeof(E) == 4 ? 16 : 32;
      const int held = p.ea.beta != 0.0f ? rows : 0;
#pragma unroll 1
      for (int i0 = 0; i0 < rows; i0 += kRows) {
        OldBits<E> old[kRows];
        float x[kRows];          // (all of them first: no load passes a store)
#pragma unroll
        for (int i = 0; i < kRows; ++i) old[i] = i0 + i < held ? reinterpret_cast<const OldBits<E>*>(out)[(i0 + i) * p.ldc] : OldBits<E>(0);
#pragma unroll
        for (int i = 0; i < kRows; ++i) x[i] = at(i0 + i);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (i0 + i < rows) epi_store_nearest(p.ea, x[i], to_f32(old[i]), out + (i0 + i) * p.ldc);
      }
    }
    __syncwarp();
  }
}

// The same in rows of whole aligned vectors: one per lane, 4 (fp16) or 8 (fp32) lanes on a row. What is fp32 leaves by TMA, from
// the box as it is (4096 x 9216 x 128 57.8 -> 45 us).
template <int kCols, typename E, typename F>
__device__ __forceinline__ void out_even(const OutParams& p, const CUtensorMap* mapC, uint32_t taddr, uint32_t stage, uint8_t* stage_gen,
                                         int m0, int n0, F release) {
  constexpr int kPer = 16 / sizeof(E), kLanes = 32 / kPer, kStep = 32 / kLanes;      // numbers of a lane, lanes and rows of an access
  const int lane = threadIdx.x & 31, row0 = lane / kLanes, col0 = lane % kLanes * kPer;
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    const int col = n0 + c + col0;
    const int rows = col < p.N ? p.M - m0 - row0 : 0;      // of this lane, one in kStep
    E* out = static_cast<E*>(p.C) + (m0 + row0) * p.ldc + col;
    uint4 old[kLanes];
#pragma unroll
    for (int t = 0; t < kLanes; ++t)
      old[t] = p.ea.beta != 0.0f && kStep * t < rows ? *reinterpret_cast<const uint4*>(out + kStep * t * p.ldc) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t r[32];
    tc_ld_32x32(taddr + c, r);
    tc_wait_ld();
    if (c + 32 >= kCols) {     // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      release();
    }
    if (m0 >= p.M || n0 + c >= p.N) continue;
    if (kPer == 4) {           // (the box before must have left)
      if (lane == 0) tma_store_wait_read<0>();
      __syncwarp();
    }
#pragma unroll
    for (int g = 0; g < 8; ++g)
      *reinterpret_cast<uint4*>(stage_gen + lane * 128 + ((g ^ (lane & 7)) << 4)) = make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
    __syncwarp();
#pragma unroll
    for (int t = 0; t < kLanes; ++t) {
      if (kStep * t >= rows) continue;
      const int row = row0 + kStep * t;
      auto piece = [&](int h) { return reinterpret_cast<float4*>(stage_gen + row * 128 + (((col0 / 4 + h) ^ (row & 7)) << 4)); };
      if constexpr (kPer == 8) {
        const float4 x = *piece(0), y = *piece(1);
        float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        uint4 w, same;
        epi_pack8<false>(p.ea, v, &old[t], static_cast<unsigned long long>(m0 + row) * p.N + col, w, same);
        *reinterpret_cast<uint4*>(out + kStep * t * p.ldc) = w;
      } else {
        float4 x = *piece(0);
        float* v = &x.x;
        const uint32_t o[4] = {old[t].x, old[t].y, old[t].z, old[t].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = epi_scale(p.ea, v[i]);
          if (p.ea.beta != 0.0f) v[i] = fmaf(p.ea.beta, __uint_as_float(o[i]), v[i]);
        }
        *piece(0) = x;
      }
    }
    if (kPer == 4) fence_async_smem();
    __syncwarp();
    if (kPer == 4 && lane == 0) {
      tma_store_5d(mapC, stage, n0 + c, m0, 0, 0, 0);
      tma_store_commit();
    }
  }
}

// Which of these a kernel has: the lean form, and the others in fp16 or fp32. (One kernel with all of them was larger than the
// instruction cache: 1001 x 4097 x 125 in fp32 15.6 -> 19.8 us.)
enum OutForm { kOutLean, kOutF16, kOutF32 };
inline OutForm out_form(const OutParams& out) {
  return out.out_f32 ? kOutF32 : out.ea.beta == 0.0f && out.ea.sr_bits == 0 ? kOutLean : kOutF16;
}
template <int kForm, int kCols, typename F>
__device__ __forceinline__ void out_tile(const OutParams& p, const CUtensorMap* mapC, uint32_t taddr, uint32_t stage, uint8_t* stage_gen,
                                         int m0, int n0, F release) {
  using E = std::conditional_t<kForm == kOutF32, float, __half>;
  if constexpr (kForm == kOutLean) out_lean<kCols>(p, mapC, taddr, stage, stage_gen, m0, n0, release);
  else if (p.store) out_even<kCols, E>(p, mapC, taddr, stage, stage_gen, m0, n0, release);
  else out_odd<kCols, E>(p, taddr, stage_gen, m0, n0, release);
}

// What an fp32 C holds in 32 rows x kCols columns to the L2 cache, a tile before it is needed: 4096 x 9216 x 128 with C added
// 90 -> 76 us (fp16, of half as many bytes, was slower with it, 48 -> 52).
template <int kForm, int kCols>
__device__ __forceinline__ void out_ahead(const OutParams& p, int m0, int n0) {
  const int row = m0 + (threadIdx.x & 31);
  if (kForm != kOutF32 || p.ea.beta == 0.0f || row >= p.M || n0 >= p.N) return;
  const float* at = static_cast<const float*>(p.C) + row * p.ldc + n0;
  for (int c = 0; c < min(kCols, p.N - n0); c += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + c));
}

}  // namespace ngb
