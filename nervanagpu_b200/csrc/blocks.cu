// Matrices in blocks of small floating-point numbers: quantisation, values, and the ReLU mask from an 8-bit record
// (the formats and the layout are described in blocks.cuh).
//
// All three move each number once and are bound by that: a quantisation reads 2 or 4 bytes per number and writes
// half a byte or one, plus a scale per block. (A call with several outputs is a launch for each, which reads A.) Two forms
// each, by how the blocks lie in the plain matrix:
//   rows      neighbours of a block are neighbours in memory: a lane takes 16 of them, two share a block of 32, or (a
//             quantisation from fp16 to 4 bits) 32
//   strided   a thread takes whole blocks, lanes run along the other axis, which is then the contiguous one (the
//             usual case: a layer's inputs, features x images, in blocks of features); any strides
#include <algorithm>
#include <cmath>

#include "blocks.cuh"
#include "blocks.h"
#include "host.h"

namespace ngb {

namespace {

// Plain matrix as a kernel sees it: element (outer o, inner l) at o * so + l * sl elements.
template <typename T>
struct PlainView {
  T* p;
  long long so, sl;
  bool wide;        // rows form: every row starts on 32 bytes
};

__device__ __forceinline__ void from_f32(float v, __half& x) { x = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, float& x) { x = v; }
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

#define NG_DEPENDENT_PROLOGUE(early) \
  grid_dependency_wait();            \
  if (early) grid_launch_dependents()

// ---- rows form: 16 numbers per lane, or 32 ------------------------------------------------------------------
constexpr int kLane = 16;

// kCount neighbours as they lie in memory
template <typename T, int kCount = kLane>
struct Raw {
  static constexpr int kVecs = kCount * sizeof(T) / 16;
  uint4 v[kVecs];
  __device__ __forceinline__ T* at() { return reinterpret_cast<T*>(v); }
  __device__ __forceinline__ const T* at() const { return reinterpret_cast<const T*>(v); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // The first n of them at a 16-byte aligned address. wide: the rows are 32-byte aligned, and whole sectors
  // are moved at a time (by halves, the two accesses of a warp each touched every sector).
  __device__ __forceinline__ void load(const T* p, int n, bool wide) {
    if (n >= kCount && wide) {
#pragma unroll
      for (int i = 0; i < kVecs; i += 2)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w), "=r"(v[i + 1].x), "=r"(v[i + 1].y),
                       "=r"(v[i + 1].z), "=r"(v[i + 1].w)
                     : "l"(reinterpret_cast<const uint4*>(p) + i));
    } else if (n >= kCount) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      // (the end of a row: whole vectors as far as they go)
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        if ((i + 1) * kPer <= n) {
          v[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
          for (int j = i * kPer; j < (i + 1) * kPer; ++j) at()[j] = j < n ? p[j] : zero_of<T>();
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int n, bool wide) const {
    if (n >= kCount && wide) {
#pragma unroll
      for (int i = 0; i < kVecs; i += 2)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint4*>(p) + i),
                     "r"(v[i].x), "r"(v[i].y), "r"(v[i].z), "r"(v[i].w), "r"(v[i + 1].x), "r"(v[i + 1].y), "r"(v[i + 1].z),
                     "r"(v[i + 1].w)
                     : "memory");
    } else if (n >= kCount) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
    } else {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        if ((i + 1) * kPer <= n) {
          reinterpret_cast<uint4*>(p)[i] = v[i];
        } else {
#pragma unroll
          for (int j = i * kPer; j < (i + 1) * kPer; ++j)
            if (j < n) p[j] = at()[j];
        }
      }
    }
  }
};

// the h-th 8 of them in fp32
template <int kCount>
__device__ __forceinline__ void to_f32x8(const Raw<__half, kCount>& r, int h, float (&x)[8]) {
  const uint32_t w[4] = {r.v[h].x, r.v[h].y, r.v[h].z, r.v[h].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <int kCount>
__device__ __forceinline__ void to_f32x8(const Raw<float, kCount>& r, int h, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 w = r.v[2 * h + i];
    x[4 * i] = __uint_as_float(w.x); x[4 * i + 1] = __uint_as_float(w.y);
    x[4 * i + 2] = __uint_as_float(w.z); x[4 * i + 3] = __uint_as_float(w.w);
  }
}

// Largest magnitude of numbers 8 h0 .. 8 h1 - 1, as the bits of an fp32 number (above those of infinity for a NaN).
template <int kCount>
__device__ __forceinline__ uint32_t top_bits(const Raw<__half, kCount>& r, int h0, int h1) {
  __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
  for (int h = h0; h < h1; ++h) {
    const uint32_t w[4] = {r.v[h].x, r.v[h].y, r.v[h].z, r.v[h].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&w[j])));
  }
  return magnitude_bits(__half2float(__hmax_nan(__low2half(top), __high2half(top))));
}
template <int kCount>
__device__ __forceinline__ uint32_t top_bits(const Raw<float, kCount>& r, int h0, int h1) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 2 * h0; i < 2 * h1; ++i)
    top = max(max(top, r.v[i].x & 0x7fffffffu), max(r.v[i].y & 0x7fffffffu, max(r.v[i].z & 0x7fffffffu, r.v[i].w & 0x7fffffffu)));
  return top;
}

// Rows at addresses that are no multiples of 16 bytes: the warp moves its 32 kCount numbers (a run of kCount <<
// log_tx of each of its rows) in order, one number per lane and access, through shared memory. (A lane that moved its
// own 16 one by one touched 32 sectors per access: 139968 x 125 fp16 read back from 8 bits took 51 us.)
template <typename T, bool kStore, int kCount>
__device__ __forceinline__ void warp_move(T* base, long long so, long long o_first, int outer, int l_first, int inner, int log_tx, T* stage) {
  const int lane = threadIdx.x + threadIdx.y * blockDim.x & 31;
  const int per_row = log_tx + (kCount == 32 ? 5 : 4) - 7;      // logarithm: pieces of 128 in a row
  if (per_row < 0) {
    // short rows, several in 128 numbers
    const int run = 128 >> -per_row;
#pragma unroll 4
    for (int i = 0; i < kCount; ++i) {
      const int e = i * 32 + lane, l = l_first + (e & (run - 1));
      const long long o = o_first + (e >> (7 + per_row));
      const bool live = o < outer && l < inner;
      if (!kStore) stage[e] = live ? base[o * so + l] : zero_of<T>();
      else if (live) base[o * so + l] = stage[e];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kCount / 4; ++i) {
    const long long o = o_first + (i >> per_row);
    const int l = l_first + (i & ((1 << per_row) - 1)) * 128 + lane;
    T* p = base + o * so + l;
    T* s = stage + i * 128 + lane;
    const int n = o < outer ? inner - l : 0;
    if (kStore) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j * 32 < n) p[j * 32] = s[j * 32];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j * 32] = j * 32 < n ? p[j * 32] : zero_of<T>();
    }
  }
}
template <typename T, int kCount>
__device__ __forceinline__ void warp_load(const T* base, long long so, long long o_first, int outer, int l_first, int inner, int log_tx,
                                          T* stage, Raw<T, kCount>& r) {
  const int lane = threadIdx.x + threadIdx.y * blockDim.x & 31;
  warp_move<T, false, kCount>(const_cast<T*>(base), so, o_first, outer, l_first, inner, log_tx, stage);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < Raw<T, kCount>::kVecs; ++i) r.v[i] = reinterpret_cast<const uint4*>(stage + lane * kCount)[i];
  __syncwarp();
}
template <typename T, int kCount>
__device__ __forceinline__ void warp_store(T* base, long long so, long long o_first, int outer, int l_first, int inner, int log_tx,
                                           T* stage, const Raw<T, kCount>& r) {
  const int lane = threadIdx.x + threadIdx.y * blockDim.x & 31;
#pragma unroll
  for (int i = 0; i < Raw<T, kCount>::kVecs; ++i) reinterpret_cast<uint4*>(stage + lane * kCount)[i] = r.v[i];
  __syncwarp();
  warp_move<T, true, kCount>(base, so, o_first, outer, l_first, inner, log_tx, stage);
  __syncwarp();
}

// One step of a rows kernel: this thread's row, and the warp's first row and first group (warp_load).
// (Rows that are moved through shared memory have CTAs of 128 threads.)
#define NG_ROWS_PROLOGUE(T, count)                                                                      \
  __shared__ __align__(16) T stage_all[kVec ? 1 : 128 * count];                                         \
  const int tid = threadIdx.x + threadIdx.y * blockDim.x;                                               \
  T* stage = kVec ? stage_all : stage_all + (tid & ~31) * count;                                        \
  const int log_tx = min(31 - __clz(blockDim.x), 5);      /* lanes of one warp in a row */              \
  const int g = blockIdx.x * blockDim.x + threadIdx.x, n = q.inner - g * count;                         \
  const int l_warp = (g - (tid & 31 & (static_cast<int>(blockDim.x) - 1))) * count;                     \
  const int y_warp = (tid & ~31) / static_cast<int>(blockDim.x);                                        \
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y

// Numbers per lane in a quantisation: 32 from fp16 to 4 bits, where what a block and a row cost besides, some 50
// instructions, counted more than the numbers themselves with 16 (4096 x 9216 nvfp4 18.1 -> 16.1 us); with the wider
// codes or numbers they take too many registers (1001 x 4097 fp32 8.3 -> 9.4, 139968 x 125 mxfp8 15.0 -> 16.3).
template <typename T, int kFmt>
__host__ __device__ constexpr int quantize_lane() {
  return BlockFormat<kFmt>::k4 && sizeof(T) == 2 ? 32 : 16;
}

// kForm: 0 rows at odd addresses; 1 aligned rows; 2 aligned rows of less than 128 numbers, with fewer lanes than share a word
// of scales (the test for that costs the others 0.8 of 10.3 us, 139968 x 128 mxfp8).
template <typename T, int kFmt, int kForm>
__global__ void __launch_bounds__(256, kForm == 0 && sizeof(T) == 4 ? 6 : 4) quantize_rows_kernel(BlockView q, PlainView<const T> a, int early) {
  NG_DEPENDENT_PROLOGUE(early);
  using F = BlockFormat<kFmt>;
  constexpr bool kVec = kForm != 0;
  constexpr int kPer = quantize_lane<T, kFmt>();
  NG_ROWS_PROLOGUE(T, kPer);
  constexpr int kUnroll = kVec ? 2 : 1;                             // rows whose loads are in flight together
  constexpr int kBlocks = kPer > F::kBlock ? kPer / F::kBlock : 1;  // of a lane
  constexpr int kDup = kPer < F::kBlock ? 2 : 1;                    // lanes that share one
  constexpr int kSharers = 4 / kBlocks;                             // lanes whose scales make a word, the sharing ones once
  constexpr int kEights = kPer / 8 / kBlocks;
  // (whole warps stay to the end of the loop: lanes exchange magnitudes and scales)
  for (long long o0 = static_cast<long long>(blockIdx.y) * blockDim.y; o0 < q.outer; o0 += kUnroll * step) {
    Raw<T, kPer> raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long o = o0 + u * step + threadIdx.y;
      if (kVec) {
        raw[u].clear();
        if (o < q.outer && n > 0) raw[u].load(a.p + o * a.so + static_cast<long long>(g) * kPer, n, a.wide);
      } else {
        warp_load(a.p, a.so, o0 + u * step + y_warp, q.outer, l_warp, q.inner, log_tx, stage, raw[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long o = o0 + u * step + threadIdx.y;
      const bool live = o < q.outer && n > 0;
      uint2 c[kPer / 8];
      uint32_t word = 0u;           // this lane's scales
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        uint32_t top = top_bits(raw[u], b * kEights, (b + 1) * kEights);
        if (kDup == 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        const BlockScale s = block_scale<kFmt, sizeof(T) == 2>(top, q.t);
        if (live && b * F::kBlock < n) word |= s.byte << (8 * b);
        bool done = false;
        if constexpr (!F::k4 && sizeof(T) == 2) {
          // (by up to 2^30 is two fp16 factors; a block of zeros needs none)
          if (!s.nan && (s.by <= 1073741824.0f || top == 0u)) {
            done = true;
            __half2 by0, by1;
            block_scale_f16(s.by, by0, by1);
#pragma unroll
            for (int h = 0; h < kEights; ++h) {
              c[h].x = block_encode4_f16(raw[u].v[h].x, raw[u].v[h].y, by0, by1);
              c[h].y = block_encode4_f16(raw[u].v[h].z, raw[u].v[h].w, by0, by1);
            }
          }
        }
        if (!done) {
#pragma unroll
          for (int h = b * kEights; h < (b + 1) * kEights; ++h) {
            float x[8];
            to_f32x8(raw[u], h, x);
            c[h] = block_encode8<kFmt, sizeof(T) == 2>(x, s);
          }
        }
      }
      // the scales of four blocks leave together
      word <<= 8 * kBlocks * (g / kDup % kSharers);
#pragma unroll
      for (int d = 1; d < kSharers; d *= 2) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, word, d * kDup);
        if (kForm == 1 || d * kDup < static_cast<int>(blockDim.x)) word |= other;
      }
      if (live) {
        uint8_t* dst = q.codes + F::code_at(q, static_cast<int>(o), g * (kPer / 8ll * F::kBytes8));
        if (!F::k4) *reinterpret_cast<uint4*>(dst) = make_uint4(c[0].x, c[0].y, c[1].x, c[1].y);
        else if (kPer == 32) *reinterpret_cast<uint4*>(dst) = make_uint4(c[0].x, c[1].x, c[kPer / 8 - 2].x, c[kPer / 8 - 1].x);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(c[0].x, c[1].x);
        if (g % (kSharers * kDup) == 0)
          *reinterpret_cast<uint32_t*>(q.scales + F::scale_at(q, static_cast<int>(o), g / kDup * kBlocks)) = word;
      }
    }
  }
}

template <typename T, int kFmt, bool kVec>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(BlockView q, PlainView<T> a, int early) {
  NG_DEPENDENT_PROLOGUE(early);
  using F = BlockFormat<kFmt>;
  NG_ROWS_PROLOGUE(T, kLane);
  constexpr int kShare = F::kNv ? 1 : 2;
  constexpr int kUnroll = kVec ? 2 : 1;
  for (long long o0 = static_cast<long long>(blockIdx.y) * blockDim.y; o0 < q.outer; o0 += kUnroll * step) {
    uint4 codes[kUnroll];
    uint32_t byte[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long o = o0 + u * step + threadIdx.y;
      codes[u] = make_uint4(0u, 0u, 0u, 0u);
      byte[u] = 0u;
      if (o < q.outer && n > 0) {
        const uint8_t* src = q.codes + F::code_at(q, static_cast<int>(o), static_cast<long long>(g) * (2 * F::kBytes8));
        if (F::k4) {
          const uint2 c = *reinterpret_cast<const uint2*>(src);
          codes[u].x = c.x;
          codes[u].z = c.y;
        } else {
          codes[u] = *reinterpret_cast<const uint4*>(src);
        }
        byte[u] = q.scales[F::scale_at(q, static_cast<int>(o), g / kShare)];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long o = o0 + u * step + threadIdx.y;
      const float scale = block_scale_value<kFmt>(byte[u], q.t);
      Raw<T> r;
      if (sizeof(T) == 2 && block_scale_fits_f16<kFmt>(scale)) {
        const __half2 by = __float2half2_rn(scale);
        r.v[0] = block_decode8_f16<kFmt>(make_uint2(codes[u].x, codes[u].y), by);
        r.v[1] = block_decode8_f16<kFmt>(make_uint2(codes[u].z, codes[u].w), by);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          block_decode8<kFmt>(h == 0 ? make_uint2(codes[u].x, codes[u].y) : make_uint2(codes[u].z, codes[u].w), scale, v);
          block_limit<kFmt, T>(scale, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) from_f32(v[i], r.at()[8 * h + i]);
        }
      }
      if (!kVec) warp_store(a.p, a.so, o0 + u * step + y_warp, q.outer, l_warp, q.inner, log_tx, stage, r);
      else if (o < q.outer && n > 0) r.store(a.p + o * a.so + static_cast<long long>(g) * kLane, n, a.wide);
    }
  }
}

// a code of a number that is not positive: 0, or with the sign bit
__device__ __forceinline__ bool not_positive(uint32_t code) { return code - 1u >= 0x7fu; }

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) relu_mask_rows_kernel(BlockView q, PlainView<T> a, int early) {
  NG_DEPENDENT_PROLOGUE(early);
  const int tid = threadIdx.x + threadIdx.y * blockDim.x, lane = tid & 31;
  const int log_tx = min(31 - __clz(blockDim.x), 5);
  const int g = blockIdx.x * blockDim.x + threadIdx.x, n = q.inner - g * kLane;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  for (long long o0 = static_cast<long long>(blockIdx.y) * blockDim.y; o0 < q.outer; o0 += step) {
    const long long o = o0 + threadIdx.y;
    const bool live = o < q.outer && n > 0;
    uint4 codes = make_uint4(0u, 0u, 0u, 0u);
    if (live) codes = *reinterpret_cast<const uint4*>(q.codes + o * q.pitch + static_cast<long long>(g) * kLane);
    uint32_t off = 0u;       // bit i: number i was not positive
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const uint32_t w = i < 4 ? codes.x : i < 8 ? codes.y : i < 12 ? codes.z : codes.w;
      off |= (not_positive(w >> (8 * (i & 3)) & 0xffu) ? 1u : 0u) << i;
    }
    if (kVec) {
      if (!live) continue;
      T* p = a.p + o * a.so + static_cast<long long>(g) * kLane;
      Raw<T> r;
      r.load(p, n, a.wide);
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if (off >> i & 1u) r.at()[i] = zero_of<T>();
      r.store(p, n, a.wide);
    } else {
      // zeros, one number per lane and access, in the order of warp_move
      const int l_warp = (g - (lane & (static_cast<int>(blockDim.x) - 1))) * kLane;
      const long long o_warp = o0 + (tid & ~31) / static_cast<int>(blockDim.x);
      if (log_tx < 3) {
#pragma unroll 4
        for (int i = 0; i < kLane; ++i) {
          const int e = i * 32 + lane, l = l_warp + (e & ((16 << log_tx) - 1));
          const long long row = o_warp + (e >> (4 + log_tx));
          const uint32_t mask = __shfl_sync(0xffffffffu, off, i * 2 + (lane >> 4));
          if ((mask >> (lane & 15) & 1u) && row < q.outer && l < q.inner) a.p[row * a.so + l] = zero_of<T>();
        }
        continue;
      }
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const long long row = o_warp + (i >> (log_tx - 3));
        const int l = l_warp + (i & ((1 << (log_tx - 3)) - 1)) * 128 + lane;
        T* p = a.p + row * a.so + l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t mask = __shfl_sync(0xffffffffu, off, i * 8 + j * 2 + (lane >> 4));
          if ((mask >> (lane & 15) & 1u) && row < q.outer && l + j * 32 < q.inner) p[j * 32] = zero_of<T>();
        }
      }
    }
  }
}

// ---- strided form --------------------------------------------------------------------------------------
// A CTA takes 64 outer rows x 4 blocks: half a tile of 4-bit scales, and 32 to 128 neighbouring bytes of codes per outer
// row, so that a quantisation leaves in whole sectors through shared memory. A warp has one block, a lane two outer
// rows: neighbours, in one access, where the outer axis is the contiguous one in aligned pairs (a quantisation
// from fp16: at any address; words put together for the way back were slower than numbers, 16.8 to 13.9 us); else 32 apart,
// one by one. (Four rows per lane were faster for large matrices by 5 % and took 6.7 us instead of 2.9 for a minibatch of
// 9216 x 128, with too few warps to hide their latency.)
constexpr int kStridedThreads = 128;
constexpr int kStridedRows = 64;

template <int kFmt>
struct StridedTile {
  using F = BlockFormat<kFmt>;
  static constexpr int kBytes = F::kBlock / 8 * F::kBytes8;     // of a block's codes
  static constexpr int kRow = 4 * kBytes;
  static constexpr int kPitch = kRow + 16;                      // (rows in shared memory, off each other's banks)
};
// Two numbers of neighbouring outer rows as they lie in memory.
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using Vec = uint32_t;
  static __device__ __forceinline__ Vec of(__half a, __half b) { return __half_as_ushort(a) | static_cast<uint32_t>(__half_as_ushort(b)) << 16; }
  static __device__ __forceinline__ float get(Vec v, int j) {
    const __half2 h = *reinterpret_cast<const __half2*>(&v);
    return j ? __high2float(h) : __low2float(h);
  }
};
template <>
struct Pair<float> {
  using Vec = uint2;
  static __device__ __forceinline__ Vec of(float a, float b) { return make_uint2(__float_as_uint(a), __float_as_uint(b)); }
  static __device__ __forceinline__ float get(Vec v, int j) { return __uint_as_float(j ? v.y : v.x); }
};
// Largest magnitudes of both rows, as the bits of fp32 numbers.
template <int kN>
__device__ __forceinline__ void top_of_pairs(const uint32_t (&raw)[kN], uint32_t (&top)[2]) {
  __half2 t = __half2half2(__ushort_as_half(0));
#pragma unroll
  for (int i = 0; i < kN; ++i) t = __hmax2_nan(t, __habs2(*reinterpret_cast<const __half2*>(&raw[i])));
  top[0] = magnitude_bits(__low2float(t));
  top[1] = magnitude_bits(__high2float(t));
}
template <int kN>
__device__ __forceinline__ void top_of_pairs(const uint2 (&raw)[kN], uint32_t (&top)[2]) {
  top[0] = top[1] = 0u;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    top[0] = max(top[0], raw[i].x & 0x7fffffffu);
    top[1] = max(top[1], raw[i].y & 0x7fffffffu);
  }
}
// How the outer rows lie in memory: anyhow; as neighbours in aligned pairs; as neighbours (fp16) at any address.
enum StridedForm { kStridedAny, kStridedPairs, kStridedShifted };
// row of the tile that is this lane's j-th
template <bool kNeighbours>
__device__ __forceinline__ int strided_row(int j) {
  const int lane = threadIdx.x & 31;
  return kNeighbours ? 2 * lane + j : lane + 32 * j;
}

template <typename T, int kFmt, int kForm>
__global__ void __launch_bounds__(kStridedThreads) quantize_strided_kernel(BlockView q, PlainView<const T> a, int early, int blocks) {
  NG_DEPENDENT_PROLOGUE(early);
  using F = BlockFormat<kFmt>;
  using S = StridedTile<kFmt>;
  using P = Pair<T>;
  __shared__ __align__(16) uint8_t codes[kStridedRows * S::kPitch];
  __shared__ __align__(16) uint8_t scales[kStridedRows * 4];
  const int which = threadIdx.x >> 5;               // of the four blocks
  const int o0 = blockIdx.x * kStridedRows;
  for (int b0 = blockIdx.y * 4; b0 < blocks; b0 += gridDim.y * 4) {
    const int b = b0 + which;
    const int n = q.inner - b * F::kBlock;          // numbers of the block that exist
    typename P::Vec raw[F::kBlock];
    const T* p = a.p + static_cast<long long>(b) * F::kBlock * a.sl;
    const int r0 = o0 + strided_row<kForm != kStridedAny>(0), r1 = o0 + strided_row<kForm != kStridedAny>(1);
    if constexpr (kForm == kStridedShifted) {
      // Numbers 2 lane and 2 lane + 1 of each run, from aligned words: where a run starts in the middle of one, a lane
      // loads the word behind that, and its first number is the second of the lane below. The first number of such a run,
      // and the last of one that ends in the middle of a word, are loaded by a lane per run. (4097 x 125 from 2.7 to 2.3
      // us, 6168 x 3385 from 15.5 to 11.8. Two loads into one register, for either case, would wait for each other: 4.1.)
      const int lane = threadIdx.x & 31, last = q.outer - 1 - o0;
      const T* run = p + o0;
      // which runs start in the middle of a word: the even ones, the odd ones
      const int odd[2] = {static_cast<int>(reinterpret_cast<uintptr_t>(run) >> 1) & 1,
                          static_cast<int>(reinterpret_cast<uintptr_t>(run + a.sl) >> 1) & 1};
      const bool whole[2] = {2 * lane + odd[0] < last, 2 * lane + odd[1] < last};
      uint32_t ends = 0u;         // first and last number of run `lane`
      if (lane < min(n, F::kBlock)) {
        const unsigned short* at = reinterpret_cast<const unsigned short*>(run + lane * a.sl);
        ends = at[0] | static_cast<uint32_t>(at[min(last, kStridedRows - 1)]) << 16;
      }
      const T* at = run + 2 * lane;
#pragma unroll
      for (int i = 0; i < F::kBlock; ++i, at += a.sl)
        raw[i] = i < n && whole[i & 1] ? *reinterpret_cast<const uint32_t*>(at + odd[i & 1]) : 0u;
#pragma unroll
      for (int i = 0; i < F::kBlock; ++i) {
        const uint32_t e = __shfl_sync(0xffffffffu, ends, i);
        if (2 * lane + odd[i & 1] == last) raw[i] = e >> 16;
        const uint32_t below = __shfl_up_sync(0xffffffffu, raw[i], 1);
        if (odd[i & 1]) raw[i] = __byte_perm(lane == 0 ? e << 16 : below, raw[i], 0x5432);
      }
    } else if (kForm == kStridedPairs) {
      const T* p0 = p + r0;
      if (r0 < q.outer && n >= F::kBlock) {
#pragma unroll
        for (int i = 0; i < F::kBlock; ++i) raw[i] = *reinterpret_cast<const typename P::Vec*>(p0 + i * a.sl);
      } else {
#pragma unroll
        for (int i = 0; i < F::kBlock; ++i) {
          raw[i] = P::of(zero_of<T>(), zero_of<T>());
          if (r0 < q.outer && i < n) raw[i] = *reinterpret_cast<const typename P::Vec*>(p0 + i * a.sl);
        }
      }
    } else {
      const T *p0 = p + r0 * a.so, *p1 = p + r1 * a.so;
#pragma unroll
      for (int i = 0; i < F::kBlock; ++i)
        raw[i] = P::of(r0 < q.outer && i < n ? p0[i * a.sl] : zero_of<T>(), r1 < q.outer && i < n ? p1[i * a.sl] : zero_of<T>());
    }
    uint32_t top[2];
    top_of_pairs(raw, top);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = strided_row<kForm != kStridedAny>(j);
      const BlockScale s = block_scale<kFmt, sizeof(T) == 2>(top[j], q.t);
      uint8_t* dst = codes + row * S::kPitch + which * S::kBytes;
#pragma unroll
      for (int h = 0; h < F::kBlock / 8; ++h) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = P::get(raw[8 * h + i], j);
        const uint2 c = block_encode8<kFmt, sizeof(T) == 2>(x, s);
        if (F::k4) *reinterpret_cast<uint32_t*>(dst + 4 * h) = c.x;
        else *reinterpret_cast<uint2*>(dst + 8 * h) = c;
      }
      scales[row * 4 + which] = n > 0 && o0 + row < q.outer ? static_cast<uint8_t>(s.byte) : 0;
    }
    __syncthreads();
    // (what lies behind the last number is zero; 4-bit rows are padded to four blocks and more, mxfp8 rows to one)
#pragma unroll
    for (int i = threadIdx.x; i < kStridedRows * (S::kRow / 16); i += kStridedThreads) {
      const int row = i / (S::kRow / 16), c = i % (S::kRow / 16);
      if (o0 + row < q.outer && (F::k4 || b0 * S::kBytes + c * 16ll < q.pitch))
        *reinterpret_cast<uint4*>(q.codes + F::code_at(q, o0 + row, static_cast<long long>(b0) * S::kBytes + c * 16)) =
            *reinterpret_cast<const uint4*>(codes + row * S::kPitch + c * 16);
    }
    const uint32_t* words = reinterpret_cast<const uint32_t*>(scales);
    if (F::k4) {
      if (threadIdx.x < 32)
        *reinterpret_cast<uint2*>(q.scales + F::scale_at(q, o0, b0) + threadIdx.x * 16) = make_uint2(words[threadIdx.x], words[threadIdx.x + 32]);
    } else if (threadIdx.x < kStridedRows && o0 + static_cast<int>(threadIdx.x) < q.outer) {
      *reinterpret_cast<uint32_t*>(q.scales + F::scale_at(q, o0 + threadIdx.x, b0)) = words[threadIdx.x];
    }
    __syncthreads();
  }
}

// (units of 16 numbers: with whole blocks of 32 per thread a minibatch of 9216 x 128 had too few warps, 3.0 us. Codes are
// read unit by unit: the warps of a CTA find each other's neighbours in the L1 cache.)
template <typename T, int kFmt, bool kVec>
__global__ void __launch_bounds__(kStridedThreads) dequantize_strided_kernel(BlockView q, PlainView<T> a, int early, int units) {
  NG_DEPENDENT_PROLOGUE(early);
  using F = BlockFormat<kFmt>;
  using P = Pair<T>;
  constexpr int kWords = F::k4 ? 2 : 4;            // of 16 codes
  const int o0 = blockIdx.x * kStridedRows;
  const int r[2] = {o0 + strided_row<kVec>(0), o0 + strided_row<kVec>(1)};
  for (int b = blockIdx.y * 4 + (threadIdx.x >> 5); b < units; b += gridDim.y * 4) {
    const int n = q.inner - b * 16;
    uint32_t w[2][kWords];
    float scale[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < kWords / 2; ++i) {
        uint2 c = make_uint2(0u, 0u);
        if (r[j] < q.outer) c = *reinterpret_cast<const uint2*>(q.codes + F::code_at(q, r[j], b * (4ll * kWords) + 8 * i));
        w[j][2 * i] = c.x;
        w[j][2 * i + 1] = c.y;
      }
      scale[j] = block_scale_value<kFmt>(r[j] < q.outer ? q.scales[F::scale_at(q, r[j], b / (F::kBlock / 16))] : 0u, q.t);
    }
    T* p = a.p + b * 16ll * a.sl;
    T *p0 = p + r[0] * a.so, *p1 = p + r[1] * a.so;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      T v[2][8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float f[8];
        block_decode8<kFmt>(F::k4 ? make_uint2(w[j][h], 0u) : make_uint2(w[j][2 * h], w[j][2 * h + 1]), scale[j], f);
        block_limit<kFmt, T>(scale[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) from_f32(f[i], v[j][i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long at = (8 * h + i) * a.sl;
        const bool live = 8 * h + i < n;
        if (kVec) {
          if (live && r[0] < q.outer) *reinterpret_cast<typename P::Vec*>(p0 + at) = P::of(v[0][i], v[1][i]);
        } else {
          if (live && r[0] < q.outer) p0[at] = v[0][i];
          if (live && r[1] < q.outer) p1[at] = v[1][i];
        }
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) relu_mask_strided_kernel(BlockView q, PlainView<T> a, int early, int blocks) {
  NG_DEPENDENT_PROLOGUE(early);
  const int o = blockIdx.x * 32 + threadIdx.x;
  if (o >= q.outer) return;
  for (int b = blockIdx.y * 8 + threadIdx.y; b < blocks; b += gridDim.y * 8) {
    T* p = a.p + o * a.so + b * 32ll * a.sl;
    const uint4* src = reinterpret_cast<const uint4*>(q.codes + o * q.pitch + b * 32ll);
    const uint4 lo = src[0], hi = src[1];
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    const int n = q.inner - b * 32;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < n && not_positive(w[i / 4] >> (8 * (i & 3)) & 0xffu)) p[i * a.sl] = zero_of<T>();
  }
}

// ---- launches ------------------------------------------------------------------------------------
struct RowGrid {
  dim3 grid, block;
};
template <typename K, typename V>
cudaError_t launch_with(const cudaLaunchConfig_t& cfg, K kernel, int early, const BlockView& q, const V& a) {
  return cudaLaunchKernelEx(&cfg, kernel, q, a, early);
}
template <typename K, typename V>
cudaError_t launch_with(const cudaLaunchConfig_t& cfg, K kernel, int early, const BlockView& q, const V& a, int blocks) {
  return cudaLaunchKernelEx(&cfg, kernel, q, a, early, blocks);
}
// Set up while the kernel before it in the stream drains; the kernel after it may do the same at once (`early`) where
// this one's blocks are all resident from the start, so that the next one's take no room from those still to come.
template <typename... P, typename... A>
int launch(const DeviceCtx* c, void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t stream, const BlockView& q, A... rest) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tuning().dependent_launch != 0 ? 1 : 0;
  const int early = static_cast<long long>(grid.x) * grid.y <= 2ll * c->sm_count;
  NG_CUDA(launch_with(cfg, kernel, early, q, rest...));
  NG_CHECK_LAUNCH();
  return NG_OK;
}
// Lanes per row: its groups of `count` numbers, over CTAs of so many threads with as few idle lanes as a power of two allows;
// the other threads take other rows. The scales of four blocks leave together, so a row has no fewer lanes than 128 numbers
// take, unless all of it fits into fewer (a shared block's two at least).
RowGrid row_grid(const DeviceCtx* c, const BlockView& q, int threads, int count, int least) {
  const int few = 128 / count;
  int groups = static_cast<int>((q.inner + count - 1ll) / count), tx = threads;
  if (groups < few) {
    for (tx = least; tx < groups; tx *= 2) {}
    groups = tx;
  } else {
    groups = (groups + few - 1) / few * few;
    while (tx > few && (groups + tx / 2 - 1) / (tx / 2) * (tx / 2) < (groups + tx - 1) / tx * tx) tx /= 2;
  }
  const int ty = threads / tx;
  RowGrid r;
  r.block = dim3(tx, ty);
  const long long gx = (groups + tx - 1) / tx, rows = (static_cast<long long>(q.outer) + ty - 1) / ty;
  const long long room = std::max(1ll, 4096ll / threads * c->sm_count / gx);
  r.grid = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(std::min(std::min(rows, room), 65535ll)));
  return r;
}
RowGrid strided_grid(const BlockView& q, int blocks) {
  RowGrid r;
  r.block = dim3(32, 8);
  r.grid = dim3(static_cast<unsigned>((q.outer + 31ll) / 32), static_cast<unsigned>(std::min((blocks + 7) / 8, 65535)));
  return r;
}

// rows that start on multiples of `bytes`
template <typename T>
bool aligned_rows(const PlainView<T>& a, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(a.p) & (bytes - 1)) == 0 && (a.so * static_cast<long long>(sizeof(T))) % bytes == 0;
}

// outer rows that lie two by two in aligned vectors
template <typename T>
bool aligned_pairs(const BlockView& q, const PlainView<T>& a) {
  return a.so == 1 && q.outer % 2 == 0 && a.sl % 2 == 0 && (reinterpret_cast<uintptr_t>(a.p) & (2 * sizeof(T) - 1)) == 0;
}

// neighbours to be quantised from any address (fp32 numbers, one per lane, fill an access as it is)
template <typename T>
constexpr int kNeighbours = sizeof(T) == 2 ? kStridedShifted : kStridedAny;

template <typename T, int kFmt>
int quantize_one(DeviceCtx* c, const BlockView& q, PlainView<const T> a, cudaStream_t stream) {
  const int blocks = (q.inner + BlockFormat<kFmt>::kBlock - 1) / BlockFormat<kFmt>::kBlock;
  int rc;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q, aligned_rows(a, 16) ? 256 : 128, quantize_lane<T, kFmt>(), quantize_lane<T, kFmt>() < BlockFormat<kFmt>::kBlock ? 2 : 1);
    a.wide = aligned_rows(a, 32);
    if (!aligned_rows(a, 16)) rc = launch(c, quantize_rows_kernel<T, kFmt, 0>, g.grid, g.block, stream, q, a);
    else if (g.block.x * quantize_lane<T, kFmt>() >= 128) rc = launch(c, quantize_rows_kernel<T, kFmt, 1>, g.grid, g.block, stream, q, a);
    else rc = launch(c, quantize_rows_kernel<T, kFmt, 2>, g.grid, g.block, stream, q, a);
  } else {
    const dim3 grid((q.outer + kStridedRows - 1) / kStridedRows, std::min((blocks + 3) / 4, 65535));
    if (aligned_pairs(q, a)) rc = launch(c, quantize_strided_kernel<T, kFmt, kStridedPairs>, grid, dim3(kStridedThreads), stream, q, a, blocks);
    else if (sizeof(T) == 2 && a.so == 1) rc = launch(c, quantize_strided_kernel<T, kFmt, kNeighbours<T>>, grid, dim3(kStridedThreads), stream, q, a, blocks);
    else rc = launch(c, quantize_strided_kernel<T, kFmt, kStridedAny>, grid, dim3(kStridedThreads), stream, q, a, blocks);
  }
  return rc;
}

template <typename T, int kFmt>
int dequantize_one(DeviceCtx* c, const BlockView& q, PlainView<T> a, cudaStream_t stream) {
  const int units = (q.inner + 15) / 16;
  int rc;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q, aligned_rows(a, 16) ? 256 : 128, kLane, 1);
    a.wide = aligned_rows(a, 32);
    if (aligned_rows(a, 16)) rc = launch(c, dequantize_rows_kernel<T, kFmt, true>, g.grid, g.block, stream, q, a);
    else rc = launch(c, dequantize_rows_kernel<T, kFmt, false>, g.grid, g.block, stream, q, a);
  } else {
    const dim3 grid((q.outer + kStridedRows - 1) / kStridedRows, std::min((units + 3) / 4, 65535));
    if (aligned_pairs(q, a)) rc = launch(c, dequantize_strided_kernel<T, kFmt, true>, grid, dim3(kStridedThreads), stream, q, a, units);
    else rc = launch(c, dequantize_strided_kernel<T, kFmt, false>, grid, dim3(kStridedThreads), stream, q, a, units);
  }
  return rc;
}

template <typename T>
int relu_mask_one(DeviceCtx* c, const BlockView& q, PlainView<T> a, cudaStream_t stream) {
  const int blocks = (q.inner + 31) / 32;
  int rc;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q, aligned_rows(a, 16) ? 256 : 128, kLane, 1);
    a.wide = aligned_rows(a, 32);
    if (aligned_rows(a, 16)) rc = launch(c, relu_mask_rows_kernel<T, true>, g.grid, g.block, stream, q, a);
    else rc = launch(c, relu_mask_rows_kernel<T, false>, g.grid, g.block, stream, q, a);
  } else {
    const RowGrid g = strided_grid(q, blocks);
    rc = launch(c, relu_mask_strided_kernel<T>, g.grid, g.block, stream, q, a, blocks);
  }
  return rc;
}

#define NG_BY_FORMAT(fmt, call)                                   \
  switch (fmt) {                                                  \
    case NG_BLOCK_MXFP4: { constexpr int kF = NG_BLOCK_MXFP4; call; } break; \
    case NG_BLOCK_NVFP4: { constexpr int kF = NG_BLOCK_NVFP4; call; } break; \
    default: { constexpr int kF = NG_BLOCK_MXFP8; call; } break;  \
  }

}  // namespace

// rows of a tile of a 4-bit format
int block_tile_rows(int outer) { return outer <= 16 ? 16 : outer <= 32 ? 32 : outer <= 64 ? 64 : 128; }

// what the sizes give, in bytes
static void block_pitches(const ng_block_desc& d, BlockView& v) {
  v.outer = d.axis ? d.rows : d.cols;
  v.inner = d.axis ? d.cols : d.rows;
  if (d.format == NG_BLOCK_MXFP8) {
    v.tile = 0;
    v.pitch = (v.inner + 31ll) / 32 * 32;
    v.spitch = (v.inner + 127ll) / 128 * 4;
  } else {
    const long long kbs = (v.inner + 255ll) / 256;
    v.tile = block_tile_rows(v.outer) * kTileRow;
    v.pitch = kbs * v.tile;
    v.spitch = kbs * (d.format == NG_BLOCK_NVFP4 ? 4 : 2) * kScaleTile;
  }
}

int check_shape(const ng_block_desc* d) {
  if (!d) return fail(NG_ERR_INVALID_ARG, "block matrix is null");
  if (d->format < NG_BLOCK_MXFP4 || d->format > NG_BLOCK_MXFP8) return fail(NG_ERR_INVALID_ARG, "unknown block format %d", d->format);
  if (d->axis != 0 && d->axis != 1) return fail(NG_ERR_INVALID_ARG, "blocks run along axis 0 or 1");
  if (d->rows < 1 || d->cols < 1) return fail(NG_ERR_INVALID_ARG, "a matrix in blocks has at least one row and column");
  if (d->rows > 0x7fff0000 || d->cols > 0x7fff0000) return fail(NG_ERR_TOO_LARGE, "a matrix in blocks has at most 2^31 - 65536 rows and columns");
  if (d->format == NG_BLOCK_NVFP4) {
    int ex = 0;
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale) || std::frexp(d->scale, &ex) != 0.5f || ex < -31 || ex > 33)
      return fail(NG_ERR_INVALID_ARG, "the scale of an nvfp4 matrix is a power of two from 2^-32 to 2^32");
  } else if (d->scale != 1.0f) {
    return fail(NG_ERR_INVALID_ARG, "only nvfp4 matrices have a scale");
  }
  return NG_OK;
}

int block_view(const DeviceCtx* c, const ng_block_desc* d, BlockView& v) {
  const int rc = check_shape(d);
  if (rc != NG_OK) return rc;
  if (!d->codes || !d->scales) return fail(NG_ERR_INVALID_ARG, "block matrix without memory");
  if ((reinterpret_cast<uintptr_t>(d->codes) | reinterpret_cast<uintptr_t>(d->scales)) & 127)
    return fail(NG_ERR_INVALID_ARG, "codes and scales must be 128-byte aligned");
  if (d->device != c->device) return fail(NG_ERR_INVALID_ARG, "block matrix of device %d, the current device is %d", d->device, c->device);
  block_pitches(*d, v);
  v.codes = static_cast<uint8_t*>(d->codes);
  v.scales = static_cast<uint8_t*>(d->scales);
  v.t = d->scale;
  return NG_OK;
}

int plain_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_cols, int box_rows, int esz) {
  const uint64_t dims[5] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1, 1, 1};
  const uint64_t row = static_cast<uint64_t>(ld) * esz, all = row * rows;
  const uint64_t strides[4] = {row, all, all, all};
  const uint32_t box[5] = {static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows), 1, 1, 1};
  return make_tensor_map(map, base, dims, strides, box, esz);
}

OutParams make_out(void* C, int m, int n, int ldc, int out_f32, const EpiArgs& ea) {
  OutParams out = {};
  out.M = m; out.N = n; out.C = C; out.ldc = ldc; out.out_f32 = out_f32; out.ea = ea;
  // (a box that leaves the matrix is cut at whole 16 bytes: rows that end inside one, in a wider matrix, would have their
  // neighbours overwritten)
  const int per16 = out_f32 ? 4 : 8;
  out.store = (reinterpret_cast<uintptr_t>(C) & 15u) == 0 && ldc % per16 == 0 && n % per16 == 0;
  return out;
}

int out_map(CUtensorMap* map, const OutParams& out) {
  return plain_map(map, out.C, out.M, out.N, out.ldc, out.out_f32 ? 32 : 64, 32, out.out_f32 ? 4 : 2);
}

int dequantize_f16(DeviceCtx* c, const ng_block_desc& d, const BlockView& q, __half* out, long long ld, cudaStream_t stream) {
  PlainView<__half> a = {out, ld, 1};
  NG_BY_FORMAT(d.format, return (dequantize_one<__half, kF>(c, q, a, stream)));
  return NG_OK;
}

}  // namespace ngb

using namespace ngb;

extern "C" {

int ng_block_bytes(const ng_block_desc* desc, size_t* codes_bytes, size_t* scales_bytes) {
  const int rc = check_shape(desc);
  if (rc != NG_OK) return rc;
  if (!codes_bytes || !scales_bytes) return fail(NG_ERR_INVALID_ARG, "no place for the sizes");
  BlockView v = {};
  block_pitches(*desc, v);
  const size_t rows = desc->format == NG_BLOCK_MXFP8 ? v.outer : (v.outer + 127ll) / 128;
  *codes_bytes = static_cast<size_t>(v.pitch) * rows;
  *scales_bytes = static_cast<size_t>(v.spitch) * rows;
  return NG_OK;
}

int ng_block_quantize(const void* A, int dtype_bytes, long long row_stride, long long col_stride,
                      const ng_block_desc* outs, int n_outs, void* stream) {
  if (!A || !outs) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (dtype_bytes != 2 && dtype_bytes != 4) return fail(NG_ERR_UNSUPPORTED, "matrices in blocks are made from fp16 and fp32");
  if (n_outs < 1 || n_outs > 4) return fail(NG_ERR_INVALID_ARG, "1 to 4 matrices in blocks from one call");
  for (int i = 0; i < n_outs; ++i) {
    const int rc = check_shape(outs + i);
    if (rc != NG_OK) return rc;
    if (outs[i].rows != outs[0].rows || outs[i].cols != outs[0].cols) return fail(NG_ERR_INVALID_ARG, "matrices of different shapes");
  }
  DeviceCtx* c = current_ctx();
  if (!c) return NG_ERR_CUDA;
  BlockView v[4];
  for (int i = 0; i < n_outs; ++i) {
    const int rc = block_view(c, outs + i, v[i]);
    if (rc != NG_OK) return rc;
  }
  for (int i = 0; i < n_outs; ++i) {
    const long long so = outs[i].axis ? row_stride : col_stride, sl = outs[i].axis ? col_stride : row_stride;
    int rc = NG_OK;
    if (dtype_bytes == 2) {
      PlainView<const __half> a = {static_cast<const __half*>(A), so, sl};
      NG_BY_FORMAT(outs[i].format, rc = (quantize_one<__half, kF>(c, v[i], a, static_cast<cudaStream_t>(stream))));
    } else {
      PlainView<const float> a = {static_cast<const float*>(A), so, sl};
      NG_BY_FORMAT(outs[i].format, rc = (quantize_one<float, kF>(c, v[i], a, static_cast<cudaStream_t>(stream))));
    }
    if (rc != NG_OK) return rc;
  }
  return NG_OK;
}

int ng_block_dequantize(const ng_block_desc* q, void* out, int dtype_bytes, long long row_stride, long long col_stride,
                        void* stream) {
  if (!out) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (dtype_bytes != 2 && dtype_bytes != 4) return fail(NG_ERR_UNSUPPORTED, "matrices in blocks are read as fp16 and fp32");
  int rc = check_shape(q);
  if (rc != NG_OK) return rc;
  DeviceCtx* c = current_ctx();
  if (!c) return NG_ERR_CUDA;
  BlockView v;
  rc = block_view(c, q, v);
  if (rc != NG_OK) return rc;
  const long long so = q->axis ? row_stride : col_stride, sl = q->axis ? col_stride : row_stride;
  if (dtype_bytes == 2) {
    PlainView<__half> a = {static_cast<__half*>(out), so, sl};
    NG_BY_FORMAT(q->format, return (dequantize_one<__half, kF>(c, v, a, static_cast<cudaStream_t>(stream))));
  } else {
    PlainView<float> a = {static_cast<float*>(out), so, sl};
    NG_BY_FORMAT(q->format, return (dequantize_one<float, kF>(c, v, a, static_cast<cudaStream_t>(stream))));
  }
  return NG_OK;
}

int ng_block_relu_mask(const ng_block_desc* q, void* E, int dtype_bytes, long long row_stride, long long col_stride,
                       void* stream) {
  if (!E) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (dtype_bytes != 2 && dtype_bytes != 4) return fail(NG_ERR_UNSUPPORTED, "deltas are fp16 or fp32");
  int rc = check_shape(q);
  if (rc != NG_OK) return rc;
  if (q->format != NG_BLOCK_MXFP8) return fail(NG_ERR_UNSUPPORTED, "only mxfp8 keeps which numbers were positive");
  DeviceCtx* c = current_ctx();
  if (!c) return NG_ERR_CUDA;
  BlockView v;
  rc = block_view(c, q, v);
  if (rc != NG_OK) return rc;
  const long long so = q->axis ? row_stride : col_stride, sl = q->axis ? col_stride : row_stride;
  if (dtype_bytes == 2) {
    PlainView<__half> a = {static_cast<__half*>(E), so, sl};
    return relu_mask_one<__half>(c, v, a, static_cast<cudaStream_t>(stream));
  }
  PlainView<float> a = {static_cast<float*>(E), so, sl};
  return relu_mask_one<float>(c, v, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
