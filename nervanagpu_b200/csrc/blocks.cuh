// Matrices held in blocks of small floating-point numbers: layout and the arithmetic of the formats.
//
// A block is a run of neighbours along one axis of the matrix (the axis that products sum over) with a scale:
//
//   mxfp4   E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6), blocks of 32, scale 2^e (E8M0: the byte is e + 127)
//   nvfp4   E2M1 numbers, blocks of 16, scale s * t: s an E4M3 byte, t one power of two for the matrix
//   mxfp8   E4M3 numbers (up to 448), blocks of 32, scale 2^e
//
//   e = the smallest with which max|x| <= top * 2^e (top = 6 or 448): nothing saturates, and the largest number
//       of a block is off by no more than its rounding
//   s = RN_E4M3(max|x| / (6 t)), kept from 2^-9 (a block that is not all zero keeps a scale) to 448
//   code = RN(x / scale), ties to even, limited to the largest number
//   mxfp8: a number that is not zero gets a code that is not zero, so that x > 0 can be told from the code.
//   Signs are kept, in mxfp4 and mxfp8 those of zeros and of what becomes zero too: the codes of a matrix are the same bytes
//   whatever its type, strides and blocked axis. (nvfp4 rounds with sums that lose the sign of a zero, fp16 numbers below
//   2^-16 of the scale theirs too, fp32 numbers not: those zeros may differ in their sign. An instruction per number that
//   puts it back took 7 % of a quantisation, 4096 x 9216 13.6 -> 14.6 us.)
//
// Values are read limited to the largest number of the type that they are read as: a number next to it may have been
// rounded to one beyond it.
//
// A block with an infinity or a NaN has the scale NaN (0xff, or 0x7f in E4M3): all of it reads back as NaN. A
// product sums over the block, so its result is lost either way. mxfp8 codes keep the signs in such blocks too.
//
// Layout. The matrix is stored along its blocked axis ("inner"), a row of codes per index of the other axis ("outer"),
// two 4-bit codes per byte (the even one in the low half).
//   mxfp8: rows of codes one behind the other, padded with zeros to whole blocks; rows of scales likewise, to 4.
//   4-bit formats: as shared and tensor memory hold them, so that a product's operands are plain contiguous copies,
//   without a tensor map to build and fetch and without a stride between their rows. Tiles of 128 outer rows (fewer
//   in a matrix of at most 64: 16, 32 or 64) x 128 bytes = 256 numbers, the tiles of 128 rows along the inner axis
//   one behind the other; the 16-byte pieces of row r are exchanged as the 128-byte swizzle wants it, piece c
//   at c ^ (r % 8). Scales: tiles of 512 bytes with 4 consecutive blocks of 128 outer rows, byte
//   (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4.
// Tiles are padded with zeros, which no call overwrites (a scale of 2^-127 or 0 with the code 0 gives zero).
#pragma once
#include "../../include/nervana_b200.h"
#include "common.cuh"

namespace ngb {

constexpr int kTileRow = 128;       // bytes of a row of a tile of 4-bit codes
constexpr int kScaleTile = 512;     // bytes of a tile of 4-bit formats' scales

// What a kernel needs to know of a matrix in blocks.
struct BlockView {
  uint8_t* codes;
  uint8_t* scales;
  long long pitch;        // bytes from one row (mxfp8) or one row of tiles of codes to the next
  int tile;               // 4-bit formats: bytes of a tile of codes
  long long spitch;       // bytes from one row (mxfp8) or one row of tiles (4-bit formats) of scales to the next
  int outer, inner;
  float t;                // nvfp4: the matrix's power of two
};

template <int kFmt>
struct BlockFormat {
  static constexpr bool k4 = kFmt != NG_BLOCK_MXFP8;
  static constexpr bool kNv = kFmt == NG_BLOCK_NVFP4;
  static constexpr int kBlock = kNv ? 16 : 32;
  static constexpr int kBytes8 = k4 ? 4 : 8;      // bytes of 8 codes

  // byte `at` of row o of the codes, within an aligned 16 bytes
  static __device__ __forceinline__ long long code_at(const BlockView& v, int o, long long at) {
    if (!k4) return o * v.pitch + at;
    const int b = static_cast<int>(at) & 127;
    return (o >> 7) * v.pitch + (at >> 7) * v.tile + (o & 127) * 128 + (b ^ ((o & 7) << 4));
  }
  static __device__ __forceinline__ long long scale_at(const BlockView& v, int o, int b) {
    if (!k4) return o * v.spitch + b;
    return (o >> 7) * v.spitch + (b >> 2) * static_cast<long long>(kScaleTile) + (o & 31) * 16 + ((o >> 5) & 3) * 4 + (b & 3);
  }
};

// Zero as bits. (A conversion of 0.0f is an instruction of its own that the compiler does not move: `p ? load : zero` became
// a branch, and the loads beside it waited for one another.)
template <typename T>
__device__ __forceinline__ T zero_of();
template <>
__device__ __forceinline__ float zero_of<float>() { return 0.0f; }
template <>
__device__ __forceinline__ __half zero_of<__half>() { return __ushort_as_half(0); }

// For a kernel that gives up: copies and MMAs in flight must end before the CTA may, and do so in microseconds, but the
// barriers that would tell may never complete, other arrivals missing. So this waits for time.
__device__ __forceinline__ void wait_for_strays() {
  const uint64_t t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 1000000ull) __nanosleep(1000);
}

// fp32 -> E4M3 / E2M1, two at a time, the first in the low half; to nearest, ties to even, limited to the largest
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&y)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}
__device__ __forceinline__ __half2 half2_of_e4m3x2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return *reinterpret_cast<__half2*>(&r);
}
__device__ __forceinline__ void half2_of_e2m1x8(uint32_t codes, __half2 (&h)[4]) {
  uint32_t r[4];
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2*>(&r[i]);
}

// Scale of a block from the bits of its largest magnitude: the byte to store, and what the numbers are multiplied
// with (powers of two, exact) or divided by (nvfp4).
struct BlockScale {
  uint32_t byte;
  float by;
  bool nan;
};
// 1 / x to within 2^-22 of it, for a normal x
__device__ __forceinline__ float rcp_near(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// kHalf: the numbers came from fp16.
template <int kFmt, bool kHalf>
__device__ __forceinline__ BlockScale block_scale(uint32_t amax_bits, float t) {
  BlockScale s;
  s.nan = amax_bits >= 0x7f800000u;
  if (BlockFormat<kFmt>::kNv) {
    // amax / 6t is rounded before it is rounded to E4M3. Neither way can that put it on the border between two of
    // those, 5 bits long, or off it: an fp32 number next to 6 t * border is more than half an ulp of the quotient away
    // from it; fp16 numbers are 2^-11 of it away, and their quotients, off by 2^-21 at most, are rounded to 16 bits.
    float quotient;
    if (kHalf) quotient = __uint_as_float((__float_as_uint(__uint_as_float(amax_bits) * rcp_near(6.0f * t)) + 0x40u) & ~0x7fu);
    else quotient = __fdiv_rn(__uint_as_float(amax_bits), 6.0f * t);
    s.byte = s.nan ? 0x7fu : cvt_e4m3x2(quotient, 0.0f);
    if (s.byte == 0u) s.byte = 1u;
    s.by = __low2float(half2_of_e4m3x2(s.byte)) * t;
  } else {
    constexpr int kEmax = BlockFormat<kFmt>::k4 ? 2 : 8;
    constexpr uint32_t kMant = BlockFormat<kFmt>::k4 ? 0x400000u : 0x600000u;   // 6 = 1.5 * 2^2, 448 = 1.75 * 2^8
    // biased exponent, one more when the mantissa is above that of the largest number
    const int e = static_cast<int>((amax_bits + (0x7fffffu - kMant)) >> 23) - kEmax;
    s.byte = s.nan ? 0xffu : static_cast<uint32_t>(max(e, 0));
    s.by = __uint_as_float(static_cast<uint32_t>(254 - min(max(e, 0), 253)) << 23);
  }
  return s;
}

// 8 numbers of a block to codes: 4 bytes in x (4-bit formats) or 8 in x and y. kHalf: they came from fp16.
template <int kFmt, bool kHalf>
__device__ __forceinline__ uint2 block_encode8(const float (&x)[8], const BlockScale& s) {
  float y[8];
  uint2 r = make_uint2(0u, 0u);
  if constexpr (BlockFormat<kFmt>::k4) {
    if constexpr (!BlockFormat<kFmt>::kNv) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i] * s.by;
    } else if constexpr (kHalf) {
      // An IEEE division per number made this kernel issue-bound (4096 x 9216: 34 us). The product with the
      // reciprocal is off by 2^-21 of the quotient, which matters on the border between two codes only; rounded to a
      // multiple of 2^-15 (the sum with 384 has that for its last bit) it is on the border when the quotient is: the
      // border times the scale has at most 7 bits, and an fp16 number that differs from it does so by 2^-11 of it.
      const float inv = rcp_near(s.by);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fmaf(x[i], inv, 384.0f) - 384.0f;
    } else {
      // An fp32 number may be closer to a border. The multiple of 2^-15 is then the border itself, its product with the
      // scale is exact, and the sign of what it leaves of x tells the side: a step of up to 2^-17 that way. (A number
      // that leaves something leaves at least 2^-26 of the scale there; elsewhere the next border is 2^-15 away, the
      // quotient's own error, 2^-21 of up to 6.5, less than half of that.)
      const float inv = rcp_near(s.by), sure = inv * 1024.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = fmaf(x[i], inv, 384.0f) - 384.0f;
        y[i] = q + fminf(fmaxf(fmaf(-q, s.by, x[i]) * sure, -7.62939453125e-06f), 7.62939453125e-06f);
      }
    }
    r.x = cvt_e2m1x8(y);
    if (s.nan) r.x = 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // not zero: no less than the smallest code; in a block with the scale NaN the smallest code of x's sign
      const float mag = s.nan ? 0.001953125f : fmaxf(fabsf(x[i]) * s.by, 0.001953125f);
      // (a zero as it is, 0 for a NaN; as the sign put on a 0 it took 7 registers more, 139968 x 128 fp16 8.0 -> 8.4 us)
      y[i] = (x[i] > 0.0f || x[i] < 0.0f) ? copysignf(mag, x[i]) : fminf(x[i], 0.0f);
    }
    r.x = cvt_e4m3x2(y[0], y[1]) | (cvt_e4m3x2(y[2], y[3]) << 16);
    r.y = cvt_e4m3x2(y[4], y[5]) | (cvt_e4m3x2(y[6], y[7]) << 16);
  }
  return r;
}

// 4 fp16 numbers of a block (two per word) to mxfp8 codes, the same codes as above. `by` as two factors that fp16
// holds (block_scale_f16): products are exact where they are not below 2^-9, the least that is encoded.
__device__ __forceinline__ uint32_t block_encode4_f16(uint32_t x0, uint32_t x1, __half2 by0, __half2 by1) {
  uint32_t r[2];
  const uint32_t x[2] = {x0, x1};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 v = *reinterpret_cast<const __half2*>(&x[i]);
    // (the least is 2^-9 for a number that is not zero: 2^15 times any such is no less)
    const __half2 least = __hmin2(__habs2(__hmul2(v, __half2half2(__ushort_as_half(0x7800)))), __half2half2(__ushort_as_half(0x1800)));
    const __half2 m = __hmax2(__habs2(__hmul2(__hmul2(v, by0), by1)), least);
    const uint32_t y = *reinterpret_cast<const uint32_t*>(&m) | (x[i] & 0x80008000u);
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(y));
    r[i] = c;
  }
  return r[0] | (r[1] << 16);
}
__device__ __forceinline__ void block_scale_f16(float by, __half2& by0, __half2& by1) {
  by0 = __float2half2_rn(fminf(by, 32768.0f));
  by1 = __float2half2_rn(fminf(fmaxf(by * (1.0f / 32768.0f), 1.0f), 32768.0f));
}

// The scale that a stored byte stands for.
template <int kFmt>
__device__ __forceinline__ float block_scale_value(uint32_t byte, float t) {
  if (BlockFormat<kFmt>::kNv) return __low2float(half2_of_e4m3x2(byte)) * t;
  if (byte == 0xffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(byte ? byte << 23 : 0x400000u);   // (2^-127 is below the normal range)
}

// The values of 8 codes.
template <int kFmt>
__device__ __forceinline__ void block_decode8(uint2 codes, float scale, float (&v)[8]) {
  __half2 h[4];
  if (BlockFormat<kFmt>::k4) {
    half2_of_e2m1x8(codes.x, h);
  } else {
    h[0] = half2_of_e4m3x2(codes.x & 0xffffu);
    h[1] = half2_of_e4m3x2(codes.x >> 16);
    h[2] = half2_of_e4m3x2(codes.y & 0xffffu);
    h[3] = half2_of_e4m3x2(codes.y >> 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
  }
}

// 8 codes as fp16 numbers times a scale that fp16 holds and with which nothing leaves its range: one rounding, the
// same results as in fp32.
template <int kFmt>
__device__ __forceinline__ bool block_scale_fits_f16(float scale) {
  // (below 2^-40 fp16 holds neither the scale nor any of the values: both are zero)
  return (scale >= 6.103515625e-05f || scale <= 9.094947e-13f) && scale * (BlockFormat<kFmt>::k4 ? 6.0f : 448.0f) <= 65504.0f;
}
template <int kFmt>
__device__ __forceinline__ uint4 block_decode8_f16(uint2 codes, __half2 scale) {
  __half2 h[4];
  if (BlockFormat<kFmt>::k4) {
    half2_of_e2m1x8(codes.x, h);
  } else {
    h[0] = half2_of_e4m3x2(codes.x & 0xffffu);
    h[1] = half2_of_e4m3x2(codes.x >> 16);
    h[2] = half2_of_e4m3x2(codes.y & 0xffffu);
    h[3] = half2_of_e4m3x2(codes.y >> 16);
  }
  uint4 r;
  uint32_t* w = &r.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hmul2(h[i], scale);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
}

// The same, limited to the largest number of the result's type (a NaN stays one).
template <int kFmt, typename T>
__device__ __forceinline__ void block_limit(float scale, float (&v)[8]) {
  constexpr float kLargest = sizeof(T) == 2 ? 65504.0f : 3.402823466e+38f;
  if (scale * (BlockFormat<kFmt>::k4 ? 6.0f : 448.0f) > kLargest) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(v[i]) > kLargest) v[i] = copysignf(kLargest, v[i]);
  }
}

}  // namespace ngb
