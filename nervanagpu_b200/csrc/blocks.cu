// Matrices in blocks of small floating-point numbers: quantisation, values, and the ReLU mask from an 8-bit record
// (the formats and the layout are described in blocks.cuh).
//
// All three move each number once and are bound by that: a quantisation reads 2 or 4 bytes per number and writes
// half a byte or one, plus a scale per block. Two forms each, by how the blocks lie in the plain matrix:
//   rows      neighbours of a block are neighbours in memory: a lane takes 8 of them (16 bytes of fp16), 2 or 4
//             lanes share a block and exchange its largest magnitude by shuffles
//   strided   a thread takes a whole block, lanes run along the other axis, which is then the contiguous one (the
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
};

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ void from_f32(float v, __half& x) { x = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, float& x) { x = v; }

// 8 neighbours at p, 16-byte aligned when kVec; only the first n exist
template <bool kVec>
__device__ __forceinline__ void load8(const __half* p, int n, float (&x)[8]) {
  if (kVec && n >= 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < n ? __half2float(p[i]) : 0.0f;
}
template <bool kVec>
__device__ __forceinline__ void load8(const float* p, int n, float (&x)[8]) {
  if (kVec && n >= 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < n ? p[i] : 0.0f;
}
template <bool kVec>
__device__ __forceinline__ void store8(__half* p, int n, const float (&v)[8]) {
  if (kVec && n >= 8) {
    uint4 w;
    __half2* h = reinterpret_cast<__half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = __float2half_rn(v[i]);
}
template <bool kVec>
__device__ __forceinline__ void store8(float* p, int n, const float (&v)[8]) {
  if (kVec && n >= 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = v[i];
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// ---- rows form. Lane g of a row takes numbers 8 g .. 8 g + 7; rows in steps of the grid.
template <typename T, int kFmt, bool kVec>
__global__ void __launch_bounds__(256) quantize_rows_kernel(BlockView q, PlainView<const T> a) {
  using F = BlockFormat<kFmt>;
  const int g = blockIdx.x * blockDim.x + threadIdx.x;
  const int n = q.inner - g * 8;                   // numbers that exist, from this lane's first on
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  // (a warp's lanes may be in different rows, but a block's are together: whole warps take part in the shuffles)
  for (long long o0 = blockIdx.y * blockDim.y; o0 < q.outer; o0 += step) {
    const int o = static_cast<int>(o0) + threadIdx.y;
    const bool live = o < q.outer && n > 0;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    if (live) load8<kVec>(a.p + o * a.so + g * 8ll, n, x);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(x[i]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if (F::kBlock == 32) top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const BlockScale s = block_scale<kFmt>(top, q.t);
    const uint2 codes = block_encode8<kFmt>(x, s);
    if (live) {
      uint8_t* dst = q.codes + o * q.pitch + g * F::kBytes8;
      if (F::k4) *reinterpret_cast<uint32_t*>(dst) = codes.x;
      else *reinterpret_cast<uint2*>(dst) = codes;
      if (g % (F::kBlock / 8) == 0) q.scales[F::scale_at(q, o, g / (F::kBlock / 8))] = static_cast<uint8_t>(s.byte);
    }
  }
}

template <typename T, int kFmt, bool kVec>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(BlockView q, PlainView<T> a) {
  using F = BlockFormat<kFmt>;
  const int g = blockIdx.x * blockDim.x + threadIdx.x;
  const int n = q.inner - g * 8;
  if (n <= 0) return;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  for (long long o = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; o < q.outer; o += step) {
    const uint8_t* src = q.codes + o * q.pitch + g * F::kBytes8;
    uint2 codes = make_uint2(0u, 0u);
    if (F::k4) codes.x = *reinterpret_cast<const uint32_t*>(src);
    else codes = *reinterpret_cast<const uint2*>(src);
    const uint32_t byte = q.scales[F::scale_at(q, static_cast<int>(o), g / (F::kBlock / 8))];
    const float scale = block_scale_value<kFmt>(byte, q.t);
    float v[8];
    block_decode8<kFmt>(codes, scale, v);
    if (sizeof(T) == 2) block_limit_f16<kFmt>(scale, v);
    store8<kVec>(a.p + o * a.so + g * 8ll, n, v);
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) relu_mask_rows_kernel(BlockView q, PlainView<T> a) {
  const int g = blockIdx.x * blockDim.x + threadIdx.x;
  const int n = q.inner - g * 8;
  if (n <= 0) return;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  for (long long o = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; o < q.outer; o += step) {
    const uint2 codes = *reinterpret_cast<const uint2*>(q.codes + o * q.pitch + g * 8);
    T* p = a.p + o * a.so + g * 8ll;
    uint32_t zero = 0u;      // bit i: number i is not positive (its code is 0 or has the sign bit)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t c = ((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) & 0xffu;
      zero |= (c - 1u >= 0x7fu ? 1u : 0u) << i;
    }
    if (kVec && n >= 8) {
      // whole vectors; fp32 in two of them
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int h = 0; h < 8 / kPer; ++h) {
        uint4 w = reinterpret_cast<uint4*>(p)[h];
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (zero >> (h * kPer + i) & 1u) e[i] = T(0.0f);
        reinterpret_cast<uint4*>(p)[h] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n && (zero >> i & 1u)) p[i] = T(0.0f);
    }
  }
}

// ---- strided form. Lanes along the outer axis, a block of numbers per thread.
template <typename T, int kFmt>
__global__ void __launch_bounds__(256) quantize_strided_kernel(BlockView q, PlainView<const T> a, int blocks) {
  using F = BlockFormat<kFmt>;
  const int o = blockIdx.x * 32 + threadIdx.x;
  if (o >= q.outer) return;
  for (int b = blockIdx.y * 8 + threadIdx.y; b < blocks; b += gridDim.y * 8) {
    const T* p = a.p + o * a.so + static_cast<long long>(b) * F::kBlock * a.sl;
    const int n = q.inner - b * F::kBlock;
    T raw[F::kBlock];
#pragma unroll
    for (int i = 0; i < F::kBlock; ++i) raw[i] = i < n ? p[i * a.sl] : T(0.0f);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < F::kBlock; ++i) top = max(top, magnitude_bits(to_f32(raw[i])));
    const BlockScale s = block_scale<kFmt>(top, q.t);
    uint8_t* dst = q.codes + o * q.pitch + static_cast<long long>(b) * (F::kBlock / 8 * F::kBytes8);
    uint32_t w[F::kBlock / 8 * F::kBytes8 / 4];
#pragma unroll
    for (int j = 0; j < F::kBlock / 8; ++j) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = to_f32(raw[8 * j + i]);
      const uint2 c = block_encode8<kFmt>(x, s);
      if (F::k4) {
        w[j] = c.x;
      } else {
        w[2 * j] = c.x;
        w[2 * j + 1] = c.y;
      }
    }
    if (F::kNv) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int j = 0; j < F::kBytes8 / 4; ++j)
        reinterpret_cast<uint4*>(dst)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
    q.scales[F::scale_at(q, o, b)] = static_cast<uint8_t>(s.byte);
  }
}

template <typename T, int kFmt>
__global__ void __launch_bounds__(256) dequantize_strided_kernel(BlockView q, PlainView<T> a, int blocks) {
  using F = BlockFormat<kFmt>;
  const int o = blockIdx.x * 32 + threadIdx.x;
  if (o >= q.outer) return;
  for (int b = blockIdx.y * 8 + threadIdx.y; b < blocks; b += gridDim.y * 8) {
    T* p = a.p + o * a.so + static_cast<long long>(b) * F::kBlock * a.sl;
    const int n = q.inner - b * F::kBlock;
    const uint8_t* src = q.codes + o * q.pitch + static_cast<long long>(b) * (F::kBlock / 8 * F::kBytes8);
    uint32_t w[F::kBlock / 8 * F::kBytes8 / 4];
    if (F::kNv) {
      const uint2 c = *reinterpret_cast<const uint2*>(src);
      w[0] = c.x;
      w[1] = c.y;
    } else {
#pragma unroll
      for (int j = 0; j < F::kBytes8 / 4; ++j) {
        const uint4 c = reinterpret_cast<const uint4*>(src)[j];
        w[4 * j] = c.x; w[4 * j + 1] = c.y; w[4 * j + 2] = c.z; w[4 * j + 3] = c.w;
      }
    }
    const float scale = block_scale_value<kFmt>(q.scales[F::scale_at(q, o, b)], q.t);
#pragma unroll
    for (int j = 0; j < F::kBlock / 8; ++j) {
      float v[8];
      block_decode8<kFmt>(F::k4 ? make_uint2(w[j], 0u) : make_uint2(w[2 * j], w[2 * j + 1]), scale, v);
      if (sizeof(T) == 2) block_limit_f16<kFmt>(scale, v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * j + i < n) from_f32(v[i], p[(8 * j + i) * a.sl]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) relu_mask_strided_kernel(BlockView q, PlainView<T> a, int blocks) {
  const int o = blockIdx.x * 32 + threadIdx.x;
  if (o >= q.outer) return;
  for (int b = blockIdx.y * 8 + threadIdx.y; b < blocks; b += gridDim.y * 8) {
    T* p = a.p + o * a.so + b * 32ll * a.sl;
    const uint8_t* src = q.codes + o * q.pitch + b * 32ll;
    const int n = min(32, q.inner - b * 32);
    for (int i = 0; i < n; ++i)
      if (src[i] - 1u >= 0x7fu) p[i * a.sl] = T(0.0f);
  }
}

// ---- launches ------------------------------------------------------------------------------------
struct RowGrid {
  dim3 grid, block;
};
// lanes per row: the number of 8-number groups, in whole blocks, over CTAs of 256 threads with as few idle lanes as
// a power of two allows; rows over the rest, several per thread once the device is full
RowGrid row_grid(const DeviceCtx* c, const BlockView& q) {
  const int groups = ((q.inner + 31) / 32) * 4;
  int tx = 256;
  while (tx > 16 && (groups + tx / 2 - 1) / (tx / 2) * (tx / 2) < (groups + tx - 1) / tx * tx) tx /= 2;
  while (tx > 4 && groups <= tx / 2) tx /= 2;
  const int ty = 256 / tx;
  RowGrid r;
  r.block = dim3(tx, ty);
  const long long gx = (groups + tx - 1) / tx, rows = (static_cast<long long>(q.outer) + ty - 1) / ty;
  const long long room = std::max(1ll, 32ll * c->sm_count / gx);
  r.grid = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(std::min(std::min(rows, room), 65535ll)));
  return r;
}
RowGrid strided_grid(const BlockView& q, int blocks) {
  RowGrid r;
  r.block = dim3(32, 8);
  r.grid = dim3(static_cast<unsigned>((q.outer + 31ll) / 32), static_cast<unsigned>(std::min((blocks + 7) / 8, 65535)));
  return r;
}

bool vectors(const void* p, long long so, long long sl, int esz) {
  return sl == 1 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (so * esz) % 16 == 0;
}

template <typename T, int kFmt>
int quantize_one(DeviceCtx* c, const BlockView& q, PlainView<const T> a, cudaStream_t stream) {
  const int blocks = (q.inner + BlockFormat<kFmt>::kBlock - 1) / BlockFormat<kFmt>::kBlock;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q);
    if (vectors(a.p, a.so, a.sl, sizeof(T))) quantize_rows_kernel<T, kFmt, true><<<g.grid, g.block, 0, stream>>>(q, a);
    else quantize_rows_kernel<T, kFmt, false><<<g.grid, g.block, 0, stream>>>(q, a);
  } else {
    const RowGrid g = strided_grid(q, blocks);
    quantize_strided_kernel<T, kFmt><<<g.grid, g.block, 0, stream>>>(q, a, blocks);
  }
  NG_CHECK_LAUNCH();
  return NG_OK;
}

template <typename T, int kFmt>
int dequantize_one(DeviceCtx* c, const BlockView& q, PlainView<T> a, cudaStream_t stream) {
  const int blocks = (q.inner + BlockFormat<kFmt>::kBlock - 1) / BlockFormat<kFmt>::kBlock;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q);
    if (vectors(a.p, a.so, a.sl, sizeof(T))) dequantize_rows_kernel<T, kFmt, true><<<g.grid, g.block, 0, stream>>>(q, a);
    else dequantize_rows_kernel<T, kFmt, false><<<g.grid, g.block, 0, stream>>>(q, a);
  } else {
    const RowGrid g = strided_grid(q, blocks);
    dequantize_strided_kernel<T, kFmt><<<g.grid, g.block, 0, stream>>>(q, a, blocks);
  }
  NG_CHECK_LAUNCH();
  return NG_OK;
}

template <typename T>
int relu_mask_one(DeviceCtx* c, const BlockView& q, PlainView<T> a, cudaStream_t stream) {
  const int blocks = (q.inner + 31) / 32;
  if (a.sl == 1) {
    const RowGrid g = row_grid(c, q);
    if (vectors(a.p, a.so, a.sl, sizeof(T))) relu_mask_rows_kernel<T, true><<<g.grid, g.block, 0, stream>>>(q, a);
    else relu_mask_rows_kernel<T, false><<<g.grid, g.block, 0, stream>>>(q, a);
  } else {
    const RowGrid g = strided_grid(q, blocks);
    relu_mask_strided_kernel<T><<<g.grid, g.block, 0, stream>>>(q, a, blocks);
  }
  NG_CHECK_LAUNCH();
  return NG_OK;
}

#define NG_BY_FORMAT(fmt, call)                                   \
  switch (fmt) {                                                  \
    case NG_BLOCK_MXFP4: { constexpr int kF = NG_BLOCK_MXFP4; call; } break; \
    case NG_BLOCK_NVFP4: { constexpr int kF = NG_BLOCK_NVFP4; call; } break; \
    default: { constexpr int kF = NG_BLOCK_MXFP8; call; } break;  \
  }

}  // namespace

// rows of codes and of scales, in bytes
static void block_pitches(const ng_block_desc& d, long long& pitch, long long& spitch) {
  const long long inner = d.axis ? d.cols : d.rows;
  if (d.format == NG_BLOCK_MXFP8) {
    pitch = (inner + kRowPad - 1) / kRowPad * kRowPad;
    spitch = pitch / 32;
  } else {
    pitch = (inner + 2 * kRowPad - 1) / (2 * kRowPad) * kRowPad;
    spitch = pitch * 2 / (d.format == NG_BLOCK_NVFP4 ? 64 : 128) * kScaleTile;
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
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale) || std::frexp(d->scale, &ex) != 0.5f || ex < -63 || ex > 65)
      return fail(NG_ERR_INVALID_ARG, "the scale of an nvfp4 matrix is a power of two from 2^-64 to 2^64");
  } else if (d->scale != 1.0f) {
    return fail(NG_ERR_INVALID_ARG, "only nvfp4 matrices have a scale");
  }
  return NG_OK;
}

int block_view(const DeviceCtx* c, const ng_block_desc* d, BlockView& v) {
  const int rc = check_shape(d);
  if (rc != NG_OK) return rc;
  if (!d->codes || !d->scales) return fail(NG_ERR_INVALID_ARG, "block matrix without memory");
  if ((reinterpret_cast<uintptr_t>(d->codes) | reinterpret_cast<uintptr_t>(d->scales)) & (kRowPad - 1))
    return fail(NG_ERR_INVALID_ARG, "codes and scales must be 128-byte aligned");
  if (d->device != c->device) return fail(NG_ERR_INVALID_ARG, "block matrix of device %d, the current device is %d", d->device, c->device);
  block_pitches(*d, v.pitch, v.spitch);
  v.codes = static_cast<uint8_t*>(d->codes);
  v.scales = static_cast<uint8_t*>(d->scales);
  v.outer = d->axis ? d->rows : d->cols;
  v.inner = d->axis ? d->cols : d->rows;
  v.t = d->scale;
  return NG_OK;
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
  long long pitch, spitch;
  block_pitches(*desc, pitch, spitch);
  const long long outer = desc->axis ? desc->rows : desc->cols;
  *codes_bytes = static_cast<size_t>(pitch) * outer;
  *scales_bytes = static_cast<size_t>(spitch) * (desc->format == NG_BLOCK_MXFP8 ? outer : (outer + 127) / 128);
  return NG_OK;
}

int ng_block_quantize(const void* A, int dtype_bytes, long long row_stride, long long col_stride,
                      const ng_block_desc* outs, int n_outs, void* stream) {
  if (!A || !outs) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (dtype_bytes != 2 && dtype_bytes != 4) return fail(NG_ERR_UNSUPPORTED, "matrices in blocks are made from fp16 and fp32");
  if (n_outs < 1 || n_outs > 4) return fail(NG_ERR_INVALID_ARG, "1 to 4 matrices in blocks from one pass");
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
