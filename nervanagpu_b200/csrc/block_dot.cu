// Products of matrices in blocks of small floating-point numbers (the formats: blocks.cuh).
//
// 4-bit x 4-bit (block_dot_kernel): C = epilogue(sum_k A[i,k] B[k,j]) on tcgen05.mma.kind::mxf4nvf4, which takes the
// packed codes from shared memory and the scales of both operands from tensor memory, multiplies each block's
// products by its two scales and accumulates in fp32. Both operands lie in memory as shared memory holds them: a k-block
// of 256 numbers (four MMAs of 64) of 128 rows is one bulk copy of 16 KB, its scales one of 1 or 2 KB, and a tcgen05.cp
// per 512 bytes takes these to tensor memory.
//
// A CTA computes a tile of 128 rows x kN columns (kN from 16 to 128). Few tiles are split along the sum over the
// CTAs of a thread-block cluster (block_share.cuh).
//
//   warp 0     producer (the first loads leave before tensor memory is allocated)
//   warp 1     tensor memory, scale copies and MMAs, by one thread
//   warps 2-9  tensor memory -> shared memory, two warps per group of 32 lanes
//   all        sum over the cluster, output stage (epilogue.cuh), stores
#include <algorithm>
#include <atomic>
#include <cmath>

#include "block_mma.cuh"
#include "block_share.cuh"
#include "blocks.h"

namespace ngb {

namespace {

constexpr uint32_t kCodesA = 128u * 128u;       // bytes of a k-block of A
constexpr int kDotThreads = 320;
constexpr uint32_t kDotSmemLimit = 232448;      // 227 KB
constexpr uint32_t kDotCtrl = 256;              // barriers, tensor-memory address, abort flag
constexpr int kDotStages = 8;                   // most

// Everything that follows from the tile's columns and the format.
template <int kN, bool kNv>
struct DotTile {
  static constexpr int kScaleTiles = kNv ? 4 : 2;            // 512-byte scale tiles per k-block and 128 rows
  static constexpr uint32_t kCodesB = kN * 128u;
  static constexpr uint32_t kScales = kScaleTiles * kScaleTile;      // of 128 rows
  static constexpr uint32_t kStageBytes = (kCodesA + kCodesB + 2 * kScales + 1023u) & ~1023u;
  static constexpr int kPitch = kSharePitch<kN>;
  static constexpr uint32_t kParts = kShareTile<kN>;
  static constexpr int kRoom = static_cast<int>((kDotSmemLimit - 1024u - kDotCtrl - kParts) / kStageBytes);
  static constexpr int kStages = kRoom < kDotStages ? kRoom : kDotStages;
  // tensor memory: the accumulator, then two buffers of scales, A's before B's
  static constexpr int kAccCols = kN < 32 ? 32 : kN;
  static constexpr int kScaleCols = kScaleTiles * 8;
  static constexpr int kColsUsed = kAccCols + 2 * kScaleCols;
  static constexpr uint32_t kCols = kColsUsed <= 128 ? 128 : 256;
  static constexpr uint32_t kSmem = kStages * kStageBytes + kParts + kDotCtrl + 1024u;
  // (this CTA's tile takes the ring's place when its products are done; the others' parts of its share have their own)
  static_assert(kParts <= kStages * kStageBytes, "the ring is smaller than the tile");
  static_assert(kSmem > kDotSmemLimit / 2, "an SM takes two CTAs: dot_room() asks for one instance only");
};

struct DotParams {
  int num_kb;
  int tiles_m;
  const uint8_t *ca, *cb;    // codes
  const uint8_t *sa, *sb;    // scales
  long long pitch_a, pitch_b;    // bytes of a row of tiles of codes
  int tile_a;                // bytes of a tile of A's codes
  long long spitch;          // bytes of a row of scale tiles (the same for both: one format, one length)
  ShareOut out;
  int swapped;               // the tile's rows are C's columns
  int* status;
  unsigned long long wait_limit_ns;
};

template <int kN, bool kNv>
__global__ void __launch_bounds__(kDotThreads, 1) block_dot_kernel(const __grid_constant__ DotParams p) {
  using T = DotTile<kN, kNv>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t parts = ring + T::kStages * T::kStageBytes, ctrl = parts + T::kParts;
  uint8_t* ring_gen = smem_raw + (ring - smem_u32(smem_raw));
  auto full_bar = [&](int s) { return ctrl + 8u * s; };
  auto empty_bar = [&](int s) { return ctrl + 8u * (kDotStages + s); };
  const uint32_t acc_bar = ctrl + 8u * (2 * kDotStages), part_bar = acc_bar + 8u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring_gen + (ctrl - ring) + 8 * (2 * kDotStages + 2));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_cta_rank());
  const int tile = blockIdx.x / splits;
  const int m0 = (tile % p.tiles_m) * 128, n0 = (tile / p.tiles_m) * kN;
  const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * rank / splits);
  const int count = static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / splits) - kb0;
  const uint32_t share_bytes = T::kParts / splits;

  // k-block i of this partition into slot i % kStages
  const int rt = m0 / 128, ct = n0 / 128;
  auto load_kb = [&](int i) {
    const int s = i % T::kStages;
    const uint32_t a = ring + s * T::kStageBytes, b = a + kCodesA, sa = b + T::kCodesB, sb = sa + T::kScales;
    const long long kb = kb0 + i;
    // (A may have tiles of fewer rows: what the MMA then reads behind them ends in rows that are not stored. B's tiles have
    // as many as this tile has columns.)
    mbar_expect_tx(full_bar(s), p.tile_a + T::kCodesB + 2 * T::kScales);
    bulk_load(a, p.ca + rt * p.pitch_a + kb * p.tile_a, p.tile_a, full_bar(s));
    bulk_load(sa, p.sa + rt * p.spitch + kb * T::kScales, T::kScales, full_bar(s));
    bulk_load(b, p.cb + ct * p.pitch_b + kb * T::kCodesB, T::kCodesB, full_bar(s));
    bulk_load(sb, p.sb + ct * p.spitch + kb * T::kScales, T::kScales, full_bar(s));
  };
  const int first = min(count, T::kStages);      // k-blocks that need no free slot
  if (warp == 0) {
    if (elect_one()) {
      for (int s = 0; s < T::kStages; ++s) {
        mbar_init(full_bar(s), 1);
        mbar_init(empty_bar(s), 1);
      }
      mbar_init(acc_bar, 1);
      mbar_init(part_bar, 1);
      *abort_flag = 0;
      mbar_fence_init();
      if (splits > 1) mbar_expect_tx(part_bar, (splits - 1) * share_bytes);
      grid_dependency_wait();
      for (int i = 0; i < first; ++i) load_kb(i);
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), T::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (splits > 1) cluster_arrive();      // (this CTA's barriers exist)
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    if (elect_one()) {
      int i = first;
      for (; i < count; ++i) {
        if (!mbar_wait(empty_bar(i % T::kStages), (i / T::kStages - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns)) {
          // given up: the loads in flight must land before the CTA may end
          int none = 0;
          for (int j = i - T::kStages; j < i; ++j)
            mbar_wait(full_bar(j % T::kStages), (j / T::kStages) & 1, &none, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns);
          break;
        }
        load_kb(i);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t scales = tmem + T::kAccCols;
      bool ok = true;
      for (int i = 0; i < count; ++i) {
        const int s = i % T::kStages;
        if (!mbar_wait(full_bar(s), (i / T::kStages) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_MMA, p.wait_limit_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = ring + s * T::kStageBytes, b = a + kCodesA, sa = b + T::kCodesB, sb = sa + T::kScales;
        mma_kblock<kNv, false, 1>(tmem, a, b, sa, sb, scales + (i & 1) * T::kScaleCols, block_idesc(128, kN, kNv), i == 0);
        tc_commit(empty_bar(s));
      }
      tc_commit(acc_bar);
      if (!ok) {     // what was issued must end before tensor memory is given back
        int none = 0;
        mbar_wait(acc_bar, 0, &none, p.status, NG_DEV_TIMEOUT_MMA, p.wait_limit_ns);
      }
    }
    __syncwarp();
  }
  if (warp >= 2) {
    const bool done = mbar_wait(acc_bar, 0, abort_flag, p.status, NG_DEV_TIMEOUT_EPILOGUE, p.wait_limit_ns);
    __syncwarp();
    if (!done) {
      wait_for_strays();
    } else if (!*abort_flag) {
      tc_fence_after();
      const int group = warp & 3, half = (warp - 2) >> 2;
      float* row = reinterpret_cast<float*>(ring_gen) + (group * 32 + lane) * T::kPitch;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(group * 32) << 16);
      if constexpr (kN < 64) {
        // 16 columns each (a tile of 16: the first of the two warps)
        if (half * 16 < kN) {
          uint32_t r[16];
          tc_ld_32x16(taddr + half * 16, r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            reinterpret_cast<uint4*>(row + half * 16)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
      } else {
#pragma unroll 1
        for (int c = half * (kN / 2); c < (half + 1) * (kN / 2); c += 32) {
          uint32_t r[32];
          tc_ld_32x32(taddr + c, r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<uint4*>(row + c)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
      }
      tc_fence_before();
    }
    fence_async_smem();      // (the parts leave by bulk copies)
  }
  __syncthreads();
  if (splits > 1) share_push(ring, parts, share_bytes, rank, splits, part_bar);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, T::kCols);
  }
  if (splits > 1) share_wait(part_bar, abort_flag, p.status, p.wait_limit_ns);
  if (!*abort_flag)
    share_store<kN, kDotThreads>(p.out, p.swapped, reinterpret_cast<float*>(ring_gen), reinterpret_cast<const float*>(ring_gen + (parts - ring)),
                                 splits, rank, m0, n0);
  __syncwarp();
  if (splits > 1) cluster_wait();
}

template <int kN, bool kNv>
int launch_dot(DeviceCtx* c, DotParams& p, int splits, cudaStream_t stream) {
  using T = DotTile<kN, kNv>;
  const long long tiles = static_cast<long long>(p.tiles_m) * ((p.out.N + kN - 1ll) / kN);
  if (tiles * splits > 0x7fffffffll) return fail(NG_ERR_TOO_LARGE, "too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
  cfg.blockDim = dim3(kDotThreads);
  cfg.dynamicSmemBytes = T::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tuning().dependent_launch != 0 ? 2 : 1;
  static std::atomic<unsigned long long> ready{0};      // devices on which this instance may use its shared memory
  if (!(ready.load(std::memory_order_relaxed) >> c->device & 1u)) {
    NG_CUDA(cudaFuncSetAttribute(block_dot_kernel<kN, kNv>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
    ready.fetch_or(1ull << c->device, std::memory_order_relaxed);
  }
  NG_CUDA(cudaLaunchKernelEx(&cfg, block_dot_kernel<kN, kNv>, p));
  NG_CHECK_LAUNCH();
  return NG_OK;
}

int pad_columns(int n) { return n <= 64 ? block_tile_rows(n) : (n + 127) / 128 * 128; }

int check_output(const void* C, int ldc, int n, int sr_bits, int out_f32) {
  if (!C) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (ldc < n) return fail(NG_ERR_INVALID_ARG, "leading dimension too small");
  if (sr_bits < 0 || sr_bits > 10) return fail(NG_ERR_INVALID_ARG, "stochastic rounding keeps 1..10 mantissa bits");
  if (sr_bits && out_f32) return fail(NG_ERR_UNSUPPORTED, "stochastic rounding is to fp16");
  return NG_OK;
}

}  // namespace

int cluster_room(const DeviceCtx* c, const void* kernel, int threads, uint32_t smem, int log) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c->sm_count >> log << log));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << log;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess)
    cudaGetLastError();
  return std::max(1, clusters << log);
}

// Of this kernel, asked once per device and cluster size. (All its instances take an SM each.)
static int dot_room(const DeviceCtx* c, int log) {
  static std::atomic<int> known[64][4];
  int n = known[c->device][log].load(std::memory_order_relaxed);
  if (n == 0) {
    n = cluster_room(c, reinterpret_cast<const void*>(block_dot_kernel<128, true>), kDotThreads, DotTile<128, true>::kSmem, log);
    known[c->device][log].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace ngb

using namespace ngb;

extern "C" {

int ng_block_dot(const ng_block_desc* A, const ng_block_desc* B, void* C, int ldc, int out_f32, float alpha,
                 float beta, int relu, int sr_bits, unsigned long long seed, unsigned int rng_offset, void* stream) {
  int rc = check_shape(A);
  if (rc == NG_OK) rc = check_shape(B);
  if (rc != NG_OK) return rc;
  if (A->format == NG_BLOCK_MXFP8 || A->format != B->format) return fail(NG_ERR_UNSUPPORTED, "both operands are in the same 4-bit format");
  if (A->axis != 1 || B->axis != 0) return fail(NG_ERR_UNSUPPORTED, "blocks run along the sum: axis 1 of A, axis 0 of B");
  if (A->cols != B->rows) return fail(NG_ERR_INVALID_ARG, "inner dimensions differ: %d and %d", A->cols, B->rows);
  const int m = A->rows, n = B->cols;
  rc = check_output(C, ldc, n, sr_bits, out_f32);
  if (rc != NG_OK) return rc;
  // The output stage multiplies once, with alpha times the operands' powers of two (themselves from 2^-64 to 2^64, 1 in mxfp4).
  const float factor = alpha * (A->scale * B->scale);
  if (std::isfinite(alpha) && static_cast<double>(factor) != static_cast<double>(alpha) * A->scale * B->scale)
    return fail(NG_ERR_UNSUPPORTED, "alpha times the operands' scales is beyond the range of fp32: %g * %g * %g", alpha, A->scale,
                B->scale);
  DeviceCtx* c = current_ctx();
  if (!c) return NG_ERR_CUDA;
  BlockView a, b;
  rc = block_view(c, A, a);
  if (rc == NG_OK) rc = block_view(c, B, b);
  if (rc != NG_OK) return rc;

  const bool nv = A->format == NG_BLOCK_NVFP4;
  DotParams p = {};
  EpiArgs& ea = p.out.ea;
  ea.alpha = factor;
  ea.beta = beta; ea.relu = relu; ea.sr_bits = sr_bits;
  ea.seed_lo = static_cast<uint32_t>(seed); ea.seed_hi = static_cast<uint32_t>(seed >> 32); ea.rng_offset = rng_offset;
  p.out.C = C; p.out.ldc = ldc; p.out.out_f32 = out_f32;
  p.out.vec_ok = (reinterpret_cast<uintptr_t>(C) & 15u) == 0 && ldc % (out_f32 ? 4 : 8) == 0;
  // The operand with more rows goes to the tile's 128 rows where that leaves less of the tiles empty.
  const long long as_is = (m + 127ll) / 128 * 128 * pad_columns(n), turned = (n + 127ll) / 128 * 128 * pad_columns(m);
  p.swapped = turned < as_is;
  if (p.swapped) std::swap(a, b);
  p.out.M = a.outer; p.out.N = b.outer;
  p.tiles_m = (p.out.M + 127) / 128;
  p.num_kb = (a.inner + 255) / 256;
  p.ca = a.codes; p.cb = b.codes; p.pitch_a = a.pitch; p.pitch_b = b.pitch; p.tile_a = a.tile;
  p.sa = a.scales; p.sb = b.scales; p.spitch = a.spitch;
  p.status = c->status; p.wait_limit_ns = c->wait_limit_ns;
  // Columns of a tile: B's rows padded, as its scales lie; a column of more has its tile in the middle of a scale tile, which
  // tensor memory cannot address. Partitions of the sum, by what they take in us: per round of tiles, the k-blocks at 135
  // bytes/ns and the output stage; when split, the exchange, at 30 bytes/ns of what each CTA gets.
  const int cols = p.out.N > 64 ? 128 : pad_columns(p.out.N);
  const long long tiles = static_cast<long long>(p.tiles_m) * ((p.out.N + cols - 1) / cols);
  int splits = 1;
  double here = 0.0;
  for (int s = 1, log = 0; s <= 8 && (s == 1 || (p.num_kb >= s && tiles * s <= dot_room(c, log))); s *= 2, ++log) {
    const double kb = (20480.0 + 128.0 * cols) * 7.4e-6, out = 0.5 + cols / 128.0;
    const double us = 4.5 + (tiles * s + c->sm_count - 1) / c->sm_count * (kb * ((p.num_kb + s - 1) / s) + out / s) +
                      (s > 1 ? 1.0 + 512.0 * cols * (s - 1) / s * 3.3e-5 : 0.0);
    if (s == 1 || us < here) {
      here = us;
      splits = s;
    }
  }
  // Or pairs of SMs on tiles of 256 x 256 (block_dot_pair.cu), by the sum of what both take in us: a start, and per round
  // of tiles its k-blocks and its output stage. Here / pairs, nvfp4: 8192^3 235 / 162, 4096^3 49 / 34, 2048^3 13.9 / 9.8,
  // 8192 x 512 x 8192 25.0 / 18.4, 1000^3 6.9 / 7.0, 1536 x 1536 x 4096 9.2 / 11.9, 4096 x 128 x 9216 10.4 / 16.4.
  const long long pair_tiles = ((m + 255ll) / 256) * ((n + 255ll) / 256);
  const double pairs = 5.5 + (pair_tiles + c->sm_count / 2 - 1) / (c->sm_count / 2) * (0.33 * p.num_kb + 0.7);
  if (m > 64 && n > 64 && pairs < here) {
    if (p.swapped) std::swap(a, b);
    return run_block_dot_pair(c, a, b, nv, make_out(C, m, n, ldc, out_f32, ea), static_cast<cudaStream_t>(stream));
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define NG_DOT(kn) (nv ? launch_dot<kn, true>(c, p, splits, s) : launch_dot<kn, false>(c, p, splits, s))
  switch (cols) {
    case 16: return NG_DOT(16);
    case 32: return NG_DOT(32);
    case 64: return NG_DOT(64);
    default: return NG_DOT(128);
  }
#undef NG_DOT
}

int ng_block_dot_f16(const void* A, int lda, const ng_block_desc* B, void* C, int m, int ldc, int out_f32, float alpha,
                     float beta, int relu, int sr_bits, unsigned long long seed, unsigned int rng_offset, void* stream) {
  int rc = check_shape(B);
  if (rc != NG_OK) return rc;
  if (!A) return fail(NG_ERR_INVALID_ARG, "null operand");
  if (B->format != NG_BLOCK_MXFP8) return fail(NG_ERR_UNSUPPORTED, "an fp16 matrix is multiplied with one in mxfp8");
  if (B->axis != 0) return fail(NG_ERR_UNSUPPORTED, "blocks run along the sum: axis 0 of B");
  const int n = B->cols, k = B->rows;
  if (m < 1) return fail(NG_ERR_INVALID_ARG, "m must be positive");
  if (lda < k) return fail(NG_ERR_INVALID_ARG, "leading dimension too small");
  rc = check_output(C, ldc, n, sr_bits, out_f32);
  if (rc != NG_OK) return rc;
  DeviceCtx* c = current_ctx();
  if (!c) return NG_ERR_CUDA;
  BlockView b;
  rc = block_view(c, B, b);
  if (rc != NG_OK) return rc;
  EpiArgs ea;
  ea.alpha = alpha; ea.beta = beta; ea.relu = relu; ea.sr_bits = sr_bits;
  ea.seed_lo = static_cast<uint32_t>(seed); ea.seed_hi = static_cast<uint32_t>(seed >> 32); ea.rng_offset = rng_offset;
  return run_block_dot_f16(c, A, lda, *B, b, C, m, ldc, out_f32, ea, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
