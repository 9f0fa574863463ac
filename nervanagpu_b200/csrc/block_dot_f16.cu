// Products of a plain fp16 matrix with one in mxfp8 (blocks.cuh): the weight gradient of a fully-connected layer from
// its deltas (m x k, k images) and the 8-bit record of its input (n x k along the images).
//
//   C[i,j] = epilogue(sum_k A[i,k] X[j,k]),   X[j,k] = code * 2^e, an fp16 number when it was made from one
//
// block_dot_f16_kernel multiplies in fp16 on tcgen05 with fp32 accumulation. The record is brought to fp16 on its way
// into shared memory: its codes come by TMA, eight warps take 64 of each row per k-block, convert them, scale them by
// their power of two (exact) and store them where the 128-byte swizzle wants them; no fp16 copy of the record is ever
// in memory. A's tiles come by TMA, or, from rows that TMA cannot address, through the same warps. A CTA
// computes tiles of 128 x kN, one after the other, with two accumulators, so that the output stage of one tile runs
// beside the products of the next: with few images the time is that of writing C. Few tiles with a long sum are split
// along it instead (kMixSplit), a tile over the CTAs of a cluster (block_share.cuh).
//
//   warp 0       TMA producer
//   warp 1       tensor memory, MMAs
//   warps 2-9    output stage: two warps per group of 32 lanes, each half of the columns
//   warps 10-17  the record to fp16
#include <algorithm>
#include <atomic>

#include "block_share.cuh"
#include "blocks.h"

namespace ngb {

namespace {

constexpr int kMixEpi = 8, kMixConv = 8;                  // warps
constexpr int kMixThreads = 32 * (2 + kMixEpi + kMixConv);
constexpr uint32_t kMixA = 128u * 128u;                   // a k-block of A: 128 rows of 64 fp16 numbers
constexpr uint32_t kMixStage = kMixEpi * 4096u;           // output staging: [32 rows][128 bytes] per warp
constexpr int kMixRaw = 3;                                // slots of codes
constexpr uint32_t kMixCtrl = 256;
constexpr uint32_t kMixSmemLimit = 232448;

constexpr int kMixSplit = 3;                              // besides the OutForms

template <int kN, bool kSplit>
struct MixTile {
  static constexpr uint32_t kB = kN * 128u;
  static constexpr uint32_t kSlot = kMixA + kB;
  static constexpr uint32_t kRaw = kN * 64u;              // a k-block of codes
  static constexpr uint32_t kOut = kSplit ? kShareTile<kN> : kMixStage;      // output staging, or the others' parts
  static constexpr int kRoom = static_cast<int>((kMixSmemLimit - 1024u - kMixCtrl - kOut - kMixRaw * kRaw) / kSlot);
  static constexpr int kStages = kRoom < 6 ? kRoom : 6;
  static constexpr uint32_t kSmem = kStages * kSlot + kMixRaw * kRaw + kOut + kMixCtrl + 1024u;
  static_assert(!kSplit || kOut <= kStages * kSlot, "the ring is smaller than the tile");
  static_assert(kSmem > kMixSmemLimit / 2, "an SM takes two CTAs: mix_room() asks for one instance only");
  static constexpr uint32_t kCols = 2 * kN;               // of tensor memory: two accumulators
  static constexpr int kEpiCols = kN > 64 ? kN / 2 : 64;  // columns of an output-stage warp (64: one of the two has them all)
};

struct MixParams {
  const __half* A;
  long long lda;
  int a_tma;
  int M, N, K;
  int tiles_n, tiles, num_kb;
  BlockView x;
  OutParams out;
  ShareOut share;
  int* status;
  unsigned long long wait_limit_ns;
};

template <int kN, int kForm>
__global__ void __launch_bounds__(kMixThreads, 1)
block_dot_f16_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapX,
                     const __grid_constant__ CUtensorMap mapC, const __grid_constant__ MixParams p) {
  constexpr bool kSplit = kForm == kMixSplit;
  using T = MixTile<kN, kSplit>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* ring_gen = smem_raw + (ring - smem_u32(smem_raw));
  const uint32_t raw = ring + T::kStages * T::kSlot, staging = raw + kMixRaw * T::kRaw;
  const uint32_t ctrl = staging + T::kOut;
  auto full_bar = [&](int s) { return ctrl + 8u * s; };
  auto empty_bar = [&](int s) { return ctrl + 8u * (6 + s); };
  auto accf_bar = [&](int a) { return ctrl + 8u * (12 + a); };
  auto acce_bar = [&](int a) { return ctrl + 8u * (14 + a); };
  auto rawf_bar = [&](int s) { return ctrl + 8u * (16 + s); };
  auto rawe_bar = [&](int s) { return ctrl + 8u * (19 + s); };
  const uint32_t part_bar = ctrl + 8u * 22;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring_gen + (ctrl - ring) + 8 * 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this CTA's tiles and its part of their sums
  const int splits = kSplit ? static_cast<int>(cluster_size()) : 1, rank = kSplit ? static_cast<int>(cluster_cta_rank()) : 0;
  const int first_tile = kSplit ? blockIdx.x / splits : blockIdx.x, step = kSplit ? p.tiles : gridDim.x;
  const int kb0 = kSplit ? static_cast<int>(static_cast<long long>(p.num_kb) * rank / splits) : 0;
  const int kb1 = kSplit ? static_cast<int>(static_cast<long long>(p.num_kb) * (rank + 1) / splits) : p.num_kb;
  const uint32_t share_bytes = T::kOut / splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::kStages; ++s) {
      mbar_init(full_bar(s), kMixConv + (p.a_tma ? 1 : 0));
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(accf_bar(a), 1);
      mbar_init(acce_bar(a), kMixEpi);
    }
    for (int s = 0; s < kMixRaw; ++s) {
      mbar_init(rawf_bar(s), 1);
      mbar_init(rawe_bar(s), kMixConv);
    }
    mbar_init(part_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    if (kSplit) mbar_expect_tx(part_bar, (splits - 1) * share_bytes);
    if (p.a_tma) tma_prefetch_desc(&mapA);
    tma_prefetch_desc(&mapX);
    if (!kSplit && p.out.store) tma_prefetch_desc(&mapC);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), T::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (kSplit) cluster_arrive();      // (this CTA's barriers exist)
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  // (slots are counted over all tiles of this CTA: `it` = k-blocks so far)
  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += step) {
        const int m0 = t / p.tiles_n * 128, n0 = t % p.tiles_n * kN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % T::kStages, x = it % kMixRaw;
          if (it >= kMixRaw && !mbar_wait(rawe_bar(x), (it / kMixRaw - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns)) {
            ok = false;
            break;
          }
          mbar_expect_tx(rawf_bar(x), T::kRaw);
          tma_load_5d(raw + x * T::kRaw, &mapX, rawf_bar(x), kb * 32, n0, 0, 0, 0);
          if (!p.a_tma) continue;
          if (it >= T::kStages && !mbar_wait(empty_bar(s), (it / T::kStages - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns)) {
            ok = false;
            break;
          }
          mbar_expect_tx(full_bar(s), kMixA);
          tma_load_5d(ring + s * T::kSlot, &mapA, full_bar(s), kb * 64, m0, 0, 0, 0);
        }
      }
      if (!ok) wait_for_strays();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29), lo = 1u << 16;
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(kN >> 3) << 17) | ((128u >> 4) << 24);
      int it = 0, local = 0;
      bool ok = true;
      for (int t = first_tile; t < p.tiles && ok; t += step, ++local) {
        const int acc = local & 1;
        if (local >= 2 && !mbar_wait(acce_bar(acc), (local / 2 - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_ACC, p.wait_limit_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          const int s = it % T::kStages;
          if (!mbar_wait(full_bar(s), (it / T::kStages) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_MMA, p.wait_limit_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = ring + s * T::kSlot;
          tc_mma_f16_run<false, 4>(tmem + acc * kN, lo | (a >> 4), hi, lo | ((a + kMixA) >> 4), hi, idesc, kb != kb0, 2u, 2u);
          tc_commit(empty_bar(s));
        }
        if (ok) tc_commit(accf_bar(acc));
      }
      if (!ok) wait_for_strays();
    }
    __syncwarp();
  } else if (warp < 2 + kMixEpi) {
    const int group = warp & 3, half = (warp - 2) >> 2;
    const uint32_t stage = staging + (warp - 2) * 4096u;
    uint8_t* stage_gen = ring_gen + (stage - ring);
    auto row_of = [&](int t) { return t / p.tiles_n * 128 + group * 32; };
    auto col_of = [&](int t) { return t % p.tiles_n * kN + half * T::kEpiCols; };
    int local = 0;
    for (int t = first_tile; t < p.tiles; t += step, ++local) {
      const int acc = local & 1;
      const int m0 = row_of(t), n0 = col_of(t);
      if (local == 0) out_ahead<kForm, T::kEpiCols>(p.out, m0, n0);
      const bool ok = mbar_wait(accf_bar(acc), (local / 2) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_EPILOGUE, p.wait_limit_ns);
      if (__any_sync(0xffffffffu, !ok)) {
        wait_for_strays();
        break;
      }
      tc_fence_after();
      if (t + step < p.tiles) out_ahead<kForm, T::kEpiCols>(p.out, row_of(t + step), col_of(t + step));
      const uint32_t taddr = tmem + (static_cast<uint32_t>(group * 32) << 16) + acc * kN + half * T::kEpiCols;
      auto release = [&] { if (lane == 0) mbar_arrive(acce_bar(acc)); };
      if constexpr (kSplit) {
        // the partial tile, where the ring was
        float* row = reinterpret_cast<float*>(ring_gen) + (group * 32 + lane) * kSharePitch<kN>;
#pragma unroll 1
        for (int c = half * (kN / 2); c < (half + 1) * (kN / 2); c += 32) {
          uint32_t r[32];
          tc_ld_32x32(tmem + (static_cast<uint32_t>(group * 32) << 16) + c, r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<uint4*>(row + c)[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
        tc_fence_before();
        fence_async_smem();      // (the parts leave by bulk copies)
      } else if (half * T::kEpiCols >= kN) release();
      else out_tile<kForm, T::kEpiCols>(p.out, &mapC, taddr, stage, stage_gen, m0, n0, release);
    }
    if (lane == 0) tma_store_wait_all();
    __syncwarp();
  } else {
    // ---- the record to fp16: a thread has a row of the tile per k-block, or (128 or 64 columns) half or a quarter of one
    constexpr int kPer = 32 * kMixConv / kN;            // threads that share a row
    constexpr int kPieces = 4 / kPer;                   // 16 codes of a k-block each
    const int tid = threadIdx.x - 32 * (2 + kMixEpi);
    const int r = tid / kPer, part = tid % kPer;
    int it = 0;
    bool ok = true;
    for (int t = first_tile; t < p.tiles && ok; t += step) {
      const int m0 = t / p.tiles_n * 128, j = t % p.tiles_n * kN + r;
      // the scales of 128 codes are a word
      const uint8_t* scales = p.x.scales + static_cast<long long>(j) * p.x.spitch;
      uint32_t word = j < p.N ? *reinterpret_cast<const uint32_t*>(scales + kb0 / 2 * 4ll) : 0u;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % T::kStages, x = it % kMixRaw;
        // A, when TMA cannot: 16 rows per warp, two numbers per lane and row, on their way while this waits
        constexpr int kRows = 128 / kMixConv;
        __half2 from_a[kRows];
        const int a_row = (warp - 2 - kMixEpi) * kRows;
        if (!p.a_tma) {
          const int k0 = kb * 64 + lane;
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const __half* row = p.A + static_cast<long long>(m0 + a_row + i) * p.lda + k0;
            const bool row_ok = m0 + a_row + i < p.M;
            from_a[i] = __halves2half2(row_ok && k0 < p.K ? row[0] : zero_of<__half>(), row_ok && k0 + 32 < p.K ? row[32] : zero_of<__half>());
          }
        }
        ok = mbar_wait(rawf_bar(x), (it / kMixRaw) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns) &&
             (it < T::kStages || mbar_wait(empty_bar(s), (it / T::kStages - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns));
        if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
        const uint8_t* src = ring_gen + (raw - ring) + x * T::kRaw + r * 64;
        uint8_t* b = ring_gen + s * T::kSlot + kMixA + r * 128;
        uint4 w[kPieces];
        float scale[(kPieces + 1) / 2];
        bool fits = true;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int piece = part * kPieces + i;                // swizzled by 64 bytes as TMA left them
          w[i] = *reinterpret_cast<const uint4*>(src + ((piece ^ (r >> 1 & 3)) << 4));
          if (i % 2 == 0) {
            scale[i / 2] = block_scale_value<NG_BLOCK_MXFP8>(word >> ((kb & 1) * 16 + (piece >> 1) * 8) & 0xffu, 1.0f);
            fits = fits && block_scale_fits_f16<NG_BLOCK_MXFP8>(scale[i / 2]);
          }
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int piece = part * kPieces + i;
          uint4 v[2];
          if (fits) {
            const __half2 by = __float2half2_rn(scale[i / 2]);
            v[0] = block_decode8_f16<NG_BLOCK_MXFP8>(make_uint2(w[i].x, w[i].y), by);
            v[1] = block_decode8_f16<NG_BLOCK_MXFP8>(make_uint2(w[i].z, w[i].w), by);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float f[8];
              block_decode8<NG_BLOCK_MXFP8>(h ? make_uint2(w[i].z, w[i].w) : make_uint2(w[i].x, w[i].y), scale[i / 2], f);
              block_limit<NG_BLOCK_MXFP8, __half>(scale[i / 2], f);
              __half2* o = reinterpret_cast<__half2*>(&v[h]);
#pragma unroll
              for (int y = 0; y < 4; ++y) o[y] = __floats2half2_rn(f[2 * y], f[2 * y + 1]);
            }
          }
          *reinterpret_cast<uint4*>(b + (((2 * piece) ^ (r & 7)) << 4)) = v[0];
          *reinterpret_cast<uint4*>(b + (((2 * piece + 1) ^ (r & 7)) << 4)) = v[1];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(rawe_bar(x));
        if ((kb & 1) && kb + 1 < kb1 && j < p.N) word = *reinterpret_cast<const uint32_t*>(scales + (kb + 1) * 2ll);
        if (!p.a_tma) {
          uint8_t* a = ring_gen + s * T::kSlot + a_row * 128 + ((lane * 2) & 15);
          const int at = (lane * 2) & 112;
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const int sw = (i & 7) << 4;         // (a_row is a multiple of 8)
            *reinterpret_cast<__half*>(a + i * 128 + (at ^ sw)) = __low2half(from_a[i]);
            *reinterpret_cast<__half*>(a + i * 128 + ((at + 64) ^ sw)) = __high2half(from_a[i]);
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(s));
      }
    }
  }
  __syncthreads();
  if (kSplit) share_push(ring, staging, share_bytes, rank, splits, part_bar);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, T::kCols);
  }
  if constexpr (kSplit) {
    share_wait(part_bar, abort_flag, p.status, p.wait_limit_ns);
    if (!*abort_flag)
      share_store<kN, kMixThreads>(p.share, false, reinterpret_cast<float*>(ring_gen), reinterpret_cast<const float*>(ring_gen + (staging - ring)),
                                   splits, rank, first_tile / p.tiles_n * 128, first_tile % p.tiles_n * kN);
    __syncwarp();
    cluster_wait();
  }
}

template <int kN, int kForm>
int launch_mix(DeviceCtx* c, MixParams& p, int splits, cudaStream_t stream) {
  constexpr bool kSplit = kForm == kMixSplit;
  using T = MixTile<kN, kSplit>;
  p.tiles_n = (p.N + kN - 1) / kN;
  const long long tiles = static_cast<long long>(p.tiles_n) * ((p.M + 127ll) / 128);
  if (tiles > 0x3fffffffll) return fail(NG_ERR_TOO_LARGE, "too many tiles");
  p.tiles = static_cast<int>(tiles);
  CUtensorMap mapA = {}, mapX, mapC = {};
  int rc = NG_OK;
  if (p.a_tma) rc = plain_map(&mapA, p.A, p.M, p.K, p.lda, 64, 128, 2);
  // (codes as 16-bit units; zeros beyond the last row)
  if (rc == NG_OK) rc = plain_map(&mapX, p.x.codes, p.N, p.x.pitch / 2, p.x.pitch / 2, 32, kN, 2);
  if (rc == NG_OK && !kSplit && p.out.store) rc = out_map(&mapC, p.out);
  if (rc != NG_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(kSplit ? tiles * splits : std::min<long long>(tiles, c->sm_count)));
  cfg.blockDim = dim3(kMixThreads);
  cfg.dynamicSmemBytes = T::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (tuning().dependent_launch != 0) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (kSplit) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = splits;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  static std::atomic<unsigned long long> ready{0};
  if (!(ready.load(std::memory_order_relaxed) >> c->device & 1u)) {
    NG_CUDA(cudaFuncSetAttribute(block_dot_f16_kernel<kN, kForm>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
    ready.fetch_or(1ull << c->device, std::memory_order_relaxed);
  }
  NG_CUDA(cudaLaunchKernelEx(&cfg, block_dot_f16_kernel<kN, kForm>, mapA, mapX, mapC, p));
  NG_CHECK_LAUNCH();
  return NG_OK;
}

}  // namespace

// CTAs of a split product that run at the same time, asked once per device and cluster size.
static int mix_room(const DeviceCtx* c, int log) {
  static std::atomic<int> known[64][4];
  int n = known[c->device][log].load(std::memory_order_relaxed);
  if (n == 0) {
    n = cluster_room(c, reinterpret_cast<const void*>(block_dot_f16_kernel<128, kMixSplit>), kMixThreads,
                     MixTile<128, true>::kSmem, log);
    known[c->device][log].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Long sums: the record as fp16 rows in scratch memory, then the product of two fp16 matrices. False, with nothing queued, when
// there is no room for the copy or for what the product needs (parts of its sum, A's odd rows in order).
static bool from_scratch(DeviceCtx* c, const void* A, int lda, const ng_block_desc& d, const BlockView& x, void* C, int m, int ldc,
                         int out_f32, const EpiArgs& ea, cudaStream_t stream, int& rc) {
  AuxClaim room;
  void* plain = nullptr;
  const long long ld = (x.inner + 7ll) / 8 * 8;
  if (room.room(c, stream, static_cast<size_t>(ld) * x.outer * 2, &plain) != NG_OK) {
    cudaGetLastError();
    return false;
  }
  GemmCall g = {};
  g.A = A; g.B = plain; g.C = C; g.b_t = 1; g.m = m; g.n = x.outer; g.k = x.inner;
  g.lda = lda; g.ldb = ld; g.ldc = ldc; g.alpha = ea.alpha; g.beta = ea.beta; g.relu = ea.relu; g.sr_bits = ea.sr_bits;
  g.seed = static_cast<unsigned long long>(ea.seed_hi) << 32 | ea.seed_lo; g.rng_offset = ea.rng_offset;
  g.batch = 1; g.loops = 1; g.out_f32 = out_f32;
  if (!reserve_gemm(c, g, stream)) return false;
  rc = dequantize_f16(c, d, x, static_cast<__half*>(plain), ld, stream);
  if (rc != NG_OK) return true;
  rc = run_gemm(g, stream);
  return true;
}

int run_block_dot_f16(DeviceCtx* c, const void* A, int lda, const ng_block_desc& d, const BlockView& x, void* C, int m, int ldc,
                      int out_f32, const EpiArgs& ea, cudaStream_t stream) {
  MixParams p = {};
  p.A = static_cast<const __half*>(A); p.lda = lda;
  p.a_tma = (reinterpret_cast<uintptr_t>(A) & 15u) == 0 && lda % 8 == 0;
  p.M = m; p.N = x.outer; p.K = x.inner;
  p.num_kb = (x.inner + 63) / 64;
  p.x = x;
  p.out = make_out(C, m, x.outer, ldc, out_f32, ea);
  p.status = c->status; p.wait_limit_ns = c->wait_limit_ns;
  // Columns of a tile: what takes the SMs least time, a tile of n columns counted as n + 64 (its rows of A, its start
  // and its end). 1001 x 4097 x 125: one round of 136 tiles of 256 columns, or four of 520 tiles of 64.
  const long long row_tiles = (m + 127ll) / 128;
  int cols = 256;
  long long best = 0;
  for (int n = 256; n >= 64; n /= 2) {
    const long long tiles = row_tiles * ((p.N + n - 1ll) / n), cost = (tiles + c->sm_count - 1) / c->sm_count * (n + 64);
    if (best == 0 || cost < best) {
      best = cost;
      cols = n;
    }
  }
  // Whole sums, sums in parts, or a copy, by what each takes in us. Measured, whole / parts / copy: 512 x 512 x 1024 10.0 / 6.7
  // / 11.9, 300 x 300 x 4000 31 / 8.9 / 14.3, x 4001 65 / 13.2 / 16.9, 5844 x 64 x 773 15.9 / 11.7 / 13.8, 512 x 512 x 8192
  // 62 / 20.5 / 16.4, 128 x 128 x 256 5.0 / 5.0 / 7.0; without room for parts, whole / copy: 1001 x 4097 x 1000 17.5 / 21.9,
  // 4096 x 4096 x 250 27 / 18, 4096 x 9216 x 128 20.0 / 20.9.
  // Whole: the tiles one after the other, k-blocks, whose conversion takes longer than their products (A's odd rows more
  // still), and output.
  const double odd = p.a_tma ? 0.0 : 0.45;
  auto kblock = [&](int n) { return 0.32 + n * 0.0013 + odd; };
  const long long rounds = best / (cols + 64);
  const double out = cols * (out_f32 ? 0.017 : 0.0085);       // a tile's; that of one tile runs beside the products of the next
  const double whole = 4.0 + rounds * std::max(p.num_kb * kblock(cols), out) + out;
  // Or the sum in parts, with their exchange at 30 bytes/ns of what each CTA gets.
  double here = whole;
  int splits = 1, split_cols = 0;
  for (int n = 64; n <= 128; n *= 2)
    for (int log = 1; log <= 3; ++log) {
      const int s = 1 << log;
      if (p.num_kb < s || row_tiles * ((p.N + n - 1ll) / n) * s > mix_room(c, log)) break;
      const double us = 3.6 + (p.num_kb + s - 1) / s * kblock(n) + 1.0 + 512.0 * n * (s - 1) / s * 3.3e-5 + 1.0 / s;
      if (us < here) {
        here = us;
        splits = s;
        split_cols = n;
      }
    }
  // Or an fp16 copy of the record, and of A's odd rows, which cost launches and traffic but leave the product alone.
  const double copy = 11.0 + std::max(2.0 * m * p.N * p.K * 1e-9, m * (out_f32 ? 4.0 : 2.0) * p.N * 2.6e-7) +
                      (3.0 * p.N * p.K + (p.a_tma ? 0.0 : 4.0 * m * p.K)) * 2e-7;
  int rc;
  if (copy < here && from_scratch(c, A, lda, d, x, C, m, ldc, out_f32, ea, stream, rc)) return rc;
  if (splits > 1) {
    p.share = {m, p.N, C, ldc, out_f32, (reinterpret_cast<uintptr_t>(C) & 15u) == 0 && ldc % (out_f32 ? 4 : 8) == 0, ea};
    return split_cols == 128 ? launch_mix<128, kMixSplit>(c, p, splits, stream) : launch_mix<64, kMixSplit>(c, p, splits, stream);
  }
#define NG_MIX(form) \
  (cols == 256 ? launch_mix<256, form>(c, p, 1, stream) : cols == 128 ? launch_mix<128, form>(c, p, 1, stream) : launch_mix<64, form>(c, p, 1, stream))
  switch (out_form(p.out)) {
    case kOutLean: return NG_MIX(kOutLean);
    case kOutF16: return NG_MIX(kOutF16);
    default: return NG_MIX(kOutF32);
  }
#undef NG_MIX
}

}  // namespace ngb
