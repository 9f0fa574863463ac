// Large products of two matrices in 4-bit blocks, on pairs of SMs (tcgen05 cta_group::2).
//
// At the rate of the 4-bit MMAs a k-block of 128 rows x 256 columns takes 512 cycles and 54 KB of operands: the SM
// cannot take them in that fast (366 ns measured, 150 bytes/ns). Two SMs on one tile of 256 x 256 share B: each
// holds 128 rows of A, half of B's columns and the scales, 38 KB per k-block. The first CTA's thread issues the MMAs for
// both; the copies of both CTAs are counted on its barriers (which TMA does for pairs, and plain bulk copies do not:
// with those, the second CTA passed the news on, which took 0.6 us per k-block as a release). CTAs stay on the device and
// take tile after tile. The accumulator and the scales leave no room for a second accumulator in tensor memory, so that a
// tile's output stage first takes the accumulator to registers, rounded to fp16, and the next tile's products start while
// it is stored.
//
//   warp 0      producer, of this CTA's operands
//   warp 1      scale copies and MMAs of both, in the first CTA
//   warps 2-9   output stage: two warps per group of 32 lanes, each half of the columns
#include <algorithm>
#include <atomic>

#include "block_mma.cuh"
#include "blocks.h"

namespace ngb {

namespace {

constexpr int kPairThreads = 320;
constexpr int kPairStages = 5;
constexpr uint32_t kPairOut = 8 * 4096;        // output staging
constexpr uint32_t kPairCtrl = 256;

template <bool kNv>
struct PairTile {
  static constexpr uint32_t kCodes = 128u * 128u;                         // of each operand, per CTA and k-block
  static constexpr uint32_t kScales = (kNv ? 4 : 2) * kScaleTile;          // of 128 rows
  static constexpr uint32_t kStage = 2 * kCodes + 3 * kScales;             // A's, and all of B's in both CTAs
  static constexpr uint32_t kStageStep = (kStage + 1023u) & ~1023u;
  static constexpr int kScaleCols = (kNv ? 4 : 2) * 12;                    // of tensor memory
  static constexpr uint32_t kSmem = kPairStages * kStageStep + kPairOut + kPairCtrl + 1024u;
  static_assert(kSmem <= 232448u, "shared memory");
  static_assert(256 + 2 * kScaleCols <= 512, "tensor memory");
};

// Codes and scales as rows of 128 bytes, one behind the other (zeros beyond the last tile), and the output.
struct PairMaps {
  CUtensorMap ca, cb, sa, sb, out;
};
struct PairParams {
  int num_kb, tiles_n, tiles;
  OutParams out;
  int* status;
  unsigned long long wait_limit_ns;
};

// Arrival at a barrier of either CTA that publishes no memory: what it orders, reads of tensor memory, has been waited
// for and fenced by tcgen05's own means. (As a release at cluster scope it takes some 0.5 us.)
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

template <bool kNv, int kForm>
__global__ void __launch_bounds__(kPairThreads, 1)
block_dot_pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairParams p) {
  using T = PairTile<kNv>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* ring_gen = smem_raw + (ring - smem_u32(smem_raw));
  const uint32_t staging = ring + kPairStages * T::kStageStep;
  const uint32_t ctrl = staging + kPairOut;
  auto full_bar = [&](int s) { return ctrl + 8u * s; };
  auto empty_bar = [&](int s) { return ctrl + 8u * (kPairStages + s); };
  const uint32_t accf_bar = ctrl + 8u * (2 * kPairStages), acce_bar = accf_bar + 8u;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring_gen + (ctrl - ring) + 8 * (2 * kPairStages + 2));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int first_tile = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(accf_bar, 1);
    mbar_init(acce_bar, 16);         // output-stage warps of both CTAs
    *abort_flag = 0;
    mbar_fence_init();
    if (p.out.store) tma_prefetch_desc(&maps.out);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                // the other CTA's barriers and tensor memory exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  bool gave_up = false;
  if (warp == 0) {
    int it = 0;
    for (int t = first_tile; t < p.tiles && !gave_up; t += step) {
      const int rt = t / p.tiles_n * 2 + rank, ct = t % p.tiles_n * 2;
      // lane by lane: A, its scales, B, the scales of B's two tiles
      const CUtensorMap* map = lane == 0 ? &maps.ca : lane == 1 ? &maps.sa : lane == 2 ? &maps.cb : &maps.sb;
      const int rows = lane == 0 || lane == 2 ? 128 : static_cast<int>(T::kScales / 128);      // of a k-block
      const int row0 = (lane < 2 ? rt : lane == 2 ? ct + rank : ct + lane - 3) * p.num_kb * rows;
      const uint32_t at = lane == 0 ? 0u : lane == 1 ? 2 * T::kCodes : lane == 2 ? T::kCodes : 2 * T::kCodes + (lane - 2) * T::kScales;
      for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
        const int s = it % kPairStages;
        if (it >= kPairStages &&
            !mbar_wait(empty_bar(s), (it / kPairStages - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_PRODUCER, p.wait_limit_ns))
          gave_up = true;
        if (__any_sync(0xffffffffu, gave_up)) {
          gave_up = true;
          break;
        }
        if (rank == 0 && lane == 0) mbar_expect_tx(full_bar(s), 2 * T::kStage);
        __syncwarp();
        if (lane < 5) tma_load_5d_pair(ring + s * T::kStageStep + at, map, map_to_cta(full_bar(s), 0), 0, row0 + kb * rows, 0, 0, 0);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      int it = 0, local = 0;
      for (int t = first_tile; t < p.tiles && !gave_up; t += step, ++local) {
        if (local > 0 && !mbar_wait(acce_bar, (local - 1) & 1, abort_flag, p.status, NG_DEV_TIMEOUT_ACC, p.wait_limit_ns)) {
          gave_up = true;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < p.num_kb; ++kb, ++it) {
          const int s = it % kPairStages, phase = (it / kPairStages) & 1;
          if (!mbar_wait(full_bar(s), phase, abort_flag, p.status, NG_DEV_TIMEOUT_MMA, p.wait_limit_ns)) {
            gave_up = true;
            break;
          }
          tc_fence_after();
          const uint32_t a = ring + s * T::kStageStep, sa = a + 2 * T::kCodes;
          mma_kblock<kNv, true, 2>(tmem, a, a + T::kCodes, sa, sa + T::kScales, tmem + 256 + (it & 1) * T::kScaleCols,
                                   block_idesc(256, 256, kNv), kb == 0);
          tc_commit_pair(map_to_cta(empty_bar(s), 0));
          tc_commit_pair(map_to_cta(empty_bar(s), 1));
        }
        if (!gave_up) {
          tc_commit_pair(map_to_cta(accf_bar, 0));
          tc_commit_pair(map_to_cta(accf_bar, 1));
        }
      }
    }
  } else {
    const int group = warp & 3, half = (warp - 2) >> 2;
    const uint32_t stage = staging + (warp - 2) * 4096u;
    uint8_t* stage_gen = ring_gen + (stage - ring);
    const uint32_t done_bar = map_to_cta(acce_bar, 0);
    auto row_of = [&](int t) { return t / p.tiles_n * 256 + rank * 128 + group * 32; };
    auto col_of = [&](int t) { return t % p.tiles_n * 256 + half * 128; };
    int local = 0;
    for (int t = first_tile; t < p.tiles; t += step, ++local) {
      const int m0 = row_of(t), n0 = col_of(t);
      if (local == 0) out_ahead<kForm, 128>(p.out, m0, n0);
      const bool ok = mbar_wait(accf_bar, local & 1, abort_flag, p.status, NG_DEV_TIMEOUT_EPILOGUE, p.wait_limit_ns);
      if (__any_sync(0xffffffffu, !ok)) {
        gave_up = true;
        break;
      }
      tc_fence_after();
      if (t + step < p.tiles) out_ahead<kForm, 128>(p.out, row_of(t + step), col_of(t + step));
      const uint32_t taddr = tmem + (static_cast<uint32_t>(group * 32) << 16) + half * 128;
      auto release = [&] { if (lane == 0) mbar_arrive_relaxed(done_bar); };
      out_tile<kForm, 128>(p.out, &maps.out, taddr, stage, stage_gen, m0, n0, release);
    }
    if (lane == 0) tma_store_wait_all();
  }
  if (gave_up) wait_for_strays();
  __syncwarp();
  __syncthreads();
  cluster_sync_all();                // nobody arrives here any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Boxes of `box_rows` rows of a run of rows of 128 bytes (as 16-bit units), as they lie.
int rows_map(CUtensorMap* map, const void* base, long long bytes, int box_rows) {
  const uint64_t dims[5] = {64, static_cast<uint64_t>(bytes / 128), 1, 1, 1};
  const uint64_t all = static_cast<uint64_t>(bytes);
  const uint64_t strides[4] = {128, all, all, all};
  const uint32_t box[5] = {64, static_cast<uint32_t>(box_rows), 1, 1, 1};
  return make_tensor_map(map, base, dims, strides, box, 2, true);
}

template <bool kNv, int kForm>
int launch_pair(DeviceCtx* c, const BlockView& a, const BlockView& b, const PairParams& p, cudaStream_t stream) {
  using T = PairTile<kNv>;
  PairMaps maps = {};
  const int rows = static_cast<int>(T::kScales / 128);
  int rc = rows_map(&maps.ca, a.codes, a.pitch * ((a.outer + 127ll) / 128), 128);
  if (rc == NG_OK) rc = rows_map(&maps.cb, b.codes, b.pitch * ((b.outer + 127ll) / 128), 128);
  if (rc == NG_OK) rc = rows_map(&maps.sa, a.scales, a.spitch * ((a.outer + 127ll) / 128), rows);
  if (rc == NG_OK) rc = rows_map(&maps.sb, b.scales, b.spitch * ((b.outer + 127ll) / 128), rows);
  if (rc == NG_OK && p.out.store) rc = out_map(&maps.out, p.out);
  if (rc != NG_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min(p.tiles, c->sm_count / 2)));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = T::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tuning().dependent_launch != 0 ? 2 : 1;
  static std::atomic<unsigned long long> ready{0};
  if (!(ready.load(std::memory_order_relaxed) >> c->device & 1u)) {
    NG_CUDA(cudaFuncSetAttribute(block_dot_pair_kernel<kNv, kForm>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
    ready.fetch_or(1ull << c->device, std::memory_order_relaxed);
  }
  NG_CUDA(cudaLaunchKernelEx(&cfg, block_dot_pair_kernel<kNv, kForm>, maps, p));
  NG_CHECK_LAUNCH();
  return NG_OK;
}

}  // namespace

int run_block_dot_pair(DeviceCtx* c, const BlockView& a, const BlockView& b, bool nv, const OutParams& out, cudaStream_t stream) {
  PairParams p = {};
  p.num_kb = (a.inner + 255) / 256;
  p.tiles_n = (b.outer + 255) / 256;
  const long long tiles = static_cast<long long>(p.tiles_n) * ((a.outer + 255ll) / 256);
  if (tiles > 0x3fffffffll) return fail(NG_ERR_TOO_LARGE, "too many tiles");
  p.tiles = static_cast<int>(tiles);
  p.out = out;
  p.status = c->status; p.wait_limit_ns = c->wait_limit_ns;
#define NG_PAIR(form) (nv ? launch_pair<true, form>(c, a, b, p, stream) : launch_pair<false, form>(c, a, b, p, stream))
  switch (out_form(out)) {
    case kOutLean: return NG_PAIR(kOutLean);
    case kOutF16: return NG_PAIR(kOutF16);
    default: return NG_PAIR(kOutF32);
  }
#undef NG_PAIR
}

}  // namespace ngb
