// The end of a product whose sum is split over the CTAs of a thread-block cluster: each holds a partial tile in shared memory,
// gets a share of the tile's rows from all the others by bulk copies between their shared memories, adds them up in the order
// of the partitions and stores them: one launch, no scratch memory, the same bits every time. (Fetched by loads from the
// others' shared memory instead, the partial tiles of 4096 x 128 x 9216 took 3.8 us of 12.2.)
#pragma once
#include <type_traits>

#include "block_out.cuh"

namespace ngb {

// Partial tiles: 128 rows of kN columns, the rows 4 floats longer, so that lanes in successive rows meet different banks.
template <int kN>
constexpr int kSharePitch = kN + 4;
template <int kN>
constexpr uint32_t kShareTile = 128u * kSharePitch<kN> * 4u;

// Where the tile goes; its rows and columns in all.
struct ShareOut {
  int M, N;
  void* C;
  long long ldc;
  int out_f32, vec_ok;       // vec_ok: C's rows are aligned vectors
  EpiArgs ea;
};

// bytes of this CTA's shared memory to another's (or its own), counted on a barrier there
__device__ __forceinline__ void bulk_push(uint32_t dst_cluster, uint32_t src, uint32_t bytes, uint32_t bar_cluster) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_cluster),
               "r"(src), "r"(bytes), "r"(bar_cluster)
               : "memory");
}
// (relaxed: neither arrival publishes memory. The barriers that the first tells of are fenced when they are made, the second
// only says that nobody reads this CTA's tile any more. As a release each took half a microsecond.)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}


// The partial tile at `tile` is written, fenced and synchronised: its shares to the others.
__device__ __forceinline__ void share_push(uint32_t tile, uint32_t parts, uint32_t share_bytes, int rank, int splits, uint32_t part_bar) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  cluster_wait();            // (with everybody's arrival long ago: the barriers that the parts count on exist)
  if (threadIdx.x < 32 && lane > 0 && lane < splits) {
    const int to = (rank + lane) % splits;
    bulk_push(map_to_cta(parts + rank * share_bytes, to), tile + to * share_bytes, share_bytes, map_to_cta(part_bar, to));
  }
  __syncwarp();
}
__device__ __forceinline__ void share_wait(uint32_t part_bar, volatile int* abort_flag, int* status, unsigned long long limit_ns) {
  if (!mbar_wait(part_bar, 0, abort_flag, status, NG_DEV_TIMEOUT_EPILOGUE, limit_ns)) {
    int none = 0;            // given up: the parts come all the same, those of a CTA that gave up too, and later than here maybe
    mbar_wait(part_bar, 0, &none, status, NG_DEV_TIMEOUT_EPILOGUE, limit_ns);
  }
  __syncwarp();
  cluster_arrive();          // (with everybody's: all parts have arrived, nobody's tile is read any more)
  __syncthreads();           // the abort flag is final
}

// The sum and the output stage. swapped: the tile's rows are C's columns.
template <int kN, int kThreads>
__device__ __forceinline__ void share_store(const ShareOut& p, bool swapped, float* tile, const float* others, int splits, int rank, int m0, int n0) {
  constexpr int kPitch = kSharePitch<kN>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = 128 / splits, r0 = rank * rows;       // this CTA's share
  // (When another partition gave up, its part holds what was there: the status word tells.)
  const bool whole = !swapped && p.vec_ok;        // rows of whole aligned vectors of C
  const int live = max(0, min(rows, p.M - m0 - r0));
  float* own = tile + r0 * kPitch;
  auto part = [&](int s) { return s == rank ? own : others + s * rows * kPitch; };
  auto sum4 = [&](auto n, int off) {
    constexpr int kParts = decltype(n)::value;
    float4 x[kParts];
#pragma unroll
    for (int s = 0; s < kParts; ++s) x[s] = *reinterpret_cast<const float4*>(part(s) + off);
#pragma unroll
    for (int s = 1; s < kParts; ++s) {
      x[0].x += x[s].x; x[0].y += x[s].y; x[0].z += x[s].z; x[0].w += x[s].w;
    }
    return x[0];
  };
  auto store_whole = [&](auto n) {
    for (int i = threadIdx.x; i < live * (kN / 8); i += kThreads) {
      const int r = i / (kN / 8), c = (i % (kN / 8)) * 8;
      const int col = n0 + c;
      const long long row = m0 + r0 + r;
      if (col >= p.N) continue;
      const float4 x = sum4(n, r * kPitch + c), y = sum4(n, r * kPitch + c + 4);
      float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      const unsigned long long lin = static_cast<unsigned long long>(row) * p.N + col;
      const int nvalid = min(8, p.N - col);
      uint8_t* crow = static_cast<uint8_t*>(p.C) + row * p.ldc * (p.out_f32 ? 4 : 2);
      if (p.out_f32) epi_store8<true>(p.ea, v, crow, crow, col, lin, nvalid, true);
      else epi_store8<false>(p.ea, v, crow, crow, col, lin, nvalid, true);
    }
  };
  auto sum_in_place = [&](auto n) {
    for (int i = threadIdx.x; i < live * (kN / 4); i += kThreads) {
      const int off = i / (kN / 4) * kPitch + i % (kN / 4) * 4;
      *reinterpret_cast<float4*>(own + off) = sum4(n, off);
    }
    __syncthreads();
  };
#define NG_BY_PARTS(call, from)                                                 \
  switch (splits) {                                                             \
    case 1: if (from <= 1) call(std::integral_constant<int, 1>()); break;       \
    case 2: call(std::integral_constant<int, 2>()); break;                      \
    case 4: call(std::integral_constant<int, 4>()); break;                      \
    default: call(std::integral_constant<int, 8>()); break;                     \
  }
  if (whole) {
    NG_BY_PARTS(store_whole, 1)
  } else {
    // C's rows are at any address, or run down the tile: one output per lane and access, neighbours in lanes
    NG_BY_PARTS(sum_in_place, 2)
    const int cols = min(kN, p.N - n0);
    const int runs = swapped ? cols : live, len = swapped ? live : cols;       // rows of C that have some, and how many
    const int run_step = swapped ? 1 : kPitch, step = swapped ? kPitch : 1;
    const long long row0 = swapped ? n0 : m0 + r0, col0 = swapped ? m0 + r0 : n0;
    const int width = swapped ? p.M : p.N;
    auto rows_of = [&](auto* base) {
      using E = std::remove_pointer_t<decltype(base)>;
      constexpr int kWarps = kThreads / 32;
      if (sizeof(E) == 2 && p.ea.sr_bits) {
        // eight neighbours at a time, which share their random bits
        const int eights = (len + 7) / 8;
#pragma unroll 1
        for (int i = threadIdx.x; i < runs * eights; i += kThreads) {
          const int u = i / eights, c = i % eights * 8;
          const float* src = own + u * run_step + c * step;
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = c + j < len ? src[j * step] : 0.0f;
          E* row = base + (row0 + u) * p.ldc;
          epi_store8_call<false>(p.ea, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], row, row, static_cast<int>(col0) + c,
                                 static_cast<unsigned long long>(row0 + u) * width + col0 + c, min(8, len - c), false);
        }
        return;
      }
      // (what C held in four rows is on its way together: one by one, 128 rows of a tile took 10 us)
#pragma unroll 1
      for (int u0 = warp; u0 < runs && p.ea.beta != 0.0f; u0 += 4 * kWarps) {
        OldBits<E> old[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int u = u0 + r * kWarps, i = j * 32 + lane;
            old[r][j] = u < runs && i < len ? reinterpret_cast<const OldBits<E>*>(base)[(row0 + u) * p.ldc + col0 + i] : OldBits<E>(0);
          }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int u = u0 + r * kWarps;
          if (u >= runs) break;
          E* out = base + (row0 + u) * p.ldc + col0 + lane;
          const float* src = own + u * run_step + lane * step;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j * 32 + lane < len) epi_store_nearest(p.ea, src[j * 32 * step], to_f32(old[r][j]), out + j * 32);
        }
      }
      for (int u = warp; u < runs && p.ea.beta == 0.0f; u += kWarps) {
        E* out = base + (row0 + u) * p.ldc + col0 + lane;
        const float* src = own + u * run_step + lane * step;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j * 32 + lane < len) epi_put(epi_scale(p.ea, src[j * 32 * step]), out + j * 32);
      }
    };
    if (p.out_f32) rows_of(static_cast<float*>(p.C));
    else rows_of(static_cast<__half*>(p.C));
  }
#undef NG_BY_PARTS
}

}  // namespace ngb
