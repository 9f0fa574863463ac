// Host-side view of matrices in blocks, shared by the element-wise kernels and the products on them.
#pragma once
#include "block_out.cuh"
#include "blocks.cuh"
#include "host.h"

namespace ngb {

// Checks what a descriptor says, without a device.
int check_shape(const ng_block_desc* d);
// Rows of a tile of codes in a 4-bit matrix of so many outer rows (128 from 65 on).
int block_tile_rows(int outer);
// Checks a descriptor against the current device and fills in what the kernels need.
int block_view(const DeviceCtx* c, const ng_block_desc* d, BlockView& v);
// The values of a checked matrix as rows of `ld` fp16 numbers along its blocked axis.
int dequantize_f16(DeviceCtx* c, const ng_block_desc& d, const BlockView& q, __half* out, long long ld, cudaStream_t stream);

// Boxes of [box_rows][box_cols] of a row-major matrix, zeros beyond it.
int plain_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_cols, int box_rows, int esz);
// Output stage of a product: its parameters, the boxes it stores, and whether its lean form will do.
OutParams make_out(void* C, int m, int n, int ldc, int out_f32, const EpiArgs& ea);
int out_map(CUtensorMap* map, const OutParams& out);
// CTAs of a kernel that run at the same time in clusters of 2^log: larger clusters leave SMs of their GPCs over (132 of 148 in
// clusters of 4, 120 in clusters of 8; 2048 x 128 x 2048 as 128 CTAs in clusters of 8 took two rounds, 12.0 us).
int cluster_room(const DeviceCtx* c, const void* kernel, int threads, uint32_t smem, int log);
// The product of block_dot_pair.cu: two 4-bit matrices of more than 64 outer rows each.
int run_block_dot_pair(DeviceCtx* c, const BlockView& a, const BlockView& b, bool nv, const OutParams& out, cudaStream_t stream);
// The product of block_dot_f16.cu, from checked operands.
int run_block_dot_f16(DeviceCtx* c, const void* A, int lda, const ng_block_desc& d, const BlockView& x, void* C, int m, int ldc,
                      int out_f32, const EpiArgs& ea, cudaStream_t stream);

}  // namespace ngb
