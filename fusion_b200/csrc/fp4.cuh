// Microscaled 4-bit floating point: the scale layout shared by the quantiser and the
// grouped product, and the element conversions.
//
// Values are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), two in a byte, the even element
// in the low four bits. A run of consecutive elements along K shares one scale byte:
//   FUS_FP4_MX: 32 elements, e8m0 (2^(byte - 127); 255 = NaN)
//   FUS_FP4_NV: 16 elements, e4m3, times one fp32 factor of the tensor (or expert)
//
// Scale tiles. tcgen05.mma reads scales from tensor memory, where lane r % 32 and column
// r / 32 hold the four bytes ("cell") of row r, and tcgen05.cp brings them there 512 bytes
// (32 lanes x 4 columns x 4 bytes: 128 rows of one cell) at a time. So scales are stored in
// exactly those atoms: a tile of `tile` rows has ceil(tile / 128) atoms for each cell, and a
// pipeline stage of 256 K elements has kCells cells. Byte of (row r of the tile, stage s,
// scale j of the stage), A = ceil(tile / 128):
//   ((s * kCells + j / 4) * A + r / 128) * 512 + (r % 32) * 16 + (r % 128 / 32) * 4 + j % 4
// A stage's scales are contiguous: one bulk copy. Tiles below 128 rows keep whole atoms: a
// 16-row block spends 2 KB of scales beside 2 KB of values in L2, nothing beside the 18 KB
// weight tile it meets. Scales past K are zero (never NaN: the values there are zero and
// 0 x NaN would spoil the sum).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace fus {

constexpr int kFp4StageK = 256;  // K elements of a pipeline stage: 128 bytes of a row

__host__ __device__ constexpr int fp4_block(int fmt) { return fmt == FUS_FP4_MX ? 32 : 16; }
// scale cells (4 bytes of a row) of a stage
__host__ __device__ constexpr int fp4_cells(int fmt) {
  return kFp4StageK / fp4_block(fmt) / 4;
}
__host__ __device__ inline long fp4_stages(long K) { return (K + kFp4StageK - 1) / kFp4StageK; }
__host__ __device__ constexpr int fp4_atoms(int tile) { return tile > 128 ? tile / 128 : 1; }
// bytes of a tile's stage
__host__ __device__ constexpr int fp4_stage_scale_bytes(int fmt, int tile) {
  return fp4_cells(fmt) * fp4_atoms(tile) * 512;
}
// byte offset of scale j (of the whole row) of row r within its tile: a row's part and a
// scale's part
FUS_DEVICE int fp4_row_offset(int r) {
  return (r >> 7) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4;
}
FUS_DEVICE long fp4_scale_offset(int tile, int r, int j) {
  return (long)(j >> 2) * fp4_atoms(tile) * 512 + fp4_row_offset(r) + (j & 3);
}

// value of a scale byte, fp32 (exact)
template <int FMT>
FUS_DEVICE float fp4_scale_value(uint32_t byte) {
  if (FMT == FUS_FP4_MX) {
    if (byte == 255u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);  // byte 0: 2^-127, subnormal
  }
  const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

}  // namespace fus
