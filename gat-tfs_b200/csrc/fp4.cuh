// 4-bit microscaled tables (E2M1 elements, one scale per block of a row).
//
// Codes: two per byte, the even column in the low half; rows of ldc bytes,
// the first ceil(width / 32) * 16 of them written (columns past the width
// hold zeros). Scales: one byte per block, in tiles of 128 rows x 4 blocks of
// 512 bytes, the tiles of 128 rows in a row, byte (r % 32) * 16 +
// (r / 32 % 4) * 4 + b % 4 of a tile: the order in which tcgen05.cp takes 32
// lanes x 16 bytes to tensor memory, where lane l of column j then holds row
// 32 j + l's four scales.
#pragma once
#include "device.cuh"

namespace gatb {

__host__ __device__ constexpr int fp4_block(int format) { return format == GAT_B200_MXFP4 ? 32 : 16; }
// Bytes of a code row as the library writes it.
__host__ __device__ constexpr int fp4_row_bytes(int width) { return (width + 31) / 32 * 16; }
// Scale tiles of 4 blocks along a row.
__host__ __device__ constexpr int fp4_tiles(int format, int width) {
    return (width + 4 * fp4_block(format) - 1) / (4 * fp4_block(format));
}

}  // namespace gatb
