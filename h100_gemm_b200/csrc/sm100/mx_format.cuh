// Microscaled 4-bit floating point: the two formats, their scale layout and the conversions.
//
// A matrix [R, C] is stored as e2m1 codes (1 sign, 2 exponent, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6)
// with one 8-bit scale per block of consecutive elements of a row:
//   MXFP4  blocks of 32, scale 2^(byte - 127)  (byte 255: NaN)
//   NVFP4  blocks of 16, scale an e4m3 number  (byte 127: NaN), times one power of two per matrix
// Codes: two to a byte, element 2i in the lower half; a row takes ceil(C / 2) bytes rounded up to 16
// (the pitch a TMA tensor map needs), the rest of it zero.
// Scales: the order the tensor cores take them in. 128 rows x 4 consecutive blocks form a group of
// 512 bytes, byte (r % 32) * 16 + (r / 32) * 4 + block % 4, which one tcgen05.cp moves to tensor
// memory as it is. The groups of one 128-row x 256-column tile lie together (two for MXFP4, four for
// NVFP4), tiles along a row follow each other, then the next 128 rows. Rows and columns are padded
// to whole tiles; the padding's scales are zero bytes.
#pragma once

#include <stdint.h>

#include "desc.cuh"

namespace b200 {

enum MxFormat : int { kMxfp4 = 0, kNvfp4 = 1 };

static constexpr int kMxTileRows = 128;  // rows of one scale tile
static constexpr int kMxTileCols = 256;  // elements of one scale tile: one 128-byte swizzle row of codes
static constexpr int kMxGroupBytes = 512;

B200_HD constexpr int mx_block(int fmt) { return fmt == kMxfp4 ? 32 : 16; }
B200_HD constexpr int mx_tile_groups(int fmt) { return kMxTileCols / (4 * mx_block(fmt)); }
B200_HD constexpr int mx_tile_bytes(int fmt) { return mx_tile_groups(fmt) * kMxGroupBytes; }
B200_HD constexpr long long mx_pitch(long long cols) { return ((cols + 1) / 2 + 15) / 16 * 16; }
B200_HD constexpr long long mx_row_tiles(long long rows) { return (rows + kMxTileRows - 1) / kMxTileRows; }
B200_HD constexpr long long mx_col_tiles(long long cols) { return (cols + kMxTileCols - 1) / kMxTileCols; }
B200_HD constexpr long long mx_scale_bytes(int fmt, long long rows, long long cols) {
  return mx_row_tiles(rows) * mx_col_tiles(cols) * mx_tile_bytes(fmt);
}
// Byte of the scale of block `block` of row `row`.
B200_HD constexpr long long mx_scale_offset(int fmt, long long row, long long block, long long col_tiles) {
  return ((row / kMxTileRows) * col_tiles * mx_tile_groups(fmt) + block / 4) * kMxGroupBytes + (row % 32) * 16 +
         (row % kMxTileRows) / 32 * 4 + block % 4;
}

#if defined(__CUDACC__)

// Eight fp32 values -> eight e2m1 codes in one word, element 0 in the lowest four bits; round to
// nearest, ties to the even code, beyond 6 saturating.
__device__ __forceinline__ uint32_t e2m1_pack8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// One code -> its value in fp32. The three magnitude bits are the top of an fp32 number with a bias
// of 1: placed at bits 22..24 and multiplied by 2^126 they read 0, 0.5, 1, ... 6 (0.5 comes out of
// the subnormal 2^-127).
__device__ __forceinline__ float e2m1_value(uint32_t code) {
  const uint32_t bits = ((code & 7u) << 22) | ((code & 8u) << 28);
  return __uint_as_float(bits) * 8.507059173023462e37f;  // 2^126
}

__device__ __forceinline__ float ue8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7FC00000u : byte << 23);
}

// e4m3 byte -> fp32: sign, 4 exponent bits (bias 7), 3 mantissa bits; no infinities, 0x7F is NaN.
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  if ((byte & 0x7Fu) == 0x7Fu) return __uint_as_float(0x7FC00000u);
  const float m = __uint_as_float((byte & 0x7Fu) << 20) * 1.329227995784916e36f;  // 2^120
  return (byte & 0x80u) ? -m : m;
}

// fp32 (not negative) -> nearest e4m3 byte, ties to even, beyond 448 saturating.
__device__ __forceinline__ uint32_t e4m3_byte(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xFFu;
}

template <int FMT>
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return FMT == kMxfp4 ? ue8m0_value(byte) : e4m3_value(byte);
}

#endif

}  // namespace b200
