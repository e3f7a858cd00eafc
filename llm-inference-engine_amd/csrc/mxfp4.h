// MXFP4 panels: the layout and device helpers that the quantisation and the
// products share.
//
// A matrix [rows, k] is held as blocks of 32 consecutive k of one row, each 32
// E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) and a scale byte
// e + 127, value = code * 2^e; scale 255 is NaN. Panels of 16 rows, k tiles of
// 128 and groups of 4 k tiles:
//   codes  [panels][tiles][64 lanes][16 bytes]   lane 16 g + r: row r, block g of the tile,
//                                                element 2i in the low half of byte i
//   scales [panels][groups][64 lanes][4 bytes]   byte j: the lane's block in the group's tile j
// with zero bytes past the rows and the blocks. This is the operand order of
// v_mfma_scale_f32_16x16x128_f8f6f4: a lane's 16 bytes are one block and its
// scale one byte of the lane's dword, so a k tile of a panel is one coalesced
// 1 KiB read, and no kernel masks a remainder.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_util.h"
#include "ehip.h"

namespace ehip {

constexpr int kMxRows = 16;     // rows of a panel
constexpr int kMxBlock = 32;    // elements of a block
constexpr int kMxTile = 128;    // k of a tile (4 blocks)
constexpr int kMxGroup = 4;     // tiles of a scale group
constexpr int kMxTileBytes = 1024;
constexpr int kMxScaleBytes = 256;  // of a panel's group

// The scale byte of a block whose largest magnitude has the bits `amax`:
// floor(log2 amax) - 2 as e + 127, at least 0; 255 with an infinity or NaN in it.
__device__ __forceinline__ uint32_t MxScaleByte(uint32_t amax) {
  const uint32_t f = amax >> 23;
  return f == 255u ? 255u : f < 2u ? 0u : f - 2u;
}

// Eight values as E2M1 codes of v / 2^(byte - 127), nearest even and at most 6
// in magnitude. The conversion takes the scale's exponent from a float's.
__device__ __forceinline__ uint32_t MxCodes(const float (&v)[8], uint32_t byte) {
  if (byte == 255u) return 0u;
  const float scale = __uint_as_float(byte << 23);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
  return r;
}

}  // namespace ehip
