// mxfp4.h -- MXFP4 on gfx950: device helpers shared by mxfp4_quant.hip,
// mxfp4_linear.hip and mxfp4_moe.hip.  Not part of the C ABI.
//
// A block is 32 values along a row: codes of four bits (sign, and 0, .5, 1, 1.5, 2, 3,
// 4, 6), the even column in a byte's low half, and a scale byte s for 2^(s - 127), 255
// for NaN.  The conversion instructions take the scale as a float of which they use the
// exponent field alone, so s << 23 is it for every s (0 is 2^-127 and 255 NaN).
//
// The products read a weight as tiles of 16 rows x 128 columns, 1 KiB: byte 16 (16 q + r)
// + b is byte b of block q of row r, which is what lane (r, q) of a matrix instruction
// takes.  A wave loads a tile with one 16-byte load a lane, whole lines in order, straight
// into registers: no LDS, no tails (rows are padded to 16, columns to 128, with zeros).
// The scale bytes of four tiles along the columns lie together, one dword a lane.
#pragma once

#include "dev_util.h"

namespace exq {
namespace mx {

constexpr int kBlock = 32;          // values of a block
constexpr int kTileK = 128;         // columns of a tile

inline int64_t tile_cols(int64_t K) { return cdiv(K, kTileK); }
// Tiles of rows of a weight; a gated one (gate rows, then up rows) pads each half and
// has its gate and up tiles in turn.
inline int64_t tile_rows(int64_t rows, int gated) {
  return gated ? 2 * cdiv(rows / 2, 16) : cdiv(rows, 16);
}

// Eight codes times the scale, in 16 bits: exact in bf16 but past its largest value, in
// f16 rounded to nearest (exact for scales from 2^-23 to 2^13).
template <bool BF>
__device__ __forceinline__ uint4 decode8(uint32_t codes, float scale) {
  uint4 o;
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (BF) {
    o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  } else {
    o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
    o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
    o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
    o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
  }
#endif
  return o;
}

// 16 rows x 16 tokens x 128 columns, both operands MXFP4: a lane's 16 bytes are block q
// of its row, its scale byte that block's.
__device__ __forceinline__ f32x4_t mfma_mx(const uint4& a, int sa, const uint4& b, int sb,
                                           f32x4_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef int i32x8_t __attribute__((ext_vector_type(8)));
  const i32x8_t A = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8_t B = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, c, 4, 4, 0, sa, 0, sb);
#else
  return c;
#endif
}

}  // namespace mx
}  // namespace exq
