// mxfp4_quant.hip -- rows to MXFP4 and back, and the order in which the products read a
// weight.  All three move bytes and are bound by HBM: 28672 x 4096 bf16 to MXFP4 63 us (4.7
// TB/s; a large copy 5.2), back 53 us (5.6, part of the codes still in the Infinity Cache);
// eight weights of 4096 x 14336 into tiles 110 us (4.6 TB/s).
#include "mxfp4.h"

namespace exq {
namespace {

using namespace mx;

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// ---- quantisation ----------------------------------------------------------------------
// A lane holds eight consecutive values (one 16-byte load, two of float32), four lanes a
// block: its largest magnitude a by two lane swaps inside the four.  The scale byte is the
// exponent field of a less 2, so that a / scale lies in [4, 8): past 6 the conversion
// saturates; a field below 2 (a < 2^-125, zero) takes the smallest scale, and a block with
// an infinity or a NaN, which no code can hold, the NaN scale, with codes of zero.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);
  v = a > v ? a : v;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);
  return b > v ? b : v;
}

template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t i, bool vec, float (&v)[8]) {
  if constexpr (DT == EXQ_DTYPE_F32) {
    const float* p = reinterpret_cast<const float*>(x) + i;
    if (vec) {
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = p[c];
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + i;
    uint32_t d[4];
    if (vec) {
      *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) d[c] = (uint32_t)p[2 * c] | (uint32_t)p[2 * c + 1] << 16;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[2 * c] = DT == EXQ_DTYPE_BF16 ? __uint_as_float(d[c] << 16) : f16_bits_to_f32(d[c] & 0xffffu);
      v[2 * c + 1] = DT == EXQ_DTYPE_BF16 ? __uint_as_float(d[c] & 0xffff0000u)
                                          : f16_bits_to_f32(d[c] >> 16);
    }
  }
}

// The codes of a lane's eight values and its block's scale byte.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8], uint32_t& s) {
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t m = __float_as_uint(v[c]) & 0x7fffffffu;
    top = m > top ? m : top;
  }
  top = quad_max(top);
  const uint32_t e = top >> 23;
  s = e == 255 ? 255u : e < 2 ? 0u : e - 2;
  uint32_t codes = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  const float scale = __uint_as_float(s << 23);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], scale, 3);
#endif
  return e == 255 ? 0u : codes;
}

constexpr int QNT = 256;

// Chunks of eight values, U in flight a lane; a block's four chunks are four lanes.
template <int DT, int U>
__global__ void __launch_bounds__(QNT) quantize_kernel(const void* __restrict__ x, int64_t chunks,
                                                       int64_t row_chunks, int64_t ld, int vec,
                                                       uint32_t* __restrict__ packed,
                                                       uint8_t* __restrict__ scales) {
  const int64_t first = (int64_t)blockIdx.x * (QNT * U) + threadIdx.x;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * QNT;
#pragma unroll
    for (int c = 0; c < 8; ++c) v[u][c] = 0.f;
    if (i < chunks) {
      // (rows that follow each other need no division)
      const int64_t row = ld == row_chunks * 8 ? 0 : i / row_chunks;
      load8<DT>(x, row * ld + (i - row * row_chunks) * 8, vec, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * QNT;
    uint32_t s;
    const uint32_t codes = encode8(v[u], s);
    if (i < chunks) {
      packed[i] = codes;
      if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
    }
  }
}

// ---- and back ------------------------------------------------------------------------------
template <int DT, int U>
__global__ void __launch_bounds__(QNT) dequantize_kernel(const uint32_t* __restrict__ packed,
                                                         const uint8_t* __restrict__ scales,
                                                         int64_t chunks, void* __restrict__ out) {
  const int64_t first = (int64_t)blockIdx.x * (QNT * U) + threadIdx.x;
  uint32_t p[U], s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * QNT;
    p[u] = i < chunks ? packed[i] : 0u;
    s[u] = i < chunks ? scales[i >> 2] : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * QNT;
    if (i >= chunks) continue;
    const float scale = __uint_as_float(s[u] << 23);
    if constexpr (DT == EXQ_DTYPE_F32) {
#if defined(__HIP_DEVICE_COMPILE__)
      float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + i * 8);
      const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p[u], scale, 0);
      const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p[u], scale, 1);
      const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p[u], scale, 2);
      const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p[u], scale, 3);
      o[0] = float4{a[0], a[1], b[0], b[1]};
      o[1] = float4{c[0], c[1], d[0], d[1]};
#endif
    } else {
      reinterpret_cast<uint4*>(out)[i] = decode8<DT == EXQ_DTYPE_BF16>(p[u], scale);
    }
  }
}

// ---- tiles -----------------------------------------------------------------------------------
// One lane a 16-byte piece (block q of row r of tile (rt, kb)), then one a dword of scales.
__global__ void __launch_bounds__(QNT) tile_kernel(const uint4* __restrict__ packed,
                                                   const uint8_t* __restrict__ scales,
                                                   int64_t mats, int64_t rows, int blocks,
                                                   int gated, int RT, int KB,
                                                   uint4* __restrict__ tiles,
                                                   uint32_t* __restrict__ tile_scales) {
  const int64_t i = (int64_t)blockIdx.x * QNT + threadIdx.x;
  const int lane = (int)(i & 63), r = lane & 15, q = lane >> 4;
  const int64_t pieces = mats * RT * KB * 64;
  const int G = (KB + 3) >> 2;
  const bool weights = i < pieces;
  const int64_t j = weights ? i >> 6 : (i - pieces) >> 6;
  const int per = weights ? KB : G;
  const int64_t m = j / ((int64_t)RT * per);
  if (m >= mats) return;
  const int64_t rem = j - m * RT * per;
  const int rt = (int)(rem / per), c = (int)(rem - (int64_t)rt * per);
  const int64_t half = rows >> 1;
  const int64_t in = gated ? (int64_t)(rt >> 1) * 16 + r : (int64_t)rt * 16 + r;
  const bool there = in < (gated ? half : rows);
  const int64_t row = m * rows + in + (gated && (rt & 1) ? half : 0);
  if (weights) {
    const int b = c * 4 + q;
    tiles[i] = there && b < blocks ? packed[row * blocks + b] : uint4{0u, 0u, 0u, 0u};
  } else {
    uint32_t s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = (c * 4 + k) * 4 + q;
      if (there && b < blocks) s |= (uint32_t)scales[row * blocks + b] << (8 * k);
    }
    tile_scales[i - pieces] = s;
  }
}

// Work-groups for n lanes' worth of work; 0: more than a launch takes.
int64_t groups_of(int64_t n, int64_t per) {
  const int64_t g = cdiv(n, per);
  return g * QNT < ((int64_t)1 << 32) ? g : 0;
}

int check_rows(const char* fn, int64_t rows, int64_t K) {
  EXQ_REQUIRE(rows >= 0 && K >= kBlock && K <= INT32_MAX / 2 && K % kBlock == 0,
              "%s: rows=%lld K=%lld: K must be a positive multiple of 32", fn, (long long)rows,
              (long long)K);
  EXQ_REQUIRE_SUPPORTED(rows <= ((int64_t)1 << 40) / K, "%s: %lld x %lld values are too many", fn,
                        (long long)rows, (long long)K);
  return EXQ_SUCCESS;
}

}  // namespace
}  // namespace exq

using namespace exq;

extern "C" int exq_quantize_mxfp4(const void* x, int dtype, int64_t rows, int64_t K,
                                  int64_t x_stride, uint8_t* packed, uint8_t* scales,
                                  exq_stream stream) {
  const char* fn = "exq_quantize_mxfp4";
  EXQ_REQUIRE(is_float_dtype(dtype), "%s: x must be f32, f16 or bf16", fn);
  const int st = check_rows(fn, rows, K);
  if (st) return st;
  EXQ_REQUIRE(x_stride >= 0, "%s: the row stride must not be negative", fn);
  if (rows == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(x && packed && scales, "%s: null pointer", fn);
  EXQ_REQUIRE((uintptr_t)packed % 16 == 0, "%s: packed must be 16-byte aligned", fn);
  const int64_t ld = rows == 1 ? K : x_stride, chunks = rows * (K / 8);
  const int vec = (uintptr_t)x % 16 == 0 && ld * dtype_bytes(dtype) % 16 == 0;
  const hipStream_t s = as_stream(stream);
  int64_t grid = 0;
  with_dtype(dtype, [&](auto dt) {
    constexpr int U = 2;
    grid = groups_of(chunks, QNT * U);
    if (grid)
      hipLaunchKernelGGL((quantize_kernel<decltype(dt)::value, U>), dim3((unsigned)grid),
                         dim3(QNT), 0, s, x, chunks, K / 8, ld, vec,
                         reinterpret_cast<uint32_t*>(packed), scales);
  });
  EXQ_REQUIRE_SUPPORTED(grid, "%s: %lld x %lld values are too many", fn, (long long)rows,
                        (long long)K);
  return check_launch("quantize_kernel");
}

extern "C" int exq_dequantize_mxfp4(const uint8_t* packed, const uint8_t* scales, int64_t rows,
                                    int64_t K, void* out, int dtype, exq_stream stream) {
  const char* fn = "exq_dequantize_mxfp4";
  EXQ_REQUIRE(is_float_dtype(dtype), "%s: out must be f32, f16 or bf16", fn);
  const int st = check_rows(fn, rows, K);
  if (st) return st;
  if (rows == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(packed && scales && out, "%s: null pointer", fn);
  EXQ_REQUIRE((uintptr_t)packed % 4 == 0 && (uintptr_t)out % 16 == 0,
              "%s: packed must be 4-byte and out 16-byte aligned", fn);
  const int64_t chunks = rows * (K / 8);
  const hipStream_t s = as_stream(stream);
  int64_t grid = 0;
  with_dtype(dtype, [&](auto dt) {
    constexpr int U = 4;
    grid = groups_of(chunks, QNT * U);
    if (grid)
      hipLaunchKernelGGL((dequantize_kernel<decltype(dt)::value, U>), dim3((unsigned)grid),
                         dim3(QNT), 0, s, reinterpret_cast<const uint32_t*>(packed), scales,
                         chunks, out);
  });
  EXQ_REQUIRE_SUPPORTED(grid, "%s: %lld x %lld values are too many", fn, (long long)rows,
                        (long long)K);
  return check_launch("dequantize_kernel");
}

extern "C" int exq_tile_mxfp4(const uint8_t* packed, const uint8_t* scales, int64_t n_matrices,
                              int64_t rows, int64_t K, int gated, uint8_t* tiles,
                              uint8_t* tile_scales, exq_stream stream) {
  const char* fn = "exq_tile_mxfp4";
  EXQ_REQUIRE(n_matrices >= 0 && rows >= 1 && rows <= (1 << 21),
              "%s: n_matrices=%lld rows=%lld out of range", fn, (long long)n_matrices,
              (long long)rows);
  EXQ_REQUIRE(!gated || rows % 2 == 0, "%s: a gated weight has an even number of rows", fn);
  EXQ_REQUIRE_SUPPORTED(n_matrices <= (1 << 20), "%s: too many matrices", fn);
  const int st = check_rows(fn, n_matrices * rows, K);
  if (st) return st;
  if (n_matrices == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(packed && scales && tiles && tile_scales, "%s: null pointer", fn);
  EXQ_REQUIRE(((uintptr_t)packed | (uintptr_t)tiles | (uintptr_t)tile_scales) % 16 == 0,
              "%s: packed, tiles and tile_scales must be 16-byte aligned", fn);
  const int64_t RT = tile_rows(rows, gated), KB = tile_cols(K);
  const int64_t lanes = n_matrices * RT * (KB + cdiv(KB, 4)) * 64;
  const int64_t grid = groups_of(lanes, QNT);
  EXQ_REQUIRE_SUPPORTED(grid, "%s: %lld x %lld x %lld values are too many", fn,
                        (long long)n_matrices, (long long)rows, (long long)K);
  hipLaunchKernelGGL(tile_kernel, dim3((unsigned)grid), dim3(QNT), 0, as_stream(stream),
                     reinterpret_cast<const uint4*>(packed), scales, n_matrices, rows,
                     (int)(K / kBlock), gated ? 1 : 0, (int)RT, (int)KB,
                     reinterpret_cast<uint4*>(tiles), reinterpret_cast<uint32_t*>(tile_scales));
  return check_launch("tile_kernel");
}
