// linear_epilogue.h -- what the dense products (linear.hip, mxfp4_linear.hip) share: their
// arguments, the activations, the epilogue of a run of consecutive output columns
// (bias, activation, gate, residual, one rounding) and the order of the tiles.
#pragma once

#include "exq_internal.h"

namespace exq {
namespace lin {

struct LinArgs {
  const uint16_t* x;
  const uint16_t* w;
  const void* bias;   // [N] ([2N] gated) or null
  const void* res;    // [T, N] or null
  void* out;
  int64_t ldx, ldw, ldr, ldo;  // elements from row to row
  int64_t T, N, K;             // N: output columns
  int bdt, rdt, odt, act;
  int vec_b, vec_r, vec_o;     // four consecutive elements may be accessed at once
  int odd;                     // rows of x or W may start at an odd 2-byte address
};

// silu(v) = v / (1 + e^-v); sigmoid(v) = 1 / (1 + e^-v); gelu_tanh(v) = v / (1 + e^-z)
// with z = 2 sqrt(2 / pi) (v + 0.044715 v^3), as (1 + tanh(z / 2)) / 2 = 1 / (1 + e^-z):
// one exponential and one division serve all three.
__device__ __forceinline__ float logistic_act(float v, int act) {
  const float z = act == EXQ_ACT_GELU_TANH
                      ? 1.5957691216057308f * (v + 0.044715f * v * v * v) : v;
  return (act == EXQ_ACT_SIGMOID ? 1.f : v) / (1.f + expf(-z));
}
__device__ __forceinline__ float erf_gelu(float v) {
  return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
}
template <int CNT>
__device__ __forceinline__ void activate_run(float (&v)[CNT], int act) {
  if (act == EXQ_ACT_NONE) return;
  if (act == EXQ_ACT_RELU) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = v[c] < 0.f ? 0.f : v[c];  // (NaN stays)
  } else if (act == EXQ_ACT_GELU) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = erf_gelu(v[c]);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = logistic_act(v[c], act);
  }
}

// CNT (a multiple of 4) consecutive values at element i.
template <int CNT>
__device__ __forceinline__ void load_run(const void* p, int dt, int64_t i, float (&v)[CNT]) {
#pragma unroll
  for (int c = 0; c < CNT; c += 4) {
    if (dt == EXQ_DTYPE_F32) {
      const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i + c);
      v[c] = f.x; v[c + 1] = f.y; v[c + 2] = f.z; v[c + 3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i + c);
      const bool bf = dt == EXQ_DTYPE_BF16;
      v[c] = bf ? __uint_as_float(u.x << 16) : f16_bits_to_f32(u.x & 0xffffu);
      v[c + 1] = bf ? __uint_as_float(u.x & 0xffff0000u) : f16_bits_to_f32(u.x >> 16);
      v[c + 2] = bf ? __uint_as_float(u.y << 16) : f16_bits_to_f32(u.y & 0xffffu);
      v[c + 3] = bf ? __uint_as_float(u.y & 0xffff0000u) : f16_bits_to_f32(u.y >> 16);
    }
  }
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf) {
  if (bf) {
    bf16x2_t h;
    h[0] = (__bf16)lo;
    h[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, h);
  }
  f16x2_t h;
  h[0] = (_Float16)lo;
  h[1] = (_Float16)hi;
  return __builtin_bit_cast(uint32_t, h);
}
template <int CNT>
__device__ __forceinline__ void store_run(void* p, int dt, int64_t i, const float (&v)[CNT]) {
  if (dt == EXQ_DTYPE_F32) {
#pragma unroll
    for (int c = 0; c < CNT; c += 4)
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i + c) =
          float4{v[c], v[c + 1], v[c + 2], v[c + 3]};
  } else {
    uint16_t* o = reinterpret_cast<uint16_t*>(p) + i;
    const bool bf = dt == EXQ_DTYPE_BF16;
    uint32_t d[CNT / 2];
#pragma unroll
    for (int c = 0; c < CNT; c += 2) d[c / 2] = pack16(v[c], v[c + 1], bf);
#pragma unroll
    for (int c = 0; c < CNT / 2; c += 2)
      *reinterpret_cast<uint2*>(o + 2 * c) = uint2{d[c], d[c + 1]};
  }
}
// The epilogue of CNT consecutive columns n.. of token m, in two parts, so that the
// residual of several runs can be on its way before the first is used.
template <int CNT>
__device__ __forceinline__ void fetch_residual(const LinArgs& a, int64_t m, int64_t n,
                                               float (&r)[CNT]) {
  if (!a.res || m >= a.T || n >= a.N) return;
  if (n + CNT <= a.N && a.vec_r) {
    load_run<CNT>(a.res, a.rdt, m * a.ldr + n, r);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      r[c] = n + c < a.N ? load_as_f32(a.res, a.rdt, m * a.ldr + n + c) : 0.f;
  }
}
template <int CNT>
__device__ __forceinline__ void add_bias(const LinArgs& a, int64_t n, int64_t off, bool whole,
                                         float (&y)[CNT]) {
  float b[CNT];
  if (whole && a.vec_b) {
    load_run<CNT>(a.bias, a.bdt, off + n, b);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      b[c] = n + c < a.N ? load_as_f32(a.bias, a.bdt, off + n + c) : 0.f;
  }
#pragma unroll
  for (int c = 0; c < CNT; ++c) y[c] += b[c];
}
template <int CNT, bool GATED>
__device__ __forceinline__ void finish_run(const LinArgs& a, int64_t m, int64_t n, float (&y)[CNT],
                                           float (&u)[CNT], const float (&r)[CNT]) {
  if (m >= a.T || n >= a.N) return;
  const bool whole = n + CNT <= a.N;
  if (a.bias) {
    add_bias<CNT>(a, n, 0, whole, y);
    if constexpr (GATED) add_bias<CNT>(a, n, a.N, whole, u);
  }
  activate_run<CNT>(y, a.act);
  if constexpr (GATED) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) y[c] *= u[c];
  } else if (a.res) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) y[c] += r[c];
  }
  if (whole && a.vec_o) {
    store_run<CNT>(a.out, a.odt, m * a.ldo + n, y);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      if (n + c < a.N) store_from_f32(a.out, a.odt, m * a.ldo + n + c, y[c]);
  }
}

// Unit (token block mt of nm, column block nt of nn) of work-group bid: work-group i
// runs on XCD i % 8, and each XCD takes an eighth of the units in a row, the token
// blocks fastest in groups of GM, so that what runs together shares rows of both
// operands in that XCD's L2.  False: none.
template <int GM>
__device__ __forceinline__ bool unit_of(int bid, int nm, int nn, int& mt, int& nt) {
  const int U = nm * nn;
  const int per = (U + 7) >> 3;
  const int local = bid >> 3;
  const int v = (bid & 7) * per + local;
  if (local >= per || v >= U) return false;
  const int g = v / (GM * nn), first = g * GM;
  const int size = nm - first < GM ? nm - first : GM;
  const int rem = v - g * GM * nn;
  nt = rem / size;
  mt = first + rem - nt * size;
  return true;
}

}  // namespace lin
}  // namespace exq
