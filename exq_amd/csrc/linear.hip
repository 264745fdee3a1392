// linear.hip -- dense products with an epilogue on gfx950 MFMA:
//   out = act(x W^T + bias) + residual           W [N, K]
//   out = act(x Wg^T + bg) * (x Wu^T + bu)       W [2N, K], gate rows first
// x [T, K] and W in f16 or bf16, sums in fp32, one rounding to the output's type.
//
// The weight rows are the MFMA's A operand and the tokens its B operand, so a lane
// ends with four consecutive output columns of one token.
#include "exq_internal.h"

namespace exq {
namespace {

struct LinArgs {
  const uint16_t* x;
  const uint16_t* w;
  const void* bias;   // [N] ([2N] gated) or null
  const void* res;    // [T, N] or null
  void* out;
  int64_t ldx, ldw, ldr, ldo;  // elements from row to row
  int64_t T, N, K;             // N: output columns
  int bdt, rdt, odt, act;
};

template <bool BF>
__device__ __forceinline__ f32x4_t mfma(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case EXQ_ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case EXQ_ACT_SILU: return silu_f32(v);
    case EXQ_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case EXQ_ACT_GELU_TANH:
      return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
    case EXQ_ACT_SIGMOID: return 1.f / (1.f + expf(-v));
    default: return v;
  }
}

// One output (token m, column n) of the product `y` (gated: `y` gate and `u` up).
template <bool GATED>
__device__ __forceinline__ float finish(const LinArgs& a, int64_t m, int64_t n, float y, float u) {
  if (a.bias) {
    y += load_as_f32(a.bias, a.bdt, n);
    if (GATED) u += load_as_f32(a.bias, a.bdt, a.N + n);
  }
  y = activate(y, a.act);
  if (GATED) return y * u;
  if (a.res) y += load_as_f32(a.res, a.rdt, m * a.ldr + n);
  return y;
}

// ---- any layout -------------------------------------------------------------
// Eight consecutive elements [k, k + 8) of a row as they lie, at any 2-byte
// alignment; zeros from K on.
struct __attribute__((packed, aligned(2))) Chunk {
  uint32_t d[4];
};
__device__ __forceinline__ uint4 load_chunk(const uint16_t* row, int64_t k, int64_t K) {
  if (k + 8 <= K) {
    const Chunk c = *reinterpret_cast<const Chunk*>(row + k);
    return uint4{c.d[0], c.d[1], c.d[2], c.d[3]};
  }
  uint32_t d[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) d[j >> 1] |= (uint32_t)row[k + j] << ((j & 1) * 16);
  return uint4{d[0], d[1], d[2], d[3]};
}

// 64 tokens x 64 weight rows (gated: 32 gate and the 32 matching up rows) by four
// waves, each 16 tokens x all weight rows; 32 k at a time through registers into
// LDS.  For rows that are not 16-byte aligned or K % 8 != 0.
constexpr int GB = 64, GK = 32, GLD = GK + 8;

template <bool BF, bool GATED>
__global__ void __launch_bounds__(256) linear_any_kernel(LinArgs a) {
  __shared__ __align__(16) uint16_t sx[GB * GLD];
  __shared__ __align__(16) uint16_t sw[GB * GLD];
  constexpr int BN = GATED ? GB / 2 : GB;  // output columns of the tile
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r16 = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * GB, n0 = (int64_t)blockIdx.y * BN;
  const int row = tid >> 2, ch = (tid & 3) * 8;
  const int64_t xr = m0 + row;
  const int64_t wn = n0 + (GATED ? row % BN : row);
  const bool xin = xr < a.T, win = wn < a.N;
  const uint16_t* xp = a.x + (xin ? xr : 0) * a.ldx;
  const uint16_t* wp = a.w + ((win ? wn : 0) + (GATED && row >= BN ? a.N : 0)) * a.ldw;
  const uint4 zero = uint4{0u, 0u, 0u, 0u};
  f32x4_t acc[4] = {};
  uint4 vx = xin ? load_chunk(xp, ch, a.K) : zero;
  uint4 vw = win ? load_chunk(wp, ch, a.K) : zero;
  for (int64_t k0 = 0; k0 < a.K; k0 += GK) {
    __syncthreads();
    *reinterpret_cast<uint4*>(sx + row * GLD + ch) = vx;
    *reinterpret_cast<uint4*>(sw + row * GLD + ch) = vw;
    __syncthreads();
    if (k0 + GK < a.K) {
      vx = xin ? load_chunk(xp, k0 + GK + ch, a.K) : zero;
      vw = win ? load_chunk(wp, k0 + GK + ch, a.K) : zero;
    }
    const uint4 b = *reinterpret_cast<const uint4*>(sx + (wave * 16 + r16) * GLD + q * 8);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      acc[t] = mfma<BF>(*reinterpret_cast<const uint4*>(sw + (t * 16 + r16) * GLD + q * 8), b,
                        acc[t]);
  }
  const int64_t m = m0 + wave * 16 + r16;
  if (m >= a.T) return;
#pragma unroll
  for (int t = 0; t < (GATED ? 2 : 4); ++t)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t n = n0 + t * 16 + q * 4 + v;
      if (n < a.N)
        store_from_f32(a.out, a.odt, m * a.ldo + n,
                       finish<GATED>(a, m, n, acc[t][v], GATED ? acc[(t + 2) & 3][v] : 0.f));
    }
}

template <bool BF, bool GATED>
int launch_linear(const LinArgs& a, hipStream_t s) {
  const int64_t bn = GATED ? GB / 2 : GB;
  const dim3 g((unsigned)cdiv(a.T, GB), (unsigned)cdiv(a.N, bn));
  hipLaunchKernelGGL((linear_any_kernel<BF, GATED>), g, dim3(256), 0, s, a);
  return check_launch("linear_any_kernel");
}

}  // namespace
}  // namespace exq

using namespace exq;

extern "C" int exq_linear(const exq_linear_problem* p, const void* x, const void* weight,
                          const void* bias, const void* residual, void* out, exq_stream stream) {
  const char* fn = "exq_linear";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  EXQ_REQUIRE(is_act_dtype(p->act_dtype), "%s: x and W must be f16 or bf16", fn);
  EXQ_REQUIRE(is_float_dtype(p->out_dtype), "%s: out dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(!bias || is_float_dtype(p->bias_dtype), "%s: bias dtype must be f32, f16 or bf16",
              fn);
  EXQ_REQUIRE(!residual || is_float_dtype(p->residual_dtype),
              "%s: residual dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(p->activation >= EXQ_ACT_NONE && p->activation <= EXQ_ACT_SIGMOID,
              "%s: unknown activation %d", fn, p->activation);
  EXQ_REQUIRE(!(p->gated && residual), "%s: a gated product takes no residual", fn);
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
  EXQ_REQUIRE(T >= 0 && T <= INT32_MAX / 2 && K >= 1 && K <= INT32_MAX / 2 && N >= 1 &&
                  N <= (1 << 20),
              "%s: sizes T=%lld K=%lld N=%lld out of range", fn, (long long)T, (long long)K,
              (long long)N);
  EXQ_REQUIRE(p->x_stride >= 0 && p->weight_stride >= 0 && p->residual_stride >= 0 &&
                  (T <= 1 || p->out_stride >= N),
              "%s: row strides must not be negative, and out's at least N", fn);
  if (T == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(x && weight && out, "%s: null pointer", fn);
  LinArgs a;
  a.x = reinterpret_cast<const uint16_t*>(x);
  a.w = reinterpret_cast<const uint16_t*>(weight);
  a.bias = bias;
  a.res = residual;
  a.out = out;
  a.ldx = p->x_stride;
  a.ldw = p->weight_stride;
  a.ldr = p->residual_stride;
  a.ldo = p->out_stride;
  a.T = T;
  a.N = N;
  a.K = K;
  a.bdt = p->bias_dtype;
  a.rdt = p->residual_dtype;
  a.odt = p->out_dtype;
  a.act = p->activation;
  const hipStream_t s = as_stream(stream);
  if (p->act_dtype == EXQ_DTYPE_BF16)
    return p->gated ? launch_linear<true, true>(a, s) : launch_linear<true, false>(a, s);
  return p->gated ? launch_linear<false, true>(a, s) : launch_linear<false, false>(a, s);
}
