// mxfp4_linear.hip -- dense products with MXFP4 weights on gfx950 matrix instructions:
//   out = act(x W^T + bias) + residual           W [N, K]
//   out = act(x Wg^T + bg) * (x Wu^T + bu)       W [2N, K], gate rows first
// x [T, K] in f16 or bf16 (W is decoded to its type) or in MXFP4 (both operands go to the
// scaled matrix instructions as they are); sums in fp32, one rounding to the output's type.
//
// Weight rows are the matrix instruction's A operand and tokens its B operand: lane (r, q)
// ends with columns 4 q .. 4 q + 3 of a tile for token r.
#include "mxfp4_tile.h"

#include <stdlib.h>
#include <type_traits>

namespace exq {
namespace {

using namespace lin;
using namespace mx;

struct MxArgs : LinArgs {   // x: 16-bit rows, or packed ones (ldx in bytes)
  const uint8_t* xs;        // [T, K / 32] scale bytes of MXFP4 x
  const uint4* tiles;       // [RT, KB] tiles of 64 pieces
  const uint32_t* wscales;  // [RT, G] of 64 dwords
  int KB, G;                // tiles along the columns, groups of four of them
};

// One wave: 16 tokens x a tile of rows (gated: a gate and an up tile).
template <bool BF, bool X4, bool GATED>
__global__ void __launch_bounds__(256) mx_simple_kernel(MxArgs a, int nm, int nn) {
  constexpr int NT = GATED ? 2 : 1;
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t mb = unit / nn;
  const int nb = (int)(unit - mb * nn);
  if (mb >= nm) return;
  const int64_t m = mb * 16 + r16 < a.T ? mb * 16 + r16 : a.T - 1;
  const int K = (int)a.K, blocks = K / kBlock;
  f32x4_t acc[NT] = {};
  for (int kb = 0; kb < a.KB; ++kb) {
    uint4 w[NT];
    uint32_t s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t rt = (int64_t)nb * NT + t;
      w[t] = a.tiles[(rt * a.KB + kb) * 64 + lane];
      s[t] = a.wscales[(rt * a.G + (kb >> 2)) * 64 + lane] >> (8 * (kb & 3)) & 0xff;
    }
    const int b = kb * 4 + q;
    if constexpr (X4) {
      uint4 x = uint4{0u, 0u, 0u, 0u};
      int sx = 0;
      if (b < blocks) {
        x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.x) + m * a.ldx +
                                            b * 16);
        sx = a.xs[m * blocks + b];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = mfma_mx(w[t], (int)s[t], x, sx, acc[t]);
    } else {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = b < blocks ? *reinterpret_cast<const uint4*>(a.x + m * a.ldx + b * 32 + j * 8)
                          : uint4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t c[4] = {w[t].x, w[t].y, w[t].z, w[t].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[t] = dev::dmfma<BF>(decode8<BF>(c[j], __uint_as_float(s[t] << 23)), x[j], acc[t]);
      }
    }
  }
  const int64_t mo = mb * 16 + r16, n = (int64_t)nb * 16 + q * 4;
  float y[4], u[4], res[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    y[v] = acc[0][v];
    u[v] = acc[NT - 1][v];
  }
  if constexpr (!GATED) fetch_residual<4>(a, mo, n, res);
  finish_run<4, GATED>(a, mo, n, y, u, res);
}

// ---- many tokens: tiles -------------------------------------------------------------------
template <bool BF, bool X4, bool GATED, int WM, int WN, int MT, int NT, int P>
__global__ void __launch_bounds__(64 * WM * WN, MT == 8 ? 1 : X4 ? 2 : 3) mx_tile_kernel(MxArgs a, int nm, int nn) {
  using T = std::conditional_t<X4, Tile4<WM, WN, MT, NT>, Tile16<BF, WM, WN, MT, NT, P>>;
  constexpr int COLS = (GATED ? 8 : 16) * NT;      // output columns of a wave
  constexpr int SUMS = T::W * wave_floats<NT>() * 4;
  constexpr int LDS = T::LDS > SUMS ? T::LDS : SUMS;
  __shared__ __align__(1024) unsigned char lds[LDS];
  int mb, nb;
  if (!unit_of<8>(blockIdx.x, nm, nn, mb, nb)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int64_t m0 = (int64_t)mb * T::BM, n0 = (int64_t)nb * COLS * WN;
  const int rows = (int)(GATED ? (a.N + 15) / 16 * 2 : (a.N + 15) / 16);
  int vo[T::D], rt[NT];
#pragma unroll
  for (int j = 0; j < T::D; ++j) {
    const int r = T::row(wave, lane, j);
    vo[j] = m0 + r < a.T ? (int)(r * a.ldx * (X4 ? 1 : 2) + T::piece(wave, lane) * 16) : kOob;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {   // (tiles past the last repeat it: what they give is not stored)
    const int i = (nb * WN + wn) * NT + t;
    rt[t] = i < rows ? i : rows - 1;
  }
  const int blocks = (int)(a.K / kBlock);
  f32x4_t acc[MT][NT] = {};
  if constexpr (X4) {
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x);
    const uint8_t* xs[MT];
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const int64_t m = m0 + (wm * MT + u) * 16 + (lane & 15);
      xs[u] = a.xs + (m < a.T ? m : a.T - 1) * blocks;
    }
    T::run(lds, uniform_rsrc(x + m0 * a.ldx), vo, xs, a.tiles,
           a.wscales, rt, a.KB, a.G, blocks, wave, lane, acc);
  } else {
    T::run(lds, uniform_rsrc(a.x + m0 * a.ldx), vo, a.tiles, a.wscales, rt, a.KB, a.G, blocks * 4,
           wave, lane, acc);
  }
  const int64_t mw = m0 + wm * MT * 16, nw = n0 + wn * COLS;
  emit_tiles<GATED, MT, NT>(reinterpret_cast<float*>(lds) + wave * wave_floats<NT>(), acc, lane,
                            [&](int m, int c, float (&y)[8], float (&up)[8]) {
                              float r[8];
                              if constexpr (!GATED) fetch_residual<8>(a, mw + m, nw + c, r);
                              finish_run<8, GATED>(a, mw + m, nw + c, y, up, r);
                            });
}

template <bool BF, bool X4, bool GATED, int WM, int WN, int MT, int NT, int P>
int launch_tile(const MxArgs& a, hipStream_t s) {
  const int64_t nm = cdiv(a.T, 16 * MT * WM), nn = cdiv(a.N, (GATED ? 8 : 16) * NT * WN);
  const int64_t grid = cdiv(nm * nn, 8) * 8;
  EXQ_REQUIRE_SUPPORTED(grid * 64 * WM * WN < ((int64_t)1 << 32),
                        "exq_linear_mxfp4: T=%lld x N=%lld is too large", (long long)a.T,
                        (long long)a.N);
  hipLaunchKernelGGL((mx_tile_kernel<BF, X4, GATED, WM, WN, MT, NT, P>), dim3((unsigned)grid),
                     dim3(64 * WM * WN), 0, s, a, (int)nm, (int)nn);
  return check_launch("mx_tile_kernel");
}

template <bool BF, bool X4, bool GATED>
int launch_products(const MxArgs& a, hipStream_t s) {
  const char* v = getenv("MXV");
  if constexpr (X4) if (v && v[0] == '0') return launch_tile<BF, X4, GATED, 2, 2, 8, 8, 2>(a, s);
  if (v && v[0] == '1') return launch_tile<BF, X4, GATED, 1, 4, 8, 4, 2>(a, s);
  if (v && v[0] == '2') return launch_tile<BF, X4, GATED, 1, 4, 4, 4, 3>(a, s);
  if (v && v[0] == '3') return launch_tile<BF, X4, GATED, 1, 4, 4, 2, 3>(a, s);
  if (v && v[0] == '4') return launch_tile<BF, X4, GATED, 1, 4, 2, 2, 6>(a, s);
  if (v && v[0] == '5') return launch_tile<BF, X4, GATED, 1, 4, 2, 4, 5>(a, s);
  if (v && v[0] == '6') return launch_tile<BF, X4, GATED, 1, 4, 4, 4, 2>(a, s);
  const int64_t nm = cdiv(a.T, 16), nn = cdiv(a.N, 16), grid = cdiv(nm * nn, 4);
  EXQ_REQUIRE_SUPPORTED(grid * 256 < ((int64_t)1 << 32),
                        "exq_linear_mxfp4: T=%lld x N=%lld is too large", (long long)a.T,
                        (long long)a.N);
  hipLaunchKernelGGL((mx_simple_kernel<BF, X4, GATED>), dim3((unsigned)grid), dim3(256), 0, s, a,
                     (int)nm, (int)nn);
  return check_launch("mx_simple_kernel");
}

}  // namespace
}  // namespace exq

using namespace exq;

extern "C" int exq_linear_mxfp4(const exq_linear_problem* p, const void* x,
                                const uint8_t* x_scales, const uint8_t* tiles,
                                const uint8_t* tile_scales, const void* bias,
                                const void* residual, void* out, exq_stream stream) {
  const char* fn = "exq_linear_mxfp4";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  const bool x4 = p->act_dtype == EXQ_DTYPE_U8;
  EXQ_REQUIRE(x4 || is_act_dtype(p->act_dtype), "%s: x must be f16, bf16 or u8 (MXFP4)", fn);
  EXQ_REQUIRE(is_float_dtype(p->out_dtype), "%s: out dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(!bias || is_float_dtype(p->bias_dtype), "%s: bias dtype must be f32, f16 or bf16",
              fn);
  EXQ_REQUIRE(!residual || is_float_dtype(p->residual_dtype),
              "%s: residual dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(p->activation >= EXQ_ACT_NONE && p->activation <= EXQ_ACT_SIGMOID,
              "%s: unknown activation %d", fn, p->activation);
  EXQ_REQUIRE(!(p->gated && residual), "%s: a gated product takes no residual", fn);
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
  EXQ_REQUIRE(T >= 0 && T <= INT32_MAX / 2 && K >= mx::kBlock && K <= (1 << 24) &&
                  K % mx::kBlock == 0 && N >= 1 && N <= (1 << 20),
              "%s: sizes T=%lld K=%lld N=%lld out of range (K a multiple of 32)", fn,
              (long long)T, (long long)K, (long long)N);
  EXQ_REQUIRE(p->x_stride >= 0 && p->residual_stride >= 0 && (T <= 1 || p->out_stride >= N),
              "%s: row strides must not be negative, and out's at least N", fn);
  if (T == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(x && tiles && tile_scales && out && (!x4 || x_scales), "%s: null pointer", fn);
  EXQ_REQUIRE(((uintptr_t)x | (uintptr_t)tiles | (uintptr_t)tile_scales) % 16 == 0 &&
                  (T == 1 || p->x_stride * (x4 ? 1 : 2) % 16 == 0),
              "%s: x's rows, tiles and tile_scales must be 16-byte aligned", fn);
  MxArgs a{};
  a.x = reinterpret_cast<const uint16_t*>(x);
  a.bias = bias;
  a.res = residual;
  a.out = out;
  a.ldx = T == 1 ? 0 : p->x_stride;
  a.ldr = p->residual_stride;
  a.ldo = p->out_stride;
  a.T = T;
  a.N = N;
  a.K = K;
  a.bdt = p->bias_dtype;
  a.rdt = p->residual_dtype;
  a.odt = p->out_dtype;
  a.act = p->activation;
  const int64_t up = p->gated ? N : 0;  // (element offset of the second half of a gated bias)
  a.vec_b = (uintptr_t)bias % 16 == 0 && up % 4 == 0;
  a.vec_r = (uintptr_t)residual % 16 == 0 && p->residual_stride % 4 == 0;
  a.vec_o = (uintptr_t)out % 16 == 0 && p->out_stride % 4 == 0;
  a.xs = x_scales;
  a.tiles = reinterpret_cast<const uint4*>(tiles);
  a.wscales = reinterpret_cast<const uint32_t*>(tile_scales);
  a.KB = (int)mx::tile_cols(K);
  a.G = (a.KB + 3) / 4;
  const hipStream_t s = as_stream(stream);
  if (x4) return p->gated ? launch_products<true, true, true>(a, s)
                          : launch_products<true, true, false>(a, s);
  if (p->act_dtype == EXQ_DTYPE_BF16)
    return p->gated ? launch_products<true, false, true>(a, s)
                    : launch_products<true, false, false>(a, s);
  return p->gated ? launch_products<false, false, true>(a, s)
                  : launch_products<false, false, false>(a, s);
}
