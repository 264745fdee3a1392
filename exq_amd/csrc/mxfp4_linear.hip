// mxfp4_linear.hip -- dense products with MXFP4 weights on gfx950 matrix instructions:
//   out = act(x W^T + bias) + residual           W [N, K]
//   out = act(x Wg^T + bg) * (x Wu^T + bu)       W [2N, K], gate rows first
// x [T, K] in f16 or bf16 (W is decoded to its type) or in MXFP4 (both operands go to the
// scaled matrix instructions as they are); sums in fp32, one rounding to the output's type.
//
// Weight rows are the matrix instruction's A operand and tokens its B operand: lane (r, q)
// ends with columns 4 q .. 4 q + 3 of a tile for token r.
#include "mxfp4_tile.h"

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

// ---- few tokens: a stream of weights --------------------------------------------------------
// 16 MT tokens x a tile of weight rows (gated: a gate tile and its up tile) by W waves that
// split the contraction; both operands straight from memory, and the sums joined through
// LDS in wave order.
template <bool BF, bool X4, bool GATED, int MT, int W>
__global__ void __launch_bounds__(64 * W) mx_stream_kernel(MxArgs a, int nn) {
  constexpr int NT = GATED ? 2 : 1, C = X4 || MT == 1 ? 4 : 2;   // tiles along K in flight
  __shared__ __align__(16) float4 red[W * MT * NT * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int mb = blockIdx.x / nn, nb = blockIdx.x - mb * nn;
  const int64_t m0 = (int64_t)mb * MT * 16;
  const int blocks = (int)(a.K / kBlock);
  const uint8_t* w8 = reinterpret_cast<const uint8_t*>(a.wscales);
  const uint8_t *x[MT], *xs[MT];   // (rows past the last repeat it: what they give is not stored)
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    const int64_t m = m0 + u * 16 + r16 < a.T ? m0 + u * 16 + r16 : a.T - 1;
    x[u] = reinterpret_cast<const uint8_t*>(a.x) + m * a.ldx * (X4 ? 1 : 2);
    xs[u] = X4 ? a.xs + m * blocks : nullptr;
  }
  const int kb0 = wave * a.KB / W, kb1 = (wave + 1) * a.KB / W;
  f32x4_t acc[MT][NT] = {};
  for (int k0 = kb0; k0 < kb1; k0 += C) {
    uint4 w[C][NT], v[C][MT][X4 ? 1 : 4];
    uint32_t s[C][NT], sx[C][MT];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int kb = k0 + c < kb1 ? k0 + c : kb1 - 1;   // (past the range: loaded again, not used)
      const int b = kb * 4 + q < blocks ? kb * 4 + q : blocks - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t rt = (int64_t)nb * NT + t;
        w[c][t] = a.tiles[(rt * a.KB + kb) * 64 + lane];
        s[c][t] = w8[((rt * a.G + (kb >> 2)) * 64 + lane) * 4 + (kb & 3)];
      }
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        if constexpr (X4) {
          v[c][u][0] = *reinterpret_cast<const uint4*>(x[u] + b * 16);
          sx[c][u] = xs[u][b];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[c][u][j] = *reinterpret_cast<const uint4*>(x[u] + b * 64 + j * 16);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (k0 + c >= kb1) break;
      const bool in = (k0 + c) * 4 + q < blocks;        // (columns past K: zeros)
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int j = 0; j < (X4 ? 1 : 4); ++j)
          if (!in) v[c][u][j] = uint4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (X4) {
#pragma unroll
          for (int u = 0; u < MT; ++u)
            acc[u][t] = mfma_mx(w[c][t], (int)s[c][t], v[c][u][0], in ? (int)sx[c][u] : 0,
                                acc[u][t]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 d = decode8<BF>(j == 0   ? w[c][t].x
                                        : j == 1 ? w[c][t].y
                                        : j == 2 ? w[c][t].z
                                                 : w[c][t].w,
                                        __uint_as_float(s[c][t] << 23));
#pragma unroll
            for (int u = 0; u < MT; ++u) acc[u][t] = dev::dmfma<BF>(d, v[c][u][j], acc[u][t]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      red[((wave * MT + u) * NT + t) * 64 + lane] =
          float4{acc[u][t][0], acc[u][t][1], acc[u][t][2], acc[u][t][3]};
  __syncthreads();
  for (int u = wave; u < MT; u += W) {
    const int64_t m = m0 + u * 16 + r16, n = (int64_t)nb * 16 + q * 4;
    float y[4], up[4], res[4];
    if constexpr (!GATED) fetch_residual<4>(a, m, n, res);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float4 sum = red[(u * NT + t) * 64 + lane];
#pragma unroll
      for (int k = 1; k < W; ++k) {
        const float4 p = red[((k * MT + u) * NT + t) * 64 + lane];
        sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
      }
      float* o = t ? up : y;
      o[0] = sum.x; o[1] = sum.y; o[2] = sum.z; o[3] = sum.w;
    }
    finish_run<4, GATED>(a, m, n, y, up, res);
  }
}

// ---- many tokens: tiles -------------------------------------------------------------------
template <bool BF, bool X4, bool GATED, int WM, int WN, int MT, int NT, int P>
__global__ void __launch_bounds__(64 * WM * WN, X4 && MT == 8 ? 2 : 3) mx_tile_kernel(MxArgs a, int nm, int nn) {
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
    const int64_t m = m0 + threadIdx.x;
    const uint8_t* xs = a.xs + (m < a.T ? m : a.T - 1) * blocks;
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

template <bool BF, bool X4, bool GATED, int MT, int W>
int launch_stream(const MxArgs& a, hipStream_t s) {
  const int64_t nm = cdiv(a.T, 16 * MT), nn = cdiv(a.N, 16), grid = nm * nn;
  EXQ_REQUIRE_SUPPORTED(grid * 64 * W < ((int64_t)1 << 32),
                        "exq_linear_mxfp4: T=%lld x N=%lld is too large", (long long)a.T,
                        (long long)a.N);
  hipLaunchKernelGGL((mx_stream_kernel<BF, X4, GATED, MT, W>), dim3((unsigned)grid), dim3(64 * W),
                     0, s, a, (int)nn);
  return check_launch("mx_stream_kernel");
}

// Which kernel: the one with the least rounds x time of a round.  ns[i]: what 128 columns of
// K take when every CU holds i + 1 of the work-groups (three is a round), measured in bf16
// and in MXFP4 tokens with K = 4096; it does not move with K.  In us for 16, 32, 64, 128, 512
// and 2048 tokens x 4096 x 4096:
//   bf16    16 x 16 stream 7.7, 12.1, 20, -, -, -      32 x 16 stream 8.7, 11.3, 19, 34, -, -
//           32 x 128 tiles 16, 17, 17, 17.7, 24.5, 79  32 x 256 23, 25, 25, 25, 26.6, 70
//           64 x 256 33, 35, 39, 39, 41, 65
//   MXFP4   16 x 16 6.0, 8.4, 12.9, -, -, -   32 x 16 6.3, 7.8, 12, 20, 37 (256), -
//           32 x 128 -, -, 13, 13.5, 15.5, 41  32 x 256 -, -, 17, 17, 18, 40
//           64 x 256 -, -, 23, 23, 24, 33      128 x 256 -, -, 29, 36, 37, 40
//           256 x 256 -, -, 37, 45, 45, 48
// and 4096 tokens x 14336 x 4096: bf16 64 x 256 351; MXFP4 64 x 256 190, 128 x 256 153, 256 x
// 256 (eight waves) 143; gated 4096 x 4096 x 14336: bf16 64 x 256 711, MXFP4 333, 294 and 301.
// A gated stream's work-group makes a gate and an up tile in the time of one (16 tokens x 2048
// x 2816 5.5 us: the tokens take it); up to four tokens cost less, as their rows are few.
struct Shape {
  int tokens, rows;
  int ns[3], ns4[3];
};
constexpr int kFewTokens = 4;
constexpr Shape kFew = {16, 16, {80, 150, 210}, {66, 120, 170}};
constexpr Shape kShapes[] = {
    {16, 16, {147, 280, 410}, {94, 170, 240}},       // streams
    {32, 16, {260, 500, 730}, {150, 280, 400}},
    {32, 128, {450, 670, 930}, {330, 390, 470}},     // tiles
    {32, 256, {740, 1140, 1590}, {480, 670, 850}},
    {64, 256, {1280, 1950, 2420}, {680, 950, 1250}},
    {128, 256, {0, 0, 0}, {1140, 1500, 2000}},
    {256, 256, {0, 0, 0}, {1400, 2720, 4080}},
};
constexpr const char* kKernels[] = {"stream 16x16", "stream 32x16", "tile 32x128", "tile 32x256",
                                    "tile 64x256",  "tile 128x256", "tile 256x256"};

// `vec`: runs of the result and the residual may be stored and loaded at once.  Where they may
// not, a tile's columns go one by one at its end, which the streams spread over more
// work-groups: counted as 5 us of any tile.  In us with a residual, streams and tiles: bf16 100
// x 1440 x 2047 8.0 and 12.2, 187 10.6 and 12.3, 400 x 512 x 1001 8.2 and 9.4, but 400 x 512 x
// 2047 13.2 and 9.8, 187 x 4096 x 2047 26.8 and 19.3; MXFP4 187 x 1440 x 2047 7.2 and 10.2, 800
// x 4096 x 14335 6 times the tiles' time.  Over 24 - 1600 tokens, K 512 - 4096 and 1001 - 14335
// columns (168 calls) the choice is 0.5 % from the faster one in the mean, 22 % at most (187 x
// 4096 x 2047 of MXFP4: 16.6 and 13.6); without the 5 us 4.4 and 76 %, by streams alone 56 % and
// 7 times.
constexpr int kUnalignedTileNs = 5000;

int pick_kernel(int64_t tokens, int64_t rows, int64_t KB, bool x4, bool gated, bool vec) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
    const Shape& k = i == 0 && tokens <= kFewTokens ? kFew : kShapes[i];
    const int* ns = x4 ? k.ns4 : k.ns;
    if (ns[0] == 0) continue;
    const int64_t rows_of = gated && k.rows == 16 ? 32 : k.rows;
    const int64_t per_cu = cdiv(cdiv(tokens, k.tokens) * cdiv(rows, rows_of), 256);
    const int64_t rest = per_cu % 3;
    const int64_t t = (per_cu / 3 * ns[2] + (rest ? ns[rest - 1] : 0)) * KB +
                      (vec || k.rows == 16 ? 0 : kUnalignedTileNs);
    if (t < least) {
      least = t;
      best = i;
    }
  }
  return best;
}

template <bool BF, bool X4, bool GATED>
int launch_products(const MxArgs& a, hipStream_t s) {
  const int kernel = pick_kernel(a.T, a.N * (GATED ? 2 : 1), a.KB, X4, GATED,
                                 a.vec_o && (a.vec_r || !a.res));
  switch (kernel) {
    case 0: return launch_stream<BF, X4, GATED, 1, 8>(a, s);
    case 1: return launch_stream<BF, X4, GATED, 2, 8>(a, s);
    case 2: return launch_tile<BF, X4, GATED, 1, 4, 2, 2, 6>(a, s);
    case 3: return launch_tile<BF, X4, GATED, 1, 4, 2, 4, 5>(a, s);
    case 4: return launch_tile<BF, X4, GATED, 1, 4, 4, 4, 3>(a, s);
    default:
      if constexpr (X4) {
        if (kernel == 5) return launch_tile<BF, X4, GATED, 1, 4, 8, 4, 2>(a, s);
        return launch_tile<BF, X4, GATED, 2, 4, 8, 4, 2>(a, s);
      }
      return EXQ_ERROR_UNSUPPORTED;  // (not reached: 16-bit tokens have no such shape)
  }
}

}  // namespace
}  // namespace exq

using namespace exq;

namespace {
int check_problem(const exq_linear_problem* p, const void* bias, const void* residual) {
  const char* fn = "exq_linear_mxfp4";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  EXQ_REQUIRE(p->act_dtype == EXQ_DTYPE_U8 || is_act_dtype(p->act_dtype),
              "%s: x must be f16, bf16 or u8 (MXFP4)", fn);
  EXQ_REQUIRE(is_float_dtype(p->out_dtype), "%s: out dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(!bias || is_float_dtype(p->bias_dtype), "%s: bias dtype must be f32, f16 or bf16",
              fn);
  EXQ_REQUIRE(!residual || is_float_dtype(p->residual_dtype),
              "%s: residual dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(p->activation >= EXQ_ACT_NONE && p->activation <= EXQ_ACT_SIGMOID,
              "%s: unknown activation %d", fn, p->activation);
  EXQ_REQUIRE(!(p->gated && residual), "%s: a gated product takes no residual", fn);
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
  EXQ_REQUIRE(T >= 0 && T <= INT32_MAX / 2 && K >= mx::kBlock && K <= (1 << 22) &&
                  K % mx::kBlock == 0 && N >= 1 && N <= (1 << 20),
              "%s: sizes T=%lld K=%lld N=%lld out of range (K a multiple of 32)", fn,
              (long long)T, (long long)K, (long long)N);
  EXQ_REQUIRE(p->x_stride >= 0 && p->residual_stride >= 0 && (T <= 1 || p->out_stride >= N),
              "%s: row strides must not be negative, and out's at least N", fn);
  // (a tile's rows of x lie in one buffer resource)
  EXQ_REQUIRE_SUPPORTED(T <= 1 || p->x_stride <= (1 << 22), "%s: x's row stride %lld is too large",
                        fn, (long long)p->x_stride);
  return EXQ_SUCCESS;
}
}  // namespace

extern "C" int exq_linear_mxfp4(const exq_linear_problem* p, const void* x,
                                const uint8_t* x_scales, const uint8_t* tiles,
                                const uint8_t* tile_scales, const void* bias,
                                const void* residual, void* out, exq_stream stream) {
  const char* fn = "exq_linear_mxfp4";
  const int status = check_problem(p, bias, residual);
  if (status != EXQ_SUCCESS) return status;
  const bool x4 = p->act_dtype == EXQ_DTYPE_U8;
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
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

extern "C" const char* exq_linear_mxfp4_kernel(const exq_linear_problem* p) {
  if (check_problem(p, nullptr, nullptr) != EXQ_SUCCESS || p->n_tokens == 0) return nullptr;
  return kKernels[pick_kernel(p->n_tokens, p->out_features * (p->gated ? 2 : 1),
                              mx::tile_cols(p->in_features), p->act_dtype == EXQ_DTYPE_U8,
                              p->gated != 0, (p->out_stride | p->residual_stride) % 4 == 0)];
}
