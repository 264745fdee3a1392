// mxfp4_moe.hip -- the MoE layer with MXFP4 experts:
//   out[t] = sum_j w[t, j] * W2_e (silu(Wg_e x_t) * (Wu_e x_t)),  e = ids[t, j]
#include "mxfp4_stream.h"

#include <stdlib.h>

namespace exq {
namespace {

using namespace mx;

constexpr int kGroup = 16;  // rows of a token group

struct MoeArgs {
  const int* hdr;            // [0]: token groups
  const TgEntry* tg;
  const int* sorted;         // expert-sorted position -> slot
  const uint16_t* x;         // gate/up: hidden [T, H]; down: mid [n, I]
  const uint4* tiles;        // [E, RT, KB]
  const uint32_t* wscales;   // [E, RT, G]
  int K, KB, G, RT, top_k, N;  // N: columns of the result
  uint16_t* mid;
  float* part;               // [slots, H]
};

// One wave: a token group x a tile of rows.
template <bool BF, bool GATEUP>
__global__ void __launch_bounds__(256) moe_simple_kernel(MoeArgs a) {
  constexpr int NT = GATEUP ? 2 : 1;
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  if ((int)blockIdx.y >= a.hdr[0]) return;
  const TgEntry g = a.tg[blockIdx.y];
  const int nb = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (nb * NT >= a.RT) return;
  const int pos = g.pos0 + (r16 < g.cnt ? r16 : 0);
  const int slot = a.sorted[pos];
  const uint16_t* x = a.x + (int64_t)(GATEUP ? slot / a.top_k : pos) * a.K;
  const int blocks = a.K / kBlock;
  f32x4_t acc[NT] = {};
  for (int kb = 0; kb < a.KB; ++kb) {
    const int b = kb * 4 + q;
    uint4 xv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      xv[j] = b < blocks ? *reinterpret_cast<const uint4*>(x + b * 32 + j * 8)
                         : uint4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t rt = (int64_t)g.e * a.RT + nb * NT + t;
      const uint4 w = a.tiles[(rt * a.KB + kb) * 64 + lane];
      const float s = __uint_as_float(
          (a.wscales[(rt * a.G + (kb >> 2)) * 64 + lane] >> (8 * (kb & 3)) & 0xff) << 23);
      const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t] = dev::dmfma<BF>(decode8<BF>(c[j], s), xv[j], acc[t]);
    }
  }
  if (r16 >= g.cnt) return;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int n = nb * 16 + q * 4 + v;
    if (n >= a.N) break;
    if constexpr (GATEUP)  // (rounded to the activations' type: the next product's operand)
      a.mid[(int64_t)pos * a.N + n] = (uint16_t)dev::to_act_bits<BF>(silu_f32(acc[0][v]) * acc[NT - 1][v]);
    else
      a.part[(int64_t)slot * a.N + n] = acc[0][v];
  }
}

// ---- many tokens: tiles -------------------------------------------------------------------
// Token groups of up to 64 expert-sorted rows x 64 NT weight rows: as many tokens as the
// group has, by halves, and the fewer they are the more stages are on their way.
constexpr int kTileGroup = 64;
constexpr int kTileLds = 48 * 1024;

// Unit (token group, weight tile) of work-group bid, which runs on XCD bid % 8: blocks of
// eight token groups x one weight tile go round the XCDs, so that the groups of an expert
// that lie together share its weights in one L2, and the work of an expert with many rows
// is every XCD's.
__device__ __forceinline__ bool spread_unit(int bid, int n, int n_tiles, int& tgi, int& nt) {
  const int local = bid >> 3, block = (local >> 3) * 8 + (bid & 7);
  const int g8 = block / n_tiles;
  nt = block - g8 * n_tiles;
  tgi = g8 * 8 + (local & 7);
  return tgi < n;
}
inline int64_t spread_grid(int64_t n, int64_t n_tiles) {
  return cdiv(cdiv(n, 8) * n_tiles, 8) * 64;
}

template <bool BF, bool GATEUP, int NT, int MT, int P>
__device__ __forceinline__ void moe_tile(const MoeArgs& a, unsigned char* lds, const TgEntry& g,
                                         int nb, int wave, int lane) {
  using T = Tile16<BF, 1, 4, MT, NT, P>;
  constexpr int COLS = (GATEUP ? 8 : 16) * NT;     // result columns of a wave
  static_assert(T::LDS <= kTileLds && T::W * wave_floats<NT>() * 4 <= kTileLds, "LDS");
  const int pc = T::piece(wave, lane);
  int vo[T::D], rt[NT];
#pragma unroll
  for (int j = 0; j < T::D; ++j) {
    const int r = T::row(wave, lane, j);
    if (r >= g.cnt) vo[j] = kOob;
    else if (GATEUP) vo[j] = (a.sorted[g.pos0 + r] / a.top_k) * (a.K * 2) + pc * 16;
    else vo[j] = r * (a.K * 2) + pc * 16;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {   // (tiles past the last repeat it: what they give is not stored)
    const int i = (nb * 4 + wave) * NT + t;
    rt[t] = g.e * a.RT + (i < a.RT ? i : a.RT - 1);
  }
  f32x4_t acc[MT][NT] = {};
  T::run(lds, uniform_rsrc(GATEUP ? a.x : a.x + (int64_t)g.pos0 * a.K), vo, a.tiles, a.wscales, rt,
         a.KB, a.G, a.K / 8, wave, lane, acc);
  const int nw = (nb * 4 + wave) * COLS;
  emit_tiles<GATEUP, MT, NT>(
      reinterpret_cast<float*>(lds) + wave * wave_floats<NT>(), acc, lane,
      [&](int r, int c, float (&y)[8], float (&up)[8]) {
        const int n = nw + c;
        if (r >= g.cnt || n >= a.N) return;   // (N is a multiple of 32)
        if constexpr (GATEUP) {   // (rounded to the activations' type: the next product's operand)
          uint32_t d[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            d[i] = pack16(silu_f32(y[2 * i]) * up[2 * i], silu_f32(y[2 * i + 1]) * up[2 * i + 1], BF);
          *reinterpret_cast<uint4*>(a.mid + (int64_t)(g.pos0 + r) * a.N + n) =
              uint4{d[0], d[1], d[2], d[3]};
        } else {
          float4* p = reinterpret_cast<float4*>(a.part + (int64_t)a.sorted[g.pos0 + r] * a.N + n);
          p[0] = float4{y[0], y[1], y[2], y[3]};
          p[1] = float4{y[4], y[5], y[6], y[7]};
        }
      });
}

template <bool BF, bool GATEUP, int NT>
__global__ void __launch_bounds__(256, 3) moe_tile_kernel(MoeArgs a, int n_tiles) {
  __shared__ __align__(1024) unsigned char lds[kTileLds];
  int tgi, nb;
  if (!spread_unit(blockIdx.x, a.hdr[0], n_tiles, tgi, nb)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TgEntry at = a.tg[tgi];
  const TgEntry g{__builtin_amdgcn_readfirstlane(at.e), __builtin_amdgcn_readfirstlane(at.pos0),
                  __builtin_amdgcn_readfirstlane(at.cnt), 2};
  if (g.cnt > 32) moe_tile<BF, GATEUP, NT, 4, 3>(a, lds, g, nb, wave, lane);
  else moe_tile<BF, GATEUP, NT, 2, NT == 2 ? 5 : 4>(a, lds, g, nb, wave, lane);
}

// CPL columns a lane, eight slots' ids, weights and then rows in flight.  Bound: bytes, or
// for few tokens the two round trips.
template <bool BF, int CPL>
__global__ void __launch_bounds__(256) moe_combine_kernel(const float* part, const void* ids,
                                                          int ids_dtype, const void* weights,
                                                          int w_dtype, int k, int E, int H, int T,
                                                          uint16_t* out) {
  constexpr int JB = 8;
  const int per = H / CPL;   // lanes of a token
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / per;
  const int h = (int)(i - t * per) * CPL;
  if (t >= T) return;
  typedef float vec_t __attribute__((ext_vector_type(CPL)));
  vec_t acc = {};
  for (int j0 = 0; j0 < k; j0 += JB) {
    int64_t e[JB];
    float w[JB];
    vec_t p[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const int64_t slot = t * k + (j0 + j < k ? j0 + j : k - 1);
      e[j] = load_index(ids, ids_dtype, slot);
      w[j] = load_as_f32(weights, w_dtype, slot);
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const bool there = j0 + j < k && e[j] >= 0 && e[j] < E;   // (no row, nor a weight, elsewhere)
      w[j] = there ? w[j] : 0.f;
      p[j] = vec_t{};
      if (there) p[j] = *reinterpret_cast<const vec_t*>(part + (t * k + j0 + j) * H + h);
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) acc += w[j] * p[j];
  }
  uint32_t d[CPL / 2];
#pragma unroll
  for (int c = 0; c < CPL; c += 2) d[c / 2] = pack16(acc[c], acc[c + 1], BF);
  if constexpr (CPL == 2)
    *reinterpret_cast<uint32_t*>(out + t * H + h) = d[0];
  else
    *reinterpret_cast<uint2*>(out + t * H + h) = uint2{d[0], d[CPL / 2 - 1]};
}

struct Layout {
  size_t hdr, tg, sorted, ends, blk, mid, part, total;
  int64_t tg_cap;
};
Layout layout(const exq_moe_problem* p) {
  const int64_t n = p->n_tokens * p->top_k;
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at = align_up(at + bytes, 256);
    return o;
  };
  l.tg_cap = tg_capacity(n, p->n_experts, kGroup);
  l.hdr = take(64);
  l.tg = take((size_t)l.tg_cap * sizeof(TgEntry));
  l.sorted = take((size_t)n * 4);
  l.ends = take((size_t)(p->n_experts + 1) * 4);
  l.blk = take((size_t)route_plan_blocks(n) * p->n_experts * 4);
  l.mid = take((size_t)n * p->inter_size * 2);
  l.part = take((size_t)n * p->hidden_size * 4);
  l.total = at;
  return l;
}

int check_moe(const exq_moe_problem* p) {
  const char* fn = "exq_moe_mxfp4_forward";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  const int64_t T = p->n_tokens, H = p->hidden_size, I = p->inter_size, k = p->top_k;
  EXQ_REQUIRE(is_act_dtype(p->act_dtype), "%s: hidden must be f16 or bf16", fn);
  EXQ_REQUIRE(is_index_dtype(p->ids_dtype), "%s: ids must be i32 or i64", fn);
  EXQ_REQUIRE(is_float_dtype(p->weights_dtype), "%s: weights must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(H >= 32 && H % 32 == 0 && I >= 32 && I % 32 == 0 && H <= (1 << 20) &&
                  I <= (1 << 20),
              "%s: H=%lld and I=%lld must be multiples of 32", fn, (long long)H, (long long)I);
  EXQ_REQUIRE(p->n_experts >= 1 && p->n_experts <= 1024 && k >= 1 && k <= 64 && T >= 0,
              "%s: T=%lld E=%lld k=%lld out of range", fn, (long long)T,
              (long long)p->n_experts, (long long)k);
  EXQ_REQUIRE(p->n_shared == 0 && p->group_size == 32,
              "%s: no shared experts, and groups of 32", fn);
  EXQ_REQUIRE_SUPPORTED(T <= ((int64_t)1 << 24) / k, "%s: T=%lld x k=%lld slots are too many", fn,
                        (long long)T, (long long)k);
  return EXQ_SUCCESS;
}

}  // namespace
}  // namespace exq

using namespace exq;

extern "C" size_t exq_moe_mxfp4_workspace_size(const exq_moe_problem* p) {
  if (check_moe(p) != EXQ_SUCCESS) return 0;
  return layout(p).total;
}

extern "C" int exq_moe_mxfp4_forward(const exq_moe_problem* p, const void* hidden,
                                     const void* topk_ids, const void* topk_weights,
                                     const uint8_t* w13_tiles, const uint8_t* w13_scales,
                                     const uint8_t* w2_tiles, const uint8_t* w2_scales, void* out,
                                     void* workspace, size_t workspace_bytes, exq_stream stream) {
  const char* fn = "exq_moe_mxfp4_forward";
  int st = check_moe(p);
  if (st) return st;
  const int64_t T = p->n_tokens, H = p->hidden_size, I = p->inter_size;
  const int k = (int)p->top_k, E = (int)p->n_experts;
  if (T == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(hidden && topk_ids && topk_weights && w13_tiles && w13_scales && w2_tiles &&
                  w2_scales && out && workspace, "%s: null pointer", fn);
  EXQ_REQUIRE(((uintptr_t)hidden | (uintptr_t)w13_tiles | (uintptr_t)w13_scales |
               (uintptr_t)w2_tiles | (uintptr_t)w2_scales | (uintptr_t)out |
               (uintptr_t)workspace) % 16 == 0,
              "%s: hidden, weights, out and workspace must be 16-byte aligned", fn);
  const Layout l = layout(p);
  if (workspace_bytes < l.total)
    return set_error(EXQ_ERROR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu needed", fn,
                     workspace_bytes, l.total);
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  const hipStream_t s = as_stream(stream);
  RoutePlanParams rp{};
  rp.ids = topk_ids;
  rp.ids_dtype = p->ids_dtype;
  rp.T = (int)T;
  rp.k = rp.kp = k;
  rp.E = rp.Ep = E;
  rp.n = (int)(T * k);
  rp.all_tier = 2;
  rp.hdr = reinterpret_cast<int*>(ws + l.hdr);
  rp.ends = reinterpret_cast<int*>(ws + l.ends);
  rp.sorted = reinterpret_cast<int*>(ws + l.sorted);
  rp.tg = reinterpret_cast<TgEntry*>(ws + l.tg);
  rp.tg_cap = (int)l.tg_cap;
  const bool tile = T > (getenv("MXTH") ? atoi(getenv("MXTH")) : 64) && getenv("MXS") == nullptr;
  rp.i4_group = rp.bf_group = rp.i8_group = rp.i4_big_group = tile ? kTileGroup : kGroup;
  if (tile) rp.i4_big_rows = getenv("MXB") ? atoi(getenv("MXB")) : 33;
  rp.out = out;
  rp.out_bytes = T * H * 2;
  rp.blk_cnt = reinterpret_cast<int*>(ws + l.blk);
  const bool st_ = getenv("MXS") == nullptr && !tile;
  const int64_t n = T * k;
  const bool by_slot = st_ && T <= (getenv("MXT") ? atoi(getenv("MXT")) : 1) && n <= kOwnedSlots;
  const bool all = st_ && !by_slot && T <= 16 && n <= 128 && E <= 256 && H <= 2048;
  const bool route8 = st_ && !all && n <= 512 && E <= 512, route16 = st_ && !all && !route8 && n <= 1024 && E <= 256;
  const bool route = by_slot || all || route8 || route16;
  const bool owned = st_ && n <= kOwnedSlots;
  if (!route) {
    st = launch_route_plan(rp, s);
    if (st) return st;
  }
  MoeArgs a{};
  a.hdr = rp.hdr;
  a.tg = rp.tg;
  a.sorted = rp.sorted;
  a.top_k = k;
  a.mid = reinterpret_cast<uint16_t*>(ws + l.mid);
  a.part = reinterpret_cast<float*>(ws + l.part);
  const bool bf = p->act_dtype == EXQ_DTYPE_BF16;
  auto run = [&](bool gateup) {
    a.x = gateup ? reinterpret_cast<const uint16_t*>(hidden) : a.mid;
    a.tiles = reinterpret_cast<const uint4*>(gateup ? w13_tiles : w2_tiles);
    a.wscales = reinterpret_cast<const uint32_t*>(gateup ? w13_scales : w2_scales);
    a.K = (int)(gateup ? H : I);
    a.N = (int)(gateup ? I : H);
    a.KB = (int)tile_cols(a.K);
    a.G = (a.KB + 3) / 4;
    a.RT = (int)(gateup ? mx::tile_rows(2 * I, 1) : mx::tile_rows(H, 0));
    if (getenv("MXS") == nullptr && !tile) {
      if (!gateup && owned) {
        OwnedArgs o{by_slot ? nullptr : a.hdr, a.tg, a.sorted, a.mid, a.tiles, reinterpret_cast<const uint8_t*>(a.wscales), topk_ids, topk_weights,
          p->ids_dtype, p->weights_dtype, (int)T, k, E, (int)I, (int)H, a.KB, a.G, a.RT, reinterpret_cast<uint16_t*>(out)};
        if (bf) hipLaunchKernelGGL((moe_owned_down_kernel<true, 3>), dim3((unsigned)(H / 16)), dim3(512), 0, s, o);
        else hipLaunchKernelGGL((moe_owned_down_kernel<false, 3>), dim3((unsigned)(H / 16)), dim3(512), 0, s, o);
        return check_launch("moe_owned_down_kernel");
      }
      StreamArgs b{rp.hdr, rp.tg, rp.sorted, topk_ids, p->ids_dtype, (int)(T * k), E, a.x, a.tiles, reinterpret_cast<const uint8_t*>(a.wscales), a.K, a.KB, a.G, a.RT, a.top_k, a.N,
                   0, 1, a.mid, a.part};
      auto go = [&](auto kernel, int KS, int C) {
        b.n_rt = (int)cdiv(a.RT / 2, 4 / KS);
        b.chunks = (int)cdiv(cdiv(a.KB, KS), C);
        const int64_t cap = tg_capacity(T * k, E, 16) * b.n_rt;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(cap < 512 ? cap : 512)), dim3(256), 0, s, b);
        return check_launch("moe_stream_kernel");
      };
#define GO(UP, NSEG, ALL, KS, C) return bf ? go(moe_stream_kernel<true, UP, NSEG, ALL, KS, C>, KS, C) : go(moe_stream_kernel<false, UP, NSEG, ALL, KS, C>, KS, C)
      if (gateup) {
        if (by_slot) GO(true, kBySlot, false, 4, 4);
        if (all) GO(true, 2, true, 4, 4);
        if (route8) GO(true, 8, false, 4, 4);
        if (route16) GO(true, 16, false, 4, 4);
        GO(true, 0, false, 4, 4);
      }
      if (a.KB <= 6) GO(false, 0, false, 2, 3);
      if (a.KB <= 8) GO(false, 0, false, 4, 2);
      if (a.KB <= 12) GO(false, 0, false, 4, 3);
      GO(false, 0, false, 4, 4);
    }
    if (tile) {
      const int64_t cap = tg_capacity(T * k, E, kTileGroup);
      const int rows = cap * cdiv(a.RT, 16) < (getenv("MXU") ? atoi(getenv("MXU")) : 512) ? 128 : 256;
      auto go = [&](auto kernel) {
        const int64_t nt = cdiv(a.RT, rows / 16);
        hipLaunchKernelGGL(kernel, dim3((unsigned)spread_grid(cap, nt)), dim3(256), 0, s, a, (int)nt);
        return check_launch("moe_tile_kernel");
      };
#define GT(UP) return rows == 128 ? bf ? go(moe_tile_kernel<true, UP, 2>) : go(moe_tile_kernel<false, UP, 2>) : bf ? go(moe_tile_kernel<true, UP, 4>) : go(moe_tile_kernel<false, UP, 4>)
      if (gateup) GT(true);
      GT(false);
    }
    const dim3 grid((unsigned)cdiv(cdiv(a.N, 16), 4), (unsigned)l.tg_cap);
    if (gateup) {
      if (bf) hipLaunchKernelGGL((moe_simple_kernel<true, true>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((moe_simple_kernel<false, true>), grid, dim3(256), 0, s, a);
    } else {
      if (bf) hipLaunchKernelGGL((moe_simple_kernel<true, false>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((moe_simple_kernel<false, false>), grid, dim3(256), 0, s, a);
    }
    return check_launch("moe_simple_kernel");
  };
  st = run(true);
  if (st) return st;
  st = run(false);
  if (st || owned) return st;
  auto combine = [&](auto kernel, int cpl) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(T * (H / cpl), 256)), dim3(256), 0, s, a.part,
                       topk_ids, p->ids_dtype, topk_weights, p->weights_dtype, k, E, (int)H, (int)T,
                       reinterpret_cast<uint16_t*>(out));
    return check_launch("moe_combine_kernel");
  };
  if (T * H <= 256 * 512)
    return bf ? combine(moe_combine_kernel<true, 2>, 2) : combine(moe_combine_kernel<false, 2>, 2);
  return bf ? combine(moe_combine_kernel<true, 4>, 4) : combine(moe_combine_kernel<false, 4>, 4);
}
