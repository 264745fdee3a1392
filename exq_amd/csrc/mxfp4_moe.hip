// mxfp4_moe.hip -- the MoE layer with MXFP4 experts:
//   out[t] = sum_j w[t, j] * W2_e (silu(Wg_e x_t) * (Wu_e x_t)),  e = ids[t, j]
//
// Few slots are bound by the latency of a chain of kernels and by the active experts' bytes,
// many by the matrix instructions, so the number of slots n = T k says which kernels run
// (path_of):
//   few (runs_by_slot) a slot is a group: two kernels, no routing, the second one sums all
//                      slots of its columns (1 token x 8 of 128 experts of 2048 x 768 13.6 us)
//   n <= 512           gate/up tiles route, down tiles write fp32 rows, a third kernel adds a
//                      token's (64 tokens 50 us, floor 26; 16 x 8 of 64 of 2048 x 1024 34 - 42, 21)
//   more               the plan is made first (2001 tokens x 6 of 64 of 2048 x 1408 251 us, floor
//                      149 at the rate of a large bf16 product; the plan 15, the sums 27)
// mid = silu(gate) * up is rounded to the activations' type, which the second product's matrix
// instructions take; all sums are in 32 bits, each in a fixed order.
#include "mxfp4_route.h"
#include "mxfp4_stream.h"

namespace exq {
namespace {

using namespace mx;

struct MoeArgs {
  int* hdr;                  // [0]: token groups
  TgEntry* tg;
  int* sorted;         // expert-sorted position -> slot
  const uint16_t* x;         // gate/up: hidden [T, H]; down: mid [n, I]
  const uint4* tiles;        // [E, RT, KB]
  const uint32_t* wscales;   // [E, RT, G]
  int K, KB, G, RT, top_k, N;  // N: columns of the result
  uint16_t* mid;
  float* part;               // [slots, H]
};

// ---- tiles ----------------------------------------------------------------------------------
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
                                         const int* tokens, int nb, int wave, int lane) {
  using T = Tile16<BF, 1, 4, MT, NT, P>;
  constexpr int COLS = (GATEUP ? 8 : 16) * NT;     // result columns of a wave
  static_assert(T::LDS <= kTileLds && T::W * wave_floats<NT>() * 4 <= kTileLds, "LDS");
  const int pc = T::piece(wave, lane);
  int vo[T::D], rt[NT];
#pragma unroll
  for (int j = 0; j < T::D; ++j) {
    const int r = T::row(wave, lane, j);
    if (r >= g.cnt) vo[j] = kOob;
    else if (GATEUP) vo[j] = (tokens ? tokens[r] : a.sorted[g.pos0 + r] / a.top_k) * (a.K * 2) + pc * 16;
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

// NSEG > 0: the kernel routes (gate/up).
template <bool BF, bool GATEUP, int NT, int NSEG>
__global__ void __launch_bounds__(256, 3) moe_tile_kernel(MoeArgs a, RouteArgs ra, int n_tiles) {
  __shared__ __align__(1024) unsigned char lds[kTileLds];
  int tgi, nb;
  TgEntry at;
  const int* tokens = nullptr;
  if constexpr (NSEG > 0) {
    using R = Router<NSEG>;
    __shared__ TgEntry own;
    __shared__ int rows[kTileGroup];
    static_assert(R::kWords * 4 <= kTileLds && kTileGroup == 64, "routing scratch");
    if (!R::here(ra, reinterpret_cast<uint32_t*>(lds), &own, rows, [&](int n) {
          return spread_unit(blockIdx.x, n, n_tiles, tgi, nb) ? tgi : -1;
        }))
      return;
    at = own;
    tokens = rows;
  } else {
    if (!spread_unit(blockIdx.x, a.hdr[0], n_tiles, tgi, nb)) return;
    at = a.tg[tgi];
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TgEntry g{__builtin_amdgcn_readfirstlane(at.e), __builtin_amdgcn_readfirstlane(at.pos0),
                  __builtin_amdgcn_readfirstlane(at.cnt), 2};
  if (g.cnt > 32) moe_tile<BF, GATEUP, NT, 4, 3>(a, lds, g, tokens, nb, wave, lane);
  else if (g.cnt > 16) moe_tile<BF, GATEUP, NT, 2, NT == 4 ? 4 : 5>(a, lds, g, tokens, nb, wave, lane);
  else moe_tile<BF, GATEUP, NT, 1, NT == 4 ? 5 : 8>(a, lds, g, tokens, nb, wave, lane);
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

// Weight tiles of a wave: four (a work-group 256 weight rows), as its tokens are read least
// so, fewer where the work-groups would not fill the CUs twice.
int wave_tiles(int64_t groups, int64_t RT, int least) {
  constexpr int64_t kFull = 512;
  for (int nt = 4; nt > least; nt /= 2)
    if (groups * cdiv(RT, 4 * nt) >= kFull) return nt;
  return least;
}
template <typename Kernel>
int launch_moe_tile(Kernel kernel, const MoeArgs& a, const RouteArgs& ra, int64_t groups, int nt,
                    hipStream_t s) {
  const int64_t n_tiles = cdiv(a.RT, 4 * nt), grid = spread_grid(groups, n_tiles);
  EXQ_REQUIRE_SUPPORTED(grid * 256 < ((int64_t)1 << 32),
                        "exq_moe_mxfp4_forward: %lld token groups x %d rows are too many",
                        (long long)groups, a.RT * 16);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, s, a, ra, (int)n_tiles);
  return check_launch("moe_tile_kernel");
}
template <bool BF, int NSEG>
int launch_gateup_as(const MoeArgs& a, const RouteArgs& ra, hipStream_t s) {
  const int64_t groups = tg_capacity(ra.n, ra.E, kTileGroup);
  if (wave_tiles(groups, a.RT, 2) == 4)
    return launch_moe_tile(moe_tile_kernel<BF, true, 4, NSEG>, a, ra, groups, 4, s);
  return launch_moe_tile(moe_tile_kernel<BF, true, 2, NSEG>, a, ra, groups, 2, s);
}
template <bool BF>
int launch_down(const MoeArgs& a, int64_t groups, hipStream_t s) {
  switch (wave_tiles(groups, a.RT, 1)) {
    case 4: return launch_moe_tile(moe_tile_kernel<BF, false, 4, 0>, a, RouteArgs{}, groups, 4, s);
    case 2: return launch_moe_tile(moe_tile_kernel<BF, false, 2, 0>, a, RouteArgs{}, groups, 2, s);
    default: return launch_moe_tile(moe_tile_kernel<BF, false, 1, 0>, a, RouteArgs{}, groups, 1, s);
  }
}

// How a batch runs.
struct Path {
  int64_t n;       // slots
  bool by_slot;    // no routing, down by output columns without partial rows
  int nseg;        // the gate/up tiles route, 64 nseg slots at most; 0: a plan kernel first
};
Path path_of(const exq_moe_problem* p) {
  Path r;
  r.n = p->n_tokens * p->top_k;
  r.by_slot = runs_by_slot(r.n, p->hidden_size, p->inter_size);
  r.nseg = r.by_slot ? 0 : r.n <= 64 ? 1 : r.n <= 128 ? 2
           : r.n <= 512 && p->n_experts <= Router<8>::kExperts ? 8 : 0;
  return r;
}

template <bool BF>
int launch_gateup(const MoeArgs& a, const RouteArgs& ra, const Path& r, hipStream_t s) {
  switch (r.nseg) {
    case 1: return launch_gateup_as<BF, 1>(a, ra, s);
    case 2: return launch_gateup_as<BF, 2>(a, ra, s);
    case 8: return launch_gateup_as<BF, 8>(a, ra, s);
    default: return launch_gateup_as<BF, 0>(a, ra, s);
  }
}

struct Layout {
  size_t hdr, tg, sorted, ends, blk, mid, part, total;
  int64_t tg_cap;
};
Layout layout(const exq_moe_problem* p) {
  const Path r = path_of(p);
  Layout l;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at = align_up(at + bytes, 256);
    return o;
  };
  l.tg_cap = tg_capacity(r.n, p->n_experts, kTileGroup);
  l.hdr = take(64);
  l.tg = take((size_t)l.tg_cap * sizeof(TgEntry));
  l.sorted = take((size_t)r.n * 4);
  l.ends = take((size_t)(p->n_experts + 1) * 4);
  l.blk = take((size_t)route_plan_blocks(r.n) * p->n_experts * 4);
  l.mid = take((size_t)r.n * p->inter_size * 2);
  l.part = take(r.by_slot ? 0 : (size_t)r.n * p->hidden_size * 4);
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
  // (one buffer resource covers it: lin::kSpan bytes)
  EXQ_REQUIRE_SUPPORTED(T <= (((int64_t)1 << 30) - 256) / H,
                        "%s: T=%lld x H=%lld: hidden is past 2 GiB", fn, (long long)T, (long long)H);
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
  const Path r = path_of(p);
  const bool bf = p->act_dtype == EXQ_DTYPE_BF16;
  MoeArgs a{};
  a.hdr = reinterpret_cast<int*>(ws + l.hdr);
  a.tg = reinterpret_cast<TgEntry*>(ws + l.tg);
  a.sorted = reinterpret_cast<int*>(ws + l.sorted);
  a.top_k = k;
  a.mid = reinterpret_cast<uint16_t*>(ws + l.mid);
  a.part = reinterpret_cast<float*>(ws + l.part);
  if (!r.by_slot && r.nseg == 0) {
    RoutePlanParams rp{};   // (no rp.out: the combine kernel writes all of it, zeros too)
    rp.ids = topk_ids;
    rp.ids_dtype = p->ids_dtype;
    rp.T = (int)T;
    rp.k = rp.kp = k;
    rp.E = rp.Ep = E;
    rp.n = (int)r.n;
    rp.all_tier = 2;
    rp.hdr = a.hdr;
    rp.ends = reinterpret_cast<int*>(ws + l.ends);
    rp.sorted = a.sorted;
    rp.tg = a.tg;
    rp.tg_cap = (int)l.tg_cap;
    rp.i4_group = rp.bf_group = rp.i8_group = rp.i4_big_group = kTileGroup;
    rp.i4_big_rows = kTileGroup / 2 + 1;   // (the groups that take longest first)
    rp.blk_cnt = reinterpret_cast<int*>(ws + l.blk);
    st = launch_route_plan(rp, s);
    if (st) return st;
  }
  auto weights_of = [&](const uint8_t* tiles, const uint8_t* scales, int64_t K, int64_t N,
                        int64_t rows, int gated) {
    a.tiles = reinterpret_cast<const uint4*>(tiles);
    a.wscales = reinterpret_cast<const uint32_t*>(scales);
    a.K = (int)K;
    a.N = (int)N;
    a.KB = (int)tile_cols(K);
    a.G = (a.KB + 3) / 4;
    a.RT = (int)mx::tile_rows(rows, gated);
  };
  weights_of(w13_tiles, w13_scales, H, I, 2 * I, 1);
  a.x = reinterpret_cast<const uint16_t*>(hidden);
  if (r.by_slot) {
    const SlotArgs b{topk_ids, p->ids_dtype, E, k, a.x, a.tiles,
                     reinterpret_cast<const uint8_t*>(a.wscales), a.K, a.KB, a.G, a.RT, (int)I,
                     a.mid};
    const dim3 grid((unsigned)(I / 16), (unsigned)r.n);
    if (bf) hipLaunchKernelGGL((moe_slot_gateup_kernel<true>), grid, dim3(256), 0, s, b);
    else hipLaunchKernelGGL((moe_slot_gateup_kernel<false>), grid, dim3(256), 0, s, b);
    st = check_launch("moe_slot_gateup_kernel");
  } else {
    const RouteArgs ra{topk_ids, p->ids_dtype, (int)r.n, E, k, a.hdr, a.tg, a.sorted};
    st = bf ? launch_gateup<true>(a, ra, r, s) : launch_gateup<false>(a, ra, r, s);
  }
  if (st) return st;
  weights_of(w2_tiles, w2_scales, I, H, H, 0);
  a.x = a.mid;
  if (r.by_slot) {
    const OwnedArgs o{a.mid, a.tiles, reinterpret_cast<const uint8_t*>(a.wscales), topk_ids,
                      topk_weights, p->ids_dtype, p->weights_dtype, (int)T, k, E, (int)I, (int)H,
                      a.KB, a.G, a.RT, reinterpret_cast<uint16_t*>(out)};
    const dim3 grid((unsigned)(H / 16));
    if (bf) hipLaunchKernelGGL((moe_owned_down_kernel<true, 3>), grid, dim3(64 * kOwnedWaves), 0, s, o);
    else hipLaunchKernelGGL((moe_owned_down_kernel<false, 3>), grid, dim3(64 * kOwnedWaves), 0, s, o);
    return check_launch("moe_owned_down_kernel");
  }
  st = bf ? launch_down<true>(a, l.tg_cap, s) : launch_down<false>(a, l.tg_cap, s);
  if (st) return st;
  auto combine = [&](auto kernel, int cpl) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(T * (H / cpl), 256)), dim3(256), 0, s, a.part,
                       topk_ids, p->ids_dtype, topk_weights, p->weights_dtype, k, E, (int)H, (int)T,
                       reinterpret_cast<uint16_t*>(out));
    return check_launch("moe_combine_kernel");
  };
  // two columns a lane until four fill the chip: 64 tokens x 2048 6.9 and 4.5 us
  if (T * H <= 256 * 512)
    return bf ? combine(moe_combine_kernel<true, 2>, 2) : combine(moe_combine_kernel<false, 2>, 2);
  return bf ? combine(moe_combine_kernel<true, 4>, 4) : combine(moe_combine_kernel<false, 4>, 4);
}
