// mxfp4_moe.hip -- the MoE layer with MXFP4 experts:
//   out[t] = sum_j w[t, j] * W2_e (silu(Wg_e x_t) * (Wu_e x_t)),  e = ids[t, j]
#include "mxfp4.h"

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

// out[t] = sum_j w[t, j] * part[t, j] in the order of j; ids outside [0, E) have no row.
template <bool BF>
__global__ void __launch_bounds__(256) moe_combine_kernel(const float* part, const void* ids,
                                                          int ids_dtype, const void* weights,
                                                          int w_dtype, int k, int E, int H,
                                                          uint16_t* out) {
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y * 256 + threadIdx.x;
  if (h >= H) return;
  float acc = 0.f;
  for (int j = 0; j < k; ++j) {
    const int64_t e = load_index(ids, ids_dtype, t * k + j);
    if (e < 0 || e >= E) continue;
    acc += load_as_f32(weights, w_dtype, t * k + j) * part[(t * k + j) * H + h];
  }
  out[t * H + h] = (uint16_t)dev::to_act_bits<BF>(acc);
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
  rp.i4_group = rp.bf_group = rp.i8_group = rp.i4_big_group = kGroup;
  rp.out = out;
  rp.out_bytes = T * H * 2;
  rp.blk_cnt = reinterpret_cast<int*>(ws + l.blk);
  st = launch_route_plan(rp, s);
  if (st) return st;
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
  if (st) return st;
  const dim3 grid((unsigned)T, (unsigned)cdiv(H, 256));
  if (bf)
    hipLaunchKernelGGL((moe_combine_kernel<true>), grid, dim3(256), 0, s, a.part, topk_ids,
                       p->ids_dtype, topk_weights, p->weights_dtype, k, E, (int)H,
                       reinterpret_cast<uint16_t*>(out));
  else
    hipLaunchKernelGGL((moe_combine_kernel<false>), grid, dim3(256), 0, s, a.part, topk_ids,
                       p->ids_dtype, topk_weights, p->weights_dtype, k, E, (int)H,
                       reinterpret_cast<uint16_t*>(out));
  return check_launch("moe_combine_kernel");
}
