// router.hip -- routing with groups of experts: softmax or sigmoid scores, an
// optional bias on the ranking, the best groups, the best experts inside them,
// renormalised and scaled weights.
//
// For a token's logits l[e] and G groups of E / G consecutive experts:
//   there(e)  l[e] and bias[e] are neither NaN nor -inf; l is capped at FLT_MAX
//   s(e)      exp(l - max l) / sum exp(l - max l), or 1 / (1 + exp(-l))
//   r(e)      s(e) + bias[e]; without a bias the order of l, which is that of s
//   group     max r, or the sum of the two best r, over its experts that are there
// The topk_group best groups stay, then the k best r in them are the ids (equal
// values to the lower index), and slots that no expert is left for get id -1 and
// weight 0.  Weights are s, or s over the sum of the chosen ones.
#include <float.h>

#include "exq_internal.h"

namespace exq {
namespace {

struct RouteArgs {
  const void* logits;
  const void* bias;          // [E] or null
  const int32_t* n_valid;    // rows from *n_valid on are padding, or null
  void* ids;
  void* wts;
  int ldt, bdt, idt, wdt;
  int T, E, k, G, gs, top_groups;
  int sigmoid, top2, renorm;
  float scale;
};

template <int CTRL, int ROWS, uint32_t ID>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)ID, (int)v, CTRL, ROWS, 0xf, false);
}
// Wave-wide reduction: quad swaps and rotations inside the 16-lane rows, then the
// row broadcasts; lane 63 ends with the result.  `ID` is the operation's identity.
template <uint32_t ID, typename Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, Op op) {
  v = op(v, dpp<0xB1, 0xf, ID>(v));   // quad_perm [1, 0, 3, 2]
  v = op(v, dpp<0x4E, 0xf, ID>(v));   // quad_perm [2, 3, 0, 1]
  v = op(v, dpp<0x124, 0xf, ID>(v));  // row_ror 4
  v = op(v, dpp<0x128, 0xf, ID>(v));  // row_ror 8
  v = op(v, dpp<0x142, 0xa, ID>(v));  // row_bcast 15 -> rows 1, 3
  v = op(v, dpp<0x143, 0xc, ID>(v));  // row_bcast 31 -> rows 2, 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return wave_reduce<0u>(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  return wave_reduce<0xffffffffu>(v, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  const uint32_t hi = wave_max((uint32_t)(v >> 32));
  const uint32_t lo = wave_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// Order-preserving key of a rank value (-0 and +0 share one); 0 lies below every
// key and marks an expert that is not there, or taken.
__device__ __forceinline__ uint64_t rank_key(double r) {
  uint64_t b = (uint64_t)__double_as_longlong(r);
  if ((b << 1) == 0u) b = 0u;
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double key_rank(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}

// The best remaining key of the wave and its expert (lane l holds experts l + 64 c):
// the lowest id among equal keys.  Key 0: none is left.
template <int MAXC>
__device__ __forceinline__ uint64_t wave_best(const uint64_t (&key)[MAXC], int lane, int lo,
                                              int hi, int& expert) {
  uint64_t bk = 0u;
  int be = 0;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = lane + 64 * c;
    if (e >= lo && e < hi && key[c] > bk) {  // strict: the lower id keeps a tie
      bk = key[c];
      be = e;
    }
  }
  const uint64_t K = wave_max64(bk);
  expert = (int)wave_min(bk == K && K ? (uint32_t)be : 0xffffffffu);
  return K;
}

__device__ __forceinline__ void store_choice(const RouteArgs& a, int64_t row, int j, int id,
                                             float w) {
  const int64_t at = row * a.k + j;
  if (a.idt == EXQ_DTYPE_I64)
    reinterpret_cast<int64_t*>(a.ids)[at] = id;
  else
    reinterpret_cast<int32_t*>(a.ids)[at] = id;
  store_from_f32(a.wts, a.wdt, at, w);
}

// One token, by one wave, ranked in 64 bits: neither an expert nor a group is
// decided by the rounding of a score.  The weights are the chosen scores:
// exp(u - U) / sum with u = l (softmax) or log(sigmoid(l)) = min(l, 0) -
// log1p(exp(-|l|)), and U the largest chosen u where they are renormalised, so
// that scores which all underflow still have their ratio.
template <int MAXC>
__device__ void route_row(const RouteArgs& a, int64_t row, int lane) {
  uint64_t key[MAXC];
  float lg[MAXC];
  float m = -FLT_MAX;
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = lane + 64 * c;
    lg[c] = -INFINITY;
    if (e < a.E) {
      const float l = load_as_f32(a.logits, a.ldt, row * a.E + e);
      const float b = a.bias ? load_as_f32(a.bias, a.bdt, e) : 0.f;
      if (l > -INFINITY && b > -INFINITY) lg[c] = fminf(l, FLT_MAX);
    }
    m = fmaxf(m, lg[c]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  double S = 0.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
      if (lg[c] > -INFINITY) S += exp((double)lg[c] - (double)m);
    S = wave_sum64(S);
  }
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    key[c] = 0u;
    if (lg[c] > -INFINITY) {
      double r = lg[c];
      if (a.bias) {
        const double s = a.sigmoid ? 1.0 / (1.0 + exp(-(double)lg[c]))
                                   : exp((double)lg[c] - (double)m) / S;
        r = s + (double)load_as_f32(a.bias, a.bdt, lane + 64 * c);
      }
      key[c] = rank_key(r);
    }
  }

  if (a.top_groups < a.G) {
    // lane g: the value of group g
    uint64_t gkey = 0u;
    for (int g = 0; g < a.G; ++g) {
      int e1, e2;
      const int lo = g * a.gs, hi = lo + a.gs;
      uint64_t v = wave_best<MAXC>(key, lane, lo, hi, e1);
      if (a.top2 && v) {
        // the two best scores, not the logits that rank them where there is no bias
        uint64_t rest[MAXC];
#pragma unroll
        for (int c = 0; c < MAXC; ++c) rest[c] = lane + 64 * c == e1 ? 0u : key[c];
        const uint64_t v2 = wave_best<MAXC>(rest, lane, lo, hi, e2);
        double r1 = key_rank(v), r2 = v2 ? key_rank(v2) : 0.0;
        if (!a.bias) {
          r1 = a.sigmoid ? 1.0 / (1.0 + exp(-r1)) : exp(r1 - (double)m) / S;
          if (v2) r2 = a.sigmoid ? 1.0 / (1.0 + exp(-r2)) : exp(r2 - (double)m) / S;
        }
        v = rank_key(r1 + r2);
      }
      if (lane == g) gkey = v;
    }
    uint64_t keep = 0u;
    for (int j = 0; j < a.top_groups; ++j) {
      const uint64_t K = wave_max64(gkey);
      if (K == 0u) break;
      const int g = (int)wave_min(gkey == K ? (uint32_t)lane : 0xffffffffu);
      keep |= 1ull << g;
      if (lane == g) gkey = 0u;
    }
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {
      const int e = lane + 64 * c;
      if (e < a.E && !(keep >> (e / a.gs) & 1u)) key[c] = 0u;
    }
  }

  int my_id = -1;
  float my_l = -INFINITY;
  for (int j = 0; j < a.k; ++j) {
    int e;
    const uint64_t K = wave_best<MAXC>(key, lane, 0, a.E, e);
    if (K == 0u) break;
    float l = 0.f;
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
      if (lane + 64 * c == e) {
        key[c] = 0u;
        l = lg[c];
      }
    l = __shfl(l, e & 63, 64);
    if (lane == j) {
      my_id = e;
      my_l = l;
    }
  }
  double w = 0.0;
  if (my_id >= 0) {
    w = my_l;
    if (a.sigmoid) w = fmin(w, 0.0) - log1p(exp(-fabs(w)));
  }
  if (a.renorm) {
    double U = my_id >= 0 ? w : -INFINITY;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) U = fmax(U, __shfl_xor(U, d, 64));
    w = my_id >= 0 ? exp(w - U) : 0.0;
    const double sum = wave_sum64(w);
    w = my_id >= 0 ? w / sum : 0.0;
  } else if (my_id >= 0) {
    w = a.sigmoid ? exp(w) : exp(w - (double)m) / S;
  }
  if (lane < a.k) store_choice(a, row, lane, my_id, (float)(w * (double)a.scale));
}

template <int MAXC>
__global__ void __launch_bounds__(256) route_rows_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;  // (wave-uniform)
  if (a.n_valid && row >= *a.n_valid) {
    if (lane < a.k) store_choice(a, row, lane, -1, 0.f);
    return;
  }
  route_row<MAXC>(a, row, lane);
}

}  // namespace
}  // namespace exq

using namespace exq;

extern "C" int exq_grouped_topk(const exq_route_problem* p, const void* logits, const void* bias,
                                const int32_t* n_valid, void* topk_ids, void* topk_weights,
                                exq_stream stream) {
  const char* fn = "exq_grouped_topk";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  EXQ_REQUIRE(is_float_dtype(p->logits_dtype), "%s: logits dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(!bias || is_float_dtype(p->bias_dtype), "%s: bias dtype must be f32, f16 or bf16",
              fn);
  EXQ_REQUIRE(is_index_dtype(p->ids_dtype), "%s: ids dtype must be i32 or i64", fn);
  EXQ_REQUIRE(is_float_dtype(p->weights_dtype), "%s: weights dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(p->scoring == EXQ_SCORE_SOFTMAX || p->scoring == EXQ_SCORE_SIGMOID,
              "%s: scoring=%d is neither softmax nor sigmoid", fn, p->scoring);
  EXQ_REQUIRE(p->group_score == EXQ_GROUP_MAX || p->group_score == EXQ_GROUP_TOP2,
              "%s: group_score=%d is neither max nor top2", fn, p->group_score);
  EXQ_REQUIRE(p->n_tokens >= 0 && p->n_tokens <= INT32_MAX / 4, "%s: n_tokens=%lld out of range",
              fn, (long long)p->n_tokens);
  EXQ_REQUIRE(p->n_experts >= 1 && p->n_experts <= 1024, "%s: n_experts=%lld must be in [1, 1024]",
              fn, (long long)p->n_experts);
  EXQ_REQUIRE(p->n_groups >= 1 && p->n_groups <= 64 && p->n_experts % p->n_groups == 0,
              "%s: n_groups=%lld must divide n_experts and be at most 64", fn,
              (long long)p->n_groups);
  EXQ_REQUIRE(p->topk_group >= 1 && p->topk_group <= p->n_groups,
              "%s: topk_group=%lld must be in [1, n_groups]", fn, (long long)p->topk_group);
  EXQ_REQUIRE(p->top_k >= 1 && p->top_k <= 64 &&
                  p->top_k <= p->n_experts / p->n_groups * p->topk_group,
              "%s: top_k=%lld must be in [1, 64] and fit the experts of topk_group groups", fn,
              (long long)p->top_k);
  if (p->n_tokens == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(logits && topk_ids && topk_weights, "%s: null pointer", fn);
  RouteArgs a;
  a.logits = logits;
  a.bias = bias;
  a.n_valid = n_valid;
  a.ids = topk_ids;
  a.wts = topk_weights;
  a.ldt = p->logits_dtype;
  a.bdt = p->bias_dtype;
  a.idt = p->ids_dtype;
  a.wdt = p->weights_dtype;
  a.T = (int)p->n_tokens;
  a.E = (int)p->n_experts;
  a.k = (int)p->top_k;
  a.G = (int)p->n_groups;
  a.gs = a.E / a.G;
  a.top_groups = (int)p->topk_group;
  a.sigmoid = p->scoring == EXQ_SCORE_SIGMOID;
  a.top2 = p->group_score == EXQ_GROUP_TOP2;
  a.renorm = p->renormalize != 0;
  a.scale = p->scale;
  const dim3 g((unsigned)cdiv(a.T, 4));
  const hipStream_t s = as_stream(stream);
  if (a.E <= 256)
    hipLaunchKernelGGL(route_rows_kernel<4>, g, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(route_rows_kernel<16>, g, dim3(256), 0, s, a);
  return check_launch("route_rows_kernel");
}
