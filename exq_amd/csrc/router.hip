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
  int chunk, vec;            // experts of a lane; runs of four may be loaded at once
  int lanes2, chunk2;        // lanes of a kept group, and experts of a lane then
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
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  return wave_reduce<0xffffffffu>(v, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dppd(double v) {  // (-inf in lanes that the step leaves out)
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = dpp<CTRL, ROWS, 0u>((uint32_t)u);
  const uint32_t hi = dpp<CTRL, ROWS, 0xfff00000u>((uint32_t)(u >> 32));
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_max64(double v) {
  v = fmax(v, dppd<0xB1, 0xf>(v));
  v = fmax(v, dppd<0x4E, 0xf>(v));
  v = fmax(v, dppd<0x124, 0xf>(v));
  v = fmax(v, dppd<0x128, 0xf>(v));
  v = fmax(v, dppd<0x142, 0xa>(v));
  v = fmax(v, dppd<0x143, 0xc>(v));
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// LDS that holds floats or candidates first and doubles later: accesses by this type are
// ordered with all others.  Its arrays are declared 16-byte aligned.
typedef double __attribute__((may_alias)) lds_double;

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
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

// Weight of a chosen expert with logit x, not yet divided by the sum of a renormalised
// row: s(x), times e^-U where it will be, U = the largest of the chosen x (sigmoid: at
// most 0), so that scores which all underflow still have their ratio.
__device__ __forceinline__ float choice_weight(const RouteArgs& a, float x, float U, float m,
                                               float S) {
  const float d = a.renorm ? U : a.sigmoid ? 0.f : m;
  float e;
  if (a.sigmoid && x > 0.f) {
    e = expf(-x);
  } else {
    // (with the rounding of the difference, which is up to 2^-18 of a score of 1e-37)
    const double wide = (double)x - (double)d;
    const float near = (float)wide;
    e = expf(near);
    if (near > -120.f) e = fmaf(e, (float)(wide - (double)near), e);
  }
  if (!a.sigmoid) return a.renorm ? e : e / S;
  return x > 0.f ? 1.f / (1.f + e) : e / (1.f + expf(x));
}

// One token, by one wave, ranked in 64 bits: neither an expert nor a group is
// decided by the rounding of a score.  Lane l holds experts l + 64 c; `mem` is E doubles
// of the wave's own LDS.  The loops over c stay rolled where they hold an exponential:
// as the rare part of route_tokens_kernel this runs from a cold instruction cache.
template <int MAXC>
__device__ void route_row(const RouteArgs& a, int64_t row, int lane, lds_double* mem) {
  float b[MAXC];
  float m = -FLT_MAX;
  wave_sync();  // (mem: of the row before, or the keys)
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {  // mem: the logits, -inf where the expert is masked
    const int e = lane + 64 * c;
    b[c] = 0.f;
    if (e < a.E) {
      const float l = load_as_f32(a.logits, a.ldt, row * a.E + e);
      if (a.bias) b[c] = load_as_f32(a.bias, a.bdt, e);
      const float x = l > -INFINITY && b[c] > -INFINITY ? fminf(l, FLT_MAX) : -INFINITY;
      m = fmaxf(m, x);
      mem[e] = x;
    }
  }
  double S = 1.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    S = 0.0;
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) S += exp(mem[e] - (double)m);  // (0 for -inf)
    S = wave_sum64(S);
  }
  auto score = [&](double l) {
    const double e = exp(a.sigmoid ? -l : l - (double)m);
    return a.sigmoid ? 1.0 / (1.0 + e) : e / S;
  };
  if (a.bias) {
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double l = mem[e];
      mem[e] = l > -INFINITY ? score(l) : l;
    }
#pragma unroll
    for (int c = 0; c < MAXC; ++c) {  // (a masked expert's bias may be infinite or NaN)
      const int e = lane + 64 * c;
      if (e < a.E && mem[e] > -INFINITY) mem[e] += (double)b[c];
    }
  }
  wave_sync();

  uint64_t keep = ~0ull;
  if (a.top_groups < a.G) {
    // lane g: the value of group g, and how many groups come before it
    double v1 = -INFINITY, v2 = -INFINITY;
    if (lane < a.G) {
      auto take = [&](double x) {
        v2 = fmax(v2, fmin(v1, x));
        v1 = fmax(v1, x);
      };
      const lds_double* at = mem + lane * a.gs;
      int i = 0;
      for (; i + 4 <= a.gs; i += 4) {  // (four reads in flight)
        const double x0 = at[i], x1 = at[i + 1], x2 = at[i + 2], x3 = at[i + 3];
        take(x0);
        take(x1);
        take(x2);
        take(x3);
      }
      for (; i < a.gs; ++i) take(at[i]);
    }
    if (a.top2 && v1 > -INFINITY) {
      if (!a.bias) {  // the sum is of scores, not of the logits that rank them
#pragma unroll 1
        for (int q = 0; q < 2; ++q) {
          const double t = v1;
          v1 = v2;
          v2 = t > -INFINITY ? score(t) : t;
        }
        // (twice swapped: v1 and v2 are the scores of what they were)
      }
      if (v2 > -INFINITY) v1 += v2;
    }
    int before = 0;
    for (int g = 0; g < a.G; ++g) {
      const double o = __shfl(v1, g, 64);
      before += o > v1 || (o == v1 && g < lane) ? 1 : 0;
    }
    keep = __ballot(lane < a.G && before < a.top_groups);
  }
  double r[MAXC];  // rank values, -inf where an expert is masked, out of the groups or taken
#pragma unroll
  for (int c = 0; c < MAXC; ++c) {
    const int e = lane + 64 * c;
    r[c] = -INFINITY;
    if (e < a.E && (a.top_groups >= a.G || keep >> (e / a.gs) & 1u)) r[c] = mem[e];
  }

  int my_id = -1;
  for (int j = 0; j < a.k; ++j) {
    double bv = -INFINITY;
    int be = 0;
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
      if (r[c] > bv) {  // strict: the lower id keeps a tie
        bv = r[c];
        be = lane + 64 * c;
      }
    const double M = wave_max64(bv);
    if (M == -INFINITY) break;
    const uint64_t at = __ballot(bv == M);
    const int e = __popcll(at) == 1
                      ? __builtin_amdgcn_readlane(
                            be, __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)at) - 1))
                      : (int)wave_min(bv == M ? (uint32_t)be : 0xffffffffu);
#pragma unroll
    for (int c = 0; c < MAXC; ++c)
      if (lane + 64 * c == e) r[c] = -INFINITY;
    if (lane == j) my_id = e;
  }
  const float x =
      my_id >= 0 ? fminf(load_as_f32(a.logits, a.ldt, row * a.E + my_id), FLT_MAX) : -INFINITY;
  float U = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) U = fmaxf(U, __shfl_xor(U, d, 64));
  if (a.sigmoid) U = fminf(U, 0.f);
  float w = my_id >= 0 ? choice_weight(a, x, U, m, (float)S) : 0.f;
  if (a.renorm) {
    float sum = w;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    w = my_id >= 0 ? w / sum : 0.f;
  }
  if (lane < a.k) store_choice(a, row, lane, my_id, w * a.scale);
}

constexpr int kRowsGrid = 1 << 23;  // work-groups in x: 2^32 threads are more than a launch takes
template <int MAXC>
__global__ void __launch_bounds__(256) route_rows_kernel(RouteArgs a) {
  __shared__ double s_mem[4][64 * MAXC];
  const int lane = threadIdx.x & 63;
  const int row = (blockIdx.y * kRowsGrid + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= a.T) return;  // (wave-uniform; the waves never meet)
  if (a.n_valid && row >= *a.n_valid) {
    if (lane < a.k) store_choice(a, row, lane, -1, 0.f);
    return;
  }
  route_row<MAXC>(a, row, lane, s_mem[threadIdx.x >> 6]);
}

// ---- four tokens a wave ------------------------------------------------------------
// A token is a 16-lane row of the wave.  Scores in fp32; what their roundings could
// decide, the wave ranks again in 64 bits (route_row).  In order:
//   the groups, 16 / G lanes each: their values by butterflies over their lanes, each
//     one's rank by counting, row rotations against all others; the keys of the kept
//     groups are dealt out again over all lanes, through LDS;
//   a threshold: the k + 1-th best of the lanes' two best keys, which at least k + 1
//     experts reach, and rarely many more;
//   the experts that reach it, packed into 16 KC slots of LDS, and their ranks by
//     counting again: no round per choice, and no lane is searched twice.
template <int CTRL>
__device__ __forceinline__ float rowf(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ int rowi(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true);
}
// Every lane of an aligned run of N lanes gets the run's reduction: pairs, quads, then
// mirrored halves of lanes that agree within them.
template <int N, typename Op>
__device__ __forceinline__ float row_reduce(float v, Op op) {
  if constexpr (N >= 2) v = op(v, rowf<0xB1>(v));
  if constexpr (N >= 4) v = op(v, rowf<0x4E>(v));
  if constexpr (N >= 8) v = op(v, rowf<0x141>(v));
  if constexpr (N >= 16) v = op(v, rowf<0x140>(v));
  return v;
}
__device__ __forceinline__ float max_op(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float min_op(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float sum_op(float a, float b) { return a + b; }
// f(constant I), ... f(constant N - 1)
template <int I, int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<I + 1, N>(f);
  }
}

struct Candidate {
  float key;
  int id;
};

constexpr float kLog2e = 1.4426950408889634f;

// Four consecutive values of a float-typed array, aligned to their size.
__device__ __forceinline__ float4 load4(const void* p, int dt, int64_t i) {
  if (dt == EXQ_DTYPE_F32)
    return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
  if (dt == EXQ_DTYPE_BF16)
    return float4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                  __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
  return float4{f16_bits_to_f32(u.x & 0xffffu), f16_bits_to_f32(u.x >> 16),
                f16_bits_to_f32(u.y & 0xffffu), f16_bits_to_f32(u.y >> 16)};
}

// n >= 1 consecutive values, all loads on their way before the first is used (the last one
// again from n on): with the type decided at each they waited for one another.
template <int CH>
__device__ __forceinline__ void load_each(const void* p, int dt, int64_t i, int n,
                                          float (&v)[CH]) {
  if (dt == EXQ_DTYPE_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c] = f[c < n ? c : n - 1];
    return;
  }
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
  uint32_t u[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) u[c] = h[c < n ? c : n - 1];
#pragma unroll
  for (int c = 0; c < CH; ++c)
    v[c] = dt == EXQ_DTYPE_BF16 ? __uint_as_float(u[c] << 16) : f16_bits_to_f32(u[c]);
}

// The k best of a row's keys, lane l holding those of experts e0 .. e0 + CH - 1 (-inf:
// none): candidates c[i], every key from V on, with their ranks, slot i * 16 + l of `total`.
template <int CH, int KC>
__device__ __forceinline__ void rank_experts(const float (&key)[CH], int e0, int k, int lane,
                                             Candidate* cand, Candidate (&c)[KC], int (&rank)[KC],
                                             int& total, float& V) {
  const int l16 = lane & 15;
  // V: the largest of the lanes' two best that k + 1 of them reach
  float m1 = -INFINITY, m2 = -INFINITY;
#pragma unroll
  for (int p = 0; p < CH; ++p) {
    m2 = fmaxf(m2, fminf(m1, key[p]));
    m1 = fmaxf(m1, key[p]);
  }
  int c1 = m2 >= m1 ? 2 : 1, c2 = 2;
  unrolled<1, 16>([&](auto j) {
    constexpr int CTRL = 0x120 + decltype(j)::value;  // rotate the row
    const float o1 = rowf<CTRL>(m1), o2 = rowf<CTRL>(m2);
    c1 += (o1 >= m1 ? 1 : 0) + (o2 >= m1 ? 1 : 0);
    c2 += (o1 >= m2 ? 1 : 0) + (o2 >= m2 ? 1 : 0);
  });
  V = row_reduce<16>(c1 > k ? m1 : c2 > k ? m2 : -INFINITY, max_op);
  V = fmaxf(V, -FLT_MAX);  // (an expert that is there has a key above -inf)
  int cnt = 0;
#pragma unroll
  for (int p = 0; p < CH; ++p) cnt += key[p] >= V ? 1 : 0;
  int upto = cnt;  // inclusive prefix over the row (row_shr, zeros shifted in)
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
  upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
  total = __shfl(upto, lane | 15, 64);
  int at = upto - cnt;
#pragma unroll
  for (int p = 0; p < CH; ++p)
    if (key[p] >= V) {
      if (at < 16 * KC) cand[at] = Candidate{key[p], e0 + p};
      ++at;
    }
  wave_sync();
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int slot = i * 16 + l16;
    c[i] = slot < total ? cand[slot] : Candidate{-INFINITY, 4096 + slot};
    rank[i] = 0;
  }
  auto first_of = [](float ok, int oid, const Candidate& x) {
    return ok > x.key || (ok == x.key && oid < x.id) ? 1 : 0;
  };
#pragma unroll
  for (int i = 0; i < KC; ++i)
#pragma unroll
    for (int j = 0; j < KC; ++j)
      if (i != j) rank[i] += first_of(c[j].key, c[j].id, c[i]);
  unrolled<1, 16>([&](auto r) {
    constexpr int CTRL = 0x120 + decltype(r)::value;
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const float ok = rowf<CTRL>(c[j].key);
      const int oid = rowi<CTRL>(c[j].id);
#pragma unroll
      for (int i = 0; i < KC; ++i) rank[i] += first_of(ok, oid, c[i]);
    }
  });
}

// Roundings.  In units of 2^-24: e^x as exp2(x log2 e) is off by 2.5 |x| + 2 of itself,
// and |x| e^-|x| <= 0.37, x s (1 - s) <= 0.23, so a sigmoid s is off by at most 4, and e / S
// by 4 / S beside what S is off by: 58 of itself (a weighted mean of |x| is at most ln 512, 36
// additions), which moves the difference of two scores by 58 of that difference, and that
// is no more than their biases differ by where the rounding could turn their order round.
// Adding the bias rounds once.  A ranking between two values no further apart than this
// is made in 64 bits (`tol`: 9 for sigmoid scores, 10 / S + 64 times the span of the biases
// for softmax, a little over 2 |r| for the rounded sums): among the candidates where it
// is theirs, by route_row otherwise.  A group's sum of two has twice the bound of the scores,
// and the roundings of both addends.  With
// logits as they come and a small bias that is one row in some thousands, but then most
// batches have one, and the wave that does is the last to end: 4,096 tokens 12.7 us with
// route_row alone.
// The largest instances have room for one of the two widths of the second deal (two groups
// always fit half of it).
template <int CH, int G, int KC>
constexpr bool kHalfOnly = CH == 32 && (G == 2 || G == 16) && KC == 2;
template <int CH, int G, int KC>
constexpr bool kFullOnly = CH == 32 && (G == 4 || G == 8) && KC == 2;

template <int CH, int G, int KC, int MAXC>
__global__ void __launch_bounds__(256, 3) route_tokens_kernel(RouteArgs a) {
  constexpr int LG = 16 / G;       // lanes of a group
  constexpr int KEYS = 16 * CH + 4;  // floats of a token's keys in LDS
  __shared__ __align__(16) Candidate s_cand[16][16 * KC + 1];
  __shared__ float s_sorted[16][16 * KC + 1];
  __shared__ __align__(16) float s_key[16][KEYS];  // (route_row: 16 CH doubles a wave)
  static_assert(4 * KEYS * sizeof(float) >= 16 * CH * sizeof(double) && KEYS % 4 == 0, "s_key");
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int tok = threadIdx.x >> 4;   // token of the work-group
  const int row0 = blockIdx.x * 16 + (threadIdx.x >> 6) * 4;  // first row of the wave
  if (row0 >= a.T) return;            // (wave-uniform; the waves never meet)
  const int row = blockIdx.x * 16 + tok;
  const int64_t rr = row < a.T ? row : a.T - 1;
  const int g = l16 / LG, sub = l16 % LG;
  const int chunk = a.chunk, first = sub * chunk;
  const int n = first >= a.gs ? 0 : a.gs - first < chunk ? a.gs - first : chunk;
  int e0 = g * a.gs + first;

  float l[CH], key[CH], b[CH];
#pragma unroll
  for (int p = 0; p < CH; ++p) {
    l[p] = -INFINITY;
    b[p] = 0.f;
  }
  if (a.vec) {  // runs of four start at multiples of four, and n is one
#pragma unroll
    for (int p = 0; p < CH; p += 4)
      if (p < n) {
        const float4 v = load4(a.logits, a.ldt, rr * a.E + e0 + p);
        l[p] = v.x; l[p + 1] = v.y; l[p + 2] = v.z; l[p + 3] = v.w;
        if (a.bias) {
          const float4 u = load4(a.bias, a.bdt, e0 + p);
          b[p] = u.x; b[p + 1] = u.y; b[p + 2] = u.z; b[p + 3] = u.w;
        }
      }
  } else {
    if (n > 0) {
      load_each<CH>(a.logits, a.ldt, rr * a.E + e0, n, l);
      if (a.bias) load_each<CH>(a.bias, a.bdt, e0, n, b);
    }
  }
#pragma unroll
  for (int p = 0; p < CH; ++p) {
    const bool there = l[p] > -INFINITY && b[p] > -INFINITY;  // (false for NaN)
    l[p] = p < n && there ? fminf(l[p], FLT_MAX) : -INFINITY;
  }

  // softmax: largest logit and sum, where a score of it is needed
  float m = 0.f, S = 1.f;
  if (!a.sigmoid && (a.bias || !a.renorm || (G > 1 && a.top2))) {
    m = -FLT_MAX;
#pragma unroll
    for (int p = 0; p < CH; ++p) m = fmaxf(m, l[p]);
    m = row_reduce<16>(m, max_op);
    S = 0.f;
#pragma unroll
    for (int p = 0; p < CH; ++p) {
      key[p] = __builtin_amdgcn_exp2f((l[p] - m) * kLog2e);  // (0 where masked)
      S += key[p];
    }
    S = row_reduce<16>(S, sum_op);
  }
  const float rS = __builtin_amdgcn_rcpf(S);
  auto score = [&](float x) __attribute__((always_inline)) {  // (0 for -inf)
    return a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x * kLog2e))
                     : __builtin_amdgcn_exp2f((x - m) * kLog2e) * rS;
  };
  float tol0 = a.sigmoid ? 0x1.2p-21f : 0x1.4p-21f * rS;
  if (a.bias && !a.sigmoid) {
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int p = 0; p < CH; ++p) {
      lo = fminf(lo, l[p] > -INFINITY ? b[p] : INFINITY);
      hi = fmaxf(hi, l[p] > -INFINITY ? b[p] : -INFINITY);
    }
    const float span = row_reduce<16>(hi, max_op) - row_reduce<16>(lo, min_op);
    tol0 += 0x1p-18f * fmaxf(fminf(span, rS), 0.f);
  }
  if (a.bias) {
    if (a.sigmoid) {
#pragma unroll
      for (int p = 0; p < CH; ++p) key[p] = score(l[p]);
    } else {
#pragma unroll
      for (int p = 0; p < CH; ++p) key[p] *= rS;
    }
#pragma unroll
    for (int p = 0; p < CH; ++p) key[p] = l[p] > -INFINITY ? key[p] + b[p] : -INFINITY;
  } else {
#pragma unroll
    for (int p = 0; p < CH; ++p) key[p] = l[p];
  }
  bool unsure = false;
  Candidate c[KC];
  int rank[KC], total;
  float V;

  if constexpr (G > 1) {
    float v1 = -INFINITY, v2 = -INFINITY;
#pragma unroll
    for (int p = 0; p < CH; ++p) {
      v2 = fmaxf(v2, fminf(v1, key[p]));
      v1 = fmaxf(v1, key[p]);
    }
    float v, size;  // a group's value, and the size of what it is the sum of
    if (a.top2) {
      auto merge = [&](float o1, float o2) {
        v2 = fmaxf(fminf(v1, o1), fmaxf(v2, o2));
        v1 = fmaxf(v1, o1);
      };
      if constexpr (LG >= 2) merge(rowf<0xB1>(v1), rowf<0xB1>(v2));
      if constexpr (LG >= 4) merge(rowf<0x4E>(v1), rowf<0x4E>(v2));
      if constexpr (LG >= 8) merge(rowf<0x141>(v1), rowf<0x141>(v2));
      const float s1 = a.bias ? v1 : score(v1), s2 = a.bias ? v2 : score(v2);
      v = v1 > -INFINITY ? s1 + (v2 > -INFINITY ? s2 : 0.f) : -INFINITY;
      size = fabsf(s1) + (v2 > -INFINITY ? fabsf(s2) : 0.f);
    } else {
      v = row_reduce<LG>(v1, max_op);
      size = fabsf(v);
    }
    int before = 0;  // groups that come first
    unrolled<1, G>([&](auto j) {
      constexpr int CTRL = 0x120 + decltype(j)::value * LG;
      const float o = rowf<CTRL>(v);
      const int og = rowi<CTRL>(g);
      before += o > v || (o == v && og < g) ? 1 : 0;
    });
    const bool keep = before < a.top_groups;
    if (a.bias || a.top2) {
      // `err`: how far v may be from its value in 64 bits, by the errors of its scores, the
      // rounding of each addend at the addend's own size (opposed ones have a small sum and
      // large roundings), and those of the sum and of v -+ err
      const float err = tol0 + 0x1.2p-24f * size + 0x1.2p-23f * fabsf(v);
      // (past the largest float, also below: then v may be -inf and the group not empty)
      const bool known = err < INFINITY, empty = !((a.top2 ? v1 : v) > -INFINITY);
      const float least = known ? v - err : -INFINITY;
      const float most = known ? v + err : empty ? -INFINITY : INFINITY;
      const float worst = row_reduce<16>(keep ? least : INFINITY, min_op);
      const float next = row_reduce<16>(keep ? -INFINITY : most, max_op);
      unsure = next > -INFINITY && !(worst > next);
    }
    // the kept groups, again over all lanes: lanes2 lanes for each of them
    float* keys = s_key[tok];
    if (CH <= 16 && a.vec) {
#pragma unroll
      for (int p = 0; p < CH; p += 4)
        if (p < n)
          *reinterpret_cast<float4*>(keys + e0 + p) =
              float4{key[p], key[p + 1], key[p + 2], key[p + 3]};
    } else {
#pragma unroll
      for (int p = 0; p < CH; ++p)
        if (p < n) keys[e0 + p] = key[p];
    }
    uint32_t kept = (uint32_t)(__ballot(keep && sub == 0) >> (lane & 48)) & 0xffffu;
    const int j = l16 / a.lanes2, sub2 = l16 - j * a.lanes2;
    for (int i = 0; i + 1 < a.top_groups; ++i)
      if (i < j) kept &= kept - 1;  // (unused lanes end with none, or with the last)
    const int g2 = kept ? (__ffs((int)kept) - 1) / LG : 0, first2 = sub2 * a.chunk2;
    int n2 = first2 >= a.gs ? 0 : a.gs - first2 < a.chunk2 ? a.gs - first2 : a.chunk2;
    if (j >= a.top_groups) n2 = 0;
    e0 = g2 * a.gs + first2;
    wave_sync();
    auto deal = [&](auto& to, auto size) __attribute__((always_inline)) {
      constexpr int N = decltype(size)::value;
      if (CH <= 16 && a.vec) {
#pragma unroll
        for (int p = 0; p < N; p += 4) {
          const float4 v = p < n2 ? *reinterpret_cast<const float4*>(keys + e0 + p)
                                  : float4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          to[p] = v.x; to[p + 1] = v.y; to[p + 2] = v.z; to[p + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int p = 0; p < N; ++p) to[p] = p < n2 ? keys[e0 + p] : -INFINITY;
      }
      rank_experts<N, KC>(to, e0, a.k, lane, s_cand[tok], c, rank, total, V);
    };
    constexpr int H = CH >= 8 ? CH / 2 : CH;
    if constexpr (kHalfOnly<CH, G, KC>) {
      float half[H];
      deal(half, std::integral_constant<int, H>{});
    } else if (!kFullOnly<CH, G, KC> && CH >= 8 && a.chunk2 <= H) {
      float half[H];
      deal(half, std::integral_constant<int, H>{});
    } else {
      deal(key, std::integral_constant<int, CH>{});
    }
  } else {
    rank_experts<CH, KC>(key, e0, a.k, lane, s_cand[tok], c, rank, total, V);
  }
  unsure |= total > 16 * KC;
  if (a.bias) {  // keys are rounded scores: is one of the first k next to its follower?
    float* sorted = s_sorted[tok];
#pragma unroll
    for (int i = 0; i < KC; ++i) sorted[rank[i]] = c[i].key;
    wave_sync();
    bool close = false;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const float tol = tol0 + 0x1.2p-23f * fabsf(c[i].key);
      if (rank[i] < a.k && rank[i] + 1 < total) close |= !(c[i].key - sorted[rank[i] + 1] > tol);
      // next to what is no candidate: then the row is not these candidates' to decide
      if (rank[i] == a.k - 1 && i * 16 + l16 < total) unsure |= !(c[i].key - V > tol);
    }
    if (const uint64_t some = __ballot(close)) {
      // the candidates again, ranked by their scores in 64 bits
      double r[KC];
      float x[KC];
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        r[i] = -INFINITY;
        x[i] = 0.f;
        if (i * 16 + l16 < total) {
          x[i] = fminf(load_as_f32(a.logits, a.ldt, rr * a.E + c[i].id), FLT_MAX);
          const double e = exp(a.sigmoid ? -(double)x[i] : (double)x[i] - (double)m);
          r[i] = (a.sigmoid ? 1.0 / (1.0 + e) : e / (double)S) +
                 (double)load_as_f32(a.bias, a.bdt, c[i].id);
        }
        rank[i] = 0;
      }
      auto first_of = [](double o, int oid, double x, int id) {
        return o > x || (o == x && oid < id) ? 1 : 0;
      };
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int j = 0; j < KC; ++j)
          if (i != j) rank[i] += first_of(r[j], c[j].id, r[i], c[i].id);
      unrolled<1, 16>([&](auto n) {
        constexpr int CTRL = 0x120 + decltype(n)::value;
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          const uint64_t u = (uint64_t)__double_as_longlong(r[j]);
          const double o = __longlong_as_double(
              (long long)((uint64_t)(uint32_t)rowi<CTRL>((int)(u >> 32)) << 32 |
                          (uint32_t)rowi<CTRL>((int)(uint32_t)u)));
          const int oid = rowi<CTRL>(c[j].id);
#pragma unroll
          for (int i = 0; i < KC; ++i) rank[i] += first_of(o, oid, r[i], c[i].id);
        }
      });
      if (!a.sigmoid) {
        // S has the rounding of 32 bits, 2^-18 of it, which moves the difference of two
        // values by that much of the difference of their scores; the scores of both are
        // within 2^-16 of themselves.  Neighbours that are further apart than this are in
        // order, and with them all; equal logits are in any case.
        static_assert(sizeof(Candidate) == sizeof(double), "a double per slot");
        lds_double* by_rank = reinterpret_cast<lds_double*>(s_cand[tok]);
        wave_sync();  // (the candidates and `sorted` have been read)
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          by_rank[rank[i]] = r[i];
          sorted[rank[i]] = x[i];
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < KC; ++i)
          if (rank[i] + 1 < total && (some >> (lane & 48) & 0xffffu)) {
            const float y = sorted[rank[i] + 1], s0 = score(x[i]), s1 = score(y);
            const double tol = 0x1p-18 * (double)fabsf(s0 - s1) + 0x1p-33 * (double)(s0 + s1) +
                               0x1p-50 * fabs(r[i]) + 0x1p-140;
            unsure |= x[i] != y && !(r[i] - by_rank[rank[i] + 1] > tol);
          }
      }
    }
  }

  // weights of the chosen: rank < k and an expert in the slot
  bool in[KC];
  float x[KC], w[KC], U = -INFINITY;
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    in[i] = rank[i] < a.k && i * 16 + l16 < total;
    x[i] = c[i].key;  // the logit itself, without a bias
    if (a.bias)
      x[i] = in[i] ? fminf(load_as_f32(a.logits, a.ldt, rr * a.E + c[i].id), FLT_MAX) : -INFINITY;
    U = fmaxf(U, in[i] ? x[i] : -INFINITY);
  }
  U = row_reduce<16>(U, max_op);
  if (a.sigmoid) U = fminf(U, 0.f);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    w[i] = choice_weight(a, x[i], U, m, S);
    if (!in[i]) w[i] = 0.f;
    sum += w[i];
  }
  const float total_w = row_reduce<16>(sum, sum_op);
  const bool padding = a.n_valid && row >= *a.n_valid;
  const uint64_t again = __ballot(unsure && row < a.T && !padding);
  if (row < a.T && !(again >> (lane & 48) & 0xffffu)) {
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const bool use = in[i] && !padding;
      const float v = a.renorm ? w[i] / total_w : w[i];
      if (rank[i] < a.k) store_choice(a, row, rank[i], use ? c[i].id : -1, use ? v * a.scale : 0.f);
    }
  }
#pragma unroll 1
  for (int t = 0; t < 4; ++t)
    if (again >> (16 * t) & 0xffffu)  // (the keys of the wave's tokens are not needed any more)
      route_row<MAXC>(a, row0 + t, lane,
                      reinterpret_cast<lds_double*>(s_key[(threadIdx.x >> 6) * 4]));
}

// The fast kernel's sizes: 1, 2, 4, 8 or 16 groups, at most 32 experts a lane and 24
// choices.  The threshold is the k + 1-th of 32 values, so the nearer k is to 32 the more
// experts pass it, and a row with more of them than slots goes to route_row after it has
// been through here: with 512 experts in one group no row at k = 16, 1 to 3 of 100 at
// k = 20 and more than half at k = 24.  us, here / route_rows_kernel, softmax, one group:
//               512 tokens x 256   4,096 x 256    4,096 x 512    16,384 x 256   16,384 x 512
//     k = 16         8.8 /  9.0     8.8 / 14.3    11.2 /  26.2    13.5 / 37.6    24.9 /  85.7
//     k = 20        15.8 /  9.9    22.2 / 16.3    30.6 /  31.0    27.4 / 44.5    44.6 / 101.8
//     k = 22        31.0 / 10.4    37.7 / 18.0    51.7 /  33.9    46.0 / 47.9    73.4 / 109.5
//     k = 24        40.6 / 10.9    41.1 / 18.8    56.3 /  35.6    70.5 / 50.2   123.0 / 115.6
// One token: 8 and 8 to 10.  So past k = 20 this kernel is the slower one for most batches
// between a few tokens and some ten thousand.
template <int CH, int G, int KC>
int launch_tokens(const RouteArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((route_tokens_kernel<CH, G, KC, CH / 4 < 1 ? 1 : CH / 4>),
                     dim3((unsigned)cdiv(a.T, 16)), dim3(256), 0, s, a);
  return check_launch("route_tokens_kernel");
}
int launch_rows(const RouteArgs& a, hipStream_t s) {
  const int64_t n = cdiv(a.T, 4);
  const dim3 g((unsigned)(n < kRowsGrid ? n : kRowsGrid), (unsigned)cdiv(n, kRowsGrid));
  if (a.E <= 256)
    hipLaunchKernelGGL(route_rows_kernel<4>, g, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(route_rows_kernel<16>, g, dim3(256), 0, s, a);
  return check_launch("route_rows_kernel");
}
template <int CH, int G>
int launch_slots(const RouteArgs& a, hipStream_t s) {
  // 16 slots up to k = 10, 32 beyond: 4,096 tokens x 256 softmax, k = 8 6.3 us and 8.7, k = 9
  // 6.4 and 8.7, k = 10 8.7 with 32 and 6.4 or 10.6 with 16, by whether a row has more; one
  // token 5.4 and 7.8.
  if (a.k <= 10) return launch_tokens<CH, G, 1>(a, s);
  if (kHalfOnly<CH, G, 2> && a.chunk2 > CH / 2) return launch_rows(a, s);
  return launch_tokens<CH, G, 2>(a, s);
}
template <int G>
int launch_chunk(RouteArgs a, hipStream_t s) {
  a.chunk = (int)cdiv(a.gs, 16 / G);
  a.lanes2 = 16 / a.top_groups;
  a.chunk2 = (int)cdiv(a.gs, a.lanes2);
  a.vec = 0;
  const int up = (a.chunk + 3) / 4 * 4;
  if (a.gs % 4 == 0 && a.E % 4 == 0 && up <= 32 &&
      (uintptr_t)a.logits % (4 * dtype_bytes(a.ldt)) == 0 &&
      (!a.bias || (uintptr_t)a.bias % (4 * dtype_bytes(a.bdt)) == 0)) {
    a.chunk = up;
    a.chunk2 = (a.chunk2 + 3) / 4 * 4;  // (no more than chunk: a kept group has as many lanes)
    a.vec = 1;
  }
  if (a.chunk <= 4) return launch_slots<4, G>(a, s);
  if (a.chunk <= 8) return launch_slots<8, G>(a, s);
  if (a.chunk <= 16) return launch_slots<16, G>(a, s);
  return launch_slots<32, G>(a, s);
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
  EXQ_REQUIRE(p->n_tokens >= 0 && p->n_tokens < (1 << 26), "%s: n_tokens=%lld out of range",
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
  const hipStream_t s = as_stream(stream);
  if (a.k <= 24) {
    // (with all groups kept they are one; their value is not asked for)
    const int G = a.top_groups == a.G ? 1 : a.G;
    RouteArgs f = a;
    if (G == 1) {
      f.G = f.top_groups = 1;
      f.gs = a.E;
    }
    if (cdiv(f.gs, 16 / (G <= 16 ? G : 16)) <= 32) {
      if (G == 1) return launch_chunk<1>(f, s);
      if (G == 2) return launch_chunk<2>(f, s);
      if (G == 4) return launch_chunk<4>(f, s);
      if (G == 8) return launch_chunk<8>(f, s);
      if (G == 16) return launch_chunk<16>(f, s);
    }
  }
  return launch_rows(a, s);
}
