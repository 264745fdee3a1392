// mxfp4_stream.h -- the MoE projections of few rows per expert: streams of weights.
//
// A unit is a token group (up to 16 MT rows of one expert) x two tiles of weight rows (a
// gate and the up tile of the same columns, or 32 output columns).  One resident round of
// work-groups takes the units in contiguous runs, so a run stays with an expert and its
// tokens mostly.  The four waves of a work-group split the contraction: each holds its
// columns of the group's tokens in LDS of its own, so no wave waits for another before the
// partial sums are joined, and streams its weight tiles through registers, two items (of C
// tiles along the columns each) ahead of the multiplication, also past the end of a unit.
// Bound: HBM.
#pragma once

#include "mxfp4_tile.h"

namespace exq {
namespace mx {

constexpr int kStreamWaves = 4;
constexpr int kStreamGroups = 16;    // token groups that a work-group's run of units touches

struct StreamArgs {
  int* hdr;                  // plan: [0] token groups
  TgEntry* tg;
  int* sorted;               // expert-sorted position -> slot
  const void* ids;           // [n] (routing in the kernel)
  int ids_dtype, n, E;
  const uint16_t* x;         // gate/up: hidden [T, H]; down: mid [n, I]
  const uint4* tiles;        // [E, RT, KB]
  const uint8_t* wscales;    // [E, RT, G] of 256 bytes
  int K, KB, G, RT, top_k, N, n_rt, chunks;
  uint16_t* mid;             // [n, I]
  float* part;               // [slots, H]
};

constexpr int kBySlot = -1;

// The work-group's run of units and the token groups that it touches.
struct Run {
  int u0, u1, g0, gn;
};
__device__ __forceinline__ Run run_of(int n_groups, int n_rt) {
  Run r;
  const int64_t U = (int64_t)n_groups * n_rt;
  r.u0 = (int)(U * blockIdx.x / gridDim.x);
  r.u1 = (int)(U * (blockIdx.x + 1) / gridDim.x);
  r.g0 = r.u0 / n_rt;
  r.gn = r.u1 > r.u0 ? (r.u1 - 1) / n_rt - r.g0 + 1 : 0;
  return r;
}

// Routing by each work-group for itself, n <= 64 NSEG slots: a bit per slot in its expert's
// masks, whose population counts give the experts' rows and a slot's rank among them in
// ascending order, a scan over the experts the places.  The same in every work-group; the
// first one writes the plan down for the next kernel.  The launch in front, 7.5 us at 64
// tokens x 8 of 128 experts, and the wait between the two are saved.
// The plan's groups are of 16 rows.  ALL: the kernel's own are all of an expert's rows, and
// slots holds for each of 16 tokens first its row in the sorted order, then how many rows
// it has (a token that repeats an id has consecutive ones).
template <int NSEG>
struct Route {
  static constexpr int kExperts = NSEG == 2 ? 256 : 4096 / NSEG;   // at most
  static constexpr int kWords = 2 * NSEG * kExperts + kExperts + 4;  // of scratch
  static constexpr int kIds = (64 * NSEG + 255) / 256;

  // rows, groups of 16 rows and experts with rows, counted in one word
  __device__ __forceinline__ static uint32_t counts(int rows) {
    return (uint32_t)rows | (uint32_t)((rows + 15) >> 4) << 12 | (uint32_t)(rows > 0) << 22;
  }
  __device__ __forceinline__ static int row_at(uint32_t c) { return c & 0xfff; }
  __device__ __forceinline__ static int group_at(uint32_t c) { return c >> 12 & 0x3ff; }
  __device__ __forceinline__ static int expert_at(uint32_t c) { return c >> 22; }

  template <bool ALL>
  __device__ __forceinline__ static Run here(const StreamArgs& a, uint32_t* scratch,
                                             TgEntry* entry, int* slots) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t* masks = reinterpret_cast<uint64_t*>(scratch);   // [E][NSEG]
    uint32_t* first = scratch + 2 * NSEG * kExperts;          // [E]: what lies before it
    uint32_t* total = first + kExperts;                       // [4]
    int id[kIds];
#pragma unroll
    for (int c = 0; c < kIds; ++c) {
      const int i = c * 256 + tid;
      id[c] = -1;
      if (i < a.n) {
        const int64_t e = load_index(a.ids, a.ids_dtype, i);
        if (e >= 0 && e < a.E) id[c] = (int)e;
      }
    }
    for (int i = tid; i < a.E * NSEG / 2; i += 256)
      reinterpret_cast<uint4*>(masks)[i] = uint4{0u, 0u, 0u, 0u};
    if (tid == 0) masks[a.E * NSEG - 1] = 0;   // (an odd number of masks)
    if (ALL && tid < kStreamGroups * 16) {
      slots[tid * 2] = 0x7fffffff;
      slots[tid * 2 + 1] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kIds; ++c) {
      const int i = c * 256 + tid;
      if (id[c] >= 0)
        atomicOr(reinterpret_cast<uint32_t*>(masks + id[c] * NSEG + (i >> 6)) + ((i >> 5) & 1),
                 1u << (i & 31));
    }
    __syncthreads();
    const int per = (a.E + 255) >> 8, e0 = tid * per;   // the thread's experts
    constexpr int PER = (kExperts + 255) / 256;
    int cnt[PER];
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      cnt[k] = 0;
      if (k < per && e0 + k < a.E) {
#pragma unroll
        for (int w = 0; w < NSEG; ++w) cnt[k] += __popcll(masks[(e0 + k) * NSEG + w]);
        mine += counts(cnt[k]);
      }
    }
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    if (lane == 63) total[wave] = sum;
    __syncthreads();
    uint32_t at = sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += total[w];
      all += total[w];
    }
    const Run run = run_of(ALL ? expert_at(all) : group_at(all), a.n_rt);
    const bool writer = blockIdx.x == 0;
    if (writer && tid == 0) a.hdr[0] = group_at(all);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (k >= per || e0 + k >= a.E) break;
      first[e0 + k] = at;
      if (ALL && cnt[k] > 0) {
        const int g = expert_at(at) - run.g0;
        if (g >= 0 && g < run.gn) entry[g] = TgEntry{e0 + k, row_at(at), cnt[k], 2};
      }
      if (!ALL || writer) {
        for (int r = 0; r < cnt[k]; r += 16) {
          const TgEntry t{e0 + k, row_at(at) + r, cnt[k] - r < 16 ? cnt[k] - r : 16, 2};
          const int g = group_at(at) + (r >> 4);
          if (writer) a.tg[g] = t;
          if (!ALL && g >= run.g0 && g < run.g0 + run.gn) entry[g - run.g0] = t;
        }
      }
      at += counts(cnt[k]);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kIds; ++c) {
      const int i = c * 256 + tid, e = id[c];
      if (e < 0) continue;
      const uint64_t* m = masks + e * NSEG;
      int rank = __popcll(m[i >> 6] & (((uint64_t)1 << (i & 63)) - 1));
#pragma unroll
      for (int w = 0; w < NSEG - 1; ++w)
        if (w < (i >> 6)) rank += __popcll(m[w]);
      const int row = row_at(first[e]) + rank;
      if (writer) a.sorted[row] = i;
      const int g = (ALL ? expert_at(first[e]) : group_at(first[e]) + (rank >> 4)) - run.g0;
      if (g < 0 || g >= run.gn) continue;
      if constexpr (!ALL) {
        slots[g * 16 + (rank & 15)] = i / a.top_k;
      } else {
        int* s = slots + (g * 16 + i / a.top_k) * 2;
        atomicMin(s, row);
        atomicAdd(s + 1, 1);
      }
    }
    __syncthreads();
    return run;
  }
};

// Every slot a group of its own: no routing.  The experts that two tokens share are read
// twice (from the caches), dropped slots read the first expert's weights for nothing.
__device__ __forceinline__ Run slot_groups(const StreamArgs& a, TgEntry* entry, int* slots) {
  const int tid = threadIdx.x;
  const Run run = run_of(a.n, a.n_rt);
  if (tid < run.gn) {
    const int slot = run.g0 + tid;
    const int64_t e = load_index(a.ids, a.ids_dtype, slot);
    const bool there = e >= 0 && e < a.E;
    entry[tid] = TgEntry{there ? (int)e : 0, slot, there ? 1 : 0, 2};
    slots[tid * 16] = slot / a.top_k;
  }
  __syncthreads();
  return run;
}

// The same from the plan in memory; slots: of `tokens` their tokens.
template <int R>
__device__ __forceinline__ Run read_plan(const StreamArgs& a, bool tokens, TgEntry* entry,
                                         int* slots) {
  const int tid = threadIdx.x;
  const Run run = run_of(a.hdr[0], a.n_rt);
  if (tid < run.gn) entry[tid] = a.tg[run.g0 + tid];
  __syncthreads();
  for (int i = tid; i < run.gn * R; i += 256) {
    const TgEntry& e = entry[i / R];
    const int r = i % R;
    if (r < e.cnt) slots[i] = tokens ? a.sorted[e.pos0 + r] / a.top_k : a.sorted[e.pos0 + r];
  }
  __syncthreads();
  return run;
}

// NSEG > 0: the kernel routes (gate/up); kBySlot: it need not.  ALL: up to 16 tokens, whose rows are all in LDS
// before the routing is known and stay there: a column of the matrix instruction is a
// token, and the columns of tokens that an expert was not chosen for are not stored.
// KS waves share a unit's contraction, 4 / KS sets of them take tile pairs side by side.
template <bool BF, bool GATEUP, int NSEG, bool ALL, int KS, int C>
__global__ void __launch_bounds__(256, 2) moe_stream_kernel(StreamArgs a) {
  constexpr int NT = 2, R = 16, W = kStreamWaves, L = C * NT, SETS = W / KS;
  constexpr int XW = C * R * 256;   // bytes of a wave's tokens
  __shared__ __align__(1024) unsigned char lds[W * XW];
  __shared__ __align__(16) float4 red[W * NT * 64];
  __shared__ TgEntry entry[kStreamGroups];
  __shared__ int slots[kStreamGroups * R * (ALL ? 2 : 1)];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4, part = wave % KS, set = wave / KS;
  const int kb0 = part * a.KB / KS, kb1 = (part + 1) * a.KB / KS;   // the wave's columns
  unsigned char* xl = lds + wave * XW;
  const uint32_t xl0 = lds_offset(xl);
  const __amdgpu_buffer_rsrc_t xr = uniform_rsrc(a.x);
  const int pieces = a.K >> 3;
  // rows of x, columns of chunk ch: a copy is four rows x 256 bytes
  auto copy_rows = [&](int cnt, int ch, auto row_of) {
    for (int r0 = 0; r0 < cnt; r0 += 4) {
      const int r = r0 + (lane >> 4);
      const int pc = (lane & 15) ^ fold(r & 15);
      const uint32_t row = r < cnt ? (uint32_t)row_of(r) : 0u;
      const uint32_t off = row * (uint32_t)(a.K * 2) + (uint32_t)pc * 16;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int kb = kb0 + ch * C + c;
        if (kb < kb1)
          dma16(xr, xl0 + (c * R + r0) * 256,
                r < cnt && kb * 16 + pc < pieces ? (int)off : kOob, kb * 256);
      }
    }
  };
  if constexpr (ALL) copy_rows(a.n / a.top_k, 0, [](int r) { return r; });
  Run run;
  if constexpr (NSEG > 0) {
    using RT = Route<NSEG>;
    uint32_t* scratch = reinterpret_cast<uint32_t*>(ALL ? reinterpret_cast<unsigned char*>(red) : lds);
    static_assert((ALL ? sizeof(red) : sizeof(lds)) >= RT::kWords * 4, "routing scratch");
    run = RT::template here<ALL>(a, scratch, entry, slots);
  } else if constexpr (NSEG == kBySlot) {
    run = slot_groups(a, entry, slots);
  } else {
    run = read_plan<R>(a, GATEUP, entry, slots);
  }
  const int u0 = run.u0, u1 = run.u1, g0 = run.g0;
  if (u0 >= u1) {
    wait_vm<0>();   // (copies into LDS that is given back)
    return;
  }
  const int items = (u1 - u0) * a.chunks;
  uint4 w[2][L];
  uint32_t s[2][L];
  // where the loads are: group (of the run), tile pairs, chunk
  int lg = 0, lrt = u0 - g0 * a.n_rt, lch = 0, li = 0;
  auto load = [&](uint4 (&wb)[L], uint32_t (&sb)[L]) {
    const int e = __builtin_amdgcn_readfirstlane(entry[lg].e);
    int t0 = (lrt * SETS + set) * NT;
    t0 = t0 < a.RT ? t0 : a.RT - NT;           // (past the last tiles: not stored)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      int kb = kb0 + lch * C + c;
      kb = kb < kb1 ? kb : kb1 - 1;            // (past the range: loaded again, not used)
      kb = kb < 0 ? 0 : kb;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t rt = (int64_t)e * a.RT + t0 + t;
        wb[c * NT + t] = a.tiles[(rt * a.KB + kb) * 64 + lane];
        sb[c * NT + t] = a.wscales[((rt * a.G + (kb >> 2)) * 64 + lane) * 4 + (kb & 3)];
      }
    }
    if (++li < items) {
      if (++lch == a.chunks) {
        lch = 0;
        if (++lrt == a.n_rt) {
          lrt = 0;
          ++lg;
        }
      }
    }
  };
  auto stage = [&](int g, int ch) {
    const int cnt = __builtin_amdgcn_readfirstlane(entry[g].cnt);
    const int pos0 = __builtin_amdgcn_readfirstlane(entry[g].pos0);
    wait_lds();   // (the rows before have been read)
    copy_rows(cnt, ch, [&](int r) { return GATEUP ? slots[g * R + r] : pos0 + r; });
  };
  // the first tokens go before the first weights and are waited for alone
  if constexpr (!ALL) stage(0, 0);
  load(w[0], s[0]);
  load(w[1], s[1]);
  wait_vm<4 * L>();
  f32x4_t acc[NT] = {};
  int g = 0, rt = u0 - g0 * a.n_rt, ch = 0, staged = 0, staged_ch = 0;
  const int fr = fold(r16);
  auto item = [&](uint4 (&wb)[L], uint32_t (&sb)[L]) {
    if (!ALL && (staged != g || staged_ch != ch)) {
      stage(g, ch);
      wait_vm<0>();
      staged = g;
      staged_ch = ch;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (kb0 + ch * C + c < kb1) {
        const unsigned char* at = xl + c * R * 256 + r16 * 256;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 x = *reinterpret_cast<const uint4*>(at + (((4 * q + j) ^ fr) * 16));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint4& v = wb[c * NT + t];
            acc[t] = dev::dmfma<BF>(decode8<BF>(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w,
                                                __uint_as_float(sb[c * NT + t] << 23)),
                                    x, acc[t]);
          }
        }
      }
    }
    load(wb, sb);
    if (++ch < a.chunks) return;
    ch = 0;
    __syncthreads();   // the sums before have been read
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      red[(wave * NT + t) * 64 + lane] = float4{acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
      acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    // the sums of a set's waves in their order, by the wave whose turn it is
    if ((rt % KS) == part) {
      float4 v[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        v[t] = red[(set * KS * NT + t) * 64 + lane];
#pragma unroll
        for (int k = 1; k < KS; ++k) {
          const float4 p = red[((set * KS + k) * NT + t) * 64 + lane];
          v[t].x += p.x; v[t].y += p.y; v[t].z += p.z; v[t].w += p.w;
        }
      }
      const int pair = rt * SETS + set;
      if constexpr (GATEUP) {   // (rounded to the activations' type: the next product's operand)
        int row = entry[g].pos0 + r16, rows = r16 < entry[g].cnt;
        if constexpr (ALL) {
          row = slots[(g * 16 + r16) * 2];
          rows = slots[(g * 16 + r16) * 2 + 1];
        }
        if (pair * NT < a.RT) {
          const uint2 d = uint2{pack16(silu_f32(v[0].x) * v[1].x, silu_f32(v[0].y) * v[1].y, BF),
                                pack16(silu_f32(v[0].z) * v[1].z, silu_f32(v[0].w) * v[1].w, BF)};
          for (int k = 0; k < rows; ++k)
            *reinterpret_cast<uint2*>(a.mid + (int64_t)(row + k) * a.N + pair * 16 + q * 4) = d;
        }
      } else if (r16 < entry[g].cnt && pair * NT < a.RT) {
        float* p = a.part + (int64_t)slots[g * R + r16] * a.N + pair * 32 + q * 4;
        *reinterpret_cast<float4*>(p) = v[0];
        *reinterpret_cast<float4*>(p + 16) = v[1];
      }
    }
    if (++rt == a.n_rt) {
      rt = 0;
      ++g;
    }
  };
  for (int i = 0; i < items; i += 2) {
    item(w[0], s[0]);
    if (i + 1 < items) item(w[1], s[1]);
  }
}

// ---- few slots: the down projection by output columns --------------------------------------
// A work-group owns 16 output columns and takes every token group: wave w the groups w, w +
// 8, ..., whose results it weighs into LDS, a row a slot; then a token's k rows are added in
// the order of its slots.  No partial rows in memory and no launch to add them.  The rows
// of mid are few and come straight from memory.
constexpr int kOwnedWaves = 8;
constexpr int kOwnedSlots = 64;

struct OwnedArgs {
  const int* hdr;            // null: every slot a group of its own
  const TgEntry* tg;
  const int* sorted;
  const uint16_t* mid;       // [n, I]
  const uint4* tiles;
  const uint8_t* wscales;
  const void* ids;
  const void* weights;
  int ids_dtype, w_dtype, T, k, E, I, H, KB, G, RT;
  uint16_t* out;
};

template <bool BF, int C>
__global__ void __launch_bounds__(64 * kOwnedWaves) moe_owned_down_kernel(OwnedArgs a) {
  constexpr int W = kOwnedWaves;
  __shared__ __align__(16) float rows[kOwnedSlots * 16];
  __shared__ float wts[kOwnedSlots];
  __shared__ int experts[kOwnedSlots];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4, n = a.T * a.k;
  const int n_groups = a.hdr ? a.hdr[0] : n, blocks = a.I / kBlock;
  if (tid < n) {   // (a dropped slot's weight is not looked at)
    const int64_t e = load_index(a.ids, a.ids_dtype, tid);
    const bool there = e >= 0 && e < a.E;
    wts[tid] = there ? load_as_f32(a.weights, a.w_dtype, tid) : 0.f;
    experts[tid] = there ? (int)e : -1;
  }
  for (int i = tid; i < n * 16; i += 64 * W) rows[i] = 0.f;
  __syncthreads();
  const int chunks = (a.KB + C - 1) / C;
  const int items = n_groups > wave ? ((n_groups - wave + W - 1) / W) * chunks : 0;
  uint4 w[2][C], x[2][C][4];
  uint32_t s[2][C];
  int slot[2], li = 0;       // slot: the lane's row of the result, -1: none
  auto load = [&](int p) {
    const int i = li < items ? li : items - 1, gi = i / chunks, ch = i - gi * chunks;
    TgEntry t;
    if (a.hdr) {
      t = a.tg[wave + gi * W];
      slot[p] = r16 < t.cnt ? a.sorted[t.pos0 + r16] : -1;
    } else {
      t.pos0 = wave + gi * W;
      t.e = experts[t.pos0];
      t.cnt = t.e < 0 ? 0 : 1;
      t.e = t.e < 0 ? 0 : t.e;
      slot[p] = r16 < t.cnt ? t.pos0 : -1;
    }
    const int er = __builtin_amdgcn_readfirstlane(t.e);
    const uint16_t* xr = a.mid + (int64_t)(t.pos0 + (r16 < t.cnt ? r16 : 0)) * a.I;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int kb = ch * C + c < a.KB ? ch * C + c : a.KB - 1;
      const int64_t rt = (int64_t)er * a.RT + blockIdx.x;
      w[p][c] = a.tiles[(rt * a.KB + kb) * 64 + lane];
      s[p][c] = a.wscales[((rt * a.G + (kb >> 2)) * 64 + lane) * 4 + (kb & 3)];
      const int b = kb * 4 + q < blocks ? kb * 4 + q : blocks - 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[p][c][j] = *reinterpret_cast<const uint4*>(xr + b * 32 + j * 8);
    }
    ++li;
  };
  f32x4_t acc = {};
  int ch = 0;
  auto item = [&](int p) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int kb = ch * C + c;
      if (kb < a.KB) {
        const bool in = kb * 4 + q < blocks;   // (columns past I: zeros)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4& v = w[p][c];
          const uint4 d = decode8<BF>(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w,
                                      __uint_as_float(s[p][c] << 23));
          acc = dev::dmfma<BF>(d, in ? x[p][c][j] : uint4{0u, 0u, 0u, 0u}, acc);
        }
      }
    }
    if (++ch == chunks) {
      ch = 0;
      if (slot[p] >= 0)
        *reinterpret_cast<float4*>(rows + slot[p] * 16 + q * 4) =
            float4{acc[0], acc[1], acc[2], acc[3]};
      acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    load(p);
  };
  if (items > 0) {
    load(0);
    load(1);
    for (int i = 0; i < items; i += 2) {
      item(0);
      if (i + 1 < items) item(1);
    }
  }
  __syncthreads();
  for (int i = tid; i < a.T * 16; i += 64 * W) {
    const int t = i >> 4, c = i & 15, h = blockIdx.x * 16 + c;
    float sum = 0.f;
    for (int j = 0; j < a.k; ++j) sum += wts[t * a.k + j] * rows[(t * a.k + j) * 16 + c];
    a.out[(int64_t)t * a.H + h] = (uint16_t)dev::to_act_bits<BF>(sum);
  }
}

}  // namespace mx
}  // namespace exq
