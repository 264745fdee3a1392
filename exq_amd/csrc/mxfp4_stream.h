// mxfp4_stream.h -- the MoE projections of a few slots: streams of weights.
#pragma once

#include "mxfp4_tile.h"

namespace exq {
namespace mx {

// ---- a few slots: gate and up by slots -------------------------------------------------------
// Every slot is a group of its own, so nothing has to be routed; experts that two tokens share
// are read twice, from the caches.  A unit is a slot x a gate tile and the up tile of the same
// columns; the four waves of a work-group share its contraction and add their sums through LDS
// in wave order.  A dropped slot reads the first expert's weights and is not stored.  Bound:
// latency, the ids' and then the weights' (1 x 8 of 2048 x 768 6.3 us, the down kernel 7.1).
constexpr int kSlotWaves = 4;

// Whether a layer of n slots runs by slots, with the down projection below, or routes and runs
// on tiles.  Slots save the routing and a launch, tiles keep more of the weights on their way.
// us a layer by slots and on tiles, weights not in the caches:
//   1024 x 512   8 slots 11.2 and 16.7, 16 14.4 and 17.6, 24 18.3 and 19.3, 32 21.9 and 20.5
//   2048 x 768   8 15.3 and 21.2, 16 20.5 and 23.9, 24 26.7 and 28.8, 32 31.4 and 30.8
//   2048 x 2048  4 17.6 and 23.5, 8 25.3 and 26.0, 12 32.7 and 31.3, 16 40.4 and 33.9
//   4096 x 1024  4 17.2 and 27.1, 8 21.5 and 28.6, 12 26.1 and 31.1, 16 33.2 and 33.3
//   8192 x 1024  4 27.2 and 37.7, 8 36.0 and 41.2, 16 58.7 and 50.7
//   4096 x 4096  2 25.0 and 37.6, 4 33.5 and 40.1, 8 54.5 and 52.6, 16 94.8 and 85.0
//   6144 x 2048  2 28.1 and 35.0, 4 32.5 and 36.3, 8 52.4 and 43.7, 16 88.1 and 64.2
//   4096 x 14336 2 67 and 83, 4 91 and 96, 8 162 and 143, 16 301 and 190
//   8192 x 8192  1 59 and 84, 2 76 and 81, 3 90 and 84, 4 105 and 92, 8 188 and 157
// So up to four slots, and up to 16 where all their experts' values are few.
constexpr int kSlotSlots = 16;
constexpr int kSlotAlways = 4;
constexpr int64_t kSlotValues = (int64_t)3 << 24;     // slots x hidden x intermediate size
inline bool runs_by_slot(int64_t slots, int64_t H, int64_t I) {
  return slots <= kSlotAlways || (slots <= kSlotSlots && slots * H * I <= kSlotValues);
}

struct SlotArgs {
  const void* ids;           // [n]
  int ids_dtype, E, top_k;
  const uint16_t* x;         // hidden [T, K]
  const uint4* tiles;        // [E, RT, KB]
  const uint8_t* wscales;    // [E, RT, G] of 256 bytes
  int K, KB, G, RT, I;
  uint16_t* mid;             // [n, I]
};

template <bool BF>
__global__ void __launch_bounds__(64 * kSlotWaves) moe_slot_gateup_kernel(SlotArgs a) {
  constexpr int W = kSlotWaves, C = 4;             // tiles along the columns in flight
  __shared__ __align__(16) float4 red[W * 2 * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int pair = blockIdx.x, slot = blockIdx.y, blocks = a.K / kBlock;
  const int64_t id = load_index(a.ids, a.ids_dtype, slot);
  const bool there = id >= 0 && id < a.E;
  const int e = __builtin_amdgcn_readfirstlane(there ? (int)id : 0);
  const uint16_t* x = a.x + (int64_t)(slot / a.top_k) * a.K;
  const int kb0 = wave * a.KB / W, kb1 = (wave + 1) * a.KB / W;
  f32x4_t acc[2] = {};
  for (int k0 = kb0; k0 < kb1; k0 += C) {
    uint4 w[C][2], xv[C][4];
    uint32_t s[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int kb = k0 + c < kb1 ? k0 + c : kb1 - 1;   // (past the range: loaded again, not used)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t rt = (int64_t)e * a.RT + pair * 2 + t;
        w[c][t] = a.tiles[(rt * a.KB + kb) * 64 + lane];
        s[c][t] = a.wscales[((rt * a.G + (kb >> 2)) * 64 + lane) * 4 + (kb & 3)];
      }
      const int b = kb * 4 + q < blocks ? kb * 4 + q : blocks - 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) xv[c][j] = *reinterpret_cast<const uint4*>(x + b * 32 + j * 8);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (k0 + c >= kb1) break;
      const bool in = (k0 + c) * 4 + q < blocks;        // (columns past K: zeros)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = in ? xv[c][j] : uint4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int t = 0; t < 2; ++t)
          acc[t] = dev::dmfma<BF>(decode8<BF>(j == 0   ? w[c][t].x
                                              : j == 1 ? w[c][t].y
                                              : j == 2 ? w[c][t].z
                                                       : w[c][t].w,
                                              __uint_as_float(s[c][t] << 23)),
                                  v, acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
    red[(wave * 2 + t) * 64 + lane] = float4{acc[t][0], acc[t][1], acc[t][2], acc[t][3]};
  __syncthreads();
  if (wave || r16 || !there) return;   // (all columns of the matrix instruction are the token)
  float4 v[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    v[t] = red[t * 64 + lane];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      const float4 p = red[(k * 2 + t) * 64 + lane];
      v[t].x += p.x; v[t].y += p.y; v[t].z += p.z; v[t].w += p.w;
    }
  }
  // (rounded to the activations' type: the next product's operand)
  *reinterpret_cast<uint2*>(a.mid + (int64_t)slot * a.I + pair * 16 + q * 4) =
      uint2{pack16(silu_f32(v[0].x) * v[1].x, silu_f32(v[0].y) * v[1].y, BF),
            pack16(silu_f32(v[0].z) * v[1].z, silu_f32(v[0].w) * v[1].w, BF)};
}

// ---- a few slots: the down projection by output columns ------------------------------------
// A work-group owns 16 output columns and takes every slot: wave w the slots w, w + 8, ...,
// whose results it weighs into LDS, a row a slot; then a token's k rows are added in the order
// of its slots.  No partial rows in memory and no launch to add them.  The rows of mid are few
// and come straight from memory.
constexpr int kOwnedWaves = 8;

struct OwnedArgs {
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
  __shared__ __align__(16) float rows[kSlotSlots * 16];
  __shared__ float wts[kSlotSlots];
  __shared__ int experts[kSlotSlots];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, q = lane >> 4, n = a.T * a.k, blocks = a.I / kBlock;
  if (tid < n) {   // (a dropped slot's weight is not looked at)
    const int64_t e = load_index(a.ids, a.ids_dtype, tid);
    const bool there = e >= 0 && e < a.E;
    wts[tid] = there ? load_as_f32(a.weights, a.w_dtype, tid) : 0.f;
    experts[tid] = there ? (int)e : -1;
  }
  for (int i = tid; i < n * 16; i += 64 * W) rows[i] = 0.f;
  __syncthreads();
  const int chunks = (a.KB + C - 1) / C;
  const int items = n > wave ? ((n - wave + W - 1) / W) * chunks : 0;
  uint4 w[2][C], x[2][C][4];
  uint32_t s[2][C];
  int slot[2], li = 0;       // slot: the lane's row of the result, -1: none
  auto load = [&](int p) {
    const int i = li < items ? li : items - 1, gi = i / chunks, ch = i - gi * chunks;
    const int at = wave + gi * W, e = experts[at];
    slot[p] = r16 == 0 && e >= 0 ? at : -1;
    const int er = __builtin_amdgcn_readfirstlane(e < 0 ? 0 : e);
    const uint16_t* xr = a.mid + (int64_t)at * a.I;
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
