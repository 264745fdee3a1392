// mxfp4_tile.h -- the products of many tokens with MXFP4 weights: what the dense and the
// MoE kernels share.
//
// A work-group of WM x WN waves makes 16 MT WM tokens x 16 NT WN weight rows, a wave 16 MT
// x 16 NT of them.  Tokens go through LDS, copied straight into one of its stages while
// another is multiplied; the waves meet once a stage.  Weights never do: a wave loads its
// tiles of the stages ahead into registers, whole lines, so LDS holds and serves one operand
// only, and a decoded weight serves MT products.  Three work-groups a CU: 64 tokens x 256
// rows reach what the library's bf16 product reaches (4096 x 4096 x 28672 1,355 TFLOP/s, the
// library's 8192^3 1,390 on that card), two of 128 x 256 1,230, one of 256 x 256 1,044.
//
// LDS rows: a 16-bit stage is 128 columns, 256 bytes a row, sixteen 16-byte pieces; lane
// (r, q) reads piece 4 q + j of its row for step j.  A ds_read_b128 is served 16 lanes at a
// time (equal bit 5 and equal parity of bits 2..4 of the lane id), 256 bytes a cycle:
// with piece c of row r at place c ^ fold(r) those 16 lanes lie in 16 different units.
#pragma once

#include "lds_copy.h"
#include "linear_epilogue.h"
#include "mxfp4.h"

namespace exq {
namespace mx {

using namespace lin;

__device__ __forceinline__ int fold(int r) { return (r & 7) | ((r & 4) << 1); }

// Buffer resource from a pointer that is the same in every lane (the compiler may hold it
// in vector registers).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_rsrc(const void* p) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)p >> 32));
  return make_rsrc(reinterpret_cast<const uint16_t*>((uintptr_t)hi << 32 | lo));
}

// Use of loaded values without an instruction.
__device__ __forceinline__ void keep(const uint4& v, uint32_t s) {
  asm volatile("" ::"v"(v.x), "v"(v.y), "v"(v.z), "v"(v.w), "v"(s));
}

// Tokens of a work-group in 16 bits.  vo[j]: byte offset from xr's base of piece
// `piece` of the row that the lane copies in copy j (kOob: none); a copy is four rows.
// P >= 3 stages: P - 1 are on their way while one is multiplied.
template <bool BF, int WM, int WN, int MT, int NT, int P>
struct Tile16 {
  static constexpr int W = WM * WN;
  static constexpr int BM = 16 * MT * WM, BR = 16 * NT * WN;   // tokens, weight rows
  static constexpr int STAGE = BM * 256;
  static constexpr int D = BM / 4 / W;                         // copies of a wave and stage
  static constexpr int LDS = P * STAGE;
  static constexpr int AHEAD = D + 2 * NT;                     // a wave's loads of a stage
  static_assert(BM % (4 * W) == 0 && W % 4 == 0 && LDS <= 160 * 1024, "copies");
  static_assert(P >= 3 && (P - 1) * AHEAD < 64, "loads in flight");

  // Row of the work-group that the lane copies in copy j, and the piece of it.
  __device__ __forceinline__ static int row(int wave, int lane, int j) {
    return (j * W + wave) * 4 + (lane >> 4);
  }
  __device__ __forceinline__ static int piece(int wave, int lane) {
    return (lane & 15) ^ fold((wave * 4 + (lane >> 4)) & 15);
  }

  // rt[t]: the wave's weight tiles' rows of tiles.  wave: uniform.
  __device__ __forceinline__ static void run(unsigned char* lds, __amdgpu_buffer_rsrc_t xr,
                                             const int (&vo)[D], const uint4* tiles,
                                             const uint32_t* scales, const int (&rt)[NT], int KB,
                                             int G, int pieces, int wave, int lane,
                                             f32x4_t (&acc)[MT][NT]) {
    const int r16 = lane & 15, q = lane >> 4, wm = wave / WN;
    const int pc = piece(wave, lane);
    const uint32_t lds0 = lds_offset(lds) + wave * 1024;
    const int rd = (wm * MT * 16 + r16) * 256, fr = fold(r16);
    auto copy = [&](int kb, uint32_t at) {
      const bool in = kb * 16 + pc < pieces;   // (columns past K are zeros)
#pragma unroll
      for (int j = 0; j < D; ++j)
        dma16(xr, at + j * W * 1024, in ? vo[j] : kOob, kb < KB ? kb * 256 : 0);
    };
    auto load = [&](int kb, uint4 (&w)[NT], uint32_t (&s)[NT]) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[t] = tiles[((int64_t)rt[t] * KB + kb) * 64 + lane];
        s[t] = scales[((int64_t)rt[t] * G + (kb >> 2)) * 64 + lane];
      }
    };
    auto multiply = [&](const unsigned char* at, const uint4 (&w)[NT], const uint32_t (&s)[NT]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 x[MT], d[NT];
#pragma unroll
        for (int u = 0; u < MT; ++u)
          x[u] = *reinterpret_cast<const uint4*>(at + u * 4096 + (((4 * q + j) ^ fr) * 16));
#pragma unroll
        for (int t = 0; t < NT; ++t)
          d[t] = decode8<BF>(j == 0 ? w[t].x : j == 1 ? w[t].y : j == 2 ? w[t].z : w[t].w,
                             __uint_as_float(s[t]));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < MT; ++u) acc[u][t] = dev::dmfma<BF>(d[t], x[u], acc[u][t]);
        if (j == 1) __builtin_amdgcn_sched_barrier(0);  // (or more operands than registers)
      }
    };
    auto scale = [](uint32_t four, int kb) { return (four >> (8 * (kb & 3)) & 0xffu) << 23; };
    uint4 w[P][NT];
    uint32_t s[P][NT];
    // stage kb into place p; past the last one zeros, and its weights once more
    auto fetch = [&](int kb, int p) {
      copy(kb, lds0 + p * STAGE);
      load(kb < KB ? kb : KB - 1, w[p], s[p]);
    };
#pragma unroll
    for (int p = 0; p < P - 1; ++p) fetch(p, p);
    for (int k0 = 0; k0 < KB; k0 += P) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int kb = k0 + p;
        if (p > 0 && kb >= KB) break;
        wait_lds();   // (what the stage before read has arrived: its place is written next)
        wait_vm<(P - 2) * AHEAD>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        uint32_t sc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t] = scale(s[p][t], kb);
        fetch(kb + P - 1, (p + P - 1) % P);   // (over the stage that all have just left)
        multiply(lds + p * STAGE + rd, w[p], sc);
      }
    }
    // (the waits above count every load: none may be dropped because no stage uses it)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int t = 0; t < NT; ++t) keep(w[p][t], s[p][t]);
    wait_vm<0>();
    __syncthreads();
  }
};

// The same with tokens in MXFP4: a stage is 256 columns, 128 bytes a row, eight pieces,
// piece c of row r at place c ^ swz8(r); a copy is eight rows.  Both operands go to the
// matrix instructions as they are.  A token's eight scale bytes of a stage are one load of
// one lane, a stage ahead, and lie behind the rows in LDS: straight from memory they were
// 2 MT one-byte loads of every wave, 16 lines each, which took longer than the products.
__device__ __forceinline__ int swz8(int r) { return (r >> 1) & 7; }
struct __attribute__((packed, aligned(1))) Bytes8 {
  uint32_t d[2];
};

template <int WM, int WN, int MT, int NT>
struct Tile4 {
  static constexpr int W = WM * WN;
  static constexpr int BM = 16 * MT * WM, BR = 16 * NT * WN;
  static constexpr int ROWS = BM * 128, STAGE = ROWS + BM * 8;
  static constexpr int D = BM / 8 / W;
  static constexpr int LDS = 2 * STAGE;
  static_assert(BM % (8 * W) == 0 && W % 2 == 0 && BM <= 64 * W && LDS <= 160 * 1024, "copies");

  __device__ __forceinline__ static int row(int wave, int lane, int j) {
    return (j * W + wave) * 8 + (lane >> 3);
  }
  __device__ __forceinline__ static int piece(int wave, int lane) {
    return (lane & 7) ^ swz8((wave * 8 + (lane >> 3)) & 15);
  }

  // xs: the scale bytes of token 64 wave + lane of the work-group, `blocks` of them.
  __device__ __forceinline__ static void run(unsigned char* lds, __amdgpu_buffer_rsrc_t xr,
                                             const int (&vo)[D], const uint8_t* xs,
                                             const uint4* tiles, const uint32_t* scales,
                                             const int (&rt)[NT], int KB, int G, int blocks,
                                             int wave, int lane, f32x4_t (&acc)[MT][NT]) {
    const int r16 = lane & 15, q = lane >> 4, wm = wave / WN, tid = wave * 64 + lane;
    const int pc = piece(wave, lane);
    const uint32_t lds0 = lds_offset(lds) + wave * 1024;
    uint4 w[2][NT];
    uint32_t s[2][NT];
    uint2 b = uint2{0u, 0u};
    // the tokens of stage kk and their scales
    auto copy = [&](int kk) {
      const uint32_t at = lds0 + (kk & 1) * STAGE;
      const bool in = kk * 8 + pc < blocks;
#pragma unroll
      for (int j = 0; j < D; ++j) dma16(xr, at + j * W * 1024, in ? vo[j] : kOob, kk * 128);
      if (tid < BM) {
        if (kk * 8 + 8 <= blocks) {
          const Bytes8 v = *reinterpret_cast<const Bytes8*>(xs + kk * 8);
          b = uint2{v.d[0], v.d[1]};
        } else {
          b = uint2{0u, 0u};
          for (int i = 0; kk * 8 + i < blocks; ++i) {
            const uint32_t v = (uint32_t)xs[kk * 8 + i] << (8 * (i & 3));
            if (i < 4) b.x |= v; else b.y |= v;
          }
        }
      }
    };
    // the weights of its half h (columns past K: x is zero)
    auto load = [&](int kk, int h) {
      const int kb = 2 * kk + h < KB ? 2 * kk + h : KB - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[h][t] = tiles[((int64_t)rt[t] * KB + kb) * 64 + lane];
        s[h][t] = scales[((int64_t)rt[t] * G + (kb >> 2)) * 64 + lane];
      }
    };
    copy(0);
    load(0, 0);
    load(0, 1);
    const int m0 = wm * MT * 16 + r16, fr = swz8(r16);
    const int KK = (KB + 1) >> 1;
    for (int kk = 0; kk < KK; ++kk) {
      unsigned char* stage = lds + (kk & 1) * STAGE;
      wait_vm<4 * NT>();   // all but the weights, whose registers the compiler waits for
      if (tid < BM) *reinterpret_cast<uint2*>(stage + ROWS + tid * 8) = b;
      wait_lds();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (kk + 1 < KK) copy(kk + 1);
      const unsigned char* at = stage + m0 * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 x[MT];
        int sx[MT];
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          x[u] = *reinterpret_cast<const uint4*>(at + u * 2048 + (((4 * h + q) ^ fr) * 16));
          sx[u] = stage[ROWS + (m0 + u * 16) * 8 + h * 4 + q];
        }
        const int shift = 8 * ((2 * kk + h) & 3);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int sw = (int)(s[h][t] >> shift);
#pragma unroll
          for (int u = 0; u < MT; ++u) acc[u][t] = mfma_mx(w[h][t], sw, x[u], sx[u], acc[u][t]);
        }
        __builtin_amdgcn_sched_barrier(0);  // (or more operands than registers)
        load(kk + 1, h);   // (past the last stage: its last columns once more, not used)
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t) keep(w[h][t], s[h][t]);   // (the waits above count every load)
    wait_vm<0>();
    __syncthreads();
  }
};

// A wave's sums through LDS of its own, 16 tokens at a time: a row of 16 NT + 4 floats a
// token, eight consecutive columns a lane, so that what emit(m, c, y, up) reads and writes
// for columns c .. c + 7 of the wave's token m are runs of 16 or 32 bytes in whole lines.
// Gated: the tiles are gate (y) and up in turn.
template <int NT>
constexpr int wave_floats() { return 16 * (16 * NT + 4); }
template <bool GATED, int MT, int NT, typename Emit>
__device__ __forceinline__ void emit_tiles(float* sums, const f32x4_t (&acc)[MT][NT], int lane,
                                           Emit emit) {
  constexpr int P = 16 * NT + 4;
  constexpr int LPR = (GATED ? 1 : 2) * NT;       // lanes of a token
  constexpr int IT = (16 * LPR + 63) / 64;        // runs of a lane
  const int r16 = lane & 15, q = lane >> 4;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      *reinterpret_cast<float4*>(sums + r16 * P + t * 16 + q * 4) =
          float4{acc[u][t][0], acc[u][t][1], acc[u][t][2], acc[u][t][3]};
    __builtin_amdgcn_sched_barrier(0);  // (a few sums at a time leave the accumulators)
    wave_sync();
#pragma unroll 1
    for (int i = 0; i < IT; ++i) {
      const int at = i * 64 + lane, m = at / LPR, c = at % LPR;
      if (16 * LPR < 64 && m >= 16) break;
      const float* p = sums + m * P + (GATED ? (c >> 1) * 32 + (c & 1) * 8 : c * 8);
      float y[8], up[8];
      *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(p);
      *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(p + 4);
      if (GATED) {
        *reinterpret_cast<float4*>(up) = *reinterpret_cast<const float4*>(p + 16);
        *reinterpret_cast<float4*>(up + 4) = *reinterpret_cast<const float4*>(p + 20);
      }
      emit(u * 16 + m, c * 8, y, up);
    }
    wave_sync();
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace mx
}  // namespace exq
