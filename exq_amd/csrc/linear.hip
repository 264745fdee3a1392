// linear.hip -- dense products with an epilogue on gfx950 MFMA:
//   out = act(x W^T + bias) + residual           W [N, K]
//   out = act(x Wg^T + bg) * (x Wu^T + bu)       W [2N, K], gate rows first
// x [T, K] and W in f16 or bf16, sums in fp32, one rounding to the output's type.
//
// The weight rows are the MFMA's A operand and the tokens its B operand, so a lane
// ends with four consecutive output columns of one token.
#include "exq_internal.h"

namespace exq {
namespace {

struct LinArgs {
  const uint16_t* x;
  const uint16_t* w;
  const void* bias;   // [N] ([2N] gated) or null
  const void* res;    // [T, N] or null
  void* out;
  int64_t ldx, ldw, ldr, ldo;  // elements from row to row
  int64_t T, N, K;             // N: output columns
  int bdt, rdt, odt, act;
  int vec_b, vec_r, vec_o;     // four consecutive elements may be accessed at once
  int odd;                     // rows of x or W may start at an odd 2-byte address
};

template <bool BF>
__device__ __forceinline__ f32x4_t mfma(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

// silu(v) = v / (1 + e^-v); sigmoid(v) = 1 / (1 + e^-v); gelu_tanh(v) = v / (1 + e^-z)
// with z = 2 sqrt(2 / pi) (v + 0.044715 v^3), as (1 + tanh(z / 2)) / 2 = 1 / (1 + e^-z):
// one exponential and one division serve all three.
__device__ __forceinline__ float logistic_act(float v, int act) {
  const float z = act == EXQ_ACT_GELU_TANH
                      ? 1.5957691216057308f * (v + 0.044715f * v * v * v) : v;
  return (act == EXQ_ACT_SIGMOID ? 1.f : v) / (1.f + expf(-z));
}
__device__ __forceinline__ float erf_gelu(float v) {
  return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
}
template <int CNT>
__device__ __forceinline__ void activate_run(float (&v)[CNT], int act) {
  if (act == EXQ_ACT_NONE) return;
  if (act == EXQ_ACT_RELU) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = v[c] < 0.f ? 0.f : v[c];  // (NaN stays)
  } else if (act == EXQ_ACT_GELU) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = erf_gelu(v[c]);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c) v[c] = logistic_act(v[c], act);
  }
}

// ---- aligned rows: copies straight into LDS ----------------------------------
// 16 bytes per lane from buffer `r` at byte offset voff + soff into LDS at
// lds + 16 * lane; `lds` and `soff` are wave-uniform.  A voff past the resource
// writes zeros and reads nothing.  Inline asm (it has no output register), as the
// compiler puts a wait for all copies in flight before the next LDS read after its
// own builtin, which ends the overlap that the stages are for; every copy here is
// waited for by count (wait_vm) and, across waves, by a barrier.  The LDS address is
// an operand in m0, so the compiler knows that m0 changes here.
typedef void __attribute__((address_space(3)))* lptr_t;
__device__ __forceinline__ uint32_t lds_offset(const unsigned char* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)p);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t lds, int voff, int soff) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"{m0}"(lds), "v"(voff),
               "s"(r), "s"(soff)
               : "memory");
#endif
}
// The same for four bytes a lane from anywhere.
__device__ __forceinline__ void touch(const uint16_t* p, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" ::"{m0}"(lds), "v"(p) : "memory");
#endif
}
constexpr int kOob = 0x7ffffff0;          // a voff past every resource
constexpr int64_t kSpan = 0x7fffff00;     // bytes that one resource covers at most
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const uint16_t* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), (short)0, (int)kSpan,
                                           0x00020000);
}
// LDS written by a copy is ordered only by the vmcnt wait, which the compiler does
// not see as a dependency: volatile asm that no memory access moves across.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// LDS rows are 128 bytes (64 k), eight 16-byte columns; column c of row r holds the
// row's chunk c ^ swz(r).  A ds_read_b128 is served 16 lanes at a time (equal bit 5
// and equal parity of bits 2..4 of the lane id), 256 bytes a cycle; with lane
// (r, q) reading chunk 4 s + q of row r those 16 lanes cover all 16 units.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

// Output column, inside a run of 16 * TILES columns, of row i of weight tile t: row
// 4 q + v of a tile is result v of lane quarter q, so with this order a lane's
// results of all tiles are 4 * TILES consecutive columns.
template <int TILES>
__device__ __forceinline__ int run_col(int t, int i) {
  return (i >> 2) * (4 * TILES) + t * 4 + (i & 3);
}

// CNT (a multiple of 4) consecutive values at element i.
template <int CNT>
__device__ __forceinline__ void load_run(const void* p, int dt, int64_t i, float (&v)[CNT]) {
#pragma unroll
  for (int c = 0; c < CNT; c += 4) {
    if (dt == EXQ_DTYPE_F32) {
      const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i + c);
      v[c] = f.x; v[c + 1] = f.y; v[c + 2] = f.z; v[c + 3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i + c);
      const bool bf = dt == EXQ_DTYPE_BF16;
      v[c] = bf ? __uint_as_float(u.x << 16) : f16_bits_to_f32(u.x & 0xffffu);
      v[c + 1] = bf ? __uint_as_float(u.x & 0xffff0000u) : f16_bits_to_f32(u.x >> 16);
      v[c + 2] = bf ? __uint_as_float(u.y << 16) : f16_bits_to_f32(u.y & 0xffffu);
      v[c + 3] = bf ? __uint_as_float(u.y & 0xffff0000u) : f16_bits_to_f32(u.y >> 16);
    }
  }
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf) {
  if (bf) {
    bf16x2_t h;
    h[0] = (__bf16)lo;
    h[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, h);
  }
  f16x2_t h;
  h[0] = (_Float16)lo;
  h[1] = (_Float16)hi;
  return __builtin_bit_cast(uint32_t, h);
}
template <int CNT>
__device__ __forceinline__ void store_run(void* p, int dt, int64_t i, const float (&v)[CNT]) {
  if (dt == EXQ_DTYPE_F32) {
#pragma unroll
    for (int c = 0; c < CNT; c += 4)
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i + c) =
          float4{v[c], v[c + 1], v[c + 2], v[c + 3]};
  } else {
    uint16_t* o = reinterpret_cast<uint16_t*>(p) + i;
    const bool bf = dt == EXQ_DTYPE_BF16;
    uint32_t d[CNT / 2];
#pragma unroll
    for (int c = 0; c < CNT; c += 2) d[c / 2] = pack16(v[c], v[c + 1], bf);
#pragma unroll
    for (int c = 0; c < CNT / 2; c += 2)
      *reinterpret_cast<uint2*>(o + 2 * c) = uint2{d[c], d[c + 1]};
  }
}
// The epilogue of CNT consecutive columns n.. of token m, in two parts, so that the
// residual of several runs can be on its way before the first is used.
template <int CNT>
__device__ __forceinline__ void fetch_residual(const LinArgs& a, int64_t m, int64_t n,
                                               float (&r)[CNT]) {
  if (!a.res || m >= a.T || n >= a.N) return;
  if (n + CNT <= a.N && a.vec_r) {
    load_run<CNT>(a.res, a.rdt, m * a.ldr + n, r);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      r[c] = n + c < a.N ? load_as_f32(a.res, a.rdt, m * a.ldr + n + c) : 0.f;
  }
}
template <int CNT>
__device__ __forceinline__ void add_bias(const LinArgs& a, int64_t n, int64_t off, bool whole,
                                         float (&y)[CNT]) {
  float b[CNT];
  if (whole && a.vec_b) {
    load_run<CNT>(a.bias, a.bdt, off + n, b);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      b[c] = n + c < a.N ? load_as_f32(a.bias, a.bdt, off + n + c) : 0.f;
  }
#pragma unroll
  for (int c = 0; c < CNT; ++c) y[c] += b[c];
}
template <int CNT, bool GATED>
__device__ __forceinline__ void finish_run(const LinArgs& a, int64_t m, int64_t n, float (&y)[CNT],
                                           float (&u)[CNT], const float (&r)[CNT]) {
  if (m >= a.T || n >= a.N) return;
  const bool whole = n + CNT <= a.N;
  if (a.bias) {
    add_bias<CNT>(a, n, 0, whole, y);
    if constexpr (GATED) add_bias<CNT>(a, n, a.N, whole, u);
  }
  activate_run<CNT>(y, a.act);
  if constexpr (GATED) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) y[c] *= u[c];
  } else if (a.res) {
#pragma unroll
    for (int c = 0; c < CNT; ++c) y[c] += r[c];
  }
  if (whole && a.vec_o) {
    store_run<CNT>(a.out, a.odt, m * a.ldo + n, y);
  } else {
#pragma unroll
    for (int c = 0; c < CNT; ++c)
      if (n + c < a.N) store_from_f32(a.out, a.odt, m * a.ldo + n + c, y[c]);
  }
}

// Unit (token block mt of nm, column block nt of nn) of work-group bid: work-group i
// runs on XCD i % 8, and each XCD takes an eighth of the units in a row, the token
// blocks fastest in groups of GM, so that what runs together shares rows of both
// operands in that XCD's L2.  False: none.
template <int GM>
__device__ __forceinline__ bool unit_of(int bid, int nm, int nn, int& mt, int& nt) {
  const int U = nm * nn;
  const int per = (U + 7) >> 3;
  const int local = bid >> 3;
  const int v = (bid & 7) * per + local;
  if (local >= per || v >= U) return false;
  const int g = v / (GM * nn), first = g * GM;
  const int size = nm - first < GM ? nm - first : GM;
  const int rem = v - g * GM * nn;
  nt = rem / size;
  mt = first + rem - nt * size;
  return true;
}

// The sums of W waves over their parts of the contraction, joined through LDS in wave
// order, and their epilogue: 16 MT tokens x 16 NT weight rows.
template <bool GATED, int MT, int NT, int W>
__device__ __forceinline__ void join_waves(const LinArgs& a, float4* red,
                                           const f32x4_t (&acc)[MT][NT], int64_t m0, int64_t n0,
                                           int wave, int lane) {
  constexpr int TILES = GATED ? NT / 2 : NT;
#pragma unroll
  for (int u = 0; u < MT; ++u)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      red[((wave * MT + u) * NT + t) * 64 + lane] =
          float4{acc[u][t][0], acc[u][t][1], acc[u][t][2], acc[u][t][3]};
  __syncthreads();
  for (int u = wave; u < MT; u += W) {
    const int64_t m = m0 + u * 16 + (lane & 15), n = n0 + (lane >> 4) * 4 * TILES;
    float y[4 * TILES], up[4 * TILES], res[4 * TILES];
    if constexpr (!GATED) fetch_residual<4 * TILES>(a, m, n, res);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float4 s = red[(u * NT + t) * 64 + lane];
#pragma unroll
      for (int w = 1; w < W; ++w) {
        const float4 p = red[((w * MT + u) * NT + t) * 64 + lane];
        s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
      }
      float* o = GATED && t >= TILES ? up + (t - TILES) * 4 : y + (t % TILES) * 4;
      o[0] = s.x; o[1] = s.y; o[2] = s.z; o[3] = s.w;
    }
    finish_run<4 * TILES, GATED>(a, m, n, y, up, res);
  }
}

// ---- few tokens: a stream of weights -------------------------------------------
// 16 MT tokens x 16 NT weight rows by W waves that split the contraction: wave w
// takes the 64-k steps w, w + W, ... of all the tile's rows through an LDS ring of
// its own (whole 128-byte lines of each row, NST steps deep), so no wave waits for
// another before the sums are joined through LDS at the end, in wave order.
template <bool BF, bool GATED, int MT, int NT, int W, int NST>
__global__ void __launch_bounds__(64 * W) linear_stream_kernel(LinArgs a, int nm, int nn) {
  constexpr int TILES = GATED ? NT / 2 : NT;   // weight tiles that make output columns
  constexpr int D = 2 * (MT + NT);             // copies of a step
  constexpr int STEP = (MT + NT) * 2048;       // bytes of a step
  constexpr int RED = W * MT * NT * 1024;
  constexpr int LDS = W * NST * STEP > RED ? W * NST * STEP : RED;
  static_assert(LDS <= 160 * 1024 && (NST - 1) * D < 64, "LDS and copies in flight");
  __shared__ __align__(1024) unsigned char lds[LDS];
  int mb, nb;
  if (!unit_of<4>(blockIdx.x, nm, nn, mb, nb)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)mb * MT * 16, n0 = (int64_t)nb * TILES * 16;
  const int K = (int)a.K;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x + m0 * a.ldx);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(a.w + n0 * a.ldw);
  const __amdgpu_buffer_rsrc_t ur = make_rsrc(a.w + (n0 + (GATED ? a.N : 0)) * a.ldw);
  // copy j of a tile fills its rows 8 j .. 8 j + 7
  int vx[MT][2], vw[NT][2], ck[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = j * 8 + (lane >> 3);
    ck[j] = ((lane & 7) ^ swz(i)) * 8;
#pragma unroll
    for (int t = 0; t < MT; ++t)
      vx[t][j] = m0 + t * 16 + i < a.T ? (int)((t * 16 + i) * a.ldx + ck[j]) * 2 : kOob;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c = run_col<TILES>(t % TILES, i);
      vw[t][j] = n0 + c < a.N ? (int)(c * a.ldw + ck[j]) * 2 : kOob;
    }
  }
  const unsigned char* ring = lds + wave * NST * STEP;
  const uint32_t ring0 = lds_offset(ring);
  const int n_it = (K + 64 * W - 1) / (64 * W);
  auto copy = [&](int it) {
    const int k0 = (it * W + wave) * 64;
    const uint32_t at = ring0 + (it % NST) * STEP;
    const bool in[2] = {k0 + ck[0] < K, k0 + ck[1] < K};  // (a step past K copies zeros)
    const int so = k0 < K ? k0 * 2 : 0;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) dma16(xr, at + (t * 2 + j) * 1024, in[j] ? vx[t][j] : kOob, so);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        dma16(GATED && t >= TILES ? ur : wr, at + ((MT + t) * 2 + j) * 1024,
              in[j] ? vw[t][j] : kOob, so);
  };
  f32x4_t acc[MT][NT] = {};
  const int rd = r16 * 128, sw = swz(r16);
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) copy(i);
  for (int it = 0; it < n_it; ++it) {
    wait_lds();  // the step that the next copies overwrite has been read
    copy(it + NST - 1);
    wait_vm<(NST - 1) * D>();
    const unsigned char* at = ring + (it % NST) * STEP + rd;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int col = ((4 * s + q) ^ sw) * 16;
      uint4 b[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) b[t] = *reinterpret_cast<const uint4*>(at + t * 2048 + col);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 w = *reinterpret_cast<const uint4*>(at + (MT + t) * 2048 + col);
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[u][t] = mfma<BF>(w, b[u], acc[u][t]);
      }
    }
  }
  wait_vm<0>();
  __syncthreads();
  join_waves<GATED, MT, NT, W>(a, reinterpret_cast<float4*>(lds), acc, m0, n0, wave, lane);
}

// ---- many tokens: tiles ------------------------------------------------------------
typedef float f32x16_t __attribute__((ext_vector_type(16)));
template <bool BF>
__device__ __forceinline__ f32x16_t mfma32(const uint4& a, const uint4& b, f32x16_t c) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
}

// Epilogue of a wave's 32 tokens x 32 NT weight rows of sums that lie in its LDS, a
// row of kPitch floats per token: eight columns a lane, a token's row across lanes,
// so every access to out and residual is a run of 16 or 32 bytes in a whole line.
template <int NT>
constexpr int pitch() { return 32 * NT + 4; }
template <bool GATED, int NT>
__device__ __forceinline__ void finish_wave(const LinArgs& a, const float* sums, int64_t m0,
                                            int64_t n0, int lane) {
  constexpr int LPR = (GATED ? 2 : 4) * NT;  // lanes per token
  constexpr int IT = LPR / 2;                // runs of a lane
  constexpr int B = IT < 4 ? IT : NT < 4 ? 4 : 2;         // residual runs in flight
#pragma unroll 1
  for (int i = 0; i < IT; i += B) {
    float r[B][8];
    if constexpr (!GATED) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int at = (i + b) * 64 + lane;
        fetch_residual<8>(a, m0 + at / LPR, n0 + at % LPR * 8, r[b]);
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int at = (i + b) * 64 + lane, m = at / LPR, c = at % LPR;
      const float* p = sums + m * pitch<NT>() + (GATED ? (c >> 1) * 32 + (c & 1) * 8 : c * 8);
      float y[8], up[8];
      *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(p);
      *reinterpret_cast<float4*>(y + 4) = *reinterpret_cast<const float4*>(p + 4);
      if (GATED) {
        *reinterpret_cast<float4*>(up) = *reinterpret_cast<const float4*>(p + 16);
        *reinterpret_cast<float4*>(up + 4) = *reinterpret_cast<const float4*>(p + 20);
      }
      finish_run<8, GATED>(a, m0 + m, n0 + c * 8, y, up, r[b]);
    }
  }
}

// A wave's sums, through memory of its own in LDS 32 tokens at a time.
template <bool GATED, int MT, int NT>
__device__ __forceinline__ void store_sums(const LinArgs& a, float* sums,
                                           const f32x16_t (&acc)[MT][NT], int64_t m0, int64_t n0,
                                           int lane) {
  const int r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<float4*>(sums + r32 * pitch<NT>() + t * 32 + 2 * v + 4 * h) =
            float4{acc[u][t][v], acc[u][t][v + 1], acc[u][t][v + 2], acc[u][t][v + 3]};
    __builtin_amdgcn_sched_barrier(0);  // (a few sums at a time leave the accumulators)
    wave_sync();
    finish_wave<GATED, NT>(a, sums, m0 + u * 32, n0, lane);
    wave_sync();
    __builtin_amdgcn_sched_barrier(0);
  }
}

// 32 MT WM tokens x 32 NT WN weight rows by WM x WN waves, each 32 MT x 32 NT, in
// blocks of 64 k through NST LDS stages.  A block is four 16-k steps.  AHEAD: the
// operands of a whole block are read from LDS while the block before is multiplied;
// otherwise those of a step during the step before.  Once a block the waves meet:
// one block has then been read by all of them and the next has landed; the stage
// just read takes the copies of block b + NST.  LDS reads and copies are issued
// between the matrix instructions, evenly.
// A gated tile of 32 weight rows is 16 gate rows and the 16 up rows of the same
// columns.
template <bool BF, bool GATED, int WM, int WN, int MT, int NT, int NST, int PF, bool AHEAD>
__global__ void __launch_bounds__(64 * WM * WN) linear_tile_kernel(LinArgs a, int nm, int nn) {
  constexpr int W = WM * WN;
  constexpr int BM = 32 * MT * WM, BR = 32 * NT * WN;  // tokens, weight rows
  constexpr int WC = (GATED ? 16 : 32) * NT;           // output columns of a wave
  constexpr int KB = 64, ROW = 2 * KB, STEPS = KB / 16;  // k of a block, bytes of a row, steps
  constexpr int STAGE = (BM + BR) * ROW;
  constexpr int RC = 1024 / ROW;                       // rows of a copy
  constexpr int DX = BM / RC / W, DW = BR / RC / W, D = DX + DW;  // copies of a wave
  constexpr int F = MT * NT, R = MT + NT;              // products and reads of a step
  constexpr int SUMS = W * 32 * pitch<NT>() * 4;
  constexpr int G = PF ? 1 : 0;                        // prefetches of a wave and block
  constexpr int STAGES = NST * STAGE + (PF ? W * 256 : 0);
  constexpr int LDS = STAGES > SUMS ? STAGES : SUMS;
  static_assert(LDS <= 160 * 1024 && (NST - 1) * (D + G) + G < 64, "LDS and copies in flight");
  static_assert(W % 2 == 0 && BM % (RC * W) == 0 && BR % (RC * W) == 0, "copies");
  __shared__ __align__(1024) unsigned char lds[LDS];
  int mb, nb;
  if (!unit_of<8>(blockIdx.x, nm, nn, mb, nb)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  const int64_t m0 = (int64_t)mb * BM, n0 = (int64_t)nb * WC * WN;
  const int K = (int)a.K;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x + m0 * a.ldx);
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(a.w + n0 * a.ldw);
  const __amdgpu_buffer_rsrc_t ur = make_rsrc(a.w + (n0 + (GATED ? a.N : 0)) * a.ldw);
  // copy j of wave w fills rows RC (w + W j) .. + RC - 1 (RC W is a multiple of 16, so a
  // lane's chunk of its row is the same for every j)
  const int lr = lane / (KB / 8);
  const int ck = ((lane % (KB / 8)) ^ swz(wave * RC + lr)) * 8;
  int vo[D];
#pragma unroll
  for (int j = 0; j < DX; ++j) {
    const int r = (j * W + wave) * RC + lr;
    vo[j] = m0 + r < a.T ? (int)(r * a.ldx + ck) * 2 : kOob;
  }
#pragma unroll
  for (int j = 0; j < DW; ++j) {
    const int r = (j * W + wave) * RC + lr;
    const int c = GATED ? (r >> 5) * 16 + (r & 15) : r;
    vo[DX + j] = n0 + c < a.N ? (int)(c * a.ldw + ck) * 2 : kOob;
  }
  const uint32_t lds0 = lds_offset(lds) + wave * 1024;
  auto copy = [&](int slot, int b, int j) {
    const int k0 = b * KB, so = k0 < K ? k0 * 2 : 0;  // (a block past K copies zeros)
    const int voff = k0 + ck < K ? vo[j] : kOob;
    // (a copy's rows are all gate or all up rows: a gate run is 16 rows)
    const bool up = GATED && j >= DX && ((((j - DX) * W + wave) * RC) >> 4) & 1;
    dma16(j < DX ? xr : up ? ur : wr,
          lds0 + slot + (j < DX ? j * W * 1024 : BM * ROW + (j - DX) * W * 1024), voff, so);
  };
  const int nk = (K + KB - 1) / KB;
  // The lines of block b on their way into the L2: a copy that finds its line there
  // takes a third of the time that one from memory takes, which two stages do not
  // cover.  Work-groups of a row or column of tiles run together on an XCD and read the
  // same rows, so each asks for a quarter of its token rows and an eighth of its weight
  // rows, a few rows a wave.  (Four bytes of each line go to LDS that nothing reads; rows
  // past the end repeat the last one, and blocks past K.)
  const uint16_t* line = nullptr;
  if constexpr (PF > 0) {
    constexpr int PX = BM / 4, P = (PX + BR / 8) / W;
    const int i = wave * P + (lane < P ? lane : P - 1);
    const int rw = (mb & 7) * (BR / 8) + i - PX, c = GATED ? (rw >> 5) * 16 + (rw & 15) : rw;
    const int64_t m = m0 + (nb & 3) * PX + i, n = n0 + c;
    line = i < PX ? a.x + (m < a.T ? m : a.T - 1) * a.ldx
                  : a.w + ((n < a.N ? n : a.N - 1) + (GATED && (rw >> 4) & 1 ? a.N : 0)) * a.ldw;
  }
  const uint32_t sink = lds_offset(lds) + NST * STAGE + wave * 256;
  auto prefetch = [&](int b) {
    if constexpr (PF > 0) touch(line + (b < nk ? b : nk - 1) * KB, sink);
  };
  f32x16_t acc[MT][NT] = {};
  constexpr int SETS = AHEAD ? 2 * STEPS : 2;  // steps whose operands are in registers
  uint4 fx[SETS][MT], fw[SETS][NT];
  const int xo = (wm * MT * 32 + r32) * ROW, wo = BM * ROW + (wn * NT * 32 + r32) * ROW;
  const int sw = swz(r32) * 16, hb = h * 16;
  auto read = [&](int slot, int s, int p, int i) {  // operand i of step s into set p
    const unsigned char* at = lds + slot + ((s * 32 + hb) ^ sw);
    if (i < NT)
      fw[p][i] = *reinterpret_cast<const uint4*>(at + wo + i * 32 * ROW);
    else
      fx[p][i - NT] = *reinterpret_cast<const uint4*>(at + xo + (i - NT) * 32 * ROW);
  };
  // Set p's products, with nr LDS reads in the first three quarters of them and nc
  // copies evenly between them.
  auto multiply = [&](int p, int nr, auto read_op, int nc, auto copy_op) {
    constexpr int FR = F >= 4 ? F * 3 / 4 : F;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int u = f / NT, t = f % NT;
      acc[u][t] = mfma32<BF>(fw[p][t], fx[p][u], acc[u][t]);
      if (f < FR)
#pragma unroll
        for (int o = f * nr / FR; o < (f + 1) * nr / FR; ++o) read_op(o);
#pragma unroll
      for (int o = f * nc / F; o < (f + 1) * nc / F; ++o) copy_op(o);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto meet = [&]() {
    wait_lds();
    wait_vm<(NST - 2) * (D + G) + G>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto after = [&](int s) { return s + STAGE == NST * STAGE ? 0 : s + STAGE; };
#pragma unroll
  for (int i = 0; i < NST; ++i) {
#pragma unroll
    for (int j = 0; j < D; ++j) copy(i * STAGE, i, j);
    prefetch(NST + i);
  }
  wait_vm<(NST - 1) * (D + G) + G>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  int slot = 0;
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < STEPS * R; ++i) read(0, i / R, i / R, i % R);
    for (int kb = 0; kb < nk; kb += 2) {
#pragma unroll
      for (int o = 0; o < 2 * STEPS; o += STEPS) {
        if (o && kb + 1 >= nk) break;
        meet();
        const int next = after(slot);
        const int b = kb + o / STEPS + NST;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int c0 = s * D / STEPS;
          multiply(
              o + s, R, [&](int i) { read(next, s, (o ^ STEPS) + s, i); },
              (s + 1) * D / STEPS - c0, [&](int i) { copy(slot, b, c0 + i); });
        }
        prefetch(b + PF);
        slot = next;
      }
    }
  } else {
    // The copies of a block: over the step that follows the meeting and the next CS - 1.
    // With two stages the last ones need the rest of the block to land; four waves, with
    // twice the copies each, stall on issue when they are closer together (192 x 256, 8
    // waves: two steps 55.1 us, three 56.3; 256 x 256, 4 waves: 95.8 and 90.0).
    constexpr int CS = NST > 2 ? STEPS : W == 8 ? 2 : 3;
#pragma unroll
    for (int i = 0; i < R; ++i) read(0, 0, 0, i);
    int prev = (NST - 1) * STAGE;  // (before the first meeting: its last blocks once more)
    for (int kb = 0; kb < nk; ++kb) {
#pragma unroll
      for (int s = 0; s + 1 < STEPS; ++s) {
        const int c0 = (s + 1) * D / CS, c1 = s + 2 <= CS ? (s + 2) * D / CS : c0;
        multiply(
            s & 1, R, [&](int i) { read(slot, s + 1, (s + 1) & 1, i); }, c1 - c0,
            [&](int i) { copy(prev, kb + NST - 1, c0 + i); });
      }
      prefetch(kb + NST - 1 + PF);
      meet();
      const int next = after(slot);
      multiply(
          1, R, [&](int i) { read(next, 0, 0, i); }, D / CS,
          [&](int i) { copy(slot, kb + NST, i); });
      prev = slot;
      slot = next;
    }
  }
  wait_vm<0>();
  __syncthreads();
  store_sums<GATED, MT, NT>(a, reinterpret_cast<float*>(lds) + wave * 32 * pitch<NT>(), acc,
                            m0 + wm * MT * 32, n0 + wn * WC, lane);
}

// ---- any layout --------------------------------------------------------------------
// Rows that are not 16-byte aligned, or K % 8 != 0: no copies into LDS, but 16-byte
// loads.  From 4-byte aligned addresses they cost little more than aligned ones, from odd
// 2-byte addresses twice as much; a row at an odd one (`odd`: there may be such) is read
// from two bytes before, and its pieces are shifted together (60 tokens x 2049 x 5632 53 ->
// 23 us).  All bytes read lie within the tensors' storage.  The tiles load odd rows as
// they lie: shifting took them longer (4096 x 4095 x 4096 249 -> 286 us).
struct __attribute__((packed, aligned(2))) Chunk {
  uint32_t d[4];
};
__device__ __forceinline__ uint4 load_unaligned(const uint16_t* p) {
  const Chunk c = *reinterpret_cast<const Chunk*>(p);
  return uint4{c.d[0], c.d[1], c.d[2], c.d[3]};
}
struct __attribute__((aligned(4))) Quad {
  uint32_t d[4];
};
__device__ __forceinline__ uint4 load_quad(const uint16_t* p) {
  const Quad c = *reinterpret_cast<const Quad*>((uintptr_t)p & ~(uintptr_t)3);
  return uint4{c.d[0], c.d[1], c.d[2], c.d[3]};
}
// Bits [sh, sh + 128) of c followed by `next`, sh = 0 or 16.
__device__ __forceinline__ uint4 shift_quad(const uint4& c, uint32_t next, uint32_t sh) {
  return uint4{__builtin_amdgcn_alignbit(c.y, c.x, sh), __builtin_amdgcn_alignbit(c.z, c.y, sh),
               __builtin_amdgcn_alignbit(c.w, c.z, sh), __builtin_amdgcn_alignbit(next, c.w, sh)};
}
__device__ __forceinline__ uint32_t odd_shift(const uint16_t* p) {
  return (uint32_t)((uintptr_t)p & 2) * 8;
}
// Eight consecutive elements [k, k + 8) of a row, one by one, zeros from K on.
__device__ __forceinline__ uint4 load_tail(const uint16_t* row, int k, int K) {
  uint32_t d[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) d[j >> 1] |= (uint32_t)row[k + j] << ((j & 1) * 16);
  return uint4{d[0], d[1], d[2], d[3]};
}
// U chunks of eight from element k on.
template <int U>
__device__ __forceinline__ void load_chunks(const uint16_t* row, int k, int K, bool odd,
                                            uint4 (&v)[U]) {
  if (k + 8 * U <= K) {
    const uint32_t last = odd ? row[k + 8 * U - 1] : 0u;
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = load_quad(row + k + 8 * i);
    const uint32_t sh = odd ? odd_shift(row + k) : 0u;
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = shift_quad(v[i], i + 1 < U ? v[i + 1].x : last, sh);
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i)
      v[i] = k + 8 * i + 8 <= K ? load_unaligned(row + k + 8 * i) : load_tail(row, k + 8 * i, K);
  }
}

// Few tokens: as linear_stream_kernel, the matrix operands straight from memory.  Wave
// w takes the 32 U-k steps w, w + W, ...; lane quarter q holds 8 U consecutive k of each
// row, eight of them in each matrix instruction.
template <bool BF, bool GATED, int MT, int NT, int W, int U>
__global__ void __launch_bounds__(64 * W) linear_stream_any_kernel(LinArgs a, int nm, int nn) {
  constexpr int TILES = GATED ? NT / 2 : NT;
  __shared__ __align__(16) float4 red[W * MT * NT * 64];
  int mb, nb;
  if (!unit_of<4>(blockIdx.x, nm, nn, mb, nb)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)mb * MT * 16, n0 = (int64_t)nb * TILES * 16;
  const int K = (int)a.K;
  // (rows past the last repeat it: what they give is not stored)
  const uint16_t *xp[MT], *wp[NT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + t * 16 + r16;
    xp[t] = a.x + (m < a.T ? m : a.T - 1) * a.ldx;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = n0 + run_col<TILES>(t % TILES, r16);
    wp[t] = a.w + ((n < a.N ? n : a.N - 1) + (t >= TILES ? a.N : 0)) * a.ldw;
  }
  f32x4_t acc[MT][NT] = {};
  for (int k0 = wave * 32 * U; k0 < K; k0 += 32 * U * W) {
    const int k = k0 + q * 8 * U;
    uint4 x[MT][U], w[NT][U];
#pragma unroll
    for (int t = 0; t < NT; ++t) load_chunks<U>(wp[t], k, K, a.odd, w[t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) load_chunks<U>(xp[t], k, K, a.odd, x[t]);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[u][t] = mfma<BF>(w[t][i], x[u][i], acc[u][t]);
  }
  join_waves<GATED, MT, NT, W>(a, red, acc, m0, n0, wave, lane);
}

// Many tokens: 32 MT WM x 32 NT WN tiles as in linear_tile_kernel, a block's rows
// through registers into one of two LDS stages.
template <bool BF, bool GATED, int WM, int WN, int MT, int NT>
__global__ void __launch_bounds__(64 * WM * WN) linear_tile_any_kernel(LinArgs a, int nm, int nn) {
  constexpr int W = WM * WN, THREADS = 64 * W;
  constexpr int BM = 32 * MT * WM, BR = 32 * NT * WN;
  constexpr int WC = (GATED ? 16 : 32) * NT;
  constexpr int KB = 64, STAGE = (BM + BR) * 2 * KB;
  constexpr int D = (BM + BR) * 8 / THREADS;       // 16-byte chunks of a thread and block
  constexpr int SUMS = W * 32 * pitch<NT>() * 4;
  constexpr int LDS = 2 * STAGE > SUMS ? 2 * STAGE : SUMS;
  __shared__ __align__(1024) unsigned char lds[LDS];
  int mb, nb;
  if (!unit_of<8>(blockIdx.x, nm, nn, mb, nb)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int wm = wave / WN, wn = wave % WN;
  const int64_t m0 = (int64_t)mb * BM, n0 = (int64_t)nb * WC * WN;
  const int K = (int)a.K;
  const int ch = tid & 7;                          // chunk of the thread's rows
  const uint16_t* rows[D];                         // (rows past the last repeat it)
  int at[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int r = j * (THREADS / 8) + (tid >> 3);
    const int rw = r - BM, c = GATED ? (rw >> 5) * 16 + (rw & 15) : rw;
    const int64_t m = m0 + r, n = n0 + c;
    rows[j] = r < BM ? a.x + (m < a.T ? m : a.T - 1) * a.ldx
                     : a.w + ((n < a.N ? n : a.N - 1) + (GATED && (rw >> 4) & 1 ? a.N : 0)) * a.ldw;
    at[j] = r * 128 + (ch ^ swz(r)) * 16;
  }
  f32x16_t acc[MT][NT] = {};
  const int xo = (wm * MT * 32 + r32) * 128, wo = BM * 128 + (wn * NT * 32 + r32) * 128;
  const int sw = swz(r32) * 16, hb = h * 16;
  uint4 v[D];
  auto load = [&](int b) {
    const int k = b * KB + ch * 8;
#pragma unroll
    for (int j = 0; j < D; ++j)
      v[j] = k + 8 <= K ? load_unaligned(rows[j] + k) : load_tail(rows[j], k, K);
  };
  load(0);
  const int nk = (K + KB - 1) / KB;
  for (int kb = 0; kb < nk; ++kb) {
    unsigned char* stage = lds + (kb & 1) * STAGE;
#pragma unroll
    for (int j = 0; j < D; ++j) *reinterpret_cast<uint4*>(stage + at[j]) = v[j];
    __syncthreads();  // (the stage written next was read before this)
    if (kb + 1 < nk) load(kb + 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const unsigned char* p = stage + ((s * 32 + hb) ^ sw);
      uint4 fx[MT], fw[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) fw[t] = *reinterpret_cast<const uint4*>(p + wo + t * 4096);
#pragma unroll
      for (int u = 0; u < MT; ++u) fx[u] = *reinterpret_cast<const uint4*>(p + xo + u * 4096);
#pragma unroll
      for (int u = 0; u < MT; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[u][t] = mfma32<BF>(fw[t], fx[u], acc[u][t]);
    }
  }
  __syncthreads();
  store_sums<GATED, MT, NT>(a, reinterpret_cast<float*>(lds) + wave * 32 * pitch<NT>(), acc,
                            m0 + wm * MT * 32, n0 + wn * WC, lane);
}

// Whether `rows` rows of stride ld fit one buffer resource.
inline bool span_fits(int64_t rows, int64_t ld, int64_t K) {
  return ((rows - 1) * ld + K + 64) * 2 < kSpan;
}

// Work-groups of a grid of nm x nn tiles, a multiple of the XCDs; 0: more than a launch
// takes.
int64_t tile_grid(int64_t nm, int64_t nn, int threads) {
  const int64_t n = cdiv(nm * nn, 8) * 8;
  return n * threads < ((int64_t)1 << 32) ? n : 0;
}
template <typename Kernel>
int launch_tiles(Kernel kernel, const LinArgs& a, int64_t tokens, int64_t cols, int threads,
                 hipStream_t s) {
  const int64_t nm = cdiv(a.T, tokens), nn = cdiv(a.N, cols), grid = tile_grid(nm, nn, threads);
  EXQ_REQUIRE_SUPPORTED(grid > 0, "exq_linear: T=%lld x N=%lld is too large", (long long)a.T,
                        (long long)a.N);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3((unsigned)threads), 0, s, a, (int)nm,
                     (int)nn);
  return check_launch("linear kernel");
}
template <bool BF, bool GATED, int MT, int NT, int W, int NST>
int launch_stream(const LinArgs& a, hipStream_t s) {
  return launch_tiles(linear_stream_kernel<BF, GATED, MT, NT, W, NST>, a, 16 * MT,
                      (GATED ? 8 : 16) * NT, 64 * W, s);
}
template <bool BF, bool GATED, int MT, int NT, int W, int U>
int launch_stream_any(const LinArgs& a, hipStream_t s) {
  return launch_tiles(linear_stream_any_kernel<BF, GATED, MT, NT, W, U>, a, 16 * MT,
                      (GATED ? 8 : 16) * NT, 64 * W, s);
}
template <bool BF, bool GATED, int WM, int WN, int MT, int NT, int NST, int PF, bool AHEAD>
int launch_tile(const LinArgs& a, hipStream_t s) {
  return launch_tiles(linear_tile_kernel<BF, GATED, WM, WN, MT, NT, NST, PF, AHEAD>, a,
                      32 * MT * WM, (GATED ? 16 : 32) * NT * WN, 64 * WM * WN, s);
}
template <bool BF, bool GATED, int WM, int WN, int MT, int NT>
int launch_tile_any(const LinArgs& a, hipStream_t s) {
  return launch_tiles(linear_tile_any_kernel<BF, GATED, WM, WN, MT, NT>, a, 32 * MT * WM,
                      (GATED ? 16 : 32) * NT * WN, 64 * WM * WN, s);
}

// Which kernel: the one with the least rounds x time of a round, where a round is as
// many work-groups as the CUs hold.  `ns` is what 64 k of a work-group take when all
// CUs hold one, `ns2` when they hold two (0: they cannot), measured in bf16 with K = 2048
// (256 x 256: 4096 and 14336); it does not move with K.  The stream kernels win while
// their rounds are few (64 tokens x 2816 gated columns: 64-token streams 11.8 us, 64 x 64
// tiles 14.0; 100 tokens: 17.5 and 13.0), those of 16 rows while they fit one round (16
// tokens x 4096 x 4096: 16 rows 9.6 us, 32 rows 13.6; x 8192 x 8192: 31.7 and 30.4; 64
// tokens x 2816 x 2048: 32 x 16 8.5, 32 x 32 9.8, 64 x 32 12.7), small tiles until they
// need a further round (1024 tokens x 2048 x 2048: 64 x 128 18.4 us, 128 x 128 21.5, 256 x
// 256 59; 2001 tokens x 2048 x 5632: 192 x 256 56.5 us, 256 x 256 60, 128 x 256 and 128 x
// 128 66; 2048 x 4096 x 4096: 128 x 256 64 us, 128 x 128 78, 256 x 256 92).
struct Shape {
  int tokens, rows, ns, ns2;
};
constexpr Shape kShapes[] = {
    {16, 32, 140, 0},   {32, 32, 175, 0},    {64, 32, 240, 0},     // streams
    {64, 64, 340, 540}, {64, 128, 470, 0},   {128, 128, 590, 0},   // tiles
    {128, 256, 950, 0}, {192, 256, 1500, 0}, {256, 256, 1740, 0},
    {16, 16, 100, 0},   {32, 16, 135, 0},    // streams of one weight tile, not for gated rows
};
constexpr int kCus = 256;

int pick_shape(int64_t tokens, int64_t rows, bool gated) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < (int)(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
    const Shape& k = kShapes[i];
    if (gated && k.rows == 16) continue;
    const int64_t units = cdiv(tokens, k.tokens) * cdiv(rows, k.rows);
    const int64_t round = k.ns2 ? 2 * kCus : kCus, rest = units % round;
    const int64_t ns = units / round * (k.ns2 ? k.ns2 : k.ns) +
                       (rest == 0 ? 0 : rest > kCus ? k.ns2 : k.ns);
    if (ns < least) {
      least = ns;
      best = i;
    }
  }
  return best;
}

// The kernels by tokens x weight rows of a work-group: kShapes, then those of any layout.
constexpr const char* kKernels[] = {
    "stream 16x32",     "stream 32x32",     "stream 64x32",     "tile 64x64",
    "tile 64x128",      "tile 128x128",     "tile 128x256",     "tile 192x256",
    "tile 256x256",     "stream 16x16",     "stream 32x16",     "any stream 16x16",
    "any stream 16x32", "any stream 32x32", "any tile 64x64",   "any tile 128x128",
};

int pick_kernel(const LinArgs& a, bool gated) {
  const int64_t rows = a.N * (gated ? 2 : 1);
  if ((((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0 && a.ldx % 8 == 0 && a.ldw % 8 == 0 &&
      a.K % 8 == 0 && span_fits(256, a.ldx, a.K) && span_fits(256, a.ldw, a.K))
    return pick_shape(a.T, rows, gated);
  // 16 rows a work-group while they fit one round: 7 tokens x 8801 x 1664 22.0 us, 32 rows
  // 29.6.  32 x 32 streams while two rounds hold them, which is where they and the 64 x 64
  // tiles meet (K = 1001, 2047, 4095: 256 tokens x 2048, two rounds, 11.7, 22.9, 40.9 us and
  // 12.6, 21.9, 47.0; 300 x 2048 15.1, 30.8, 56.1 and 12.9, 22.4, 51.3; 100 x 2048 8.2, 14.1,
  // 22.4 and 13.0, 22.3, 38.3); 128 x 128 tiles from more than one round of them (2048 x 2048,
  // one round, 26.0, 54.7, 88.8 us and 64 x 64 27.4, 53.7, 99.6; 2048 x 2200 31.5, 57.2, 96.9
  // and 36.6, 71.5, 130.6; 1500 x 2048 29.2, 53.4, 87.0 and 23.3, 42.2, 74.8).
  if (a.T <= 16) return !gated && a.N <= 16 * kCus ? 11 : 12;
  if (cdiv(a.T, 32) * cdiv(rows, 32) <= 2 * kCus) return 13;
  return cdiv(a.T, 128) * cdiv(rows, 128) <= kCus ? 14 : 15;
}

template <bool BF, bool GATED>
int launch_linear(const LinArgs& a, hipStream_t s) {
  const int kernel = pick_kernel(a, GATED);
  switch (kernel) {
    case 0: return launch_stream<BF, GATED, 1, 2, 8, 3>(a, s);
    case 1: return launch_stream<BF, GATED, 2, 2, 8, 2>(a, s);
    case 2: return launch_stream<BF, GATED, 4, 2, 4, 3>(a, s);
    case 3: return launch_tile<BF, GATED, 2, 2, 1, 1, 4, 0, true>(a, s);
    case 4: return launch_tile<BF, GATED, 2, 2, 1, 2, 6, 0, true>(a, s);
    case 5: return launch_tile<BF, GATED, 2, 4, 2, 1, 4, 0, true>(a, s);
    case 6: return launch_tile<BF, GATED, 2, 4, 2, 2, 3, 0, false>(a, s);
    case 7: return launch_tile<BF, GATED, 2, 4, 3, 2, 2, 3, false>(a, s);
    case 8: return launch_tile<BF, GATED, 2, 2, 4, 4, 2, 4, false>(a, s);
    case 12: return launch_stream_any<BF, GATED, 1, 2, 8, 4>(a, s);
    case 13: return launch_stream_any<BF, GATED, 2, 2, 8, 2>(a, s);
    case 14: return launch_tile_any<BF, GATED, 2, 2, 1, 1>(a, s);
    case 15: return launch_tile_any<BF, GATED, 2, 2, 2, 2>(a, s);
    default:
      if constexpr (!GATED) {
        if (kernel == 9) return launch_stream<BF, GATED, 1, 1, 16, 2>(a, s);
        if (kernel == 10) return launch_stream<BF, GATED, 2, 1, 8, 3>(a, s);
        if (kernel == 11) return launch_stream_any<BF, GATED, 1, 1, 16, 4>(a, s);
      }
      return EXQ_ERROR_UNSUPPORTED;  // (not reached: every kernel that is picked is above)
  }
}

}  // namespace
}  // namespace exq

using namespace exq;

namespace {
int check_problem(const exq_linear_problem* p, const void* bias, const void* residual) {
  const char* fn = "exq_linear";
  EXQ_REQUIRE(p, "%s: null problem", fn);
  EXQ_REQUIRE(is_act_dtype(p->act_dtype), "%s: x and W must be f16 or bf16", fn);
  EXQ_REQUIRE(is_float_dtype(p->out_dtype), "%s: out dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(!bias || is_float_dtype(p->bias_dtype), "%s: bias dtype must be f32, f16 or bf16",
              fn);
  EXQ_REQUIRE(!residual || is_float_dtype(p->residual_dtype),
              "%s: residual dtype must be f32, f16 or bf16", fn);
  EXQ_REQUIRE(p->activation >= EXQ_ACT_NONE && p->activation <= EXQ_ACT_SIGMOID,
              "%s: unknown activation %d", fn, p->activation);
  EXQ_REQUIRE(!(p->gated && residual), "%s: a gated product takes no residual", fn);
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
  EXQ_REQUIRE(T >= 0 && T <= INT32_MAX / 2 && K >= 1 && K <= INT32_MAX / 2 && N >= 1 &&
                  N <= (1 << 20),
              "%s: sizes T=%lld K=%lld N=%lld out of range", fn, (long long)T, (long long)K,
              (long long)N);
  EXQ_REQUIRE(p->x_stride >= 0 && p->weight_stride >= 0 && p->residual_stride >= 0 &&
                  (T <= 1 || p->out_stride >= N),
              "%s: row strides must not be negative, and out's at least N", fn);
  return EXQ_SUCCESS;
}
}  // namespace

extern "C" int exq_linear(const exq_linear_problem* p, const void* x, const void* weight,
                          const void* bias, const void* residual, void* out, exq_stream stream) {
  const char* fn = "exq_linear";
  const int status = check_problem(p, bias, residual);
  if (status != EXQ_SUCCESS) return status;
  const int64_t T = p->n_tokens, K = p->in_features, N = p->out_features;
  if (T == 0) return EXQ_SUCCESS;
  EXQ_REQUIRE(x && weight && out, "%s: null pointer", fn);
  LinArgs a;
  a.x = reinterpret_cast<const uint16_t*>(x);
  a.w = reinterpret_cast<const uint16_t*>(weight);
  a.bias = bias;
  a.res = residual;
  a.out = out;
  a.ldx = p->x_stride;
  a.ldw = p->weight_stride;
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
  a.odd = ((uintptr_t)x | (uintptr_t)weight) % 4 != 0 || (a.ldx | a.ldw) % 2 != 0;
  const hipStream_t s = as_stream(stream);
  if (p->act_dtype == EXQ_DTYPE_BF16)
    return p->gated ? launch_linear<true, true>(a, s) : launch_linear<true, false>(a, s);
  return p->gated ? launch_linear<false, true>(a, s) : launch_linear<false, false>(a, s);
}

extern "C" const char* exq_linear_kernel(const exq_linear_problem* p, const void* x,
                                         const void* weight) {
  if (check_problem(p, nullptr, nullptr) != EXQ_SUCCESS || p->n_tokens == 0) return nullptr;
  LinArgs a = {};
  a.x = reinterpret_cast<const uint16_t*>(x);
  a.w = reinterpret_cast<const uint16_t*>(weight);
  a.ldx = p->x_stride;
  a.ldw = p->weight_stride;
  a.T = p->n_tokens;
  a.N = p->out_features;
  a.K = p->in_features;
  return kKernels[pick_kernel(a, p->gated != 0)];
}
