// mxfp4_route.h -- routing of a few slots by every work-group for itself.
//
// A bit per slot in its expert's masks, whose population counts give the experts' rows and
// a slot's rank among them in ascending order, and a scan over the experts the places: the
// same in every work-group.  The first one writes the plan down for the next kernel.  The
// launch in front, 7.5 us at 64 tokens x 8 of 128 experts, and the wait between the two
// are saved for about 2.5 us in the kernel.
#pragma once

#include "mxfp4.h"

namespace exq {
namespace mx {

struct RouteArgs {
  const void* ids;           // [n]
  int ids_dtype, n, E, top_k;
  int* hdr;                  // the plan: [0] token groups
  TgEntry* tg;
  int* sorted;               // expert-sorted position -> slot
};

// n <= 64 NSEG slots, E <= kExperts.
template <int NSEG>
struct Router {
  static constexpr int kExperts = NSEG <= 4 ? 1024 : 4096 / NSEG;
  static constexpr int kWords = 2 * NSEG * kExperts + kExperts + 4;  // of scratch
  static constexpr int kIds = (64 * NSEG + 255) / 256;

  // rows and groups of 64 rows, counted in one word
  __device__ __forceinline__ static uint32_t counts(int rows) {
    return (uint32_t)rows | (uint32_t)((rows + 63) >> 6) << 16;
  }
  __device__ __forceinline__ static int row_at(uint32_t c) { return c & 0xffff; }
  __device__ __forceinline__ static int group_at(uint32_t c) { return c >> 16; }

  // The work-group's own token group, pick(groups) of the groups of 64 rows (-1: none), with
  // its tokens, and the plan from the first work-group.
  template <typename Pick>
  __device__ __forceinline__ static bool here(const RouteArgs& a, uint32_t* scratch, TgEntry* own,
                                              int* tokens, Pick pick) {
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
    for (int i = tid; i < a.E * NSEG; i += 256) masks[i] = 0;
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
    const int g0 = pick(group_at(all));
    const bool writer = blockIdx.x == 0;
    if (writer && tid == 0) a.hdr[0] = group_at(all);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (k >= per || e0 + k >= a.E) break;
      first[e0 + k] = at;
      const int g = g0 - group_at(at);
      if (g0 >= 0 && g >= 0 && g * 64 < cnt[k])
        *own = TgEntry{e0 + k, row_at(at) + g * 64, cnt[k] - g * 64 < 64 ? cnt[k] - g * 64 : 64, 2};
      if (writer)
        for (int r = 0; r < cnt[k]; r += 64)
          a.tg[group_at(at) + r / 64] =
              TgEntry{e0 + k, row_at(at) + r, cnt[k] - r < 64 ? cnt[k] - r : 64, 2};
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
      if (writer) a.sorted[row_at(first[e]) + rank] = i;
      if (group_at(first[e]) + (rank >> 6) == g0) tokens[rank & 63] = i / a.top_k;
    }
    __syncthreads();
    return g0 >= 0;
  }
};

}  // namespace mx
}  // namespace exq
