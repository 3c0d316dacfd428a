// What the attention kernels share.
//
// Rows.  The G = Hq / Hkv query heads that share a key head are folded into rows: row r of (sample, key head) is query
// r / G, head r % G of the group.  Statistics are laid out by row: lse[(b * Hkv + g) * rows_padded + r] =
// log2 sum_j 2^(S_j log2 e), +infinity for a row without keys, so that 2^(S - lse) is zero there, NaN for a row whose scores
// are not numbers or all -infinity.
#pragma once
#include "fbev_device.cuh"
#include "fbev_query.h"

namespace fbev {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;  // statistic of a part whose keys all score -infinity

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__host__ __device__ __forceinline__ long long att_rows(const FbevAttention& p) { return (long long)p.Lq * (p.Hq / p.Hkv); }
__host__ __device__ __forceinline__ long long att_rows_padded(const FbevAttention& p) { return (att_rows(p) + 3) / 4 * 4; }

__device__ __forceinline__ int att_keys(const FbevAttention& p, int b) {
  if (p.key_lengths == nullptr) return p.Lk;
  const int n = p.key_lengths[b];
  return n < 0 ? 0 : n > p.Lk ? p.Lk : n;
}
__device__ __forceinline__ bool att_allowed(const FbevAttention& p, int b, int j) {
  return p.key_mask == nullptr || p.key_mask[(long long)b * p.mask_stride + j] != 0;
}

// The key tiles t0 .. t0 + n - 1 (n <= kSkipTiles) in which the mask leaves something: their numbers, less t0, go to `list`,
// their count is returned.  All warps of a block call it.  What masks take away comes in runs (a camera that is missing, a
// padded one), so whole tiles are empty: with one camera of six gone 33 tiles become 28 or 29, and 4 x 901 queries x 4219
// keys x 8 heads of 32 take 55 us instead of 63.  A mask that empties nothing costs its block about 1 us.
constexpr int kSkipTiles = 256;
template <int WARPS>
__device__ __forceinline__ int att_tiles_left(const uint8_t* mask, int keys, int t0, int n, uint8_t* list, int* count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = warp; t < n; t += WARPS) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = (t0 + t) * 128 + 32 * i + lane;
      any |= j < keys && mask[j] != 0;
    }
    any = __any_sync(kFull, any);
    if (lane == 0) list[t] = any;
  }
  __syncthreads();
  if (warp == 0) {  // in place: a tile's number goes to its own place or one before it
    int k = 0;
    for (int t = 0; t < n; t += 32) {
      const bool on = t + lane < n && list[t + lane] != 0;
      const uint32_t w = __ballot_sync(kFull, on);
      if (on) list[k + __popc(w & ((1u << lane) - 1))] = (uint8_t)(t + lane);
      k += __popc(w);
      __syncwarp();
    }
    if (lane == 0) *count = k;
  }
  __syncthreads();
  return *count;
}

}  // namespace fbev
