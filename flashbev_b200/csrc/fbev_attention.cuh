// What the attention kernels share.
//
// Rows.  The G = Hq / Hkv query heads that share a key head are folded into rows: row r of (sample, key head) is query
// r / G, head r % G of the group.  Statistics are laid out by row: lse[(b * Hkv + g) * rows_padded + r] =
// log2 sum_j 2^(S_j log2 e), +infinity for a row without keys, so that 2^(S - lse) is zero there.
#pragma once
#include "fbev_device.cuh"
#include "fbev_query.h"

namespace fbev {

constexpr float kLog2e = 1.44269504088896340736f;

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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}

}  // namespace fbev
