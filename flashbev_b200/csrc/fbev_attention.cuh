// Attention, one warp per row.
//
// Rows.  The G = Hq / Hkv query heads that share a key head are folded into rows: row r of (sample, key head) is query
// r / G, head r % G of the group.  Statistics are laid out by row: lse[(b * Hkv + g) * rows_padded + r] =
// log2 sum_j 2^(S_j log2 e), +infinity for a row without keys, so that 2^(S - lse) is zero there.
//
// Running maximum m and sum l of a row, base 2: a new score s rescales l and the output by 2^(m - max(m, s)).
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

// elements lane, lane + 32, ... of a head
template <typename T>
__device__ __forceinline__ void load_head(float (&v)[4], const T* src, int D, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lane + 32 * i < D ? to_float(src[lane + 32 * i]) : 0.0f;
}
__device__ __forceinline__ float dot_head(const float (&a)[4], const float (&b)[4]) {
  return warp_sum(fmaf(a[0], b[0], fmaf(a[1], b[1], fmaf(a[2], b[2], a[3] * b[3]))));
}

template <typename T>
__device__ __forceinline__ const T* q_head(const FbevAttention& p, int b, long long l, int h) {
  return reinterpret_cast<const T*>(p.q) + (p.q_shared ? 0 : b * p.q_stride[0]) + l * p.q_stride[1] + h * p.q_stride[2];
}

template <typename T>
__global__ void __launch_bounds__(128) att_row_kernel(const __grid_constant__ FbevAttention p, T* out, float* lse) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long rows = att_rows(p);
  if (unit >= rows * p.B * p.Hkv) return;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const long long bg = unit / rows, row = unit - bg * rows;
  const int b = (int)(bg / p.Hkv), g = (int)(bg % p.Hkv);
  const long long l = row / G;
  const int h = g * G + (int)(row % G);
  float q[4], o[4] = {}, kv[4];
  load_head(q, q_head<T>(p, b, l, h), p.D, lane);
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_stride[0] + g * p.k_stride[2];
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_stride[0] + g * p.v_stride[2];
  const float c = p.scale * kLog2e;
  float m = -INFINITY, sum = 0.0f;
  const int n = att_keys(p, b);
  for (int j = 0; j < n; ++j) {
    if (!att_allowed(p, b, j)) continue;
    load_head(kv, k + (long long)j * p.k_stride[1], p.D, lane);
    const float s = dot_head(q, kv) * c;
    const float mn = fmaxf(m, s);
    const float back = m == -INFINITY ? 0.0f : exp2_fast(m - mn), e = exp2_fast(s - mn);
    m = mn;
    sum = sum * back + e;
    load_head(kv, v + (long long)j * p.v_stride[1], p.D, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(e, kv[i], o[i] * back);
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : NAN;
  T* dst = out + (((long long)b * p.Lq + l) * p.Hq + h) * p.D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.D) dst[lane + 32 * i] = from_float<T>(o[i] * inv);
  if (lse != nullptr && lane == 0) lse[bg * att_rows_padded(p) + row] = sum == 0.0f ? INFINITY : m + log2f(sum);
}

// delta[row] = <out, grad_out>, laid out like lse
template <typename T>
__global__ void __launch_bounds__(128) att_delta_kernel(const __grid_constant__ FbevAttention p, const T* __restrict__ out,
                                                        const T* __restrict__ go, float* __restrict__ delta) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long rows = att_rows(p);
  if (unit >= rows * p.B * p.Hkv) return;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const long long bg = unit / rows, row = unit - bg * rows;
  const int b = (int)(bg / p.Hkv), g = (int)(bg % p.Hkv);
  const long long at = (((long long)b * p.Lq + row / G) * p.Hq + g * G + row % G) * p.D;
  float x[4], y[4];
  load_head(x, out + at, p.D, lane);
  load_head(y, go + at, p.D, lane);
  const float d = dot_head(x, y);
  if (lane == 0) delta[bg * att_rows_padded(p) + row] = d;
}

template <typename T>
__global__ void __launch_bounds__(128) att_row_grad_q_kernel(const __grid_constant__ FbevAttention p, const float* lse,
                                                             const float* delta, const T* go, T* gq) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long rows = att_rows(p);
  if (unit >= rows * p.B * p.Hkv) return;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const long long bg = unit / rows, row = unit - bg * rows;
  const int b = (int)(bg / p.Hkv), g = (int)(bg % p.Hkv);
  const long long l = row / G;
  const int h = g * G + (int)(row % G);
  const long long at = (((long long)b * p.Lq + l) * p.Hq + h) * p.D;
  float q[4], d[4], acc[4] = {}, kk[4], vv[4];
  load_head(q, q_head<T>(p, b, l, h), p.D, lane);
  load_head(d, go + at, p.D, lane);
  const float lr = lse[bg * att_rows_padded(p) + row], dr = delta[bg * att_rows_padded(p) + row];
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_stride[0] + g * p.k_stride[2];
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_stride[0] + g * p.v_stride[2];
  const int n = att_keys(p, b);
  for (int j = 0; j < n; ++j) {
    if (!att_allowed(p, b, j)) continue;
    load_head(kk, k + (long long)j * p.k_stride[1], p.D, lane);
    load_head(vv, v + (long long)j * p.v_stride[1], p.D, lane);
    const float e = exp2_fast(dot_head(q, kk) * p.scale * kLog2e - lr);
    const float ds = e * (dot_head(d, vv) - dr);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(ds, kk[i], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.D) gq[at + lane + 32 * i] = from_float<T>(acc[i] * p.scale);
}

template <typename T>
__global__ void __launch_bounds__(128) att_row_grad_kv_kernel(const __grid_constant__ FbevAttention p, const float* lse,
                                                              const float* delta, const T* go, T* gk, T* gv) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= (long long)p.B * p.Lk * p.Hkv) return;
  const int lane = threadIdx.x & 31, G = p.Hq / p.Hkv;
  const int g = (int)(unit % p.Hkv);
  const long long bj = unit / p.Hkv;
  const int b = (int)(bj / p.Lk), j = (int)(bj % p.Lk);
  float dk[4] = {}, dv[4] = {};
  if (j < att_keys(p, b) && att_allowed(p, b, j)) {
    float kk[4], vv[4], q[4], d[4];
    load_head(kk, reinterpret_cast<const T*>(p.k) + b * p.k_stride[0] + j * p.k_stride[1] + g * p.k_stride[2], p.D, lane);
    load_head(vv, reinterpret_cast<const T*>(p.v) + b * p.v_stride[0] + j * p.v_stride[1] + g * p.v_stride[2], p.D, lane);
    const long long rows = att_rows(p), st = ((long long)b * p.Hkv + g) * att_rows_padded(p);
    for (long long row = 0; row < rows; ++row) {
      const long long l = row / G;
      const int h = g * G + (int)(row % G);
      load_head(q, q_head<T>(p, b, l, h), p.D, lane);
      load_head(d, go + (((long long)b * p.Lq + l) * p.Hq + h) * p.D, p.D, lane);
      const float e = exp2_fast(dot_head(q, kk) * p.scale * kLog2e - lse[st + row]);
      const float ds = e * (dot_head(d, vv) - delta[st + row]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dv[i] = fmaf(e, d[i], dv[i]);
        dk[i] = fmaf(ds, q[i], dk[i]);
      }
    }
  }
  const long long at = unit * p.D;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < p.D) {
      gk[at + lane + 32 * i] = from_float<T>(dk[i] * p.scale);
      gv[at + lane + 32 * i] = from_float<T>(dv[i]);
    }
}

}  // namespace fbev
