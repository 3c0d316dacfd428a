// Residual addition + root-mean-square norm, its 8-bit output and its gradient.
//
//   h = x + r,  s = (mean(h^2) + eps)^(-1/2),  n = h s,  y = n w
//   dx = dr = dh + s (w dy - n mean(w dy n)),  dw = sum over rows of dy n
//
// Bound by memory: a row is read once, kept in registers and written once.  A row belongs to a group of LANES threads
// (8, 16 or 32 of one warp, or a block of 256) that hold NV chunks of VE elements each, the smallest group whose
// registers take the row.  Sums run in float32, within a thread first, then across the group in a fixed order.
//
// y comes from the unrounded sum: rounding h to 16 bits first would add an error as large as y's own rounding.  The
// gradient re-reads the rounded h (the tensor the residual stream keeps anyway) but takes s from the unrounded one.
//
// dw: each block walks rows at a stride and keeps its sums in registers; one partial row per block goes to the
// workspace and a second small kernel adds them in block order, so the result does not depend on who arrives first.
#pragma once
#include <cuda_fp8.h>

#include "fbev_device.cuh"
#include "fbev_query.h"
#include "fbev_rotary.cuh"

namespace fbev {

struct NormArgs {
  const void *x, *r, *w;       // backward: x = h
  void *y, *h;                 // y: T or E4M3 bytes
  float *rstd, *scales;
  const float* rstd_in;
  const void *dy, *dh;
  void* dx;
  float* dw_part;              // [blocks][C] or null
  long long rows;
  int C;
  float eps;
};

// sum (or maximum) over a group of LANES threads; `red` has room for one float per warp when the group is a block
template <int LANES, bool MAX>
__device__ __forceinline__ float group_reduce(float v, float* red) {
#pragma unroll
  for (int d = (LANES < 32 ? LANES : 32) / 2; d > 0; d >>= 1) {
    const float o = __shfl_xor_sync(kFull, v, d);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  if (LANES > 32) {
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the words may still be read from the reduction before
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < LANES / 32; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

// fmaxf drops NaN; the scale of a row with one has to show it
__device__ __forceinline__ float max_keep_nan(float a, float b) { return (a > b || a != a) ? a : b; }

constexpr int kNormThreads = 256;

template <typename T, int VE, int NV, int LANES, bool QUANT>
__global__ void __launch_bounds__(kNormThreads) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const int lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * (kNormThreads / LANES) + threadIdx.x / LANES;
  const bool live = row < a.rows;  // every thread takes part in the shuffles
  const long long base = row * a.C;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* r = reinterpret_cast<const T*>(a.r);
  const T* w = reinterpret_cast<const T*>(a.w);
  float h[NV][VE];
  float sum = 0.0f;
  Pack<T, VE> px[NV], pr[NV], pw[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * LANES + lane) * VE;
    if (!live || c >= a.C) continue;
    px[n] = *reinterpret_cast<const Pack<T, VE>*>(x + base + c);
    if (r) pr[n] = *reinterpret_cast<const Pack<T, VE>*>(r + base + c);
    if (w) pw[n] = *reinterpret_cast<const Pack<T, VE>*>(w + c);
  }
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * LANES + lane) * VE;
    const bool in = live && c < a.C;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      h[n][e] = in ? to_float(px[n].v[e]) + (r ? to_float(pr[n].v[e]) : 0.0f) : 0.0f;
      sum = fmaf(h[n][e], h[n][e], sum);
    }
    if (in && a.h) {
      Pack<T, VE> ph;
#pragma unroll
      for (int e = 0; e < VE; ++e) ph.v[e] = from_float<T>(h[n][e]);
      *reinterpret_cast<Pack<T, VE>*>(reinterpret_cast<T*>(a.h) + base + c) = ph;
    }
  }
  sum = group_reduce<LANES, false>(sum, red);
  const float s = 1.0f / sqrtf(sum / (float)a.C + a.eps);
  if (live && lane == 0 && a.rstd) a.rstd[row] = s;
  float top = 0.0f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * LANES + lane) * VE;
    if (!live || c >= a.C) continue;
    Pack<T, VE> py;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      h[n][e] *= s;
      if (w) h[n][e] *= to_float(pw[n].v[e]);
      if (QUANT) top = max_keep_nan(fabsf(h[n][e]), top);
      else py.v[e] = from_float<T>(h[n][e]);
    }
    if (!QUANT) *reinterpret_cast<Pack<T, VE>*>(reinterpret_cast<T*>(a.y) + base + c) = py;
  }
  if (QUANT) {
    // the maximum over a group drops NaN: whether there is one is a reduction of its own
    const float any_nan = group_reduce<LANES, true>(top != top ? 1.0f : 0.0f, red);
    top = group_reduce<LANES, true>(top, red);
    if (any_nan > 0.0f) top = __int_as_float(0x7fc00000);
    float scale = top / 448.0f;
    if (scale == 0.0f) scale = 1.0f;  // a row of zeros (or of values whose scale underflows)
    if (live && lane == 0) a.scales[row] = scale;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * LANES + lane) * VE;
      if (!live || c >= a.C) continue;
      Pack<uint8_t, VE> pq;
#pragma unroll
      for (int e = 0; e < VE; ++e) pq.v[e] = __nv_cvt_float_to_fp8(__fdiv_rn(h[n][e], scale), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<Pack<uint8_t, VE>*>(reinterpret_cast<uint8_t*>(a.y) + base + c) = pq;
    }
  }
}

// Rows of any length: a block per row reads it once per pass.  Serves rows too long for the registers of a block.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(kNormThreads) norm_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const long long row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.C;
  const T* r = a.r ? reinterpret_cast<const T*>(a.r) + row * a.C : nullptr;
  const T* w = reinterpret_cast<const T*>(a.w);
  T* hp = a.h ? reinterpret_cast<T*>(a.h) + row * a.C : nullptr;
  float sum = 0.0f;
  for (int c = threadIdx.x; c < a.C; c += kNormThreads) {
    const float h = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
    sum = fmaf(h, h, sum);
  }
  sum = group_reduce<kNormThreads, false>(sum, red);
  const float s = 1.0f / sqrtf(sum / (float)a.C + a.eps);
  if (threadIdx.x == 0 && a.rstd) a.rstd[row] = s;
  float scale = 1.0f;
  if (QUANT) {
    float top = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += kNormThreads) {
      const float h = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
      top = max_keep_nan(fabsf(h * s * (w ? to_float(w[c]) : 1.0f)), top);
    }
    const float any_nan = group_reduce<kNormThreads, true>(top != top ? 1.0f : 0.0f, red);
    top = group_reduce<kNormThreads, true>(top, red);
    if (any_nan > 0.0f) top = __int_as_float(0x7fc00000);
    scale = top / 448.0f;
    if (scale == 0.0f) scale = 1.0f;
    if (threadIdx.x == 0) a.scales[row] = scale;
  }
  // each element is read before its own thread overwrites it (h may be written over x or r)
  for (int c = threadIdx.x; c < a.C; c += kNormThreads) {
    const float h = to_float(x[c]) + (r ? to_float(r[c]) : 0.0f);
    const float y = h * s * (w ? to_float(w[c]) : 1.0f);
    if (hp) hp[c] = from_float<T>(h);
    if (QUANT)
      reinterpret_cast<uint8_t*>(a.y)[row * a.C + c] = __nv_cvt_float_to_fp8(__fdiv_rn(y, scale), __NV_SATFINITE, __NV_E4M3);
    else
      reinterpret_cast<T*>(a.y)[row * a.C + c] = from_float<T>(y);
  }
}

// A row's values are unpacked twice rather than kept unpacked: four blocks of one chunk a lane fit an SM then (the grid is
// that many), and what hides the memory's latency here is their number.  The limit of 64 registers costs the bfloat16 forms
// 24 to 32 bytes of spills a thread.
template <typename T, int VE, int NV, int LANES>
__global__ void __launch_bounds__(kNormThreads, NV == 1 ? 4 : NV == 2 ? 2 : 1) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  extern __shared__ float s_dw[];  // [C], only with dw_part
  constexpr int kGroups = kNormThreads / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const T* hp = reinterpret_cast<const T*>(a.x);
  const T* w = reinterpret_cast<const T*>(a.w);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const T* dh = reinterpret_cast<const T*>(a.dh);
  Pack<T, VE> pw[NV];
  float dw[NV][VE] = {};
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * LANES + lane) * VE;
    if (w && c < a.C) pw[n] = *reinterpret_cast<const Pack<T, VE>*>(w + c);
  }
  for (long long first = (long long)blockIdx.x * kGroups; first < a.rows; first += (long long)gridDim.x * kGroups) {
    const long long row = first + group;
    const bool live = row < a.rows;
    const long long base = row * a.C;
    Pack<T, VE> ph[NV], py[NV], pd[NV];
    const float s = live ? a.rstd_in[row] : 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * LANES + lane) * VE;
      if (!live || c >= a.C) continue;
      ph[n] = *reinterpret_cast<const Pack<T, VE>*>(hp + base + c);
      if (dy) py[n] = *reinterpret_cast<const Pack<T, VE>*>(dy + base + c);
      if (dh) pd[n] = *reinterpret_cast<const Pack<T, VE>*>(dh + base + c);
    }
    float dot = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * LANES + lane) * VE;
      if (!live || c >= a.C || !dy) continue;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = to_float(py[n].v[e]), nv = to_float(ph[n].v[e]) * s;
        dw[n][e] = fmaf(d, nv, dw[n][e]);
        dot = fmaf(w ? d * to_float(pw[n].v[e]) : d, nv, dot);
      }
    }
    if (!a.dx) continue;  // uniform
    dot = group_reduce<LANES, false>(dot, red) / (float)a.C;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * LANES + lane) * VE;
      if (!live || c >= a.C) continue;
      Pack<T, VE> po;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float d = dy ? to_float(py[n].v[e]) : 0.0f, nv = to_float(ph[n].v[e]) * s;
        const float g = w ? d * to_float(pw[n].v[e]) : d;
        po.v[e] = from_float<T>(fmaf(s, fmaf(-nv, dot, g), dh ? to_float(pd[n].v[e]) : 0.0f));
      }
      *reinterpret_cast<Pack<T, VE>*>(reinterpret_cast<T*>(a.dx) + base + c) = po;
    }
  }
  if (a.dw_part) {
    // the block's groups add one after another
    for (int gi = 0; gi < kGroups; ++gi) {
      if (group == gi) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const int c = (n * LANES + lane) * VE;
          if (c >= a.C) continue;
#pragma unroll
          for (int e = 0; e < VE; ++e) s_dw[c + e] = gi == 0 ? dw[n][e] : s_dw[c + e] + dw[n][e];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.C; c += kNormThreads) a.dw_part[(long long)blockIdx.x * a.C + c] = s_dw[c];
  }
  grid_dependency_trigger();
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_grad_long_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[kNormThreads / 32];
  const T* w = reinterpret_cast<const T*>(a.w);
  bool first = true;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
    const T* hp = reinterpret_cast<const T*>(a.x) + row * a.C;
    const T* dy = a.dy ? reinterpret_cast<const T*>(a.dy) + row * a.C : nullptr;
    const T* dh = a.dh ? reinterpret_cast<const T*>(a.dh) + row * a.C : nullptr;
    const float s = a.rstd_in[row];
    float dot = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += kNormThreads) {
      const float n = to_float(hp[c]) * s, d = dy ? to_float(dy[c]) : 0.0f;
      dot = fmaf(w ? d * to_float(w[c]) : d, n, dot);
      if (a.dw_part) {
        float* acc = a.dw_part + (long long)blockIdx.x * a.C + c;  // this thread's own word of the block's row
        *acc = fmaf(d, n, first ? 0.0f : *acc);
      }
    }
    if (!a.dx) continue;
    dot = group_reduce<kNormThreads, false>(dot, red) / (float)a.C;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.C;
    for (int c = threadIdx.x; c < a.C; c += kNormThreads) {
      const float n = to_float(hp[c]) * s, d = dy ? to_float(dy[c]) : 0.0f;
      const float g = w ? d * to_float(w[c]) : d;
      dx[c] = from_float<T>(fmaf(s, fmaf(-n, dot, g), dh ? to_float(dh[c]) : 0.0f));
    }
  }
  grid_dependency_trigger();
}

// dw[c] = sum over blocks of part[block][c]: 32 columns per block, 32 threads share a column's rows
template <typename T>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ part, int blocks, int C, T* __restrict__ dw) {
  __shared__ float s[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, g = threadIdx.x >> 5;
  float v = 0.0f;
  if (c < C)
#pragma unroll 8
    for (int i = g; i < blocks; i += 32) v += part[(long long)i * C + c];
  s[g][lane] = v;
  __syncthreads();
  v = s[lane][g];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  if (lane == 0 && blockIdx.x * 32 + g < C) dw[blockIdx.x * 32 + g] = from_float<T>(v);
}

// Blocks of the gradient kernel, the rows of its dw workspace: four per SM, and no more than there are rows.
static long long norm_grad_blocks(long long rows) { return rows < 148 * 4 ? rows : 148 * 4; }

template <typename T, int VE, int NV, int LANES>
static int norm_run(const NormArgs& a, bool quant, bool grad, long long grad_blocks, cudaStream_t st) {
  constexpr int kGroups = kNormThreads / LANES;
  const long long blocks = (a.rows + kGroups - 1) / kGroups;
  if (grad) {
    const size_t smem = a.dw_part ? (size_t)a.C * 4 : 0;
    norm_grad_kernel<T, VE, NV, LANES><<<(unsigned)grad_blocks, kNormThreads, smem, st>>>(a);
  } else if (blocks >= (1ll << 31)) {
    return FBEV_ERR_RANGE;
  } else if (quant) {
    norm_kernel<T, VE, NV, LANES, true><<<(unsigned)blocks, kNormThreads, 0, st>>>(a);
  } else {
    norm_kernel<T, VE, NV, LANES, false><<<(unsigned)blocks, kNormThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T>
static int norm_dispatch(const NormArgs& a, bool quant, bool grad, long long grad_blocks, cudaStream_t st) {
  constexpr int W = 16 / sizeof(T);
  uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.r | (uintptr_t)a.w | (uintptr_t)a.h | (uintptr_t)a.dy | (uintptr_t)a.dh |
                  (uintptr_t)a.dx;
  const bool q_fits = !quant || (uintptr_t)a.y % W == 0;
  if (!quant) all |= (uintptr_t)a.y;
  if (a.C % W == 0 && all % 16 == 0 && q_fits) {
    const int n = a.C / W;  // 16-byte chunks of a row
    if (n <= 8) return norm_run<T, W, 1, 8>(a, quant, grad, grad_blocks, st);
    if (n <= 16) return norm_run<T, W, 1, 16>(a, quant, grad, grad_blocks, st);
    if (n <= 32) return norm_run<T, W, 1, 32>(a, quant, grad, grad_blocks, st);
    if (n <= 64) return norm_run<T, W, 2, 32>(a, quant, grad, grad_blocks, st);
    if (n <= 128) return norm_run<T, W, 4, 32>(a, quant, grad, grad_blocks, st);
    if (n <= 256) return norm_run<T, W, 1, 256>(a, quant, grad, grad_blocks, st);
    if (n <= 512) return norm_run<T, W, 2, 256>(a, quant, grad, grad_blocks, st);
    if (n <= 1024) return norm_run<T, W, 4, 256>(a, quant, grad, grad_blocks, st);
  } else {
    if (a.C <= 64) return norm_run<T, 1, 2, 32>(a, quant, grad, grad_blocks, st);
    if (a.C <= 256) return norm_run<T, 1, 8, 32>(a, quant, grad, grad_blocks, st);
    if (a.C <= 1024) return norm_run<T, 1, 4, 256>(a, quant, grad, grad_blocks, st);
    if (a.C <= 4096) return norm_run<T, 1, 16, 256>(a, quant, grad, grad_blocks, st);
  }
  if (grad) norm_grad_long_kernel<T><<<(unsigned)grad_blocks, kNormThreads, 0, st>>>(a);
  else if (a.rows >= (1ll << 31)) return FBEV_ERR_RANGE;
  else if (quant) norm_long_kernel<T, true><<<(unsigned)a.rows, kNormThreads, 0, st>>>(a);
  else norm_long_kernel<T, false><<<(unsigned)a.rows, kNormThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

static int norm_any(int dtype, const NormArgs& a, bool quant, bool grad, long long grad_blocks, cudaStream_t st) {
  switch (dtype) {
    case FBEV_F32: return norm_dispatch<float>(a, quant, grad, grad_blocks, st);
    case FBEV_BF16: return norm_dispatch<__nv_bfloat16>(a, quant, grad, grad_blocks, st);
    default: return norm_dispatch<__half>(a, quant, grad, grad_blocks, st);
  }
}

}  // namespace fbev
