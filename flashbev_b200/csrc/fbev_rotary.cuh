// Rotary positions with several axes.
//
// A block owns TB tokens.  It first leaves cos and sin of its tokens' angles in shared memory, one (token, pair) per
// thread and turn, then rotates the tokens' heads from there: an angle is evaluated once per token and pair, not once
// per head, and the element loop is loads, four multiply-adds per pair and stores.
//
// Angles.  positions * 2 pi * turns is needed modulo 2 pi.  A float32 product would lose the fraction of a turn once a
// position is large (at 10^5 a float32 step is 2^-7), so the product is formed in float64 in units of turns, its
// integer part is taken off exactly, and only the remainder (|t| <= 1/2) is rounded to float32 for sincospif.
//
// Bound by memory: each element is read and written once.
#pragma once
#include "fbev_device.cuh"
#include "fbev_query.h"

namespace fbev {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryItems = 4;  // chunks a thread has in flight

// VE consecutive elements of T as they lie in memory
template <typename T, int VE>
struct alignas(sizeof(T) * VE) Pack {
  T v[VE];
};

template <typename T, typename P, int VE, bool INTER>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ FbevRotary p, T* __restrict__ out, int TB) {
  extern __shared__ float2 s_cs[];  // [TB][pairs]: cos, sin
  const long long tokens = (long long)p.B * p.L;
  const long long t0 = (long long)blockIdx.x * TB;
  const int nt = (int)(tokens - t0 < TB ? tokens - t0 : TB);
  const T* x = reinterpret_cast<const T*>(p.x);
  // chunks of a head: rotated ones (a chunk of the split layout covers VE elements of both halves), then copied ones
  const int rot = INTER ? 2 * p.pairs / VE : p.pairs / VE;
  const int per_head = rot + (p.D - 2 * p.pairs) / VE;
  const int items = nt * p.H * per_head;

  const T* src[kRotaryItems];
  T* dst[kRotaryItems];
  int tok[kRotaryItems], ch[kRotaryItems];
  Pack<T, VE> a[kRotaryItems], b[kRotaryItems];
  auto fetch = [&](int k, int i) {
    ch[k] = i % per_head;
    const int th = i / per_head;
    tok[k] = th / p.H;
    const int h = th - tok[k] * p.H;
    const long long t = t0 + tok[k];
    const long long bb = t / p.L, l = t - bb * p.L;
    src[k] = x + bb * p.x_stride[0] + l * p.x_stride[1] + h * p.x_stride[2];
    dst[k] = out + (t * p.H + h) * p.D;
    const int at = ch[k] < rot ? ch[k] * VE : 2 * p.pairs + (ch[k] - rot) * VE;
    a[k] = *reinterpret_cast<const Pack<T, VE>*>(src[k] + at);
    if (!INTER && ch[k] < rot) b[k] = *reinterpret_cast<const Pack<T, VE>*>(src[k] + p.pairs + at);
  };
  // the first chunks travel while the angles are evaluated
#pragma unroll
  for (int k = 0; k < kRotaryItems; ++k) {
    const int i = threadIdx.x + k * kRotaryThreads;
    if (i < items) fetch(k, i);
  }
  const P* pos = reinterpret_cast<const P*>(p.positions);
  for (int i = threadIdx.x; i < nt * p.pairs; i += kRotaryThreads) {
    const int lt = i / p.pairs, pr = i - lt * p.pairs;
    const long long t = t0 + lt, bb = t / p.L, l = t - bb * p.L;
    double turns = (double)pos[bb * p.pos_stride + l * p.axes + p.pair_axis[pr]] * p.pair_turns[pr];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    s_cs[i] = make_float2(c, p.inverse ? -s : s);
  }
  __syncthreads();
  for (int base = 0; base < items; base += kRotaryItems * kRotaryThreads) {
#pragma unroll
    for (int k = 0; k < kRotaryItems; ++k) {
      const int i = base + threadIdx.x + k * kRotaryThreads;
      if (i >= items) continue;
      if (base > 0) fetch(k, i);
      if (ch[k] >= rot) {
        *reinterpret_cast<Pack<T, VE>*>(dst[k] + 2 * p.pairs + (ch[k] - rot) * VE) = a[k];
        continue;
      }
      const int at = ch[k] * VE;
      const float2* cs = s_cs + tok[k] * p.pairs + (INTER ? at / 2 : at);
      if (INTER) {
#pragma unroll
        for (int e = 0; e + 1 < VE; e += 2) {
          const float2 w = cs[e / 2];
          const float u = to_float(a[k].v[e]), v = to_float(a[k].v[e + 1]);
          a[k].v[e] = from_float<T>(u * w.x - v * w.y);
          a[k].v[e + 1] = from_float<T>(u * w.y + v * w.x);
        }
        *reinterpret_cast<Pack<T, VE>*>(dst[k] + at) = a[k];
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float2 w = cs[e];
          const float u = to_float(a[k].v[e]), v = to_float(b[k].v[e]);
          a[k].v[e] = from_float<T>(u * w.x - v * w.y);
          b[k].v[e] = from_float<T>(u * w.y + v * w.x);
        }
        *reinterpret_cast<Pack<T, VE>*>(dst[k] + at) = a[k];
        *reinterpret_cast<Pack<T, VE>*>(dst[k] + p.pairs + at) = b[k];
      }
    }
  }
}

template <typename T, typename P, int VE>
static int rotary_launch_ve(const FbevRotary* p, T* out, cudaStream_t st) {
  const int per_head = (p->interleaved ? 2 * p->pairs : p->pairs) / VE + (p->D - 2 * p->pairs) / VE;
  const long long tokens = (long long)p->B * p->L, item_tok = (long long)p->H * per_head;
  // enough tokens for four chunks a thread and a bounded table; fewer when that would leave SMs without a block
  long long tb = kRotaryItems * kRotaryThreads / item_tok;
  const long long table = 2048 / (p->pairs > 0 ? p->pairs : 1);
  if (tb > table) tb = table;
  const long long spread = (tokens + 148 * 2 - 1) / (148 * 2);
  if (tb > spread) tb = spread;
  if (tb < 1) tb = 1;
  if (tb * item_tok >= (1ll << 30)) return FBEV_ERR_RANGE;
  const long long blocks = (tokens + tb - 1) / tb;
  if (blocks >= (1ll << 31)) return FBEV_ERR_RANGE;
  const size_t smem = (size_t)tb * p->pairs * sizeof(float2);
  if (p->interleaved) {
    if constexpr (VE >= 2) rotary_kernel<T, P, VE, true><<<(unsigned)blocks, kRotaryThreads, smem, st>>>(*p, out, (int)tb);
  } else {
    rotary_kernel<T, P, VE, false><<<(unsigned)blocks, kRotaryThreads, smem, st>>>(*p, out, (int)tb);
  }
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T, typename P>
static int rotary_launch(const FbevRotary* p, T* out, cudaStream_t st) {
  // the widest chunk that divides the halves, the copied rest, the strides and the addresses
  constexpr int kWide = 16 / sizeof(T);
  const auto fits = [&](int ve) {
    const int unit = p->interleaved ? 2 * p->pairs : p->pairs;
    bool ok = unit % ve == 0 && (p->D - 2 * p->pairs) % ve == 0 && p->D % ve == 0;
    for (int i = 0; i < 3; ++i) ok = ok && p->x_stride[i] % ve == 0;
    return ok && (uintptr_t)p->x % (ve * sizeof(T)) == 0 && (uintptr_t)out % (ve * sizeof(T)) == 0;
  };
  if (fits(kWide)) return rotary_launch_ve<T, P, kWide>(p, out, st);
  if (fits(kWide / 2)) return rotary_launch_ve<T, P, kWide / 2>(p, out, st);
  if (p->interleaved) {
    if (fits(2)) return rotary_launch_ve<T, P, 2>(p, out, st);
    return FBEV_ERR_ALIGN;  // interleaved pairs are loaded whole
  }
  return rotary_launch_ve<T, P, 1>(p, out, st);
}

template <typename T>
static int rotary_pos(const FbevRotary* p, void* out, cudaStream_t st) {
  switch (p->pos_dtype) {
    case FBEV_POS_F32: return rotary_launch<T, float>(p, reinterpret_cast<T*>(out), st);
    case FBEV_POS_I32: return rotary_launch<T, int32_t>(p, reinterpret_cast<T*>(out), st);
    default: return rotary_launch<T, int64_t>(p, reinterpret_cast<T*>(out), st);
  }
}

}  // namespace fbev
