// Rotary positions with several axes.
//
// A block owns TB tokens.  It first leaves cos and sin of its tokens' angles in shared memory, one (token, pair) per
// thread and turn, then rotates the tokens' heads from there: an angle is evaluated once per token and pair, not once
// per head, and the element loop is loads, four multiply-adds per pair and stores.
//
// Angles.  positions * 2 pi * turns is needed modulo 2 pi.  A float32 product would lose the fraction of a turn once a
// position is large (at 10^5 a float32 step is 2^-7), so the product is formed in float64 in units of turns, its
// integer part is taken off exactly, and only the remainder (|t| <= 1/2) is rounded to float32 for sincospif.  What float64
// rounds on the way (the exponent -j / S, which weighs ln(base) times, the frequency, the product) is at most
// |angle| * 2^-49 for a base of 10^4: below float32's own rounding up to angles of 2^24.
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

// n / d for n < 2^31 by a multiplication: mul = ceil(2^(32 + s) / d) with 2^s >= d > 2^(s-1)
struct Divisor {
  unsigned d, mul, shift;
};
static Divisor make_divisor(unsigned d) {
  unsigned s = 0;
  while ((1ull << s) < d) ++s;
  return Divisor{d, (unsigned)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ unsigned divide(unsigned n, const Divisor& v) { return (unsigned)(((unsigned long long)__umulhi(n, v.mul) + n) >> v.shift); }

template <typename T, typename P, int VE, bool INTER>
__global__ void __launch_bounds__(kRotaryThreads)
    rotary_kernel(const __grid_constant__ FbevRotary p, T* __restrict__ out, int TB, const Divisor by_head, const Divisor by_heads,
                  const Divisor by_pairs) {
  extern __shared__ float2 s_cs[];  // [TB][pairs]: cos, sin
  const long long tokens = (long long)p.B * p.L;
  const long long t0 = (long long)blockIdx.x * TB;
  const int nt = (int)(tokens - t0 < TB ? tokens - t0 : TB);
  const T* x = reinterpret_cast<const T*>(p.x);
  // chunks of a head: rotated ones (a chunk of the split layout covers VE elements of both halves), then copied ones
  const int rot = INTER ? 2 * p.pairs / VE : p.pairs / VE;
  const int per_head = rot + (p.D - 2 * p.pairs) / VE;
  const int items = nt * p.H * per_head;

  // sample and position of the block's first token; the others follow, wrapping into the next samples (whole divisions of
  // 64 bits for every chunk cost more than all the rest: 85 us against 54 on 160000 tokens of 8 x 32 floats)
  const long long b0 = t0 / p.L;
  const int l0 = (int)(t0 - b0 * p.L);
  const auto place = [&](int tok, long long& bb, int& l) {
    bb = b0;
    l = l0 + tok;
    while (l >= p.L) {
      l -= p.L;
      ++bb;
    }
  };
  T* dst[kRotaryItems];
  int tok[kRotaryItems], ch[kRotaryItems];
  Pack<T, VE> a[kRotaryItems], b[kRotaryItems];
  auto fetch = [&](int k, int i) {
    const int th = (int)divide(i, by_head);
    ch[k] = i - th * per_head;
    tok[k] = (int)divide(th, by_heads);
    const int h = th - tok[k] * p.H;
    long long bb;
    int l;
    place(tok[k], bb, l);
    const T* src = x + bb * p.x_stride[0] + l * p.x_stride[1] + h * p.x_stride[2];
    dst[k] = out + ((t0 + tok[k]) * p.H + h) * p.D;
    const int at = ch[k] < rot ? ch[k] * VE : 2 * p.pairs + (ch[k] - rot) * VE;
    a[k] = *reinterpret_cast<const Pack<T, VE>*>(src + at);
    if (!INTER && ch[k] < rot) b[k] = *reinterpret_cast<const Pack<T, VE>*>(src + p.pairs + at);
  };
  // the first chunks travel while the angles are evaluated
#pragma unroll
  for (int k = 0; k < kRotaryItems; ++k) {
    const int i = threadIdx.x + k * kRotaryThreads;
    if (i < items) fetch(k, i);
  }
  const P* pos = reinterpret_cast<const P*>(p.positions);
  for (int i = threadIdx.x; i < nt * p.pairs; i += kRotaryThreads) {
    const int lt = (int)divide(i, by_pairs), pr = i - lt * p.pairs;
    long long bb;
    int l;
    place(lt, bb, l);
    double turns = (double)pos[bb * p.pos_stride + (long long)l * p.axes + p.pair_axis[pr]] * p.pair_turns[pr];
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
  const Divisor by_head = make_divisor(per_head), by_heads = make_divisor(p->H), by_pairs = make_divisor(p->pairs > 0 ? p->pairs : 1);
  if (p->interleaved) {
    if constexpr (VE >= 2) rotary_kernel<T, P, VE, true><<<(unsigned)blocks, kRotaryThreads, smem, st>>>(*p, out, (int)tb, by_head, by_heads, by_pairs);
  } else {
    rotary_kernel<T, P, VE, false><<<(unsigned)blocks, kRotaryThreads, smem, st>>>(*p, out, (int)tb, by_head, by_heads, by_pairs);
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
    const int size[3] = {p->B, p->L, p->H};  // the stride of a dimension of one is never used
    for (int i = 0; i < 3; ++i) ok = ok && (size[i] == 1 || p->x_stride[i] % ve == 0);
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
