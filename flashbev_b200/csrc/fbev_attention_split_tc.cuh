// Attention with float32 accuracy on the tensor cores, and for heads and strides that TMA cannot address.
//
// A float32 number is the sum of three bfloat16 numbers (8 significant bits each): x = x0 + x1 + x2.  A product of two
// tensors is then the sum of the products of their parts; those of the order of 2^-24 and less are left out, six remain:
//
//   x y = x0 y0 + (x0 y1 + x1 y0) + (x1 y1 + x0 y2 + x2 y0)
//
// split_kernel writes the parts of q, k, v (and grad_out) once, as [sample, key head][row][part][width] in 16 bits, rows
// being (query, head of the group) as in fbev_attention.cuh; keys that may not be attended become zeros there, so
// nothing of what stood in them travels on.  Four products of one shape follow, each by att_split_kernel:
//
//   out: X0 = Q, Y0 = K, Z = V      acc += P Z    P = 2^(c S - m), running maximum m
//   dV:  X0 = K, Y0 = Q, Z = dO     acc += P Z    P = 2^(c S - lse)
//   dQ:  X = (Q, dO), Y = (K, V), Z = K           acc += dS Z, dS = P (dP - delta)
//   dK:  X = (K, V), Y = (Q, dO), Z = Q           the same transposed
//
// with S = X0 Y0^T and dP = X1 Y1^T for a tile of 128 rows of X against the tiles of Y, in six products each.  P and dS
// are split into their parts by the threads that form them and are operands from tensor memory.
//
// The tensor cores cut an accumulator off after each instruction instead of rounding it.  Over many instructions that
// becomes a bias, so a tile's product starts from zero, the small products go first, and the sum over the tiles is kept
// by the threads in registers, rounded.  What is cut off is then 8 instructions' worth at full size, about 2^-22.
//
// All operands stream through a ring of four stages (128 rows x 64 of the width x 3 parts, 48 KiB) in the order in which
// they are used; X is fetched again for each tile (from L2), which keeps any width up to 128 within shared memory.
// Tensor memory, columns: S 0, dP 128 (then the first two parts of P or dS; each half of the warps over its own half of
// the columns), third part 256, product of the tile 320.
#pragma once
#include "fbev_attention.cuh"
#include "fbev_rotary.cuh"
#include "fbev_tc.cuh"

namespace fbev {

enum { kSplitOut = 0, kSplitDv = 1, kSplitDq = 2, kSplitDk = 3 };

struct SplitArgs {
  CUtensorMap x0, y0, x1, y1, z;
  FbevAttention p;
  int x_tiles, y_tiles;   // of a (sample, key head)
  int x_rows;
  int splits, per_split;  // blocks along Y and their tiles
  const float* allowed;   // [B][key tiles][128]: 0 or -infinity
  const float* nlse;      // -lse and -delta [B * Hkv][row tiles][128]; rows that are not there: -infinity and 0
  const float* ndelta;
  float* g;               // result
  float* lse;             // out: statistics or null
  float* part;            // or parts of it: with splits > 1, and for 16-bit types, whose results the next kernel rounds
  float* part_lse;        // out
  float c;
};

constexpr int kSplitStages = 4;
constexpr uint32_t kSplitStageBytes = 3 * kTileBytes;
constexpr uint32_t kSplitSmem = kSplitStages * kSplitStageBytes + 1024;

// parts (x, y) of the six products, the largest last
__device__ __forceinline__ int split_x(int i) { return i == 0 ? 2 : i == 1 ? 0 : i == 2 ? 1 : i == 3 ? 1 : 0; }
__device__ __forceinline__ int split_y(int i) { return i == 0 ? 0 : i == 1 ? 2 : i == 2 ? 1 : i == 3 ? 0 : i == 4 ? 1 : 0; }

// NC: 64-wide chunks of a head
template <int NC, int MODE>
__global__ void __launch_bounds__(kAttThreads, 1) att_split_kernel(const __grid_constant__ SplitArgs a) {
  constexpr bool kDs = MODE == kSplitDq || MODE == kSplitDk;       // dS, not P
  constexpr bool kKeyRows = MODE == kSplitDv || MODE == kSplitDk;  // X: keys
  constexpr int W = NC == 1 ? 32 : 64;                             // columns of the result that a thread keeps
  extern __shared__ unsigned char s_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * kSplitStages + 7];
  __shared__ float s_max[2][2][128];
  __shared__ float s_sum[128];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bail;

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int u = blockIdx.x;
  const int split = u % a.splits;
  u /= a.splits;
  const int xt = u % a.x_tiles, bg = u / a.x_tiles, b = bg / a.p.Hkv, g = bg % a.p.Hkv;
  const int keys = uniform(att_keys(a.p, b));
  const int t0 = split * a.per_split;
  int n = (kKeyRows ? (xt * 128 < keys ? a.y_tiles : 0) : (keys + 127) / 128) - t0;
  n = n < 0 ? 0 : n > a.per_split ? a.per_split : n;

  const uint32_t s_ring = (smem_addr(s_raw) + 1023) & ~1023u;
  const uint32_t bars = smem_addr(s_bar);
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (kSplitStages + s); };
  const uint32_t s_full = bars + 16 * kSplitStages, s_free = s_full + 8, dp_full = s_full + 16, p_full = s_full + 24,
                 r_full = s_full + 32, top_full = s_full + 40, drained = s_full + 48;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSplitStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 8);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 8);
    mbar_init(r_full, 1);
    mbar_init(top_full, 8);
    mbar_init(drained, 1);
    s_bail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) tmem_alloc<512>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns of the SM are this block's
  const Bail bail{&s_bail, a.p.status};
  grid_dependency_wait();  // the parts come from the kernels before

  if (warp >= 8) {
    set_registers_down<80>();
    if (warp == 8 && n > 0) {
      // ---- loads -------------------------------------------------------------------------------------------------
      int slot = 0;
      const auto load = [&](const CUtensorMap* map, int chunk, int tile) {
        const int s = slot % kSplitStages;
        if (slot >= kSplitStages) warp_wait(empty(s), ((slot / kSplitStages) - 1) & 1, bail);
        mbar_expect(full(s), kSplitStageBytes);
        tma_load_4d(s_ring + s * kSplitStageBytes, map, full(s), 64 * chunk, tile * 128, 0, bg);
        ++slot;
      };
      const auto load_scores = [&](int t) {
        for (int c = 0; c < NC; ++c) {
          load(&a.x0, c, xt);
          load(&a.y0, c, t0 + t);
        }
      };
      const auto load_dprobs = [&](int t) {
        for (int c = 0; c < NC; ++c) {
          load(&a.x1, c, xt);
          load(&a.y1, c, t0 + t);
        }
      };
      load_scores(0);
      if (kDs) load_dprobs(0);
      for (int t = 0; t < n ; ++t) {
        if (t + 1 < n) load_scores(t + 1);
        for (int c = 0; c < NC; ++c) load(&a.z, c, t0 + t);
        if (kDs && t + 1 < n) load_dprobs(t + 1);
      }
      if (__any_sync(kFull, *bail.flag != 0))  // nothing may be left in flight when the block ends
        for (int i = slot > kSplitStages ? slot - kSplitStages : 0; i < slot; ++i)
          mbar_drain(full(i % kSplitStages), (i / kSplitStages) & 1);
    } else if (warp == 9 && n > 0) {
      // ---- matrix instructions -----------------------------------------------------------------------------------
      const int ksteps = (a.p.D + 15) / 16;
      const uint32_t i_dp = umma_instr<__nv_bfloat16>(128, false, false);
      const uint32_t i_s = umma_instr<__nv_bfloat16>(128, false, a.p.scale < 0.0f);
      int slot = 0;
      const auto take = [&]() {
        const int s = slot % kSplitStages;
        warp_wait(full(s), (slot / kSplitStages) & 1, bail);
        ++slot;
        return s;
      };
      const auto product = [&](uint32_t d, uint32_t instr, uint32_t done) {  // X Y^T over the head's width
        for (int c = 0; c < NC; ++c) {
          const int sx = take(), sy = take();
          tc_fence_after();
          const uint64_t dx = desc_k_major(s_ring + sx * kSplitStageBytes), dy = desc_k_major(s_ring + sy * kSplitStageBytes);
#pragma unroll
          for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c * 4 + k < ksteps)
                umma_ss(d, dx + split_x(i) * (kTileBytes / 16) + 2 * k, dy + split_y(i) * (kTileBytes / 16) + 2 * k, instr, c + i + k > 0);
          umma_commit(empty(sx));
          umma_commit(empty(sy));
        }
        umma_commit(done);
      };
      const auto accumulate = [&]() {  // the parts in tensor memory times Z, from zero
        for (int c = 0; c < NC; ++c) {
          const int s = take();
          tc_fence_after();
          const int wide = ksteps * 16 - 64 * c;  // the last chunk may be narrow
          const uint32_t instr = umma_instr<__nv_bfloat16>(wide < 64 ? wide : 64, true, false);
          const uint64_t dz = desc_mn_major(s_ring + s * kSplitStageBytes);
#pragma unroll
          for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t half = k < 4 ? 0 : 1, at = 8 * (k & 3);
              const uint32_t px = split_x(i) == 2 ? tmem + 256 + 32 * half + at : tmem + 128 + 64 * half + 32 * split_x(i) + at;
              umma_ts(tmem + 320 + 64 * c, px, dz + split_y(i) * (kTileBytes / 16) + 128 * k, instr, i + k > 0);
            }
          umma_commit(empty(s));
        }
        umma_commit(r_full);
      };
      product(tmem, i_s, s_full);
      if (kDs) product(tmem + 128, i_dp, dp_full);
      for (int t = 0; t < n ; ++t) {
        if (t + 1 < n) {
          warp_wait(s_free, t & 1, bail);
          product(tmem, i_s, s_full);
        }
        warp_wait(p_full, t & 1, bail);
        accumulate();
        if (kDs && t + 1 < n) product(tmem + 128, i_dp, dp_full);
      }
      if (__any_sync(kFull, *bail.flag != 0)) {
        umma_commit(drained);
        mbar_drain(drained, 0);
      }
    }
  } else {
    // ---- P or dS, and the sum over the tiles ---------------------------------------------------------------------------
    set_registers_up<208>();
    const int h = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int row = xt * 128 + r;
    const bool live = row < a.x_rows;
    const long long key_tiles = kKeyRows ? a.x_tiles : a.y_tiles, row_tiles = kKeyRows ? a.y_tiles : a.x_tiles;
    // added to the scores along the columns, and to dP
    const float* col = kKeyRows ? a.nlse + ((long long)bg * row_tiles + t0) * 128 : a.allowed + ((long long)b * key_tiles + t0) * 128;
    const float* col_delta = kKeyRows ? a.ndelta + ((long long)bg * row_tiles + t0) * 128 : nullptr;
    const float nl = MODE == kSplitDq ? a.nlse[((long long)bg * row_tiles + xt) * 128 + r] : 0.0f;
    const float nd = MODE == kSplitDq ? a.ndelta[((long long)bg * row_tiles + xt) * 128 + r] : 0.0f;
    float acc[W];
#pragma unroll
    for (int x = 0; x < W; ++x) acc[x] = 0.0f;
    float m = -INFINITY, sum = 0.0f;
    const auto absorb = [&](int t, float f) {  // the product of tile t, then the factor to the next maximum
      warp_wait(r_full, t & 1, bail);
      tc_fence_after();
#pragma unroll
      for (int x = 0; x < W; x += 32) {
        float part[32];
        tmem_ld32(lanes + 320 + W * h + x, part);
        tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 32; ++y) acc[x + y] = (acc[x + y] + part[y]) * f;
      }
    };
    for (int t = 0; t < n; ++t) {
      warp_wait(s_full, t & 1, bail);
      tc_fence_after();
      float p[64];
      tmem_ld32(lanes + 64 * h, p);
      tmem_ld32(lanes + 64 * h + 32, p + 32);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      float back = 1.0f, top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 64; x += 4) {
        const float4 l = *reinterpret_cast<const float4*>(col + 128 * t + 64 * h + x);
        p[x] = fmaf(p[x], a.c, l.x + nl);
        p[x + 1] = fmaf(p[x + 1], a.c, l.y + nl);
        p[x + 2] = fmaf(p[x + 2], a.c, l.z + nl);
        p[x + 3] = fmaf(p[x + 3], a.c, l.w + nl);
        if (MODE == kSplitOut) top = fmaxf(fmaxf(top, fmaxf(p[x], p[x + 1])), fmaxf(p[x + 2], p[x + 3]));
      }
      float off = 0.0f;
      if (MODE == kSplitOut) {
        // the other half of the row's columns is in another warp
        s_max[t & 1][h][r] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(top_full);
        warp_wait(top_full, t & 1, bail);
        const float mn = fmaxf(m, fmaxf(top, s_max[t & 1][h ^ 1][r]));
        back = m == -INFINITY ? 0.0f : exp2_fast(m - mn);
        m = mn;
        off = mn == -INFINITY ? 0.0f : mn;
        sum *= back;
      }
      float some[4] = {};
#pragma unroll
      for (int x = 0; x < 64; ++x) {
        p[x] = exp2_fast(p[x] - off);
        if (MODE == kSplitOut) some[x & 3] += p[x];
      }
      sum += (some[0] + some[1]) + (some[2] + some[3]);
      if (kDs) {
        warp_wait(dp_full, t & 1, bail);
        tc_fence_after();
#pragma unroll
        for (int y = 0; y < 64; y += 32) {
          float dp[32];
          tmem_ld32(lanes + 128 + 64 * h + y, dp);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            float4 d = make_float4(nd, nd, nd, nd);
            if (kKeyRows) d = *reinterpret_cast<const float4*>(col_delta + 128 * t + 64 * h + y + x);
            p[y + x] *= dp[x] + d.x;
            p[y + x + 1] *= dp[x + 1] + d.y;
            p[y + x + 2] *= dp[x + 2] + d.z;
            p[y + x + 3] *= dp[x + 3] + d.w;
          }
        }
      }
      if (t > 0) {
        absorb(t - 1, back);
      }
      // three parts; what is left after each is exact
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        uint32_t packed[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          packed[x] = pack2<__nv_bfloat16>(p[2 * x], p[2 * x + 1]);
          p[2 * x] -= __uint_as_float(packed[x] << 16);
          p[2 * x + 1] -= __uint_as_float(packed[x] & 0xffff0000u);
        }
        tmem_st32(i == 2 ? lanes + 256 + 32 * h : lanes + 128 + 64 * h + 32 * i, packed);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (n > 0) absorb(n - 1, 1.0f);
    // ---- output --------------------------------------------------------------------------------------------------------
    float f = kDs ? a.p.scale : 1.0f;
    if (MODE == kSplitOut) {
      // each half has summed its own columns
      if (h == 1) s_sum[r] = sum;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (h == 0) {
        sum += s_sum[r];
        s_max[0][0][r] = sum;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      sum = s_max[0][0][r];
    }
    const bool parted = a.part != nullptr;
    bool lost = false;                                  // no score above -infinity though there are keys (as in fbev_attention_tc.cuh)
    bool none = MODE == kSplitDq && nl == -INFINITY;    // no keys; scores that are not numbers are NaN at masked keys too
    if (MODE == kSplitOut) {
      if (__any_sync(kFull, !(sum > 0.0f))) {
        bool seen = false;
        for (int j = lane; j < 128 * n; j += 32) seen = seen || col[j] == 0.0f;
        seen = __any_sync(kFull, seen);
        none = !seen;
        lost = seen && sum == 0.0f;
      }
      if (none) sum = 0.0f;
      f = lost && !parted ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    if (kDs && parted) f = 1.0f;  // the scale is applied to the sum of the parts
    if (live) {
      const int G = a.p.Hq / a.p.Hkv;
      bool zero = n == 0 || none;
      if (kKeyRows) zero = zero || a.allowed[((long long)b * key_tiles + xt) * 128 + r] != 0.0f;
      const long long heads = (long long)a.p.B * a.p.Hkv;
      const long long at = kKeyRows ? (((long long)b * a.p.Lk + row) * a.p.Hkv + g) * a.p.D
                                    : (((long long)b * a.p.Lq + row / G) * a.p.Hq + g * G + row % G) * a.p.D;
      // parts of out are laid out by row tile for the join, those of the gradients like the gradients
      float* part = a.part;
      if (parted) {
        if (MODE == kSplitOut) part += ((split * heads + bg) * a.x_tiles * 128 + row) * a.p.D;
        else part += split * (kKeyRows ? (long long)a.p.B * a.p.Lk * a.p.Hkv : (long long)a.p.B * a.p.Lq * a.p.Hq) * a.p.D + at;
      }
      float* dst = a.g + at;
      if (parted) dst = part;
#pragma unroll
      for (int x = 0; x < W; x += 4) {
        const int d = W * h + x;
        float v[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] = zero ? 0.0f : acc[x + y] * f;
        if (a.p.D % 4 == 0) {
          if (d < a.p.D) *reinterpret_cast<float4*>(dst + d) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (d + y < a.p.D) dst[d + y] = v[y];
        }
      }
      if (MODE == kSplitOut && h == 0) {
        const long long padded = att_rows_padded(a.p);
        if (parted) a.part_lse[(split * heads + bg) * a.x_tiles * 128 + row] = lost ? kLowest : sum == 0.0f ? -INFINITY : m + log2f(sum);
        else if (a.lse != nullptr) a.lse[bg * padded + row] = lost ? NAN : sum == 0.0f ? INFINITY : m + log2f(sum);
      }
    }
    tc_fence_before();
  }
  grid_dependency_trigger();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_free<512>(s_tmem);
  }
}

struct SplitSource {
  const void* src;          // T, strided [B, L, H, D]
  long long stride[3];
  int G;                    // heads folded into rows
  int L, shared;
  int whole;                // rows and strides of whole fours of elements at such addresses
  __nv_bfloat16* parts;     // [B * Hkv][L * G][3][width]
  int width;                // D rounded up to eight
  float* allowed;           // keys: [B][tiles][128], and the rows of keys that may not be attended are zeros
  // rows of grad_out: their statistics
  const void* out;
  const float* lse;
  float* nlse;
  float* ndelta;
};

struct SplitSet {
  SplitSource of[4];
  unsigned first[5];  // blocks of each
};

// The parts of all tensors in one launch: LANES (16, or 32 for heads above 64) a row, four elements a lane.  Bound by
// memory: 4 bytes in, 6 out per element.  Both directions of 2 x 32109 rows of 64: 34 us, 65 with a warp for each row, whole
// divisions of 64 bits and loads of single elements.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ FbevAttention p, const __grid_constant__ SplitSet set) {
  int which = 0;
  while (blockIdx.x >= set.first[which + 1]) ++which;
  const SplitSource& s = set.of[which];
  // all below 2^31; whole divisions of 64 bits would be most of the kernel
  const unsigned rows = (unsigned)s.L * (unsigned)s.G, tiles = (rows + 127) / 128,
                 unit = (blockIdx.x - set.first[which]) * (256 / LANES) + threadIdx.x / LANES;
  const unsigned tile = unit >> 7, bg = tile / tiles, row = unit - bg * tiles * 128;
  const int lane = threadIdx.x % LANES, D = p.D;
  grid_dependency_trigger();
  const unsigned b = bg / (unsigned)p.Hkv, l = row / (unsigned)s.G;
  const int g = (int)(bg - b * p.Hkv), h = g * s.G + (int)(row - l * s.G);
  bool there = row < rows;
  bool clear = false;
  if (s.allowed != nullptr) {
    const bool may = there && (int)row < att_keys(p, (int)b) && att_allowed(p, (int)b, (int)row);
    if (g == 0 && lane == 0) s.allowed[(long long)b * tiles * 128 + row] = may ? 0.0f : -INFINITY;
    clear = there && !may;
    there = may;
  }
  const bool mine = 4 * lane < s.width;
  Pack<T, 4> v, o;
  float x[4] = {};
  const bool dots = s.nlse != nullptr;
  if (there && mine) {
    const T* src = reinterpret_cast<const T*>(s.src) + (s.shared ? 0 : b * s.stride[0]) + l * s.stride[1] + h * s.stride[2] + 4 * lane;
    const T* out = reinterpret_cast<const T*>(s.out) + (((long long)b * p.Lq + l) * p.Hq + h) * D + 4 * lane;
    if (s.whole) {  // four elements at once
      if (4 * lane < D) {
        v = *reinterpret_cast<const Pack<T, 4>*>(src);
        if (dots) o = *reinterpret_cast<const Pack<T, 4>*>(out);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * lane + i < D) {
          v.v[i] = src[i];
          if (dots) o.v[i] = out[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lane + i < D) x[i] = to_float(v.v[i]);
  }
  if (dots) {
    float d = 0.0f;
    if (there && mine) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * lane + i < D) d = fmaf(x[i], to_float(o.v[i]), d);
    }
#pragma unroll
    for (int k = LANES / 2; k > 0; k >>= 1) d += __shfl_xor_sync(kFull, d, k);
    if (lane == 0) {
      s.nlse[unit] = there ? -s.lse[bg * att_rows_padded(p) + row] : -INFINITY;
      s.ndelta[unit] = -d;
    }
  }
  if (!(there || clear) || !mine) return;
  __nv_bfloat16* parts = s.parts + ((long long)bg * rows + row) * 3 * s.width + 4 * lane;
#pragma unroll
  for (int i = 0; i < 3; ++i) {  // zeros where a key is cleared
    uint2 w;
    w.x = pack2<__nv_bfloat16>(x[0], x[1]);
    w.y = pack2<__nv_bfloat16>(x[2], x[3]);
    *reinterpret_cast<uint2*>(parts + i * s.width) = w;
    x[0] -= __uint_as_float(w.x << 16);
    x[1] -= __uint_as_float(w.x & 0xffff0000u);
    x[2] -= __uint_as_float(w.y << 16);
    x[3] -= __uint_as_float(w.y & 0xffff0000u);
  }
}

}  // namespace fbev
