// Attention on the tensor cores, 16-bit types.
//
// Forward.  A block owns up to two tiles of 128 rows (rows as in fbev_attention.cuh: query and head of the group) of one
// sample and key head, and a range of key tiles of 128.  Per row tile and key tile, base 2 and with c = scale * log2 e:
//
//   S = Q K^T             operands in shared memory, 128 x 128 float32 accumulator in tensor memory
//   P = 2^(c S - m)       one thread per row: tensor memory -> registers -> 16 bits, written over S
//   O += P V              P from tensor memory, V from shared memory (read across its rows), accumulator in tensor memory
//
// Roles: eight softmax warps (two groups of four, one per row tile), a warp that loads by TMA, a warp that issues the
// matrix instructions, a warp that reads the key mask and clears values that may not be attended.  Step q of a block is key
// tile q / 2 of row tile q % 2 (one row tile: q of that).  The scores of steps q + 1 .. q + kBufs - 1 are formed while a
// softmax group works on step q; P V of step q and the scores of step q + kBufs, which take P's place, follow.  With heads
// up to 64 wide tensor memory holds three score tiles, so a group finds its next one ready; with two it waits for both
// products.
//
// NaN scores do not raise the maximum, they show in the sum, from where they reach the output and the statistics.  A row whose
// keys all score -infinity has the statistic kLowest instead of the -infinity of a row without keys: its output is NaN, as a
// quotient of zeros, while the latter's is zero; of several parts of a row only those above it count.
//
// m is the row's running maximum, raised only when a tile exceeds it by more than 8: weights then stay below 2^8 (no loss
// in either type, both sides of the quotient carry the same factor) and the output, which lives in tensor memory, is
// rescaled in a few of the first tiles only.
//
// Few rows (one row tile): both groups take the same rows, one the even and one the odd key tiles, and join in shared
// memory at the end.  Whenever the row tiles leave SMs without a block the key tiles are split over several blocks, which
// leave normalised float32 outputs and their logarithmic sums for att_join_kernel.
//
// Tensor memory, columns: S/P tiles from 0 (128 each), O of the two groups behind them (64 or 128 each).
//
// Bound by the exponentials and what surrounds them in the softmax warps with heads of 64 (2 x 8100 queries x 5400 keys x 8
// heads: 235 us, 750 TFLOP/s; the unit for exponentials alone would need 150 us), by the tensor cores with heads of 128
// (2 x 8100 x 8448 x 8: 520 us, 1.09 PFLOP/s), by the memory's rate with one query a sample (64 samples, lengths up to
// 16384: 150 us, 84 % of the copy rate).
#pragma once
#include "fbev_attention.cuh"
#include "fbev_tc.cuh"

namespace fbev {

struct AttPlan {
  int G, TL;           // heads of a group, queries in a row tile (TL * G <= 128 rows)
  int row_tiles;       // of a (sample, key head)
  int pair;            // one row tile, even and odd key tiles
  int row_blocks;      // units along the rows: up to two row tiles each
  // The first `whole` units (of all samples and key heads) are a block each; each of the others is split along the keys
  // over `splits` blocks of `per_split` key tiles.
  int whole, splits, per_split;
};

struct AttFwdArgs {
  CUtensorMap q, k, v;
  FbevAttention p;
  AttPlan pl;
  void* out;
  float* lse;       // final statistics or null
  float* part;      // [splits][split units][256 rows][D]
  float* part_lse;  // [splits][split units][256 rows]
  float c;          // |scale| * log2 e
};

template <int NSUB>
struct AttFwdShape {
  static constexpr int kBufs = NSUB == 1 ? 3 : 2;      // score tiles in tensor memory
  // with two score tiles a group waits for P V and the next scores: P V then begins at half of P
  static constexpr bool kHalves = kBufs == 2;
  static constexpr int kOutAt = 128 * kBufs, kOutCols = NSUB == 1 ? 64 : 128;
  static constexpr int kStages = NSUB == 1 ? 10 : 5;
  static constexpr uint32_t kStageBytes = NSUB * kTileBytes;
  static constexpr uint32_t kSmem = 2 * kStageBytes + kStages * kStageBytes + 1024;
};

// 2^x of two numbers on the multiply-add pipe, for weights that are rounded to 16 bits: x = n + f with n whole and
// |f| <= 1/2, 2^f by the cubic with the least largest relative error on that interval (2^-13.7, Remez exchange), times 2^n,
// whose bits the rounding of x leaves in place: a product, not an addition to the exponent, so that NaN stays NaN.  The unit
// for exponentials takes 16 a clock and SM, a quarter of what it would have to take to keep pace with the rest of the
// softmax; a part of the weights goes this way instead.  What is below 2^-126 becomes 2^-126: a score of -infinity leaves a
// weight that no sum notices, and rows without any key are told by their keys.
//
// How many of eight pairs: 0, 1, 2, 3, 4 gave 258, 244, 246, 248, 276 us in the forward at 2 x 8100 queries x 5400 keys x 8
// heads of 64, and 522, 522, 526, 533, 555 us at 2 x 8100 x 8448 x 8 heads of 128.  In the gradients 2 and 3 gave 613 and
// 625 us at 2 x 10000 queries x 4224 keys x 8 heads on 4 of 64 (603 with 3 and the addition to the exponent), 607 and 615 us
// with 4 heads of 128.
constexpr int kPolyForward = 1, kPolyGrad = 2;
// eight pairs at once; the steps of the cubics side by side, the other exponentials between them
template <int OF8>
__device__ __forceinline__ void exp2_run(float2 (&x)[8]) {
  constexpr int K = OF8 > 0 ? OF8 : 1;
  float2 r[K], f[K], p[K];
  const auto unit = [&](int i) { x[i] = make_float2(exp2_fast(x[i].x), exp2_fast(x[i].y)); };
  const auto between = [&](int stage) {  // pairs OF8 .. 7, spread over six stages
#pragma unroll
    for (int i = OF8; i < 8; ++i)
      if ((i - OF8) * 6 / (8 - OF8) == stage) unit(i);
  };
  between(0);
#pragma unroll
  for (int i = 0; i < OF8; ++i) {
    x[i] = make_float2(max_nan(x[i].x, -126.0f), max_nan(x[i].y, -126.0f));
    r[i] = add2(x[i], make_float2(12583039.0f, 12583039.0f));  // 1.5 * 2^23 + 127: n + 127 in the low bits
  }
  between(1);
#pragma unroll
  for (int i = 0; i < OF8; ++i) {
    const float2 n = add2(r[i], make_float2(-12583039.0f, -12583039.0f));
    f[i] = fma2(n, make_float2(-1.0f, -1.0f), x[i]);
  }
  between(2);
#pragma unroll
  for (int i = 0; i < OF8; ++i) p[i] = fma2(f[i], make_float2(0.05517167f, 0.05517167f), make_float2(0.24261113f, 0.24261113f));
  between(3);
#pragma unroll
  for (int i = 0; i < OF8; ++i) p[i] = fma2(p[i], f[i], make_float2(0.69326097f, 0.69326097f));
  between(4);
#pragma unroll
  for (int i = 0; i < OF8; ++i) p[i] = fma2(p[i], f[i], make_float2(0.99992806f, 0.99992806f));
  between(5);
#pragma unroll
  for (int i = 0; i < OF8; ++i)
    x[i] = mul2(p[i], make_float2(__uint_as_float(__float_as_uint(r[i].x) << 23), __uint_as_float(__float_as_uint(r[i].y) << 23)));
}

constexpr int kMaskRing = 4;
constexpr int kAttThreads = 384;

// O and statistics of one row leave: rounded to T, or float32 with the base-2 logarithm of the sum for the join
template <typename T>
__device__ __forceinline__ void store_row16(T* dst, const float* o, float f, int n) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (i >= n) break;
    uint4 w;
    w.x = pack2<T>(o[i] * f, o[i + 1] * f);
    w.y = pack2<T>(o[i + 2] * f, o[i + 3] * f);
    w.z = pack2<T>(o[i + 4] * f, o[i + 5] * f);
    w.w = pack2<T>(o[i + 6] * f, o[i + 7] * f);
    *reinterpret_cast<uint4*>(dst + i) = w;
  }
}
__device__ __forceinline__ void store_row32(float* dst, const float* o, float f, int n) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    if (i >= n) break;
    *reinterpret_cast<float4*>(dst + i) = make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
  }
}

template <typename T, int NSUB>
__global__ void __launch_bounds__(kAttThreads, 1) att_fwd_kernel(const __grid_constant__ AttFwdArgs a) {
  using Shape = AttFwdShape<NSUB>;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kStageBytes = Shape::kStageBytes;
  extern __shared__ unsigned char s_raw[];
  constexpr int kBufs = Shape::kBufs;
  __shared__ __align__(8) uint64_t s_bar[3 * kStages + 3 * kBufs + 6 + 2 * kMaskRing];
  __shared__ uint32_t s_mask[kMaskRing][4];
  __shared__ float s_stat[2][128];
  __shared__ uint8_t s_list[kSkipTiles];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bail, s_count;

  const AttPlan& pl = a.pl;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // block -> (split, row block, sample, key head); row blocks of one key head are neighbours and share its keys in L2
  int u = blockIdx.x, split = 0;
  const bool parted = u >= pl.whole;
  if (parted) {
    split = (u - pl.whole) % pl.splits;
    u = pl.whole + (u - pl.whole) / pl.splits;
  }
  const int rb = u % pl.row_blocks;
  const int bg = u / pl.row_blocks, b = bg / a.p.Hkv, g = bg % a.p.Hkv;
  const int keys = uniform(att_keys(a.p, b));
  const int t0 = split * pl.per_split;
  int n = (keys + 127) / 128 - t0;  // key tiles of this block
  n = n < 0 ? 0 : parted && n > pl.per_split ? pl.per_split : n;
  const bool pair = pl.pair != 0;
  const int tiles = pair ? 1 : (pl.row_tiles - 2 * rb < 2 ? 1 : 2);  // row tiles of this block
  const bool masked = a.p.key_mask != nullptr;
  const bool skips = masked && n > 0 && n <= kSkipTiles;
  if (skips) n = uniform(att_tiles_left<kAttThreads / 32>(a.p.key_mask + (long long)b * a.p.mask_stride, keys, t0, n, s_list, &s_count));
  const auto key_tile = [&](int t) { return t0 + (skips ? uniform(s_list[t]) : t); };
  const long long rows = att_rows(a.p);
  const int tile_rows = pl.TL * pl.G;

  const uint32_t smem = (smem_addr(s_raw) + 1023) & ~1023u;
  const uint32_t s_q = smem, s_ring = smem + 2 * kStageBytes;
  const uint32_t bars = smem_addr(s_bar);
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (kStages + s); };
  const auto fixed = [&](int s) { return bars + 8 * (2 * kStages + s); };
  const uint32_t q_full = bars + 8 * (3 * kStages), drained = q_full + 8;
  const auto o_full = [&](int i) { return q_full + 16 + 8 * i; };  // the group's last product is done
  // the product of each step, by two barriers in turn.  A barrier tells only its last phase from the one before: who waits for
  // the step before its own has to know of the product two phases back.  The scores it holds came after the product kBufs
  // steps ago, and two steps are one phase.
  const auto o_step = [&](int q) { return q_full + 32 + 8 * (q & 1); };
  const auto s_full = [&](int i) { return q_full + 48 + 8 * i; };
  const auto p_half = [&](int i) { return q_full + 48 + 8 * (kBufs + i); };
  const auto p_full = [&](int i) { return q_full + 48 + 8 * (2 * kBufs + i); };
  const auto m_full = [&](int i) { return q_full + 48 + 8 * (3 * kBufs + i); };
  const auto m_empty = [&](int i) { return q_full + 48 + 8 * (3 * kBufs + kMaskRing + i); };

  // softmax warps with rows to work on: all four of a group, fewer when the only row tile is short
  const long long left = rows - (long long)(pair ? 0 : 2 * rb) * tile_rows;
  const int live_rows = pair ? (int)(left < tile_rows ? left : tile_rows) : 128;
  const int live_warps = (live_rows + 31) / 32;

  // The warp that clears values follows the ring tile by tile and has to let go of each stage too: a barrier tells only
  // the last phase from the one before, so no one may fall a round behind.
  const bool fixes = masked || keys < a.p.Lk;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), fixes ? 2 : 1);
      mbar_init(fixed(s), 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(o_full(i), 1);
      mbar_init(o_step(i), 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_half(i), live_warps);
      mbar_init(p_full(i), live_warps);
    }
    for (int i = 0; i < kMaskRing; ++i) {
      mbar_init(m_full(i), 1);
      mbar_init(m_empty(i), pair ? live_warps : 4 * tiles);
    }
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
  // a tile whose values have to be cleared in places: masked, or cut off by the sample's length inside the tensor
  const auto needs_fix = [&](int t) { return masked || ((t0 + t + 1) * 128 > keys && keys < a.p.Lk); };

  // steps, and which of them take a new tile of keys (the order of the ring: keys of the first kBufs steps, then the values
  // of step q and the keys of step q + kBufs in turn)
  const int streams = pair ? 2 : tiles, steps = pair ? n : n * tiles;
  const auto tile_of = [&](int q) { return pair || streams == 1 ? q : q >> 1; };
  const auto stream_of = [&](int q) { return streams == 1 ? 0 : q & 1; };
  const auto new_tile = [&](int q) { return pair || streams == 1 || (q & 1) == 0; };

  if (warp >= 8) {
    set_registers_down<80>();
    if (warp == 8 && n > 0) {
      // ---- loads -------------------------------------------------------------------------------------------------
      mbar_expect(q_full, (uint32_t)(tiles * NSUB * tile_rows * 128));
      for (int i = 0; i < tiles; ++i)
        for (int x = 0; x < NSUB; ++x)
          tma_load_5d(s_q + i * kStageBytes + x * kTileBytes, &a.q, q_full, 64 * x, 0, g, (2 * rb + i) * pl.TL, a.p.q_shared ? 0 : b);
      int slot = 0;
      const auto load = [&](const CUtensorMap* map, int t) {
        const int s = slot % kStages;
        if (slot >= kStages) warp_wait(empty(s), ((slot / kStages) - 1) & 1, bail);
        mbar_expect(full(s), kStageBytes);
        const int tile = key_tile(t);
        for (int x = 0; x < NSUB; ++x)
          tma_load_4d(s_ring + s * kStageBytes + x * kTileBytes, map, full(s), 64 * x, g, tile * 128, b);
        ++slot;
      };
      for (int q = 0; q < kBufs && q < steps; ++q)
        if (new_tile(q)) load(&a.k, tile_of(q));
      for (int q = 0; q < steps; ++q) {
        if (new_tile(q)) load(&a.v, tile_of(q));
        if (q + kBufs < steps && new_tile(q + kBufs)) load(&a.k, tile_of(q + kBufs));
      }
      if (__any_sync(kFull, *bail.flag != 0)) {
        // nothing may be left in flight when the block ends
        mbar_drain(q_full, 0);
        for (int i = slot > kStages ? slot - kStages : 0; i < slot; ++i) mbar_drain(full(i % kStages), (i / kStages) & 1);
      }
    } else if (warp == 9 && n > 0) {
      // ---- matrix instructions -----------------------------------------------------------------------------------
      const bool negative = a.p.scale < 0.0f;
      const int ksteps = (a.p.D + 15) / 16;
      const uint32_t i_s = umma_instr<T>(128, false, negative), i_o = umma_instr<T>(ksteps * 16, true, false);
      uint32_t fix_parity = 0;
      int slot = 0;
      warp_wait(q_full, 0, bail);
      const auto take = [&]() {  // next tile of the ring
        const int s = slot % kStages;
        warp_wait(full(s), (slot / kStages) & 1, bail);
        ++slot;
        return s;
      };
      const auto scores = [&](int q, int s) {
        tc_fence_after();
        const uint32_t d = tmem + 128 * (q % kBufs);
#pragma unroll
        for (int x = 0; x < NSUB; ++x) {
          const uint64_t da = desc_k_major(s_q + (pair ? 0 : stream_of(q)) * kStageBytes + x * kTileBytes);
          const uint64_t db = desc_k_major(s_ring + s * kStageBytes + x * kTileBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (x * 4 + k < ksteps) umma_ss(d, da + 2 * k, db + 2 * k, i_s, x + k > 0);
        }
        umma_commit(s_full(q % kBufs));
      };
      const auto values = [&](int q, int s, int half, bool first) {  // half of the keys
        tc_fence_after();
        const uint64_t db = desc_mn_major(s_ring + s * kStageBytes);
        const uint32_t d = tmem + Shape::kOutAt + Shape::kOutCols * stream_of(q), p = tmem + 128 * (q % kBufs);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int kk = 4 * half + k;
          umma_ts(d, p + 8 * kk, db + 128 * kk, i_o, !first || kk > 0);
        }
      };
      const auto fix_wait = [&](int t, int s) {
        if (!needs_fix(t)) return;
        warp_wait(fixed(s), (fix_parity >> s) & 1, bail);
        fix_parity ^= 1u << s;
      };
      int sk = 0, sv = 0;
      const auto last_use = [&](int q) { return pair || streams == 1 || (q & 1) == 1; };  // of the tile of keys or values
      for (int q = 0; q < kBufs && q < steps; ++q) {
        if (new_tile(q)) sk = take();
        scores(q, sk);
        if (last_use(q)) umma_commit(empty(sk));
      }
      for (int q = 0; q < steps; ++q) {
        const int i = stream_of(q), buf = q % kBufs, parity = (q / kBufs) & 1;
        if (new_tile(q)) {
          sv = take();
          fix_wait(tile_of(q), sv);
        }
        const bool more = q + kBufs < steps;
        if (more && new_tile(q + kBufs)) sk = take();
        if (Shape::kHalves) {
          warp_wait(p_half(buf), parity, bail);
          values(q, sv, 0, q < streams);
        }
        warp_wait(p_full(buf), parity, bail);
        if (!Shape::kHalves) values(q, sv, 0, q < streams);
        values(q, sv, 1, false);
        umma_commit(o_step(q));
        if (q + streams >= steps) umma_commit(o_full(i));
        if (last_use(q)) umma_commit(empty(sv));
        if (more) {
          scores(q + kBufs, sk);
          if (last_use(q + kBufs)) umma_commit(empty(sk));
        }
      }
      if (__any_sync(kFull, *bail.flag != 0)) {
        umma_commit(drained);
        mbar_drain(drained, 0);
      }
    } else if (warp == 10 && n > 0 && fixes) {
      // ---- key mask, values that may not be attended ---------------------------------------------------------------
      const uint8_t* mask = masked ? a.p.key_mask + (long long)b * a.p.mask_stride : nullptr;
      int slot = 0;
      const auto follow = [&]() {  // the next stage of the ring, once it is loaded
        const int s = slot % kStages;
        warp_wait(full(s), (slot / kStages) & 1, bail);
        ++slot;
        return s;
      };
      const auto release = [&](int s) {
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      };
      for (int q = 0; q < kBufs && q < steps; ++q)
        if (new_tile(q)) release(follow());
      for (int q = 0; q < steps; ++q) {
        const bool keys_next = q + kBufs < steps && new_tile(q + kBufs);
        if (!new_tile(q)) {
          if (keys_next) {
            const int sk = follow();
            release(sk);
          }
          continue;
        }
        const int t = tile_of(q);
        uint32_t word[4] = {kFull, kFull, kFull, kFull};
        const bool fix = needs_fix(t);
        if (fix) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = key_tile(t) * 128 + 32 * i + lane;
            word[i] = __ballot_sync(kFull, j < keys && (!masked || mask[j] != 0));
          }
        }
        if (masked) {
          const int m = t % kMaskRing;
          if (t >= kMaskRing) warp_wait(m_empty(m), ((t / kMaskRing) - 1) & 1, bail);
          if (lane < 4) s_mask[m][lane] = lane == 0 ? word[0] : lane == 1 ? word[1] : lane == 2 ? word[2] : word[3];
          __syncwarp();
          if (lane == 0) mbar_arrive(m_full(m));
        }
        const int s = follow();
        if (fix) {
          if ((word[0] & word[1] & word[2] & word[3]) != kFull) {
            // a row's 128 bytes: eight lanes, four rows at a time (the swizzle permutes within the row, zeros do not care)
            for (int r = lane >> 3; r < 128; r += 4) {
              const uint32_t w = r < 32 ? word[0] : r < 64 ? word[1] : r < 96 ? word[2] : word[3];
              if ((w >> (r & 31)) & 1) continue;
              for (int x = 0; x < NSUB; ++x) smem_zero16(s_ring + s * kStageBytes + x * kTileBytes + r * 128 + (lane & 7) * 16);
            }
            fence_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(fixed(s));
        }
        release(s);
        if (keys_next) {
          const int sk = follow();
          release(sk);
        }
      }
    }
  } else {
    // ---- softmax ---------------------------------------------------------------------------------------------------
    set_registers_up<208>();
    const int i = warp >> 2, w4 = warp & 3;
    const int r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)(w4 * 32) << 16);
    const uint32_t t_o = lanes + Shape::kOutAt + Shape::kOutCols * i;
    const int mine = pair ? (n - i + 1) / 2 : (i < tiles ? n : 0);  // key tiles of this group
    const bool works = w4 < live_warps && (pair || i < tiles);
    const int row_tile = pair ? 0 : 2 * rb + i;
    const long long row = (long long)row_tile * tile_rows + r;
    const bool live = works && r < tile_rows && row < rows;
    const int d16 = (a.p.D + 15) / 16 * 16;
    float m = -INFINITY, sum = 0.0f;
    bool seen = mine > 0 && !masked;  // a key that may be attended (the same for all rows)
    if (works) {
      for (int j = 0; j < mine; ++j) {
        const int q = j * streams + i, t = tile_of(q), buf = q % kBufs;
        const uint32_t t_s = lanes + 128 * buf;
        uint32_t word[4] = {kFull, kFull, kFull, kFull};
        bool cut = false;
        if (masked) {
          const int mr = t % kMaskRing;
          warp_wait(m_full(mr), (t / kMaskRing) & 1, bail);
#pragma unroll
          for (int x = 0; x < 4; ++x) word[x] = s_mask[mr][x];
          __syncwarp();
          if (lane == 0) mbar_arrive(m_empty(mr));
          cut = (word[0] & word[1] & word[2] & word[3]) != kFull;
          seen = seen || (word[0] | word[1] | word[2] | word[3]) != 0;
        } else if ((t0 + t + 1) * 128 > keys) {
          const int have = keys - (t0 + t) * 128;
#pragma unroll
          for (int x = 0; x < 4; ++x) word[x] = have >= 32 * x + 32 ? kFull : have <= 32 * x ? 0u : (1u << (have - 32 * x)) - 1u;
          cut = true;
        }
        warp_wait(s_full(buf), (q / kBufs) & 1, bail);
        tc_fence_after();
        float s[128];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld32(t_s + 32 * x, s + 32 * x);
        tmem_wait_ld();
        if (cut) {
#pragma unroll
          for (int x = 0; x < 128; ++x)
            if (!((word[x / 32] >> (x % 32)) & 1)) s[x] = -INFINITY;
        }
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int x = 4; x < 124; x += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y) top[y] = max3(top[y], s[x + 2 * y], s[x + 2 * y + 1]);
        }
        const float mt = max3(max3(top[0], top[1], top[2]), max3(top[3], s[124], s[125]), fmaxf(s[126], s[127])) * a.c;
        const bool raise = mt > m + 8.0f;
        if (__any_sync(kFull, raise)) {
          const float back = raise ? (m == -INFINITY ? 0.0f : exp2_fast(m - mt)) : 1.0f;
          if (raise) m = mt;
          sum *= back;
          // the output so far has to be complete
          if (j > 0) {
            const int last = q - streams;
            warp_wait(o_step(last), (last >> 1) & 1, bail);
            tc_fence_after();
#pragma unroll 1
            for (int x = 0; x < d16; x += 32) {
              float o[32];
              tmem_ld32(t_o + x, o);
              tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] *= back;
              tmem_st32(t_o + x, o);
            }
          }
        }
        const float off = m == -INFINITY ? 0.0f : -m;
        float2 part[4] = {};
        // in runs of eight pairs, so that the long chains of the pairs on the multiply-add pipe fill the gaps of the others
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t packed[32];
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            float2 e[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const int z = 64 * half + 2 * (x + y);
              e[y] = fma2(make_float2(s[z], s[z + 1]), make_float2(a.c, a.c), make_float2(off, off));
            }
            exp2_run<kPolyForward>(e);
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              part[y & 3] = add2(part[y & 3], e[y]);
              packed[x + y] = pack2<T>(e[y].x, e[y].y);
            }
          }
          tmem_st32(t_s + 32 * half, packed);
          if (half == 0 && Shape::kHalves) {  // the tensor cores may begin
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_half(buf));
          }
        }
        const float2 all = add2(add2(part[0], part[1]), add2(part[2], part[3]));
        sum += all.x + all.y;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(buf));
      }
      if (seen && m == -INFINITY) {  // scores, but none above -infinity
        m = kLowest;
        sum = sum * 0.0f + 1.0f;     // NaN stays
      }
      if (mine > 0) warp_wait(o_full(i), 0, bail);
      // the second group is about to write over the ring: the first group's tiles must have been consumed too
      if (pair && i == 1 && mine > 0) warp_wait(o_full(0), 0, bail);
      __syncwarp();
      tc_fence_after();
    }
    // ---- output ------------------------------------------------------------------------------------------------------
    if (pair && n > 1) {
      // the second group's rows join the first's through shared memory; the ring is idle, all tiles are consumed
      float* s_join = reinterpret_cast<float*>(s_raw + (s_ring - smem_addr(s_raw)));  // [d16][128]
      if (i == 1 && works) {
#pragma unroll 1
        for (int x = 0; x < d16; x += 32) {
          float o[32];
          tmem_ld32(t_o + x, o);
          tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 32; ++y) s_join[(x + y) * 128 + r] = o[y];
        }
        s_stat[0][r] = m;
        s_stat[1][r] = sum;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    if (i == 0 || !pair) {
      float f0 = 1.0f, f1 = 0.0f;
      const bool joins = pair && n > 1;
      if (joins && works) {
        const float m1 = s_stat[0][r], sum1 = s_stat[1][r];
        const float mm = fmaxf(m, m1);
        f0 = m == -INFINITY ? 0.0f : exp2_fast(m - mm);
        f1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - mm);
        sum = sum * f0 + sum1 * f1;
        m = mm;
      }
      const bool none = m == -INFINITY;             // no key
      if (m == kLowest && !parted) sum = NAN;  // parts: the join tells whether another one has a score
      const float inv = none ? 0.0f : 1.0f / sum;
      const long long l = row / pl.G;
      T* dst = reinterpret_cast<T*>(a.out) + (((long long)b * a.p.Lq + l) * a.p.Hq + g * pl.G + (int)(row - l * pl.G)) * a.p.D;
      const long long units = (long long)a.p.B * a.p.Hkv * pl.row_blocks - pl.whole;
      const long long at = (split * units + (u - pl.whole)) * 256 + (pair ? 0 : 128 * i) + r;
      float* dpart = parted ? a.part + at * a.p.D : nullptr;
      const float* s_join = reinterpret_cast<const float*>(s_raw + (s_ring - smem_addr(s_raw)));
      __syncwarp();
      if (works) {
#pragma unroll 1
        for (int x = 0; x < d16; x += 32) {
          float o[32];
          if (mine > 0) {
            tmem_ld32(t_o + x, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0.0f;
          }
          if (joins) {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = o[y] * f0 + s_join[(x + y) * 128 + r] * f1;
          }
          if (live) {
            if (parted)
              store_row32(dpart + x, o, inv, a.p.D - x);
            else
              store_row16<T>(dst + x, o, inv, a.p.D - x);
          }
          __syncwarp();
        }
      }
      if (live) {
        if (parted)
          a.part_lse[at] = none ? -INFINITY : m + log2f(sum);
        else if (a.lse != nullptr)
          a.lse[(long long)bg * att_rows_padded(a.p) + row] = none ? INFINITY : m + log2f(sum);
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

struct JoinArgs {
  const float* part;      // [splits][units][slots][D]
  const float* part_lse;  // [splits][units][slots]
  float* lse;             // or null
  int splits, slots;      // rows of a unit in the parts: 128 or 256
  int whole, units;       // units before the first split one, split units
  int per_head;           // units of a (sample, key head)
  int tile_rows;          // rows of a row tile of 128
  int warps;              // warps that share a row: 4 or 1
};

// out[row] = sum over splits of 2^(lse_s - L) o_s with L = log2 sum_s 2^lse_s; NaN where a part is, and where no part has a
// score above -infinity though one has keys.  Few rows: a block per row, whose warps take
// the splits in turn (in a fixed order) and add up in shared memory; many: a warp per row.
template <typename T>
__global__ void __launch_bounds__(128) att_join_kernel(const __grid_constant__ FbevAttention p, const __grid_constant__ JoinArgs a, T* __restrict__ out) {
  __shared__ float s_out[4][128], s_total[4];
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int place = a.warps == 4 ? blockIdx.x : blockIdx.x * 4 + warp;
  const int u = place / a.slots, slot = place % a.slots;
  const int unit = a.whole + u, bg = unit / a.per_head, G = p.Hq / p.Hkv;
  const long long rows = att_rows(p);
  const long long row = ((long long)(unit - bg * a.per_head) * (a.slots / 128) + slot / 128) * a.tile_rows + slot % 128;
  if (slot % 128 >= a.tile_rows || row >= rows) return;  // the whole block where it shares a row
  const long long step = (long long)a.units * a.slots, at = (long long)u * a.slots + slot;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = max_nan(top, a.part_lse[s * step + at]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(kFull, top, d));
  const bool scored = top > kLowest;  // not with NaN
  float total = scored || top == -INFINITY ? 0.0f : NAN, o[4] = {};
  if (scored) {
#pragma unroll 4
    for (int s = a.warps == 4 ? warp : 0; s < a.splits; s += a.warps) {
      const float w = exp2_fast(a.part_lse[s * step + at] - top);
      const float* src = a.part + (s * step + at) * p.D;
      total += w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.D) o[i] = fmaf(w, src[lane + 32 * i], o[i]);
    }
  }
  const long long l = row / G;
  const int b = bg / p.Hkv, h = (bg % p.Hkv) * G + (int)(row - l * G);
  T* dst = out + (((long long)b * p.Lq + l) * p.Hq + h) * p.D;
  if (a.warps == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s_out[warp][lane + 32 * i] = o[i];
    if (lane == 0) s_total[warp] = total;
    __syncthreads();
    total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    const int c = threadIdx.x;
    const float v = (s_out[0][c] + s_out[1][c]) + (s_out[2][c] + s_out[3][c]);
    if (c < p.D) dst[c] = from_float<T>(total == 0.0f ? 0.0f : v / total);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < p.D) dst[lane + 32 * i] = from_float<T>(total == 0.0f ? 0.0f : o[i] / total);
  }
  if (a.lse != nullptr && lane == 0 && (warp == 0 || a.warps == 1))
    a.lse[bg * att_rows_padded(p) + row] = total == 0.0f ? INFINITY : top + log2f(total);
}

}  // namespace fbev
