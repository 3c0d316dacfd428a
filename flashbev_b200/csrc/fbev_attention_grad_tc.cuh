// Gradients of attention on the tensor cores, 16-bit types.
//
// With the forward's statistics (lse, base 2) and delta = <out, grad_out> per row, and c = scale * log2 e:
//
//   P = 2^(c S - lse),  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,    dK = scale dS^T Q,    dV = P^T dO
//
// Two kernels of one shape, so that each sum has one owner and no atomic orders it: a block keeps a tile X of 128 rows
// and walks the tiles Y of the other side.
//
//   dQ:     X = (Q, dO) of a row tile,  Y = (K, V) of the key tiles:   S = X0 Y0^T, dP = X1 Y1^T, acc0 += dS Y0
//   dK, dV: X = (K, V) of a key tile,   Y = (Q, dO) of the row tiles:  the same transposed, and acc1 += P^T Y1
//
// S and dP are formed twice that way, seven products instead of the least of five; in exchange nothing of dQ travels to
// memory in float32 and the result is the same from run to run.
//
// In the transposed kernel lse and delta belong to the columns.  Reading them by every thread, from shared memory that the
// matrix instructions keep busy, took a third of a step.  They enter through the tensor cores instead: a 16-wide step more,
// ones times three bfloat16 parts of -lse / c (24 bits, whatever the operands' type), leaves S - lse / c in the accumulator,
// and another dP - delta.  The tile with the parts (columns 0 .. 2 and 16 .. 18) holds the ones too (columns 32 .. 34 of its
// rows).
//
// A 128 x 128 tile of S is in the hands of sixteen warps, a thread has 32 columns of a row: tensor memory -> registers ->
// P in 16 bits back over S (needed as an operand only for dV), then dP -> dS in 16 bits back over dP.  Each quarter of the
// columns writes over its own quarter only.  While the warps form P of the next tile, the tensor cores run acc0 of this one
// and dP of the next; while they form dS, acc1 and S of the next.  All warps are in the same phase of a tile, so it is their
// number that hides the latencies of a phase.
//
// For dQ, where tensor memory has the room, dP has two tiles in turn: with one, dP of the next tile waits for acc0 of this
// one, that for dS, and dS for dP, and this round trip is the length of a step.
//
// Transposed, with heads up to 64 wide, S has two tiles instead: the next one is formed before P of this one is used up.
//
// Bound by the round trip of a tile: products, the sixteen warps' two phases (tensor memory to registers, exponentials,
// packing, and back), products.  At 2 x 10000 queries x 4224 keys, 8 query heads on 4 key heads of 64, bf16, with lengths:
// dQ 212 us, dK and dV 272 us (321 with one tile of S, 400 with the statistics read by the threads), the statistics'
// kernel 16 us, the parts' sums 11 us each; the forward of the same takes 176 us.
//
// Tensor memory, columns: S/P 0, dP/dS 128 and 256, acc0 384; transposed: S/P 0 and 128, dP/dS 256, acc0 384, acc1 448, or
// with wide heads S/P 0, dP/dS 128, acc0 256, acc1 384.
#pragma once
#include "fbev_attention_tc.cuh"
#include "fbev_rotary.cuh"

namespace fbev {

struct AttGradPlan {
  int G, TL, row_tiles, key_tiles;
  int splits, per_split;  // blocks along Y and their tiles
};

struct AttGradArgs {
  CUtensorMap x0, x1, y0, y1, z;
  FbevAttention p;
  AttGradPlan pl;
  const float* nlse;    // dQ: -lse and -delta of every row, laid out by row tile: [B * Hkv][row_tiles][128], rows that are
  const float* ndelta;  // not there have a weight of zero (-infinity) and no delta; transposed: the same in the tiles of z
  void* g0;      // dQ, or dK
  void* g1;      // dV
  float* part0;  // float32 parts of g0 and g1 with splits > 1, unscaled
  float* part1;
  float c;
};

constexpr int kGradThreads = 640;  // sixteen warps for P and dS, four for loads, matrix instructions and masks

// two resident tiles and a ring of at least four: Y0 and Y1 of a tile are held while Y0 of the next is read
template <int NSUB>
struct AttGradShape {
  static constexpr int kStages = NSUB == 1 ? 10 : 4;
  static constexpr uint32_t kStageBytes = NSUB * kTileBytes;
  static constexpr uint32_t kSmem = (2 + kStages) * kStageBytes + 2 * kTileBytes + 1024;  // and two tiles of statistics
};

template <typename T, int NSUB, bool KV>
__global__ void __launch_bounds__(kGradThreads, 1) att_grad_kernel(const __grid_constant__ AttGradArgs a) {
  using Shape = AttGradShape<NSUB>;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kStageBytes = Shape::kStageBytes;
  constexpr bool kTwo = !KV;               // tiles of dP
  constexpr bool kTwoS = KV && NSUB == 1;  // and of S
  constexpr uint32_t kAcc0 = kTwo || kTwoS ? 384 : 256, kAcc1 = kTwoS ? 448 : 384;
  extern __shared__ unsigned char s_raw[];
  __shared__ __align__(8) uint64_t s_bar[3 * kStages + 11 + 2 * kMaskRing];
  __shared__ uint32_t s_mask[kMaskRing][4];
  __shared__ uint8_t s_list[kSkipTiles];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bail, s_count;

  const AttGradPlan& pl = a.pl;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  int u = blockIdx.x;
  const int split = u % pl.splits;
  u /= pl.splits;
  const int x_tiles = KV ? pl.key_tiles : pl.row_tiles;
  const int xt = u % x_tiles, bg = u / x_tiles, b = bg / a.p.Hkv, g = bg % a.p.Hkv;
  const int keys = uniform(att_keys(a.p, b));
  const bool masked = a.p.key_mask != nullptr;
  const long long rows = att_rows(a.p);
  const int tile_rows = pl.TL * pl.G;
  const int t0 = split * pl.per_split;
  int n = (KV ? (xt * 128 < keys ? pl.row_tiles : 0) : (keys + 127) / 128) - t0;  // tiles Y of this block
  n = n < 0 ? 0 : n > pl.per_split ? pl.per_split : n;
  // dQ skips the tiles of keys that the mask empties; a block of dK and dV whose keys are all masked has nothing to do
  const bool skips = masked && n > 0 && (KV || n <= kSkipTiles);
  if (skips) {
    const uint8_t* mask = a.p.key_mask + (long long)b * a.p.mask_stride;
    const int left = uniform(att_tiles_left<kGradThreads / 32>(mask, keys, KV ? xt : t0, KV ? 1 : n, s_list, &s_count));
    n = KV ? (left > 0 ? n : 0) : left;
  }
  const auto y_tile = [&](int t) { return t0 + (!KV && skips ? uniform(s_list[t]) : t); };

  const uint32_t smem = (smem_addr(s_raw) + 1023) & ~1023u;
  const uint32_t s_x = smem, s_ring = smem + 2 * kStageBytes,
                 s_z = s_ring + kStages * kStageBytes;
  const uint32_t bars = smem_addr(s_bar);
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (kStages + s); };
  const auto fixed = [&](int s) { return bars + 8 * (2 * kStages + s); };
  const uint32_t x_full = bars + 8 * (3 * kStages), acc_full = x_full + 8, drained = x_full + 16;
  // two barriers in turn where one of the sides may be a tile further than the other thinks: a barrier tells only its last
  // phase from the one before
  const auto s_full = [&](int t) { return x_full + 24 + 8 * (t & 1); };
  const auto p_done = [&](int t) { return x_full + 40 + 8 * (t & 1); };
  const auto dp_full = [&](int t) { return x_full + 56 + 8 * (t & 1); };
  const auto ds_done = [&](int t) { return x_full + 72 + 8 * (t & 1); };
  const auto s_at = [&](int t) { return kTwoS ? 128u * (t & 1) : 0u; };
  const auto dp_at = [&](int t) { return kTwo ? 128u + 128u * (t & 1) : kTwoS ? 256u : 128u; };
  const auto m_full = [&](int i) { return x_full + 88 + 8 * i; };
  const auto m_empty = [&](int i) { return x_full + 88 + 8 * (kMaskRing + i); };

  // dQ: keys that may not be attended are cleared before they meet dS, by a warp that follows the ring (as in the forward)
  const bool fixes = !KV && (masked || keys < a.p.Lk);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), fixes ? 2 : 1);
      mbar_init(fixed(s), 1);
    }
    mbar_init(x_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full(i), 1);
      mbar_init(p_done(i), 16);
      mbar_init(dp_full(i), 1);
      mbar_init(ds_done(i), 16);
    }
    mbar_init(acc_full, 1);
    mbar_init(drained, 1);
    for (int i = 0; i < kMaskRing; ++i) {
      mbar_init(m_full(i), 1);
      mbar_init(m_empty(i), KV ? 1 : 16);
    }
    s_bail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (KV && tile_rows < 128) {
    // rows that no load writes take part in the sums over rows: zeros instead of what the memory held
    for (int s = 0; s < kStages * NSUB; ++s)
      for (int i = threadIdx.x; i < (128 - tile_rows) * 8; i += kGradThreads)
        smem_zero16(s_ring + s * kTileBytes + tile_rows * 128 + i * 16);
    fence_async_smem();
  }
  if (warp == 17) tmem_alloc<512>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns of the SM are this block's
  const Bail bail{&s_bail, a.p.status};
  const uint32_t x_bytes = KV ? kStageBytes : (uint32_t)(NSUB * tile_rows * 128);
  const uint32_t y_bytes = KV ? (uint32_t)(NSUB * tile_rows * 128) : kStageBytes;
  const auto needs_fix = [&](int t) { return fixes && (masked || (t0 + t + 1) * 128 > keys); };
  grid_dependency_wait();  // delta comes from the kernel before

  if (warp >= 16) {
    set_registers_down<64>();
    if (warp == 16 && n > 0) {
      // ---- loads -------------------------------------------------------------------------------------------------
      const int qb = a.p.q_shared ? 0 : b;
      const auto load_rows = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int tile, int batch) {
        for (int x = 0; x < NSUB; ++x) tma_load_5d(dst + x * kTileBytes, map, bar, 64 * x, 0, g, tile * pl.TL, batch);
      };
      const auto load_keys = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int tile) {
        for (int x = 0; x < NSUB; ++x) tma_load_4d(dst + x * kTileBytes, map, bar, 64 * x, g, tile * 128, b);
      };
      mbar_expect(x_full, 2 * x_bytes);
      if (KV) {
        load_keys(s_x, &a.x0, x_full, xt);
        load_keys(s_x + kStageBytes, &a.x1, x_full, xt);
      } else {
        load_rows(s_x, &a.x0, x_full, xt, qb);
        load_rows(s_x + kStageBytes, &a.x1, x_full, xt, b);
      }
      int slot = 0;
      const auto load = [&](const CUtensorMap* map, int t, int batch) {
        const int s = slot % kStages;
        if (slot >= kStages) warp_wait(empty(s), ((slot / kStages) - 1) & 1, bail);
        mbar_expect(full(s), y_bytes);
        if (KV)
          load_rows(s_ring + s * kStageBytes, map, full(s), t0 + t, batch);
        else
          load_keys(s_ring + s * kStageBytes, map, full(s), y_tile(t));
        ++slot;
      };
      for (int t = 0; t < n; ++t) {
        load(&a.y0, t, qb);
        if (KV) {  // the statistics' two tiles, by the mask ring's barriers
          const int i = t & 1;
          if (t >= 2) warp_wait(m_empty(i), ((t >> 1) - 1) & 1, bail);
          mbar_expect(m_full(i), kTileBytes);
          tma_load_4d(s_z + i * kTileBytes, &a.z, m_full(i), 0, 0, (t0 + t) * 128, bg);
        }
        load(&a.y1, t, b);
      }
      if (__any_sync(kFull, *bail.flag != 0)) {
        // nothing may be left in flight when the block ends
        mbar_drain(x_full, 0);
        for (int i = slot > kStages ? slot - kStages : 0; i < slot; ++i) mbar_drain(full(i % kStages), (i / kStages) & 1);
        if (KV)
          for (int t = n > 2 ? n - 2 : 0; t < n; ++t) mbar_drain(m_full(t & 1), (t >> 1) & 1);
      }
    } else if (warp == 17 && n > 0) {
      // ---- matrix instructions -----------------------------------------------------------------------------------
      const int ksteps = (a.p.D + 15) / 16;
      const uint32_t i_s = umma_instr<T>(128, false, a.p.scale < 0.0f), i_dp = umma_instr<T>(128, false, false),
                     i_acc = umma_instr<T>(ksteps * 16, true, false);
      uint32_t fix_parity = 0;
      warp_wait(x_full, 0, bail);
      const auto stage = [&](int slot) { return s_ring + (slot % kStages) * kStageBytes; };
      const auto wait_full = [&](int slot) { warp_wait(full(slot % kStages), (slot / kStages) & 1, bail); };
      const auto product = [&](uint32_t d, uint32_t x, uint32_t y, uint32_t instr) {  // X Y^T over the head's width
#pragma unroll
        for (int i = 0; i < NSUB; ++i) {
          const uint64_t da = desc_k_major(x + i * kTileBytes), db = desc_k_major(y + i * kTileBytes);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (i * 4 + k < ksteps) umma_ss(d, da + 2 * k, db + 2 * k, instr, i + k > 0);
        }
      };
      const auto accumulate = [&](uint32_t d, uint32_t t, uint32_t y, bool first) {  // 16-bit tile in tensor memory times Y
        const uint64_t db = desc_mn_major(y);
#pragma unroll
        for (int k = 0; k < 8; ++k) umma_ts(d, t + 32 * (k / 2) + 8 * (k & 1), db + 128 * k, i_acc, !first || k > 0);
      };
      const auto add_stat = [&](uint32_t d, int t, int at) {  // ones times the parts in columns at .. at + 15
        const uint64_t z = desc_k_major(s_z + (t & 1) * kTileBytes);
        umma_ss(d, z + 4, z + at / 8, umma_instr<__nv_bfloat16>(128, false, false), true);
      };
      const auto scores = [&](int t) {
        wait_full(2 * t);
        if (KV) warp_wait(m_full(t & 1), (t >> 1) & 1, bail);
        if (needs_fix(t)) {
          const int s = (2 * t) % kStages;
          warp_wait(fixed(s), (fix_parity >> s) & 1, bail);
          fix_parity ^= 1u << s;
        }
        tc_fence_after();
        product(tmem + s_at(t), s_x, stage(2 * t), i_s);
        if (KV) add_stat(tmem + s_at(t), t, 0);
        umma_commit(s_full(t));
      };
      const auto dprobs = [&](int t) {
        wait_full(2 * t + 1);
        tc_fence_after();
        product(tmem + dp_at(t), s_x + kStageBytes, stage(2 * t + 1), i_dp);
        if (KV) add_stat(tmem + dp_at(t), t, 16);
        umma_commit(dp_full(t));
        if (KV) umma_commit(m_empty(t & 1));
        if (!KV) umma_commit(empty((2 * t + 1) % kStages));
      };
      scores(0);
      dprobs(0);
      for (int t = 0; t < n; ++t) {
        if (kTwoS && t + 1 < n) scores(t + 1);
        warp_wait(p_done(t), (t >> 1) & 1, bail);
        if (KV) {
          tc_fence_after();
          accumulate(tmem + kAcc1, tmem + s_at(t), stage(2 * t + 1), t == 0);
          umma_commit(empty((2 * t + 1) % kStages));
        }
        if (!kTwoS && t + 1 < n) {
          scores(t + 1);
          if (kTwo) dprobs(t + 1);
        }
        warp_wait(ds_done(t), (t >> 1) & 1, bail);
        tc_fence_after();
        accumulate(tmem + kAcc0, tmem + dp_at(t), stage(2 * t), t == 0);
        umma_commit(empty((2 * t) % kStages));
        if (!kTwo && t + 1 < n) dprobs(t + 1);
      }
      umma_commit(acc_full);
      if (__any_sync(kFull, *bail.flag != 0)) {
        umma_commit(drained);
        mbar_drain(drained, 0);
      }
    } else if (fixes && warp == 18 && n > 0) {
      // ---- key mask, keys that may not be attended -----------------------------------------------------------------
      const uint8_t* mask = masked ? a.p.key_mask + (long long)b * a.p.mask_stride : nullptr;
      const auto release = [&](int s) {
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      };
      for (int t = 0; t < n; ++t) {
        uint32_t word[4] = {kFull, kFull, kFull, kFull};
        const bool fix = needs_fix(t);
        if (fix) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = y_tile(t) * 128 + 32 * i + lane;
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
        const int s = (2 * t) % kStages, s1 = (2 * t + 1) % kStages;
        warp_wait(full(s), ((2 * t) / kStages) & 1, bail);
        if (fix) {
          if ((word[0] & word[1] & word[2] & word[3]) != kFull) {
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
        warp_wait(full(s1), ((2 * t + 1) / kStages) & 1, bail);
        release(s1);
      }
    }
  } else {
    // ---- P and dS ----------------------------------------------------------------------------------------------------
    set_registers_up<104>();
    const int h = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const long long row = (long long)xt * tile_rows + r;             // dQ
    const bool row_live = !KV && r < tile_rows && row < rows;
    const int key = xt * 128 + r;                                    // dK, dV
    const float nl = KV ? 0.0f : a.nlse[((long long)bg * pl.row_tiles + xt) * 128 + r];
    const float nd = KV ? 0.0f : a.ndelta[((long long)bg * pl.row_tiles + xt) * 128 + r];
    for (int t = 0; t < n; ++t) {
      const int mr = t % kMaskRing;
      const uint32_t t_s = lanes + s_at(t) + 32 * h, t_dp = lanes + dp_at(t) + 32 * h;
      uint32_t word = kFull;
      if (!KV && masked) {
        warp_wait(m_full(mr), (t / kMaskRing) & 1, bail);
        word = s_mask[mr][h];
        __syncwarp();
        if (lane == 0) mbar_arrive(m_empty(mr));
      } else if (!KV && (t0 + t + 1) * 128 > keys) {
        const int have = keys - (t0 + t) * 128 - 32 * h;
        word = have >= 32 ? kFull : have <= 0 ? 0u : (1u << have) - 1u;
      }
      warp_wait(s_full(t), (t >> 1) & 1, bail);
      tc_fence_after();
      float p[32];
      tmem_ld32(t_s, p);
      tmem_wait_ld();
      if (!KV) {  // S may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_done(t));
      }
#pragma unroll
      for (int x = 0; x < 32; x += 16) {
        float2 e[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float2 s2 = make_float2(p[x + 2 * y], p[x + 2 * y + 1]), c2 = make_float2(a.c, a.c);
          e[y] = KV ? mul2(s2, c2) : fma2(s2, c2, make_float2(nl, nl));
        }
        exp2_run<kPolyGrad>(e);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          p[x + 2 * y] = e[y].x;
          p[x + 2 * y + 1] = e[y].y;
        }
      }
      uint32_t packed[16];
      if (KV) {
#pragma unroll
        for (int x = 0; x < 16; ++x) packed[x] = pack2<T>(p[2 * x], p[2 * x + 1]);
        __syncwarp();
        tmem_st16(t_s, packed);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_done(t));
      }
      warp_wait(dp_full(t), (t >> 1) & 1, bail);
      tc_fence_after();
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float dp[16];
        tmem_ld16(t_dp + 16 * y, dp);
        tmem_wait_ld();
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          const float* q = p + 16 * y + x;
          float2 s0 = make_float2(dp[x], dp[x + 1]), s1 = make_float2(dp[x + 2], dp[x + 3]);
          if (!KV) {
            s0 = add2(s0, make_float2(nd, nd));
            s1 = add2(s1, make_float2(nd, nd));
          }
          s0 = mul2(s0, make_float2(q[0], q[1]));
          s1 = mul2(s1, make_float2(q[2], q[3]));
          if (word != kFull) {  // a select, not a product: what stands there may be NaN
            const uint32_t w = word >> (16 * y + x);
            if (!(w & 1)) s0.x = 0.0f;
            if (!(w & 2)) s0.y = 0.0f;
            if (!(w & 4)) s1.x = 0.0f;
            if (!(w & 8)) s1.y = 0.0f;
          }
          packed[8 * y + x / 2] = pack2<T>(s0.x, s0.y);
          packed[8 * y + x / 2 + 1] = pack2<T>(s1.x, s1.y);
        }
      }
      __syncwarp();
      tmem_st16(t_dp, packed);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_done(t));
    }
    if (n > 0) warp_wait(acc_full, 0, bail);
    tc_fence_after();
    // ---- output: a quarter of dQ's columns each, or dK by the even quarters and dV by the odd ones -------------------------
    const int d16 = (a.p.D + 15) / 16 * 16;
    const bool parted = pl.splits > 1;
    const bool live = KV ? key < a.p.Lk : row_live;
    bool zero = n == 0;
    if (KV && live) zero = zero || key >= keys || !att_allowed(a.p, b, key);
    const long long l = KV ? 0 : row / pl.G;
    const long long at = KV ? (((long long)b * a.p.Lk + key) * a.p.Hkv + g) * a.p.D
                            : (((long long)b * a.p.Lq + l) * a.p.Hq + g * pl.G + (row - l * pl.G)) * a.p.D;
    const long long whole = KV ? (long long)a.p.B * a.p.Lk * a.p.Hkv * a.p.D : (long long)a.p.B * a.p.Lq * a.p.Hq * a.p.D;
    const bool second = KV && (h & 1);
    T* dst = reinterpret_cast<T*>(second ? a.g1 : a.g0) + at;
    float* dpart = parted ? (second ? a.part1 : a.part0) + split * whole + at : nullptr;
    const float f = second ? 1.0f : a.p.scale;
    __syncwarp();
#pragma unroll 1
    for (int x = KV ? 32 * (h >> 1) : 32 * h; x < d16; x += KV ? 64 : 128) {
      float o[32];
      if (n > 0) {
        tmem_ld32(lanes + (second ? kAcc1 : kAcc0) + x, o);
        tmem_wait_ld();
      }
      if (zero) {
#pragma unroll
        for (int y = 0; y < 32; ++y) o[y] = 0.0f;
      }
      if (live) {
        if (parted)
          store_row32(dpart + x, o, 1.0f, a.p.D - x);
        else
          store_row16<T>(dst + x, o, f, a.p.D - x);
      }
      __syncwarp();
    }
    tc_fence_before();
  }
  grid_dependency_trigger();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_free<512>(s_tmem);
  }
}

// g[i] = f * (sum of the parts in order)
template <typename T>
__global__ void __launch_bounds__(256) att_sum_kernel(const float* __restrict__ part, int splits, long long count, float f, T* __restrict__ g) {
  grid_dependency_wait();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
    float s = 0.0f;
    for (int k = 0; k < splits; ++k) s += part[k * count + i];
    g[i] = from_float<T>(s * f);
  }
}

// -lse and -delta = -<out, grad_out> of every row of the padded row tiles: eight lanes share a row, 16 bytes a load, and have
// kStatRows rows in flight
constexpr int kStatRows = 2;
template <typename T>
__global__ void __launch_bounds__(256) att_stat_kernel(const __grid_constant__ FbevAttention p, int TL, int row_tiles, const T* __restrict__ out,
                                                       const T* __restrict__ go, const float* __restrict__ lse, float* __restrict__ nlse,
                                                       float* __restrict__ ndelta, uint4* __restrict__ parts, float inv_c) {
  const int lane = threadIdx.x & 7, G = p.Hq / p.Hkv;
  const unsigned rows = (unsigned)att_rows(p);
  // blocks of 32 * kStatRows rows of a row tile
  constexpr unsigned kBlocks = 4 / kStatRows;
  const unsigned all = blockIdx.x / kBlocks, part = blockIdx.x - all * kBlocks;
  const unsigned bg = all / (unsigned)row_tiles, tile = all - bg * (unsigned)row_tiles, b = bg / p.Hkv, g = bg - b * p.Hkv;
  const unsigned first = 32 * kStatRows * part + (threadIdx.x >> 3);
  float d[kStatRows], l[kStatRows];
  Pack<T, 8> x[kStatRows][2], y[kStatRows][2];
  bool live[kStatRows];
#pragma unroll
  for (int k = 0; k < kStatRows; ++k) {
    const unsigned r = first + 32 * k, row = tile * TL * G + r, q = row / G;
    live[k] = r < (unsigned)(TL * G) && row < rows;
    const long long head = (((long long)b * p.Lq + q) * p.Hq + g * G + (row - q * G)) * p.D;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (live[k] && lane * 8 + 64 * i < p.D) {
        x[k][i] = *reinterpret_cast<const Pack<T, 8>*>(out + head + lane * 8 + 64 * i);
        y[k][i] = *reinterpret_cast<const Pack<T, 8>*>(go + head + lane * 8 + 64 * i);
      }
    l[k] = live[k] ? lse[bg * att_rows_padded(p) + row] : INFINITY;
  }
#pragma unroll
  for (int k = 0; k < kStatRows; ++k) {
    d[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (live[k] && lane * 8 + 64 * i < p.D) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[k] = fmaf(to_float(x[k][i].v[e]), to_float(y[k][i].v[e]), d[k]);
      }
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) d[k] += __shfl_xor_sync(kFull, d[k], s);
    const long long at = (long long)all * 128 + first + 32 * k;
    if (lane == 0) {
      nlse[at] = -l[k];
      ndelta[at] = -d[k];
    }
    if (parts != nullptr) {
      // lane i: columns 8 i .. 8 i + 7 of the row's 64
      uint4 w = make_uint4(0, 0, 0, 0);
      if (lane == 0 || lane == 2) {
        float v = lane == 0 ? -l[k] * inv_c : -d[k];
        const bool finite = fabsf(v) < 3.0e38f;
        const uint32_t p0 = pack2<__nv_bfloat16>(v, 0.0f);
        v = finite ? v - __uint_as_float(p0 << 16) : 0.0f;
        const uint32_t p1 = pack2<__nv_bfloat16>(v, 0.0f);
        v = finite ? v - __uint_as_float(p1 << 16) : 0.0f;
        w.x = p0 | p1 << 16;
        w.y = pack2<__nv_bfloat16>(v, 0.0f);
      } else if (lane == 4) {
        w.x = pack2<__nv_bfloat16>(1.0f, 1.0f);
        w.y = pack2<__nv_bfloat16>(1.0f, 0.0f);
      }
      parts[at * 8 + lane] = w;
    }
  }
  grid_dependency_trigger();
}

}  // namespace fbev
