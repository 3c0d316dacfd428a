// The operators of include/fbev_query.h: argument checks, plans, launches and the C ABI.  Kernels: fbev_attention_tc.cuh and
// fbev_attention_grad_tc.cuh (16-bit attention and its gradients), fbev_attention_split_tc.cuh (float32, and what TMA cannot
// address), fbev_rotary.cuh, fbev_norm.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "fbev_query.h"
#include "fbev_attention.cuh"
#include "fbev_attention_tc.cuh"
#include "fbev_attention_grad_tc.cuh"
#include "fbev_attention_split_tc.cuh"
#include "fbev_norm.cuh"
#include "fbev_rotary.cuh"

namespace fbev {

static size_t size_of(int dtype) { return dtype == FBEV_F32 ? 4 : 2; }
static bool known_dtype(int dtype) { return dtype == FBEV_F32 || dtype == FBEV_BF16 || dtype == FBEV_F16; }

static int check_attention(const FbevAttention* p) {
  if (p == nullptr) return FBEV_ERR_NULL;
  if (p->struct_size != sizeof(FbevAttention)) return FBEV_ERR_STRUCT;
  if (!known_dtype(p->dtype)) return FBEV_ERR_DTYPE;
  if (p->B < 0 || p->Lq < 0 || p->Lk < 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv != 0 || p->D <= 0 || p->D > 128)
    return FBEV_ERR_SHAPE;
  if (!(p->scale >= -1e30f && p->scale <= 1e30f)) return FBEV_ERR_RANGE;
  if (att_rows(*p) >= (1ll << 31) || (long long)p->B * p->Hq >= (1ll << 31)) return FBEV_ERR_RANGE;
  if ((long long)p->B * p->Hkv * (att_rows(*p) + 256) >= (1ll << 31) || (long long)p->B * p->Hkv * (p->Lk + 256ll) >= (1ll << 31))
    return FBEV_ERR_RANGE;  // blocks of a launch
  if ((uintptr_t)p->key_lengths % 4 || (uintptr_t)p->status % 4) return FBEV_ERR_ALIGN;
  const size_t es = size_of(p->dtype);
  if ((uintptr_t)p->q % es || (uintptr_t)p->k % es || (uintptr_t)p->v % es) return FBEV_ERR_ALIGN;
  return FBEV_OK;
}

// rows of q and keys that are read must have an address
static bool has_pointers(const FbevAttention* p) {
  const bool queries = p->B > 0 && p->Lq > 0, keys = p->B > 0 && p->Lk > 0;
  return (!queries || p->q) && (!keys || (p->k && p->v));
}

static size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }

// ---- tensor-core path -------------------------------------------------------------------------------------------------

constexpr int kSms = 148;

static bool tma_operand(const void* ptr, const int64_t (&stride)[3], const int64_t (&size)[3], bool first_unused) {
  if ((uintptr_t)ptr % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (size[i] > 1 && !(i == 0 && first_unused) && (stride[i] <= 0 || stride[i] % 8 != 0 || stride[i] >= (1ll << 38))) return false;
  return true;
}

// 16-bit types whose rows TMA can address: heads of whole 16 bytes, strides of whole 16 bytes.  Everything else goes through
// the kernels of three-part operands.
static bool direct(const FbevAttention& p) {
  if (p.dtype == FBEV_F32 || p.D % 8 != 0 || p.Lk == 0 || p.Lq == 0 || p.B == 0 || p.Hq / p.Hkv > 128) return false;
  return tma_operand(p.q, p.q_stride, {p.B, p.Lq, p.Hq}, p.q_shared != 0) &&
         tma_operand(p.k, p.k_stride, {p.B, p.Lk, p.Hkv}, false) && tma_operand(p.v, p.v_stride, {p.B, p.Lk, p.Hkv}, false);
}

// How units of work (a block each, `tiles` steps long) are spread over the SMs.  Blocks of one length run in waves of one per
// SM, so the last wave may leave most of them idle; a unit that is split along its steps runs as several shorter blocks,
// whose parts have to be written and summed.  The choice is the shortest of: nothing split; all units split into s; where
// `tail` is set, the units of the last wave alone split into s.  Times are in steps, 3 for a block's begin and end and
// `part` for the parts of a unit (writing and reading, spread over all SMs); where the samples' lengths differ the mean over
// full, three quarter and half length counts, since all blocks of a short sample end early.  Only full waves are left whole
// by a split tail.
struct SplitChoice {
  int whole, splits, per_split;
};
static SplitChoice choose_splits(int units, int tiles, double part, bool ragged, bool tail) {
  const auto waves = [&](double blocks) { return (double)((long long)((blocks + kSms - 1) / kSms)); };
  const auto all = [&](int s, int per) {
    if (!ragged) return waves((double)units * s) * (per + 3);
    double t = 0;
    for (const double f : {1.0, 0.75, 0.5}) t += waves((long long)(f * units * s)) * (per + 3) / 3;
    return t;
  };
  SplitChoice best{units, 1, tiles > 0 ? tiles : 1};
  double cost = all(1, tiles);
  const int full = units / kSms * kSms, rest = units - full;
  for (int want = 2; want <= tiles && want <= 128; ++want) {
    const int per = (tiles + want - 1) / want, s = (tiles + per - 1) / per;
    if (s != want) continue;
    const double c = all(s, per) + (units * s / (double)kSms) * part + 2;
    if (c < 0.98 * cost) {
      cost = c;
      best = {0, s, per};
    }
    if (tail && full > 0 && rest > 0) {
      const double d = (double)(full / kSms) * (tiles + 3) + waves((double)rest * s) * (per + 3) + (rest * s / (double)kSms) * part + 2;
      if (d < 0.98 * cost) {
        cost = d;
        best = {full, s, per};
      }
    }
  }
  return best;
}

static AttPlan attention_plan(const FbevAttention& p) {
  AttPlan pl{};
  pl.G = p.Hq / p.Hkv;
  pl.TL = 128 / pl.G;
  pl.row_tiles = (p.Lq + pl.TL - 1) / pl.TL;
  pl.pair = pl.row_tiles == 1;
  pl.row_blocks = (pl.row_tiles + 1) / 2;
  const int units = p.B * p.Hkv * pl.row_blocks, key_tiles = (p.Lk + 127) / 128;
  // few rows: the memory's rate bounds a step, and splitting only pays to give every SM work
  const SplitChoice c = choose_splits(units, key_tiles, 256.0 * p.D * 4 / 40000.0, p.key_lengths != nullptr && !pl.pair, !pl.pair);
  pl.whole = c.whole;
  pl.splits = c.splits;
  pl.per_split = c.per_split;
  return pl;
}

static size_t split_output_bytes(const FbevAttention& p, const AttPlan& pl) {
  return round_up((size_t)pl.splits * (p.B * p.Hkv * pl.row_blocks - pl.whole) * 256 * p.D * 4, 256);
}
// ---- three-part operands ----------------------------------------------------------------------------------------------

struct SplitPlan {
  int x_tiles, y_tiles, x_rows, splits, per_split;
};
static SplitPlan split_plan(const FbevAttention& p, int mode) {
  const bool key_rows = mode == kSplitDv || mode == kSplitDk;
  SplitPlan pl;
  const int row_tiles = (int)((att_rows(p) + 127) / 128), key_tiles = (p.Lk + 127) / 128;
  pl.x_tiles = key_rows ? key_tiles : row_tiles;
  pl.y_tiles = key_rows ? row_tiles : key_tiles;
  pl.x_rows = key_rows ? p.Lk : (int)att_rows(p);
  // a step takes about four times as long as one of the 16-bit kernels
  const SplitChoice c = choose_splits(p.B * p.Hkv * pl.x_tiles, pl.y_tiles, 128.0 * p.D * 4 / 160000.0, p.key_lengths != nullptr, false);
  pl.splits = c.splits;
  pl.per_split = c.per_split;
  return pl;
}

// Offsets in the workspace.  The parts of one result are summed before the next is computed and share their place.
struct SplitLayout {
  int width;
  size_t q, k, v, go, allowed, nlse, ndelta, part, part_lse, bytes;
};
static SplitLayout split_layout(const FbevAttention& p, bool backward) {
  SplitLayout l{};
  l.width = (p.D + 7) / 8 * 8;
  const size_t heads = (size_t)p.B * p.Hkv, rows = heads * att_rows(p), keys = heads * p.Lk;
  const size_t row_bytes = round_up(rows * 3 * l.width * 2, 256), key_bytes = round_up(keys * 3 * l.width * 2, 256);
  const size_t stat = round_up(heads * ((att_rows(p) + 127) / 128) * 512, 256);
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t here = at;
    at += n;
    return here;
  };
  l.q = take(row_bytes);
  l.k = take(key_bytes);
  l.v = take(key_bytes);
  l.allowed = take(round_up((size_t)p.B * ((p.Lk + 127) / 128) * 512, 256));
  size_t part = 0;
  if (backward) {
    l.go = take(row_bytes);
    l.nlse = take(stat);
    l.ndelta = take(stat);
  }
  for (int mode = backward ? kSplitDv : kSplitOut; mode <= (backward ? kSplitDk : kSplitOut); ++mode) {
    const SplitPlan pl = split_plan(p, mode);
    if (pl.splits == 1 && p.dtype == FBEV_F32) continue;
    const size_t n = (size_t)pl.splits * (mode == kSplitDv || mode == kSplitDk ? keys : mode == kSplitDq ? rows : heads * pl.x_tiles * 128) * p.D * 4;
    if (n > part) part = n;
  }
  l.part = take(round_up(part, 256));
  if (!backward && part > 0) l.part_lse = take(round_up((size_t)split_plan(p, kSplitOut).splits * heads * split_plan(p, kSplitOut).x_tiles * 512, 256));
  l.bytes = at;
  return l;
}

static size_t forward_workspace(const FbevAttention& p) {
  if (!direct(p)) return split_layout(p, false).bytes;
  const AttPlan pl = attention_plan(p);
  if (pl.splits == 1) return 0;
  return split_output_bytes(p, pl) + round_up((size_t)pl.splits * (p.B * p.Hkv * pl.row_blocks - pl.whole) * 256 * 4, 256);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the driver's encoder, looked up once (the library does not link against the driver)
static EncodeTiled encode_tiled() {
  static std::atomic<void*> found{nullptr};
  void* fn = found.load(std::memory_order_acquire);
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    found.store(fn, std::memory_order_release);
  }
  return reinterpret_cast<EncodeTiled>(fn);
}

// 64 elements x rows of a [.., tokens, heads, D] tensor in 128-byte rows; a dimension of one has any stride
static int encode_map(CUtensorMap* map, int dtype, int rank, const void* ptr, const long long* dims, const long long* strides,
                      const int* box) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return FBEV_ERR_NO_DEVICE;
  cuuint64_t d[5], st[4];
  cuuint32_t bx[5], one[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    bx[i] = (cuuint32_t)box[i];
    if (i > 0) st[i - 1] = dims[i] > 1 ? (cuuint64_t)strides[i] * 2 : 128;
  }
  const CUresult rc = fn(map, dtype == FBEV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                         const_cast<void*>(ptr), d, st, bx, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? FBEV_OK : FBEV_ERR_LAUNCH;
}
// rows (query, head of the group): box of TL queries
static int encode_rows(CUtensorMap* map, const FbevAttention& p, const AttPlan& pl, const void* ptr, const int64_t* stride,
                       bool shared) {
  const long long dims[5] = {p.D, pl.G, p.Hkv, p.Lq, shared ? 1 : p.B};
  const long long strides[5] = {1, stride[2], pl.G * stride[2], stride[1], stride[0]};
  const int box[5] = {64, pl.G, 1, pl.TL, 1};
  return encode_map(map, p.dtype, 5, ptr, dims, strides, box);
}
static int encode_keys(CUtensorMap* map, const FbevAttention& p, const void* ptr, const int64_t* stride) {
  const long long dims[4] = {p.D, p.Hkv, p.Lk, p.B};
  const long long strides[4] = {1, stride[2], stride[1], stride[0]};
  const int box[4] = {64, 1, 128, 1};
  return encode_map(map, p.dtype, 4, ptr, dims, strides, box);
}

// dynamic shared memory above 48 KiB is granted once per kernel and device
template <typename K>
static int allow_smem(K* kernel, uint32_t bytes, std::atomic<uint64_t>& done) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return FBEV_ERR_NO_DEVICE;
  }
  if (done.load(std::memory_order_acquire) >> dev & 1) return FBEV_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
    cudaGetLastError();
    return FBEV_ERR_NO_DEVICE;
  }
  done.fetch_or(1ull << dev, std::memory_order_release);
  return FBEV_OK;
}

// a kernel that may be brought in while the one before it drains; it calls grid_dependency_wait() first
template <typename... KArgs, typename... Args>
static cudaError_t launch_next(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// c of the exponentials: a scale of zero still has to turn a masked score of -infinity into a weight of zero
static float score_factor(const FbevAttention& p) {
  const float c = (p.scale < 0.0f ? -p.scale : p.scale) * kLog2e;
  return c < 1e-30f ? 1e-30f : c;
}

// a block per row where that still leaves the GPU room, else a warp
template <typename T>
static void launch_join(const FbevAttention& p, JoinArgs a, T* out, cudaStream_t st) {
  const int places = a.units * a.slots;
  a.warps = a.splits > 4 && places <= kSms * 16 ? 4 : 1;
  launch_next(att_join_kernel<T>, (unsigned)(a.warps == 4 ? places : places / 4), 128, 0, st, p, a, out);
}

// ---- three-part operands: launches -------------------------------------------------------------------------------------

static int encode_parts(CUtensorMap* map, const void* ptr, long long rows, long long heads, int width) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return FBEV_ERR_NO_DEVICE;
  const cuuint64_t d[4] = {(cuuint64_t)width, (cuuint64_t)rows, 3, (cuuint64_t)heads};
  const cuuint64_t st[3] = {(cuuint64_t)width * 6, (cuuint64_t)width * 2, (cuuint64_t)rows * width * 6};
  const cuuint32_t box[4] = {64, 128, 3, 1}, one[4] = {1, 1, 1, 1};
  const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), d, st, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T>
static int split_operands(const FbevAttention& p, const SplitLayout& l, const T* out, const float* lse, const T* go, cudaStream_t st) {
  char* ws = reinterpret_cast<char*>(p.workspace);
  const int G = p.Hq / p.Hkv;
  SplitSet set{};
  const auto fill = [&](int i, const void* src, const int64_t* stride, int g, int len, int shared, size_t at) {
    SplitSource& s = set.of[i];
    s.src = src;
    for (int k = 0; k < 3; ++k) s.stride[k] = stride[k];
    s.G = g;
    s.L = len;
    s.shared = shared;
    s.whole = p.D % 4 == 0 && (uintptr_t)src % (4 * sizeof(T)) == 0;
    for (int k = 0; k < 3; ++k) s.whole = s.whole && stride[k] % 4 == 0;
    s.parts = reinterpret_cast<__nv_bfloat16*>(ws + at);
    s.width = l.width;
  };
  const int64_t go_stride[3] = {(int64_t)p.Lq * p.Hq * p.D, (int64_t)p.Hq * p.D, p.D};
  fill(0, p.q, p.q_stride, G, p.Lq, p.q_shared, l.q);
  fill(1, p.k, p.k_stride, 1, p.Lk, 0, l.k);
  fill(2, p.v, p.v_stride, 1, p.Lk, 0, l.v);
  set.of[1].allowed = set.of[2].allowed = reinterpret_cast<float*>(ws + l.allowed);  // both clear, both write the same flags
  int count = 3;
  if (go != nullptr) {
    fill(3, go, go_stride, G, p.Lq, 0, l.go);
    set.of[3].out = out;
    set.of[3].lse = lse;
    set.of[3].nlse = reinterpret_cast<float*>(ws + l.nlse);
    set.of[3].ndelta = reinterpret_cast<float*>(ws + l.ndelta);
    count = 4;
  }
  long long blocks = 0;
  for (int i = 0; i < 4; ++i) {
    set.first[i] = (unsigned)blocks;
    if (i < count) blocks += (long long)p.B * p.Hkv * (((long long)set.of[i].L * set.of[i].G + 127) / 128) * (p.D <= 64 ? 8 : 16);
    if (blocks >= (1ll << 31)) return FBEV_ERR_RANGE;
    set.first[i + 1] = (unsigned)blocks;
  }
  if (p.D <= 64)
    split_kernel<T, 16><<<(unsigned)blocks, 256, 0, st>>>(p, set);
  else
    split_kernel<T, 32><<<(unsigned)blocks, 256, 0, st>>>(p, set);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <int NC, int MODE>
static int split_launch(const FbevAttention& p, const SplitLayout& l, const SplitPlan& pl, float* g, float* part, float* lse, cudaStream_t st) {
  static std::atomic<uint64_t> granted{0};
  char* ws = reinterpret_cast<char*>(p.workspace);
  const long long heads = (long long)p.B * p.Hkv, rows = att_rows(p);
  CUtensorMap q, k, v, go;
  int rc = allow_smem(att_split_kernel<NC, MODE>, kSplitSmem, granted);
  if (rc == FBEV_OK) rc = encode_parts(&q, ws + l.q, rows, heads, l.width);
  if (rc == FBEV_OK) rc = encode_parts(&k, ws + l.k, p.Lk, heads, l.width);
  if (rc == FBEV_OK) rc = encode_parts(&v, ws + l.v, p.Lk, heads, l.width);
  if (rc == FBEV_OK) rc = MODE == kSplitOut ? FBEV_OK : encode_parts(&go, ws + l.go, rows, heads, l.width);
  if (rc != FBEV_OK) return rc;
  if (MODE == kSplitOut) go = q;
  SplitArgs a;
  const bool key_rows = MODE == kSplitDv || MODE == kSplitDk;
  a.x0 = key_rows ? k : q;
  a.y0 = key_rows ? q : k;
  a.x1 = key_rows ? v : go;
  a.y1 = key_rows ? go : v;
  a.z = MODE == kSplitOut ? v : MODE == kSplitDv ? go : MODE == kSplitDq ? k : q;
  a.p = p;
  a.x_tiles = pl.x_tiles;
  a.y_tiles = pl.y_tiles;
  a.x_rows = pl.x_rows;
  a.splits = pl.splits;
  a.per_split = pl.per_split;
  a.allowed = reinterpret_cast<const float*>(ws + l.allowed);
  a.nlse = reinterpret_cast<const float*>(ws + l.nlse);
  a.ndelta = reinterpret_cast<const float*>(ws + l.ndelta);
  a.g = g;
  a.lse = lse;
  a.part = part;
  a.part_lse = reinterpret_cast<float*>(ws + l.part_lse);
  a.c = score_factor(p);
  launch_next(att_split_kernel<NC, MODE>, (unsigned)(heads * pl.x_tiles * pl.splits), kAttThreads, kSplitSmem, st, a);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

// float32 results of one block per tile are written in place; all others pass through parts
template <typename T, int MODE>
static int split_result(const FbevAttention& p, const SplitLayout& l, T* g, float* lse, cudaStream_t st) {
  const SplitPlan pl = split_plan(p, MODE);
  const bool whole = pl.splits == 1 && std::is_same<T, float>::value;
  float* part = whole ? nullptr : reinterpret_cast<float*>(reinterpret_cast<char*>(p.workspace) + l.part);
  float* into = reinterpret_cast<float*>(whole ? g : nullptr);
  const int rc = p.D <= 64 ? split_launch<1, MODE>(p, l, pl, into, part, lse, st) : split_launch<2, MODE>(p, l, pl, into, part, lse, st);
  if (rc != FBEV_OK || whole) return rc;
  if (MODE == kSplitOut) {
    const int units = p.B * p.Hkv * pl.x_tiles;
    launch_join<T>(p, JoinArgs{part, reinterpret_cast<float*>(reinterpret_cast<char*>(p.workspace) + l.part_lse), lse, pl.splits, 128, 0, units,
                               pl.x_tiles, 128, 0}, g, st);
  } else {
    const bool key_rows = MODE == kSplitDv || MODE == kSplitDk;
    const long long count = (long long)p.B * (key_rows ? (long long)p.Lk * p.Hkv : (long long)p.Lq * p.Hq) * p.D;
    const long long want = (count + 255) / 256;
    launch_next(att_sum_kernel<T>, (unsigned)(want < kSms * 8 ? want : kSms * 8), 256, 0, st, (const float*)part, pl.splits, count,
                MODE == kSplitDv ? 1.0f : p.scale, g);
  }
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

static int clear(void* ptr, size_t bytes, cudaStream_t st) {
  if (ptr == nullptr || bytes == 0 || cudaMemsetAsync(ptr, 0, bytes, st) == cudaSuccess) return FBEV_OK;
  cudaGetLastError();
  return FBEV_ERR_LAUNCH;
}

template <typename T>
static int split_forward(const FbevAttention& p, T* out, float* lse, cudaStream_t st) {
  if (p.Lk == 0) return clear(out, (size_t)p.B * att_rows(p) * p.Hkv * p.D * sizeof(T), st);
  const SplitLayout l = split_layout(p, false);
  const int rc = split_operands<T>(p, l, nullptr, nullptr, nullptr, st);
  return rc != FBEV_OK ? rc : split_result<T, kSplitOut>(p, l, out, lse, st);
}

template <typename T>
static int split_backward(const FbevAttention& p, const T* out, const float* lse, const T* go, T* gq, T* gk, T* gv, cudaStream_t st) {
  if (p.Lq == 0 || p.Lk == 0) {
    const size_t rows = (size_t)p.B * att_rows(p) * p.Hkv * p.D * sizeof(T), keys = (size_t)p.B * p.Lk * p.Hkv * p.D * sizeof(T);
    int rc = clear(gq, rows, st);
    if (rc == FBEV_OK) rc = clear(gk, keys, st);
    return rc == FBEV_OK ? clear(gv, keys, st) : rc;
  }
  const SplitLayout l = split_layout(p, true);
  int rc = split_operands<T>(p, l, out, lse, go, st);
  if (rc == FBEV_OK && gq) rc = split_result<T, kSplitDq>(p, l, gq, nullptr, st);
  if (rc == FBEV_OK && gk) rc = split_result<T, kSplitDv>(p, l, gv, nullptr, st);
  if (rc == FBEV_OK && gk) rc = split_result<T, kSplitDk>(p, l, gk, nullptr, st);
  return rc;
}

template <typename T, int NSUB>
static int tensor_forward(const FbevAttention& p, T* out, float* lse, cudaStream_t st) {
  static std::atomic<uint64_t> granted{0};
  AttFwdArgs a;
  a.p = p;
  a.pl = attention_plan(p);
  int rc = allow_smem(att_fwd_kernel<T, NSUB>, AttFwdShape<NSUB>::kSmem, granted);
  if (rc == FBEV_OK) rc = encode_rows(&a.q, p, a.pl, p.q, p.q_stride, p.q_shared != 0);
  if (rc == FBEV_OK) rc = encode_keys(&a.k, p, p.k, p.k_stride);
  if (rc == FBEV_OK) rc = encode_keys(&a.v, p, p.v, p.v_stride);
  if (rc != FBEV_OK) return rc;
  a.out = out;
  a.lse = lse;
  a.c = score_factor(p);
  a.part = reinterpret_cast<float*>(p.workspace);
  a.part_lse = a.pl.splits > 1 ? reinterpret_cast<float*>(reinterpret_cast<char*>(p.workspace) + split_output_bytes(p, a.pl)) : nullptr;
  const int units = p.B * p.Hkv * a.pl.row_blocks - a.pl.whole;  // split ones
  const unsigned blocks = (unsigned)(a.pl.whole + units * a.pl.splits);
  att_fwd_kernel<T, NSUB><<<blocks, kAttThreads, AttFwdShape<NSUB>::kSmem, st>>>(a);
  if (units > 0)
    launch_join<T>(p, JoinArgs{a.part, a.part_lse, lse, a.pl.splits, 256, a.pl.whole, units, a.pl.row_blocks, a.pl.TL * a.pl.G, 0}, out, st);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T>
static int attention_forward(const FbevAttention& p, T* out, float* lse, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (direct(p))
      return p.D <= 64 ? tensor_forward<T, 1>(p, out, lse, st) : tensor_forward<T, 2>(p, out, lse, st);
  }
  return split_forward<T>(p, out, lse, st);
}

// blocks along the other side when this side's tiles leave SMs idle
static AttGradPlan gradient_plan(const FbevAttention& p, bool kv) {
  AttGradPlan pl{};
  pl.G = p.Hq / p.Hkv;
  pl.TL = 128 / pl.G;
  pl.row_tiles = (p.Lq + pl.TL - 1) / pl.TL;
  pl.key_tiles = (p.Lk + 127) / 128;
  const SplitChoice c = choose_splits(p.B * p.Hkv * (kv ? pl.key_tiles : pl.row_tiles), kv ? pl.row_tiles : pl.key_tiles,
                                      (kv ? 2 : 1) * 128.0 * p.D * 4 / 40000.0, p.key_lengths != nullptr, false);
  pl.splits = c.splits;
  pl.per_split = c.per_split;
  return pl;
}
static size_t gradient_part_bytes(const FbevAttention& p, bool kv) {  // of one of the gradients
  const AttGradPlan pl = gradient_plan(p, kv);
  if (pl.splits == 1) return 0;
  return round_up((size_t)pl.splits * p.B * (kv ? (size_t)p.Lk * p.Hkv : (size_t)p.Lq * p.Hq) * p.D * 4, 256);
}
static size_t stat_bytes(const FbevAttention& p) {  // -lse or -delta by row tile
  return (size_t)p.B * p.Hkv * gradient_plan(p, false).row_tiles * 512;
}
static size_t stat_tile_bytes(const FbevAttention& p) {  // and the tiles in which they meet the matrix instructions
  return 32 * stat_bytes(p);
}
// both statistics, their tiles, then the parts of dQ, and after those are summed the parts of dK and dV in the same place
static size_t backward_workspace(const FbevAttention& p) {
  if (!direct(p)) return split_layout(p, true).bytes;
  const size_t q = gradient_part_bytes(p, false), kv = 2 * gradient_part_bytes(p, true);
  return 2 * stat_bytes(p) + stat_tile_bytes(p) + (q > kv ? q : kv);
}

template <typename T, int NSUB, bool KV>
static int tensor_gradient(const FbevAttention& p, const T* go, T* g0, T* g1, cudaStream_t st) {
  static std::atomic<uint64_t> granted{0};
  AttGradArgs a;
  a.p = p;
  a.pl = gradient_plan(p, KV);
  AttPlan rows{};
  rows.G = a.pl.G;
  rows.TL = a.pl.TL;
  const int64_t go_stride[3] = {(int64_t)p.Lq * p.Hq * p.D, (int64_t)p.Hq * p.D, p.D};
  int rc = allow_smem(att_grad_kernel<T, NSUB, KV>, AttGradShape<NSUB>::kSmem, granted);
  if (rc == FBEV_OK) rc = encode_rows(KV ? &a.y0 : &a.x0, p, rows, p.q, p.q_stride, p.q_shared != 0);
  if (rc == FBEV_OK) rc = encode_rows(KV ? &a.y1 : &a.x1, p, rows, go, go_stride, false);
  if (rc == FBEV_OK) rc = encode_keys(KV ? &a.x0 : &a.y0, p, p.k, p.k_stride);
  if (rc == FBEV_OK) rc = encode_keys(KV ? &a.x1 : &a.y1, p, p.v, p.v_stride);
  char* ws = reinterpret_cast<char*>(p.workspace);
  if (KV && rc == FBEV_OK) {
    const long long rows = 128ll * a.pl.row_tiles, dims[4] = {64, 1, rows, (long long)p.B * p.Hkv}, strides[4] = {1, 64, 64, 64 * rows};
    const int box[4] = {64, 1, 128, 1};
    rc = encode_map(&a.z, p.dtype, 4, ws + 2 * stat_bytes(p), dims, strides, box);
  } else {
    a.z = a.x0;
  }
  if (rc != FBEV_OK) return rc;
  a.nlse = reinterpret_cast<const float*>(ws);
  a.ndelta = reinterpret_cast<const float*>(ws + stat_bytes(p));
  a.part0 = reinterpret_cast<float*>(ws + 2 * stat_bytes(p) + stat_tile_bytes(p));
  a.part1 = reinterpret_cast<float*>(ws + 2 * stat_bytes(p) + stat_tile_bytes(p) + gradient_part_bytes(p, KV));
  a.g0 = g0;
  a.g1 = g1;
  a.c = score_factor(p);
  const long long blocks = (long long)p.B * p.Hkv * (KV ? a.pl.key_tiles : a.pl.row_tiles) * a.pl.splits;
  launch_next(att_grad_kernel<T, NSUB, KV>, (unsigned)blocks, kGradThreads, AttGradShape<NSUB>::kSmem, st, a);
  if (a.pl.splits > 1) {
    const long long count = (long long)p.B * (KV ? (long long)p.Lk * p.Hkv : (long long)p.Lq * p.Hq) * p.D;
    const long long want = (count + 255) / 256;
    const unsigned grid = (unsigned)(want < kSms * 8 ? want : kSms * 8);
    launch_next(att_sum_kernel<T>, grid, 256, 0, st, (const float*)a.part0, a.pl.splits, count, p.scale, g0);
    if (KV) launch_next(att_sum_kernel<T>, grid, 256, 0, st, (const float*)a.part1, a.pl.splits, count, 1.0f, g1);
  }
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T, int NSUB>
static int tensor_backward(const FbevAttention& p, const T* out, const float* lse, const T* go, T* gq, T* gk, T* gv, cudaStream_t st) {
  const AttGradPlan pl = gradient_plan(p, false);
  float* nlse = reinterpret_cast<float*>(p.workspace);
  float* ndelta = reinterpret_cast<float*>(reinterpret_cast<char*>(p.workspace) + stat_bytes(p));
  const unsigned blocks = (unsigned)((long long)p.B * p.Hkv * pl.row_tiles * (4 / kStatRows));
  uint4* tiles = reinterpret_cast<uint4*>(reinterpret_cast<char*>(p.workspace) + 2 * stat_bytes(p));
  att_stat_kernel<T><<<blocks, 256, 0, st>>>(p, pl.TL, pl.row_tiles, out, go, lse, nlse, ndelta, gk ? tiles : nullptr, 1.0f / score_factor(p));
  int rc = cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
  if (rc == FBEV_OK && gq) rc = tensor_gradient<T, NSUB, false>(p, go, gq, (T*)nullptr, st);
  if (rc == FBEV_OK && gk) rc = tensor_gradient<T, NSUB, true>(p, go, gk, gv, st);
  return rc;
}

template <typename T>
static int attention_backward(const FbevAttention& p, const T* out, const float* lse, const T* go, T* gq, T* gk, T* gv,
                              cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (direct(p))
      return p.D <= 64 ? tensor_backward<T, 1>(p, out, lse, go, gq, gk, gv, st) : tensor_backward<T, 2>(p, out, lse, go, gq, gk, gv, st);
  }
  return split_backward<T>(p, out, lse, go, gq, gk, gv, st);
}

}  // namespace fbev

using namespace fbev;

extern "C" {

size_t fbev_cross_attention_lse_count(const FbevAttention* p) {
  if (check_attention(p) != FBEV_OK) return 0;
  return (size_t)p->B * p->Hkv * att_rows_padded(*p);
}

size_t fbev_cross_attention_workspace_bytes(const FbevAttention* p, int backward) {
  if (check_attention(p) != FBEV_OK) return 0;
  return backward ? backward_workspace(*p) : forward_workspace(*p);
}

static int check_workspace(const FbevAttention* p, int backward) {
  const size_t need = fbev_cross_attention_workspace_bytes(p, backward);
  if (need == 0) return FBEV_OK;
  if (p->workspace == nullptr || p->workspace_bytes < need || (uintptr_t)p->workspace % 256) return FBEV_ERR_SCRATCH;
  return FBEV_OK;
}

int fbev_cross_attention(const FbevAttention* p, void* out, float* lse, void* stream) {
  int rc = check_attention(p);
  if (rc != FBEV_OK) return rc;
  if (p->B == 0 || p->Lq == 0) return FBEV_OK;
  if (out == nullptr || !has_pointers(p)) return FBEV_ERR_NULL;
  if ((uintptr_t)out % 16 || (uintptr_t)lse % 16) return FBEV_ERR_ALIGN;
  rc = check_workspace(p, 0);
  if (rc != FBEV_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case FBEV_F32: return attention_forward<float>(*p, reinterpret_cast<float*>(out), lse, st);
    case FBEV_BF16: return attention_forward<__nv_bfloat16>(*p, reinterpret_cast<__nv_bfloat16*>(out), lse, st);
    default: return attention_forward<__half>(*p, reinterpret_cast<__half*>(out), lse, st);
  }
}

int fbev_cross_attention_grad(const FbevAttention* p, const void* out, const float* lse, const void* grad_out, void* grad_q,
                              void* grad_k, void* grad_v, void* stream) {
  int rc = check_attention(p);
  if (rc != FBEV_OK) return rc;
  if ((grad_k == nullptr) != (grad_v == nullptr)) return FBEV_ERR_NULL;
  if (p->B == 0 || (grad_q == nullptr && grad_k == nullptr)) return FBEV_OK;
  const bool queries = p->Lq > 0;
  if (!has_pointers(p) || (queries && (!out || !lse || !grad_out))) return FBEV_ERR_NULL;
  const uintptr_t all = (uintptr_t)out | (uintptr_t)grad_out | (uintptr_t)grad_q | (uintptr_t)grad_k | (uintptr_t)grad_v;
  if (all % 16 || (uintptr_t)lse % 16) return FBEV_ERR_ALIGN;
  rc = check_workspace(p, 1);
  if (rc != FBEV_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    return attention_backward<T>(*p, reinterpret_cast<const T*>(out), lse, reinterpret_cast<const T*>(grad_out),
                                 reinterpret_cast<T*>(grad_q), reinterpret_cast<T*>(grad_k), reinterpret_cast<T*>(grad_v), st);
  };
  switch (p->dtype) {
    case FBEV_F32: return go(float());
    case FBEV_BF16: return go(__nv_bfloat16());
    default: return go(__half());
  }
}

int fbev_rotary_axes(const FbevRotary* p, void* out, void* stream) {
  if (p == nullptr) return FBEV_ERR_NULL;
  if (p->struct_size != sizeof(FbevRotary)) return FBEV_ERR_STRUCT;
  if (!known_dtype(p->dtype) || p->pos_dtype < FBEV_POS_F32 || p->pos_dtype > FBEV_POS_I64) return FBEV_ERR_DTYPE;
  if (p->B < 0 || p->L < 0 || p->H < 0 || p->D <= 0 || p->D > 256 || p->pairs < 0 || 2 * p->pairs > p->D || p->axes < 1 ||
      p->axes > 8)
    return FBEV_ERR_SHAPE;
  for (int i = 0; i < p->pairs; ++i)
    if (p->pair_axis[i] >= p->axes) return FBEV_ERR_SHAPE;
  if (p->B == 0 || p->L == 0 || p->H == 0) return FBEV_OK;
  if (p->x == nullptr || out == nullptr || p->positions == nullptr) return FBEV_ERR_NULL;
  const size_t es = size_of(p->dtype);
  if ((uintptr_t)p->x % es || (uintptr_t)out % es || (uintptr_t)p->positions % (p->pos_dtype == FBEV_POS_I64 ? 8 : 4))
    return FBEV_ERR_ALIGN;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (p->dtype) {
    case FBEV_F32: return rotary_pos<float>(p, out, st);
    case FBEV_BF16: return rotary_pos<__nv_bfloat16>(p, out, st);
    default: return rotary_pos<__half>(p, out, st);
  }
}

static int check_norm(int dtype, long long rows, int C, std::initializer_list<const void*> ptrs) {
  if (!known_dtype(dtype)) return FBEV_ERR_DTYPE;
  if (rows < 0 || C <= 0) return FBEV_ERR_SHAPE;
  if (C > (1 << 20)) return FBEV_ERR_RANGE;
  for (const void* q : ptrs)
    if ((uintptr_t)q % size_of(dtype)) return FBEV_ERR_ALIGN;
  return FBEV_OK;
}

int fbev_add_rms_norm(int dtype, long long rows, int C, float eps, const void* x, const void* residual, const void* weight,
                      void* y, void* h_out, float* rstd, void* stream) {
  const int rc = check_norm(dtype, rows, C, {x, residual, weight, y, h_out});
  if (rc != FBEV_OK) return rc;
  if (rows == 0) return FBEV_OK;
  if (x == nullptr || y == nullptr) return FBEV_ERR_NULL;
  if ((uintptr_t)rstd % 4) return FBEV_ERR_ALIGN;
  NormArgs a{};
  a.x = x; a.r = residual; a.w = weight; a.y = y; a.h = h_out; a.rstd = rstd; a.rows = rows; a.C = C; a.eps = eps;
  return norm_any(dtype, a, false, false, 0, reinterpret_cast<cudaStream_t>(stream));
}

int fbev_add_rms_norm_e4m3(int dtype, long long rows, int C, float eps, const void* x, const void* residual,
                           const void* weight, uint8_t* q, float* scales, void* h_out, void* stream) {
  const int rc = check_norm(dtype, rows, C, {x, residual, weight, h_out});
  if (rc != FBEV_OK) return rc;
  if (rows == 0) return FBEV_OK;
  if (x == nullptr || q == nullptr || scales == nullptr) return FBEV_ERR_NULL;
  if ((uintptr_t)scales % 4) return FBEV_ERR_ALIGN;
  NormArgs a{};
  a.x = x; a.r = residual; a.w = weight; a.y = q; a.h = h_out; a.scales = scales; a.rows = rows; a.C = C; a.eps = eps;
  return norm_any(dtype, a, true, false, 0, reinterpret_cast<cudaStream_t>(stream));
}

size_t fbev_add_rms_norm_grad_workspace_bytes(long long rows, int C, int with_weight) {
  if (rows <= 0 || C <= 0 || C > (1 << 20) || !with_weight) return 0;
  return round_up((size_t)norm_grad_blocks(rows) * C * 4, 256);
}

int fbev_add_rms_norm_grad(int dtype, long long rows, int C, const void* h, const float* rstd, const void* weight,
                           const void* grad_y, const void* grad_h, void* grad_x, void* grad_weight, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const int rc = check_norm(dtype, rows, C, {h, weight, grad_y, grad_h, grad_x, grad_weight});
  if (rc != FBEV_OK) return rc;
  if (grad_x == nullptr && grad_weight == nullptr) return FBEV_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (grad_weight && cudaMemsetAsync(grad_weight, 0, (size_t)C * size_of(dtype), st) != cudaSuccess) {
      cudaGetLastError();
      return FBEV_ERR_LAUNCH;
    }
    return FBEV_OK;
  }
  if (h == nullptr || rstd == nullptr) return FBEV_ERR_NULL;
  if ((uintptr_t)rstd % 4) return FBEV_ERR_ALIGN;
  NormArgs a{};
  a.x = h; a.w = weight; a.rstd_in = rstd; a.dy = grad_y; a.dh = grad_h; a.dx = grad_x; a.rows = rows; a.C = C;
  const long long blocks = norm_grad_blocks(rows);
  if (grad_weight) {
    if (workspace == nullptr || workspace_bytes < fbev_add_rms_norm_grad_workspace_bytes(rows, C, 1) || (uintptr_t)workspace % 256)
      return FBEV_ERR_SCRATCH;
    a.dw_part = reinterpret_cast<float*>(workspace);
  }
  const int lrc = norm_any(dtype, a, false, true, blocks, st);
  if (lrc != FBEV_OK || !grad_weight) return lrc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((C + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const float* part = a.dw_part;
  switch (dtype) {
    case FBEV_F32: cudaLaunchKernelEx(&cfg, norm_dw_kernel<float>, part, (int)blocks, C, reinterpret_cast<float*>(grad_weight)); break;
    case FBEV_BF16: cudaLaunchKernelEx(&cfg, norm_dw_kernel<__nv_bfloat16>, part, (int)blocks, C, reinterpret_cast<__nv_bfloat16*>(grad_weight)); break;
    default: cudaLaunchKernelEx(&cfg, norm_dw_kernel<__half>, part, (int)blocks, C, reinterpret_cast<__half*>(grad_weight)); break;
  }
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

}  // extern "C"
