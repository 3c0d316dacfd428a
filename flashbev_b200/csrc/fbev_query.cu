// The operators of include/fbev_query.h: argument checks, plans, launches and the C ABI.  Kernels:
// fbev_attention.cuh, fbev_rotary.cuh, fbev_norm.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fbev_query.h"
#include "fbev_attention.cuh"
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
  if (att_rows(*p) >= (1ll << 31) || (long long)p->B * p->Hq >= (1ll << 31)) return FBEV_ERR_RANGE;
  if ((long long)p->B * p->Hkv * (att_rows(*p) / 4 + 1) >= (1ll << 31) || (long long)p->B * p->Hkv * (p->Lk / 4 + 1) >= (1ll << 31))
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

template <typename T>
static int attention_forward(const FbevAttention& p, T* out, float* lse, cudaStream_t st) {
  const long long units = att_rows(p) * p.B * p.Hkv;
  att_row_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, st>>>(p, out, lse);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
}

template <typename T>
static int attention_backward(const FbevAttention& p, const T* out, const float* lse, const T* go, T* gq, T* gk, T* gv,
                              cudaStream_t st) {
  float* delta = reinterpret_cast<float*>(p.workspace);
  const long long units = att_rows(p) * p.B * p.Hkv, keys = (long long)p.B * p.Lk * p.Hkv;
  if (units > 0) att_delta_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, st>>>(p, out, go, delta);
  if (gq && units > 0) att_row_grad_q_kernel<T><<<(unsigned)((units + 3) / 4), 128, 0, st>>>(p, lse, delta, go, gq);
  if (gk && keys > 0) att_row_grad_kv_kernel<T><<<(unsigned)((keys + 3) / 4), 128, 0, st>>>(p, lse, delta, go, gk, gv);
  return cudaGetLastError() == cudaSuccess ? FBEV_OK : FBEV_ERR_LAUNCH;
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
  return backward ? round_up(fbev_cross_attention_lse_count(p) * 4, 256) : 0;
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
  if ((uintptr_t)out % size_of(p->dtype) || (uintptr_t)lse % 16) return FBEV_ERR_ALIGN;
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
  if (all % size_of(p->dtype) || (uintptr_t)lse % 16) return FBEV_ERR_ALIGN;
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
