/*
 * fbev_query.h - C ABI of the operators for a view transform in which BEV queries attend to camera tokens:
 * cross attention, rotary positions with several axes, residual addition + root-mean-square norm.  Same library
 * (libfbev.so), status codes, element types and conventions as fbev.h: device pointers the caller owns, borrowed for
 * the asynchronous launch; nothing is allocated, freed or synchronised; an FBEV_* status instead of an exception.
 * The reference (yokosyun/FlashBEV) has no counterpart of these operators.
 */
#ifndef FBEV_QUERY_H_
#define FBEV_QUERY_H_

#include <stddef.h>
#include <stdint.h>

#include "fbev.h"

#ifdef __cplusplus
extern "C" {
#endif

/* bits a kernel of this header may OR into the optional device status word (FBEV_DEV_* of fbev.h is bit 0) */
enum { FBEV_DEV_TIMEOUT = 2 /* a wait inside an attention kernel ran out; its output is not valid */ };

/*
 * One attention call.  For every sample b, query l and head h, with g = h / (Hq / Hkv):
 *   S_j = scale * <q[b,l,h], k[b,j,g]> over the keys j that may be attended: j < key_lengths[b] (where given) and
 *   key_mask[b,j] != 0 (where given);  out[b,l,h] = sum_j softmax(S)_j v[b,j,g].
 * A row without any such key gives zeros and zero gradients; one with NaN or +infinity among its scores, or with none above
 * -infinity, gives NaN, as do the gradients it reaches.  What stands in keys and values that may not be attended
 * (infinities, NaN) has no influence.  All sums and statistics are held in float32.
 */
typedef struct FbevAttention {
  uint32_t struct_size;       /* sizeof(FbevAttention) */
  int32_t dtype;              /* FBEV_F32 / FBEV_BF16 / FBEV_F16: q, k, v, the output and all gradients */
  int32_t B, Lq, Lk;          /* samples, queries, keys; zeros are allowed */
  int32_t Hq, Hkv, D;         /* query heads, key heads (a divisor of Hq), head width 1..128 */
  float scale;                /* finite, at most 1e30 in magnitude */
  int32_t q_shared;           /* 1: the queries are the same for every sample; q_stride[0] is not used */
  int64_t q_stride[3];        /* elements from sample to sample, token to token, head to head; the head's elements */
  int64_t k_stride[3];        /*   are contiguous */
  int64_t v_stride[3];
  int64_t mask_stride;        /* bytes from one sample's key_mask to the next, 0: one mask for all */
  const void* q;
  const void* k;
  const void* v;
  const int32_t* key_lengths; /* device [B] or NULL; values outside 0..Lk are clamped */
  const uint8_t* key_mask;    /* device [B,Lk] bytes, 0 = may not be attended, or NULL */
  uint32_t* status;           /* optional device word, FBEV_DEV_* */
  void* workspace;            /* device, 256-byte aligned, not shared by calls that may overlap */
  uint64_t workspace_bytes;   /* at least fbev_cross_attention_workspace_bytes() of the same call */
} FbevAttention;

/* Number of float32 values of the statistics tensor `lse`: one per query and head, each (sample, key head) padded to a
 * multiple of four; 0 for an invalid problem.  A forward with Lk = 0 leaves them as they were (its backward reads none). */
size_t fbev_cross_attention_lse_count(const FbevAttention* p);

/* Device bytes of workspace for the forward (backward = 0) or the backward (backward = 1); 0 for an invalid problem. */
size_t fbev_cross_attention_workspace_bytes(const FbevAttention* p, int backward);

/* out: device, contiguous [B,Lq,Hq,D], 16-byte aligned.  lse: device, 16-byte aligned, fbev_cross_attention_lse_count()
 * floats for the backward, or NULL. */
int fbev_cross_attention(const FbevAttention* p, void* out, float* lse, void* stream);

/* Gradients of sum(out * grad_out).  out, grad_out: contiguous [B,Lq,Hq,D]; lse: as the forward left it.
 * grad_q [B,Lq,Hq,D], grad_k and grad_v [B,Lk,Hkv,D], contiguous, overwritten; all 16-byte aligned; grad_q, or grad_k and
 * grad_v together, may be NULL.  The results do not depend on the order in which blocks run. */
int fbev_cross_attention_grad(const FbevAttention* p, const void* out, const float* lse, const void* grad_out,
                              void* grad_q, void* grad_k, void* grad_v, void* stream);

/*
 * Rotary positions.  x, out [B,L,H,D]; the first 2 * pairs elements of a head are rotated pair by pair, the rest is
 * copied.  Pair p belongs to axis pair_axis[p] and turns by positions[b,l,axis] * 2 pi * pair_turns[p]; it consists of
 * the elements (2p, 2p+1) when interleaved, else of (p, pairs + p).  Angles are reduced in float64.  inverse turns the
 * other way: the gradient.
 */
enum { FBEV_POS_F32 = 0, FBEV_POS_I32 = 1, FBEV_POS_I64 = 2 };
#define FBEV_ROTARY_MAX_PAIRS 128
typedef struct FbevRotary {
  uint32_t struct_size;       /* sizeof(FbevRotary) */
  int32_t dtype;              /* element type of x and out */
  int32_t B, L, H, D;         /* D <= 256; zeros are allowed for B, L and H */
  int32_t pairs, axes;        /* 2 * pairs <= D, 1 <= axes <= 8 */
  int32_t interleaved, inverse;
  int32_t pos_dtype;          /* FBEV_POS_* */
  int32_t reserved;           /* 0 */
  int64_t x_stride[3];        /* elements: sample, token, head; a head's elements are contiguous */
  int64_t pos_stride;         /* elements from one sample's positions [L,axes] to the next, 0: one for all */
  const void* x;
  const void* positions;      /* device [B,L,axes] */
  double pair_turns[FBEV_ROTARY_MAX_PAIRS];
  uint8_t pair_axis[FBEV_ROTARY_MAX_PAIRS];
} FbevRotary;

/* out: device, contiguous [B,L,H,D]; may be x itself when x is contiguous. */
int fbev_rotary_axes(const FbevRotary* p, void* out, void* stream);

/*
 * h = x + residual (x alone when residual is NULL); rstd = (mean(h^2) + eps)^(-1/2); y = h * rstd * weight (ones when
 * NULL), all from the unrounded float32 sum.  Rows of C contiguous elements.  h_out [rows,C] may be NULL (and may be x
 * or residual themselves); rstd [rows] may be NULL.
 */
int fbev_add_rms_norm(int dtype, long long rows, int C, float eps, const void* x, const void* residual, const void* weight,
                      void* y, void* h_out, float* rstd, void* stream);

/* The same with y in 8 bits (E4M3): scales[row] = max|y| / 448, or 1 where that is 0, and q = y / scale rounded to
 * nearest even. */
int fbev_add_rms_norm_e4m3(int dtype, long long rows, int C, float eps, const void* x, const void* residual,
                           const void* weight, uint8_t* q, float* scales, void* h_out, void* stream);

/* Device bytes of workspace of the gradient (256-byte aligned); 0 when grad_weight is not asked for. */
size_t fbev_add_rms_norm_grad_workspace_bytes(long long rows, int C, int with_weight);

/* h and rstd: as the forward left them (h = x when there was no residual).  grad_y, grad_h [rows,C]: upstream
 * gradients of y and of the sum; either may be NULL (zero).  grad_x [rows,C] (it is the residual's gradient too) and
 * grad_weight [C]; either may be NULL.  The results do not depend on the order in which blocks run. */
int fbev_add_rms_norm_grad(int dtype, long long rows, int C, const void* h, const float* rstd, const void* weight,
                           const void* grad_y, const void* grad_h, void* grad_x, void* grad_weight, void* workspace,
                           size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FBEV_QUERY_H_ */
