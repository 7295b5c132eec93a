/*
 * chia_rope.h -- C ABI of the norm of queries and keys with the rotation to their
 * positions (sm_100a), forward and backward.
 *
 * For each row x of head_dim values (a token's query or key of one head):
 *
 *   n = x * rstd * (w + weight_offset),  rstd = 1 / sqrt(mean(x^2) + eps)
 *   y = n with its first `rot` channels turned: pair i by pos * freq_i
 *       (a, b) -> (a cos - b sin, b cos + a sin)
 *
 * Pair i is channels (i, i + rot / 2), or (2 i, 2 i + 1) where `interleaved`. A
 * frequency is given as a fraction of a turn for each position, in units of 2^-64:
 * freqs[i] = round(freq_i / (2 pi) * 2^64). The angle is then a product modulo
 * 2^64, exact for any position.
 *
 * The calls are asynchronous on `stream`, neither allocate nor synchronise, and
 * report argument errors before anything is launched.
 */
#ifndef CHIA_ROPE_H
#define CHIA_ROPE_H

#include "chia_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHIA_ROPE_ABI_VERSION 1

/* element types beside enum chia_dtype */
enum chia_rope_dtype { CHIA_DTYPE_F32 = 2 };

typedef struct chia_rope_params {
  int32_t abi_version; /* CHIA_ROPE_ABI_VERSION                              */
  int32_t dtype;       /* of q, k, their outputs and gradients: bf16, fp16, f32 */
  int32_t weight_dtype; /* of the weights and their gradients: likewise      */
  int32_t head_dim;    /* 64 or 128                                          */
  int32_t heads;       /* of q                                               */
  int32_t heads_kv;    /* of k                                               */
  int32_t rot;         /* channels that turn: a multiple of 8, 0 to head_dim */
  int32_t interleaved;
  int64_t batch;
  int64_t seqlen; /* tokens of each batch entry                              */
  const void *q;  /* unit stride on the channels                             */
  const void *k;
  void *q_out; /* may be q itself (then with its strides)                    */
  void *k_out;
  int64_t q_stride[3]; /* elements: batch, head, token; multiples of 8       */
  int64_t k_stride[3];
  int64_t q_out_stride[3];
  int64_t k_out_stride[3];
  const void *q_weight; /* [head_dim], 16-byte aligned, or NULL: none for this
                           input                                             */
  const void *k_weight;
  const uint64_t *freqs;    /* [rot / 2]                                     */
  const int32_t *positions; /* NULL: 0, 1, 2, ... in each batch entry        */
  int64_t position_stride;  /* elements between batch entries; 0: shared     */
  float eps;
  float weight_offset;
} chia_rope_params_t;

CHIA_API int chia_qk_norm_rope(const chia_rope_params_t *params, void *stream);

/* Gradients of q, k (dq, dk, strides like those of the outputs in params: element
 * strides q_out_stride, k_out_stride belong to dq and dk here) and of the weights
 * (dq_weight, dk_weight [head_dim], or NULL), from those of the outputs. q_out and
 * k_out of params are not used. The weights' gradients are summed in an order that
 * does not change from call to call. */
typedef struct chia_rope_grads {
  const void *dq_out; /* unit stride on the channels                         */
  const void *dk_out;
  int64_t dq_out_stride[3];
  int64_t dk_out_stride[3];
  void *dq;
  void *dk;
  void *dq_weight;
  void *dk_weight;
} chia_rope_grads_t;

/* workspace: chia_qk_norm_rope_bwd_workspace_bytes() bytes, 16-byte aligned; used
 * during the call only. */
CHIA_API int chia_qk_norm_rope_bwd(const chia_rope_params_t *params, const chia_rope_grads_t *grads,
                                   void *workspace, int64_t workspace_bytes, void *stream);
CHIA_API int64_t chia_qk_norm_rope_bwd_workspace_bytes(const chia_rope_params_t *params);

#ifdef __cplusplus
}
#endif

#endif /* CHIA_ROPE_H */
