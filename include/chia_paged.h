/*
 * chia_paged.h -- C ABI for serving from a paged 8-bit K/V cache (sm_100a).
 *
 * One step of a serving loop is three calls on one stream:
 *
 *   chia_page_tables   the step's new pages, slots, positions and offsets from
 *                      the requests' lengths (chia_release_pages gives the
 *                      pages of finished requests back, chia_trim_pages those
 *                      of rejected tokens)
 *   chia_cache_append  the new tokens' keys and values into the cache, in 8
 *                      bits with one scale for each (page, K/V head)
 *   chia_paged_attn    the step's queries over the cache: every operator of
 *                      chia_attn.h (score modification, mask, normaliser)
 *
 * The cache. k_cache and v_cache are [num_pages, heads_kv, page_size, head_dim]
 * bytes (e4m3 or int8), contiguous; k_scale and v_scale are fp32, not negative,
 * [num_pages, heads_kv]. A stored value q stands for q * scale. chia_cache_append
 * writes scales that are powers of two: the smallest 2^e, e >= -64, with
 * max|x| <= 448 * 2^e (e4m3) or 127 * 2^e (int8), the maximum taken over the
 * finite values of the page's tokens and the head's channels.
 *
 * Requests. Request b's keys are the first seq_lens[b] tokens of the pages
 * block_table[b][0], block_table[b][1], ...; its queries are the rows
 * [cu_q[b], cu_q[b + 1]) of q and stand for its last tokens: query i of n has
 * position seq_lens[b] - n + i, and the masks of chia_attn.h apply to positions.
 *
 * All calls are asynchronous on `stream`, never synchronise or allocate, and
 * report argument errors before anything is launched. What only the device can
 * see (a page or slot out of range, no free page left) is OR-ed into *status
 * and skipped; no call reads or writes outside the tensors it is given.
 */
#ifndef CHIA_PAGED_H
#define CHIA_PAGED_H

#include "chia_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHIA_PAGED_ABI_VERSION 1

/* further bits of *status (beside enum chia_status) */
enum chia_paged_status {
  CHIA_ERR_BAD_INDEX = 8, /* a length, page, slot or offset out of range      */
  CHIA_ERR_NO_PAGES = 16  /* a request was not served: no free page, or its
                             row of the block table is full                  */
};

/* element types of the cache */
enum chia_cache_dtype { CHIA_CACHE_E4M3 = 0, CHIA_CACHE_INT8 = 1 };

/* ------------------------------------------------------------------ tables */
typedef struct chia_tables_params {
  int32_t abi_version; /* CHIA_PAGED_ABI_VERSION                             */
  int32_t page_size;   /* 16, 32, 64 or 128                                  */
  int64_t batch;       /* requests (rows of the block table)                 */
  int64_t table_width; /* pages a row holds                                  */
  int64_t table_stride; /* elements between rows                             */
  int64_t ring_size;   /* entries of free_pages                              */
  int64_t max_tokens;  /* entries of slots and positions                     */
  const int32_t *seq_lens; /* [batch] tokens in the cache before the step    */
  const int32_t *new_lens; /* [batch] tokens the step adds (tables); non-zero:
                              the request is finished (release); tokens that
                              it keeps (trim)                                */
  int32_t *block_table;    /* [batch, table_width]; new pages are entered    */
  int32_t *free_pages;     /* ring of free pages; release writes its tail    */
  const int32_t *free_state; /* [2]: first entry of the ring, number of pages */
  int32_t *slots;     /* out [max_tokens] page * page_size + offset, -1: none */
  int32_t *positions; /* out [max_tokens]                                    */
  int32_t *cu_q;      /* out [batch + 1] offsets of each request's tokens    */
  int32_t *new_seq_lens;   /* out [batch]                                    */
  int32_t *new_free_state; /* out [2]                                        */
  int32_t *status;    /* optional                                            */
} chia_tables_params_t;

/* The tables of a step. Request b needs ceil((len + new) / page_size) -
 * ceil(len / page_size) new pages; requests take pages from the ring's head in
 * order. A request that would not fit its row of the table, or that needs pages
 * when the ring has not enough left for it and those before it, is not served:
 * its slots are -1, its length stays, and CHIA_ERR_NO_PAGES is reported (cu_q
 * counts its tokens all the same). A free_state out of range is reported and
 * taken as an empty ring. Tokens past max_tokens are reported; they have pages
 * and count in the lengths, but no slots. Entries of slots and positions past the
 * step's tokens are -1 and 0. seq_lens and free_state are not changed (the new
 * ones are outputs), so a step may be run again. */
CHIA_API int chia_page_tables(const chia_tables_params_t *params, void *stream);

/* The pages of finished requests (new_lens[b] != 0) go to the ring's tail, in
 * order; their lengths become 0 in new_seq_lens. A request whose length is more
 * than its row holds is reported and keeps length and pages; where free_state is
 * out of range all do, and new_free_state is an empty ring. The outputs slots,
 * positions and cu_q are not used. */
CHIA_API int chia_release_pages(const chia_tables_params_t *params, void *stream);

/* The same for the tail of a request, after drafted tokens were rejected: it keeps
 * its first new_lens[b] tokens (0 to seq_lens[b]; anything else is reported and
 * keeps all), and the pages past them go to the ring. A length that is lowered
 * without this call takes the pages past it out of use: chia_page_tables enters
 * new ones over them. */
CHIA_API int chia_trim_pages(const chia_tables_params_t *params, void *stream);

/* ------------------------------------------------------------------ append */
typedef struct chia_append_params {
  int32_t abi_version;
  int32_t dtype;       /* enum chia_dtype: type of k and v                   */
  int32_t cache_dtype; /* enum chia_cache_dtype                              */
  int32_t head_dim;    /* 64 or 128                                          */
  int32_t heads_kv;
  int32_t page_size;
  int64_t tokens;
  int64_t num_pages;
  const void *k; /* [tokens, heads_kv, head_dim], unit stride on head_dim     */
  const void *v;
  int64_t k_stride[2]; /* elements: token, head; multiples of 8              */
  int64_t v_stride[2];
  const int32_t *slots; /* [tokens]; -1: the token is skipped                */
  void *k_cache;
  void *v_cache;
  float *k_scale;
  float *v_scale;
  int32_t *status; /* optional                                               */
} chia_append_params_t;

/* The tokens of one page in one call are adjacent rows of k and v (as
 * chia_page_tables lays them out), skipped ones between them or not, page_size
 * rows at most. A page that comes again within so many rows is reported, and those
 * tokens are left out; further apart it is not seen, and what the page then holds
 * is not defined. Where they hold the page's first slot the
 * page begins anew: its scale comes from them alone. Otherwise the page keeps
 * its scale if that is large enough for them, or takes theirs, and then every
 * value the page holds is expressed in the new scale. Values are rounded to
 * nearest, ties to even; infinities become the largest value, NaN stays NaN
 * (e4m3) or becomes 0 (int8). */
CHIA_API int chia_cache_append(const chia_append_params_t *params, void *stream);

/* --------------------------------------------------------------- attention */
typedef struct chia_paged_params {
  int32_t abi_version;
  int32_t dtype;       /* enum chia_dtype: type of q and o                   */
  int32_t cache_dtype; /* enum chia_cache_dtype                              */
  int32_t head_dim;    /* 64 or 128                                          */
  int32_t norm;        /* enum chia_norm                                     */
  int32_t mod;         /* enum chia_mod                                      */
  int32_t heads;
  int32_t heads_kv;    /* divides heads                                      */
  int32_t page_size;   /* 16, 32, 64 or 128                                  */
  int32_t max_q;       /* most queries of any request, as far as the host
                          knows: chooses the schedule, never the result      */
  int64_t batch;
  int64_t tokens;      /* rows of q and o                                    */
  int64_t num_pages;
  int64_t table_width;
  int64_t table_stride;
  const void *q; /* [tokens, heads, head_dim], unit stride on head_dim        */
  void *o;       /* likewise                                                 */
  int64_t q_stride[2]; /* elements: token, head; multiples of 8              */
  int64_t o_stride[2];
  const void *k_cache;
  const void *v_cache;
  const float *k_scale;
  const float *v_scale;
  const int32_t *block_table;
  const int32_t *seq_lens; /* [batch] keys of each request, its queries' own
                              tokens among them                              */
  const int32_t *cu_q; /* [batch + 1], not falling, or NULL: tokens / batch
                          queries each. Where an offset falls or is out of range
                          the requests from there on may not be served          */
  float *lse;          /* optional fp32 [tokens, heads], softmax only        */
  const float *head_param; /* as in chia_attn.h                              */
  float scale;
  float softcap;
  float sig_bias;
  float out_scale;
  int64_t win_left; /* the mask of chia_attn.h, on positions                 */
  int64_t win_right;
  int64_t block;
  int64_t prefix;
  int64_t dilation;
  int32_t *status; /* optional                                               */
  void *workspace; /* chia_paged_attn_workspace_bytes() bytes, 256-byte
                      aligned, zero-filled before its first use and left so
                      that any later call may use it; calls that share one
                      must not overlap on the GPU                            */
  int64_t workspace_bytes;
  uint64_t wait_limit_ns; /* as in chia_attn.h                               */
} chia_paged_params_t;

/* Keys whose page is out of range are reported and left out, as if the mask hid
 * them; entries of pages that no query sees may be anything. A row that sees no key gets zeros (log-sum-exp -inf). Rows of q that no
 * request owns are not written. */
CHIA_API int chia_paged_attn(const chia_paged_params_t *params, void *stream);

/* Workspace bytes of chia_paged_attn on the current device (host only); -1
 * when params are invalid. */
CHIA_API int64_t chia_paged_attn_workspace_bytes(const chia_paged_params_t *params);

#ifdef __cplusplus
}
#endif

#endif /* CHIA_PAGED_H */
