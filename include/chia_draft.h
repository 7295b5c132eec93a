/*
 * chia_draft.h -- C ABI for speculative decoding over the paged 8-bit K/V cache of
 * chia_paged.h: trees of drafted tokens.
 *
 * A request's tree is its last n = cu_q[b + 1] - cu_q[b] tokens, at most
 * CHIA_TREE_NODES. Node 0 is the token that is decided already, the others are
 * drafted; parents[t] is the node (counted in the request) that node t's token
 * follows, smaller than its own number, or -1 for a root. Their keys and values
 * stand in the cache in the order of the nodes, behind the seq_lens[b] - n tokens
 * before the tree. A step is
 *
 *   chia_page_tables, chia_tree_tables   slots; positions and ancestors
 *   chia_cache_append, chia_tree_attn    in each layer
 *   chia_verify_drafts                   which path is accepted, what follows it
 *   chia_cache_compact                   in each layer: the path's keys and values
 *                                        together
 *   chia_trim_pages                      the other drafts' pages
 *
 * As in chia_paged.h, calls are asynchronous, report argument errors before they
 * launch anything, and what only the device can see is OR-ed into *status and
 * skipped.
 */
#ifndef CHIA_DRAFT_H
#define CHIA_DRAFT_H

#include "chia_paged.h"
#include "chia_rope.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHIA_DRAFT_ABI_VERSION 1
#define CHIA_COMPACT_ABI_VERSION 2
#define CHIA_TREE_NODES 64

/* ------------------------------------------------------------------ tables */
typedef struct chia_tree_params {
  int32_t abi_version; /* CHIA_DRAFT_ABI_VERSION                             */
  int32_t pad;
  int64_t batch;
  int64_t tokens;          /* entries of parents, positions and ancestors    */
  const int32_t *parents;  /* [tokens]                                       */
  const int32_t *cu_q;     /* [batch + 1], as in chia_paged.h                */
  const int32_t *seq_lens; /* [batch], the trees' tokens among them          */
  int32_t *positions;      /* out: seq_lens[b] - n + the node's depth        */
  uint64_t *ancestors; /* out: bit i: node i is an ancestor, or the node itself */
  int32_t *status;     /* optional                                           */
} chia_tree_params_t;

/* A request of more than CHIA_TREE_NODES tokens is no tree but a chunk of a prompt:
 * its tokens follow one another, its parents are not looked at and its words are 0.
 * A parent out of range is reported, its node a root. Rows that no request owns get
 * zeros. */
CHIA_API int chia_tree_tables(const chia_tree_params_t *params, void *stream);

/* --------------------------------------------------------------- attention */
/* chia_paged_attn for trees: a node sees the keys before its tree that the mask
 * shows to its position, and of the tree's keys those in its word that the mask does
 * not put too far back (win_left, the begin of a block, the dilation, of positions;
 * score modifications likewise). The workspace is that of chia_paged_attn.
 * positions and ancestors are those of chia_tree_tables; a position outside of its
 * request's tokens counts as the nearest inside. The words may hold any nodes of
 * the request. Requests of more than CHIA_TREE_NODES queries see what they see in
 * chia_paged_attn. The kernel is chosen for the call, by the mean number of rows of a
 * request: padding (requests without tokens) counts in it. */
CHIA_API int chia_tree_attn(const chia_paged_params_t *params, const int32_t *positions,
                            const uint64_t *ancestors, void *stream);

/* ------------------------------------------------------------ verification */
typedef struct chia_verify_params {
  int32_t abi_version;
  int32_t dtype; /* of the probabilities: bf16, fp16 or f32                  */
  int64_t batch;
  int64_t tokens;
  int64_t vocab;      /* at most 2^22                                        */
  int64_t max_tokens; /* width of out_tokens and path, at least 1            */
  const void *target_probs; /* [tokens, vocab]: row t, what follows node t   */
  const void *draft_probs;  /* likewise what its children were drawn from, or
                               NULL: they were not drawn at random           */
  int64_t target_stride; /* elements between rows                            */
  int64_t draft_stride;
  const int32_t *node_tokens; /* [tokens] in [0, vocab)                      */
  const int32_t *parents;
  const int32_t *cu_q;
  const float *uniforms; /* [tokens] in [0, 1)                               */
  int32_t *counts;       /* out [batch]                                      */
  int32_t *out_tokens;   /* out [batch, max_tokens]                          */
  int32_t *path;         /* out [batch, max_tokens]                          */
  int32_t *status;       /* optional                                         */
} chia_verify_params_t;

/* Which drafted tokens of each request stand, so that what comes out is distributed
 * as the target's own samples are. At a node (first node 0) the residual is
 * r = its target row, of mass Z = 1. Its children are asked in their order. Child c
 * with token x and number u, q the node's draft row, s what q gives to its earlier
 * siblings (children are drawn one after another without replacement):
 *
 *   accepted where  u Z q(x) < r(x) (1 - s)      (the walk goes on at c)
 *   else  r = max(r - Z / (1 - s) q, 0), q without x from now on,  Z = sum r
 *
 * and without draft rows: accepted where u Z < r(x), else r(x) = 0 and Z loses it.
 * Where no child is accepted (or max_tokens - 1 are) a token is drawn from r with
 * the number of node 0: the first x with sum_{y <= x} r(y) > u sum r (the last one
 * of positive r where there is none). A residual that holds nothing counts as the
 * row itself, a row that holds nothing gives -1. Entries that are not positive
 * finite numbers count as 0. Sums, products and comparisons are in 64 bits.
 *
 * out_tokens[b]: the accepted tokens, then the drawn one; path[b]: node 0, then the
 * accepted nodes; counts[b] of each, -1 behind them. counts[b] is 0 for a request
 * without tokens. A request of more than CHIA_TREE_NODES tokens is reported and
 * gets 0; a parent or token out of range is reported, its node never accepted. A
 * request of fewer is a tree whatever it holds: with chunks of prompts in a step, pass
 * the offsets of the trees alone. Rows are read four entries at a time where their
 * addresses are multiples of that. */
CHIA_API int chia_verify_drafts(const chia_verify_params_t *params, void *stream);

/* -------------------------------------------------------------- compaction */
typedef struct chia_compact_params {
  int32_t abi_version; /* CHIA_COMPACT_ABI_VERSION, or 1: without the last two */
  int32_t cache_dtype; /* enum chia_cache_dtype                              */
  int32_t head_dim;    /* 64 or 128                                          */
  int32_t heads_kv;
  int32_t page_size;
  int32_t pad;
  int64_t batch;
  int64_t max_tokens; /* width of path                                       */
  int64_t num_pages;
  int64_t table_width;
  int64_t table_stride;
  const int32_t *path;   /* [batch, max_tokens]: nodes that rise             */
  const int32_t *counts; /* [batch]                                          */
  const int32_t *cu_q;
  const int32_t *seq_lens;
  const int32_t *block_table;
  void *k_cache;
  void *v_cache;
  float *k_scale;
  float *v_scale;
  int32_t *keep_lens; /* out [batch]: seq_lens[b] - n + counts[b], what
                         chia_trim_pages takes                               */
  int32_t *status;    /* optional                                            */
  const int32_t *slots; /* [tokens], those of chia_page_tables, or NULL: every
                           request's tokens are in the cache                 */
  int64_t tokens;
} chia_compact_params_t;

/* Keys and values of node path[b][i] go to the place of node i, for i < counts[b].
 * A page takes the largest scale of the pages that its new tokens come from where
 * that is larger than its own, and what it holds is then expressed in it, as
 * chia_cache_append does. A request whose path does not rise, has nodes that are not
 * its own or pages out of range is reported and left as it is, with its seq_lens[b].
 * So, without a report, is one that chia_page_tables did not serve (a slot of its
 * tokens is -1): its seq_lens[b] has no tree in it, and the step may be run again.
 * No two requests share a page that is written. */
CHIA_API int chia_cache_compact(const chia_compact_params_t *params, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* CHIA_DRAFT_H */
