"""Speculative decoding over the paged 8-bit K/V cache (``include/chia_draft.h``): trees of drafted tokens.

A step checks a tree of drafted tokens for each request: its last ``n`` tokens, at most 64. Node 0 is the token that is
decided already; ``parents[t]`` is the node (counted within the request) that node ``t``'s token follows, ``-1`` for a
root. A row of single drafts is the tree with ``parents = -1, 0, 1, ...``. On one stream, without a synchronisation::

    step = page_tables(seq_lens, new_lens, block_table, free_pages, free_state, page_size=64, max_tokens=T)
    tree = tree_tables(parents, step.cu_q, step.seq_lens)
    # in each layer
    q, k = qk_norm_rope(q, k, q_weight, k_weight, freqs, tree.positions)
    cache_append(k, v, step.slots, *cache)
    out = paged_attention(q, *cache, block_table, step.seq_lens, step.cu_q, max_q=..., tree=tree)
    # then
    done = verify_drafts(target_probs, tokens, parents, step.cu_q, uniforms, draft_probs=..., max_tokens=...)
    # in each layer
    keep = cache_compact(done.path, done.counts, step.cu_q, step.seq_lens, block_table, *cache, step.slots)
    seq_lens, free_state = release_pages(None, step.seq_lens, block_table, free_pages, step.free_state,
                                         page_size=64, keep_lens=keep)

Chunks of prompts may stand beside the trees in all calls but ``verify_drafts``, to which every request is a tree. With the
trees first, ``n`` of them, ``verify_drafts`` and ``cache_compact`` take the first parts of the tables (``step.cu_q[:n + 1]``,
``step.seq_lens[:n]``, ``block_table[:n]``), and ``keep`` is what comes back and the others' lengths.

All computation happens in ``libchia_attn.so`` on the current CUDA stream; there is no CPU or PyTorch fallback. What only
the GPU can see (a parent or a page out of range) is skipped there and raised by ``check_device_status``.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N
from .paged import TreeStep, _status

__all__ = ["TreeStep", "Verified", "tree_tables", "verify_drafts", "cache_compact"]


class Verified(NamedTuple):
    """What ``verify_drafts`` returns; all int32 on the GPU."""

    counts: torch.Tensor  # [B] tokens that came out: the accepted ones and one more
    tokens: torch.Tensor  # [B, max_tokens] the tokens, -1 behind them
    path: torch.Tensor    # [B, max_tokens] node 0 and the accepted nodes, -1 behind them


def tree_tables(parents: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor) -> TreeStep:
    """Positions and ancestors of the trees' nodes, for the norm, the rotation and the attention of all layers.

    ``parents`` ``[T]``, ``cu_q`` ``[B + 1]`` and ``seq_lens`` ``[B]`` (with the trees' tokens, as ``page_tables`` returns
    it), int32 on the GPU. A parent comes before its children; another one is reported and its node a root. A request of
    more than 64 tokens is a chunk of a prompt: its tokens follow one another, its parents are not looked at. Rows that no
    request owns get zeros.
    """
    r = N.binding().tree_tables(parents, cu_q, seq_lens, _status(parents))
    if type(r) is int:
        N.check(r, "chia_tree_tables")
    return TreeStep(*r)


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_q: torch.Tensor,
                  uniforms: torch.Tensor, *, draft_probs: Optional[torch.Tensor] = None, max_tokens: int) -> Verified:
    """Which drafted tokens stand, and the token that follows them, so that all of them are distributed as the target's
    own samples.

    ``target_probs`` ``[T, V]`` (fp32, bf16 or fp16): row ``t``, the target's probabilities of what follows node ``t``.
    ``draft_probs``: likewise those that the children of node ``t`` were drawn from, one after another without
    replacement, in their order; ``None``: the tree was not drawn at random. ``tokens``, ``parents`` ``[T]``, ``cu_q``
    ``[B + 1]`` int32; ``uniforms`` ``[T]`` fp32 in ``[0, 1)``: each drafted node is asked with its own number, the token
    that follows is drawn with that of node 0.

    At a node the residual ``r`` begins as its target row, with the mass ``Z = 1``. Child ``c`` with token ``x`` is
    accepted where ``u Z q(x) < r(x) (1 - s)``, ``s`` being what its earlier siblings had of ``q``; else ``r = max(r - Z /
    (1 - s) q, 0)``, ``q`` loses ``x`` and ``Z = sum r``. Without draft probabilities: where ``u Z < r(x)``, else ``r``
    and ``Z`` lose it. Where no child is accepted, or ``max_tokens - 1`` tokens are, the next token is drawn from ``r``:
    the first ``x`` with ``sum_{y <= x} r(y) > u sum r``. Entries that are not positive finite numbers count as zero, an
    empty residual as the row itself; a row of zeros gives -1. All of this is computed in 64 bits. A request without
    tokens has a count of 0; so has one of more than 64, which is reported: chunks of prompts are not verified (above). Rows
    whose width is a multiple of four are read fastest (131,073 entries take a third longer than 131,072).
    """
    r = N.binding().verify(target_probs, tokens, parents, cu_q, uniforms, draft_probs, max_tokens, _status(target_probs))
    if type(r) is int:
        N.check(r, f"chia_verify_drafts(probs={tuple(target_probs.shape)}, max_tokens={max_tokens})")
    return Verified(*r)


def cache_compact(path: torch.Tensor, counts: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
                  block_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Move the keys and values of an accepted path together, in place: node ``path[b, i]``'s go to the place of node
    ``i``, for ``i < counts[b]``. Returns the lengths that the requests keep, ``[B]`` int32, for ``release_pages``.

    A page keeps its scale or, where a page that its new tokens come from has a larger one, takes that and has its values
    expressed in it, as in ``cache_append``. A path rises. One that does not, or whose pages are out of range, is
    reported, and its request left as it is; requests of more than 64 tokens (chunks) are left as they are.

    ``slots`` (``[T]`` int32, what ``page_tables`` returned): a request that it did not serve, whose tokens have no slot,
    is left as it is with its length, so that the step may be run again. Without ``slots`` the last tokens of such a request,
    which are none of the tree's, would be taken for it.
    """
    r = N.binding().compact(path, counts, cu_q, seq_lens, block_table, k_cache, v_cache, k_scale, v_scale,
                            _status(k_cache), slots)
    if type(r) is int:
        N.check(r, f"chia_cache_compact(path={tuple(path.shape)}, cache={tuple(k_cache.shape)})")
    return r
