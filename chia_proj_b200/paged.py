"""Serving from a paged 8-bit K/V cache (``include/chia_paged.h``).

One step of a serving loop, on one stream and without a synchronisation::

    step = page_tables(seq_lens, new_lens, block_table, free_pages, free_state,
                       page_size=64, max_tokens=q.shape[0])
    cache_append(k, v, step.slots, k_cache, v_cache, k_scale, v_scale)
    out = paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table,
                          step.seq_lens, step.cu_q, max_q=...)
    seq_lens, free_state = step.seq_lens, step.free_state

The cache is four tensors (``new_cache`` makes them): ``k_cache``, ``v_cache``
``[num_pages, H_kv, page_size, D]`` in float8_e4m3fn or int8, and fp32 scales
``[num_pages, H_kv]``: one scale for each block of ``page_size`` tokens and
head. A stored value ``x`` stands for ``x * scale``. All computation happens in
``libchia_attn.so`` on the current CUDA stream; there is no CPU or PyTorch
fallback. What only the GPU can see (a page out of range, an empty free list)
is skipped there and raised by ``check_device_status``.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from .ops import CAUSAL, Mask, _MODS, _NORMS, _cached_default, _param_tensor, _status_word

__all__ = ["PAGE_SIZES", "PageStep", "TreeStep", "new_cache", "page_tables", "release_pages", "cache_append",
           "paged_attention"]

PAGE_SIZES = (16, 32, 64, 128)

class PageStep(NamedTuple):
    """What ``page_tables`` returns; all int32 on the GPU."""

    slots: torch.Tensor       # [max_tokens] page * page_size + offset; -1: no place
    positions: torch.Tensor   # [max_tokens] position in the request
    cu_q: torch.Tensor        # [B + 1] offsets of the requests' tokens
    seq_lens: torch.Tensor    # [B] lengths after the step
    free_state: torch.Tensor  # [2] the ring of free pages after the step


class TreeStep(NamedTuple):
    """What ``tree_tables`` (``draft.py``) returns, for each token of the trees of drafted tokens."""

    positions: torch.Tensor  # [T] int32: the tokens before the tree, and the node's depth
    ancestors: torch.Tensor  # [T] int64: bit i: node i is an ancestor, or the node itself


def _status(t) -> int:
    """Address of the status word of a tensor's device (0 where it is on none)."""
    return _status_word(t.device).data_ptr() if isinstance(t, torch.Tensor) and t.is_cuda else 0


def new_cache(num_pages: int, heads_kv: int, head_dim: int, *, page_size: int = 64,
              dtype: torch.dtype = torch.float8_e4m3fn,
              device: Union[str, torch.device] = "cuda") -> Tuple[torch.Tensor, ...]:
    """Zero-filled ``k_cache, v_cache, k_scale, v_scale``."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} unsupported {PAGE_SIZES}")
    if dtype not in (torch.float8_e4m3fn, torch.int8):
        raise ValueError(f"cache dtype {dtype} unsupported")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim {head_dim} unsupported (64 or 128)")
    shape = (num_pages, heads_kv, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return k, v, ks, vs


def page_tables(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                free_pages: torch.Tensor, free_state: torch.Tensor, *, page_size: int,
                max_tokens: int) -> PageStep:
    """The tables of a step that adds ``new_lens[b]`` tokens to request ``b``.

    ``seq_lens``, ``new_lens`` ``[B]``; ``block_table`` ``[B, W]``, whose new
    entries are written; ``free_pages`` a ring of pages whose free part starts
    at ``free_state[0]`` and has ``free_state[1]`` entries; all int32 on the
    GPU. ``max_tokens``: the length of ``slots`` and ``positions``, at least
    the sum of ``new_lens`` (entries past it are -1 and 0).

    Request ``b`` takes ``ceil((len + new) / page_size) - ceil(len /
    page_size)`` pages from the ring's head, in request order. One that would
    not fit its row, or finds too few pages, is not served: its slots are -1,
    its length stays, and ``check_device_status`` raises. ``seq_lens`` and
    ``free_state`` are left as they are, so a step may be run again.
    """
    if max_tokens < 0:
        raise ValueError("max_tokens must be >= 0")
    r = N.binding().tables(seq_lens, new_lens, block_table, free_pages, free_state, page_size,
                           max_tokens, _status(seq_lens))
    if type(r) is int:
        N.check(r, "chia_page_tables")
    return PageStep(*r)


def release_pages(done: Optional[torch.Tensor], seq_lens: torch.Tensor, block_table: torch.Tensor,
                  free_pages: torch.Tensor, free_state: torch.Tensor, *, page_size: int,
                  keep_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Give the pages of the requests with ``done[b] != 0`` (int32) back: they
    are written to the ring's tail. Returns the new ``seq_lens`` (0 for those
    requests) and ``free_state``.

    ``keep_lens`` (int32, with ``done=None``): each request keeps its first
    ``keep_lens[b]`` tokens, and the pages past them are given back. This is how
    rejected tokens are taken out: a length that is lowered by hand leaves their
    pages in no request and not in the ring.
    """
    if (done is None) == (keep_lens is None):
        raise ValueError("release_pages takes either done or keep_lens")
    what, mode = (done, -1) if keep_lens is None else (keep_lens, -2)
    r = N.binding().tables(seq_lens, what, block_table, free_pages, free_state, page_size, mode,
                           _status(seq_lens))
    if type(r) is int:
        N.check(r, "chia_release_pages" if mode == -1 else "chia_trim_pages")
    return r


def cache_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
                 v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Write the tokens ``k, v`` ``[T, H_kv, D]`` (bf16 or fp16) to ``slots``
    ``[T]`` (int32; -1: skipped) of the cache, in place.

    The tokens of one page are adjacent rows, as ``page_tables`` lays them out;
    skipped ones may lie between them.
    Scales are powers of two, the smallest that hold the page's largest finite
    value. Tokens that hold a page's first slot begin the page anew; others
    keep its scale or, where they need a larger one, have the values that the
    page holds expressed in theirs.
    """
    r = N.binding().append(k, v, slots, k_cache, v_cache, k_scale, v_scale, _status(k_cache))
    if r is not None:
        N.check(r, f"chia_cache_append(k={tuple(k.shape)}, cache={tuple(k_cache.shape)})")


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, *,
                    max_q: Optional[int] = None, norm: str = "softmax", mod: str = "none",
                    mask: Mask = CAUSAL, scale: Optional[float] = None, softcap: float = 30.0,
                    head_param: Optional[Union[torch.Tensor, Sequence[float]]] = None,
                    sig_bias: float = 0.0, out_scale: float = 1.0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    wait_limit_ns: int = 0, tree: Optional[TreeStep] = None):
    """``attention`` of a step's queries over the paged cache.

    ``q`` ``[T, H, D]`` (bf16 or fp16), request ``b``'s queries in rows
    ``[cu_q[b], cu_q[b + 1])`` (``None``: ``T / B`` each); its keys are the
    first ``seq_lens[b]`` tokens of the pages in ``block_table[b]``, its
    queries their last ones: query ``i`` of ``n`` has position ``seq_lens[b] -
    n + i``, and ``mask`` applies to positions. ``norm``, ``mod``, ``mask``,
    ``scale``, ``softcap``, ``head_param``, ``sig_bias``, ``out_scale``,
    ``wait_limit_ns`` as in ``attention``; ``H % H_kv == 0``. ``max_q``: the
    most queries of any request, as far as the host knows (``None``: ``T -
    B + 1``, or ``T / B`` without ``cu_q``); it chooses the schedule, never the result.
    Keys whose page is out of range are left out and reported, and so are requests
    from an offset on that falls. A row that sees no key is zero. ``return_lse``: also the natural log-sum-exp,
    fp32 ``[T, H]`` (softmax only). Forward only.

    ``tree`` (what ``tree_tables`` returns): a request's queries are a tree of
    drafted tokens. Each sees the keys before the tree that ``mask`` shows to its
    position, and of the tree's itself and its ancestors, as far as the mask does not
    put them too far back. Requests of more than 64 queries are chunks, as without.
    """
    if norm not in _NORMS or mod not in _MODS:
        raise ValueError(f"unknown norm/mod {norm!r}/{mod!r}")
    if norm != "softmax":
        if return_lse:
            raise ValueError("return_lse needs norm='softmax'")
        if mod != "none":
            raise ValueError(f"mod {mod!r} needs norm='softmax'")
    if wait_limit_ns < 0:
        raise ValueError("wait_limit_ns must be >= 0")
    mask.validate()
    hp = None
    if mod == "alibi" or mod == "temp":
        hp = head_param
        if hp is None:
            hp = _cached_default(mod, q.shape[1], q.device)
        elif not isinstance(hp, torch.Tensor):
            hp = _param_tensor(hp, q.shape[1], q.device)
    r = N.binding().attention(
        q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_q, max_q, _NORMS[norm],
        _MODS[mod], (mask.left, mask.right, mask.block, mask.prefix, mask.dilation), scale, softcap,
        hp, sig_bias, out_scale, out, return_lse, wait_limit_ns, _status(k_cache), tree)
    if type(r) is int:  # the message is formatted only on failure
        N.check(r, f"chia_{'paged' if tree is None else 'tree'}_attn(norm={norm}, mod={mod}, mask={mask}, q={tuple(q.shape)}, "
                   f"cache={tuple(k_cache.shape)})")
    return r
