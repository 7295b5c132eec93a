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

import ctypes
import math
from typing import Dict, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from .ops import (CAUSAL, Mask, _MODS, _NORMS, _cached_default, _param_tensor, _prep,
                  _status_word)

__all__ = ["PAGE_SIZES", "PageStep", "new_cache", "page_tables", "release_pages", "cache_append",
           "paged_attention"]

PAGE_SIZES = (16, 32, 64, 128)
_CACHE_TYPES = {torch.float8_e4m3fn: N.CACHE_E4M3, torch.int8: N.CACHE_INT8}
_TYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}

_pack_tables = N.packer(N.TablesParams)
_pack_append = N.packer(N.AppendParams)
_pack_paged = N.packer(N.PagedParams)
_workspaces: Dict[tuple, torch.Tensor] = {}
_workspace_bytes: Dict[int, int] = {}
_functions: Dict[str, object] = {}
_stream = torch._C._cuda_getCurrentRawStream  # of a device index; current_stream() builds an object


class PageStep(NamedTuple):
    """What ``page_tables`` returns; all int32 on the GPU."""

    slots: torch.Tensor       # [max_tokens] page * page_size + offset; -1: no place
    positions: torch.Tensor   # [max_tokens] position in the request
    cu_q: torch.Tensor        # [B + 1] offsets of the requests' tokens
    seq_lens: torch.Tensor    # [B] lengths after the step
    free_state: torch.Tensor  # [2] the ring of free pages after the step


def _on_gpu(name: str, t, dim: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != dim:
        raise ValueError(f"{name} must be a {dim}-D tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: the library runs on CUDA only "
                           "(no CPU fallback)")


def _int32(name: str, t, shape: tuple, dev: torch.device) -> None:
    _on_gpu(name, t, len(shape))
    if t.dtype is not torch.int32 or t.shape != shape or t.device != dev:
        raise ValueError(f"{name} must be int32 {shape} on {dev}, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have unit stride")


def _call(name: str, dev: torch.device, packed: bytes, stream: int, what) -> None:
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(N.load(), name)
    if torch.cuda.current_device() == dev.index:
        code = fn(packed, stream)
    else:
        with torch.cuda.device(dev):
            code = fn(packed, stream)
    if code:  # the message is formatted only on failure
        N.check(code, f"{name}({', '.join(str(tuple(t.shape)) for t in what)})")


def _page_size(page: int) -> int:
    if page not in PAGE_SIZES:
        raise ValueError(f"page_size {page} unsupported {PAGE_SIZES}")
    return page


def new_cache(num_pages: int, heads_kv: int, head_dim: int, *, page_size: int = 64,
              dtype: torch.dtype = torch.float8_e4m3fn,
              device: Union[str, torch.device] = "cuda") -> Tuple[torch.Tensor, ...]:
    """Zero-filled ``k_cache, v_cache, k_scale, v_scale``."""
    _page_size(page_size)
    if dtype not in _CACHE_TYPES:
        raise ValueError(f"cache dtype {dtype} unsupported")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim {head_dim} unsupported (64 or 128)")
    shape = (num_pages, heads_kv, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return k, v, ks, vs


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    _on_gpu("k_cache", k_cache, 4)
    _on_gpu("v_cache", v_cache, 4)
    ct = _CACHE_TYPES.get(k_cache.dtype)
    shape, dev = k_cache.shape, k_cache.device
    if ct is None or v_cache.dtype is not k_cache.dtype:
        raise ValueError(f"k_cache, v_cache must share a type, float8_e4m3fn or int8; got "
                         f"{k_cache.dtype}, {v_cache.dtype}")
    if v_cache.shape != shape or v_cache.device != dev:
        raise ValueError("k_cache, v_cache must match in shape and device")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache, v_cache must be contiguous")
    _page_size(shape[2])
    if shape[3] not in (64, 128):
        raise ValueError(f"head_dim {shape[3]} unsupported (64 or 128)")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        _on_gpu(name, s, 2)
        if s.dtype is not torch.float32 or s.shape != shape[:2] or s.device != dev or \
                not s.is_contiguous():
            raise ValueError(f"{name} must be contiguous fp32 {tuple(shape[:2])} on {dev}")
    return ct, shape, dev


def _tables_call(name, seq_lens, lens, block_table, free_pages, free_state, page_size, max_tokens,
                 outs):
    _page_size(page_size)
    _on_gpu("seq_lens", seq_lens, 1)
    dev, B = seq_lens.device, seq_lens.shape[0]
    _on_gpu("block_table", block_table, 2)
    _on_gpu("free_pages", free_pages, 1)
    if B < 1 or block_table.shape[1] < 1 or free_pages.shape[0] < 1:
        raise ValueError("empty seq_lens, block_table or free_pages")
    _int32("seq_lens", seq_lens, (B,), dev)
    _int32("new_lens" if outs else "done", lens, (B,), dev)
    _int32("block_table", block_table, (B, block_table.shape[1]), dev)
    _int32("free_pages", free_pages, (free_pages.shape[0],), dev)
    _int32("free_state", free_state, (2,), dev)
    if B > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("the rows of block_table must not overlap")
    # one allocation for all outputs
    T = max_tokens if outs else 0
    buf = torch.empty(2 * T + 2 * B + 3, dtype=torch.int32, device=dev)
    base = buf.data_ptr()
    o = (base, base + 4 * T, base + 8 * T, base + 8 * T + 4 * (B + 1),
         base + 8 * T + 4 * (2 * B + 1))
    stream = _stream(dev.index)
    packed = _pack_tables(
        N.PAGED_ABI_VERSION, page_size, B, block_table.shape[1],
        max(block_table.stride(0), block_table.shape[1]), free_pages.shape[0], T,
        seq_lens.data_ptr(), lens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(),
        free_state.data_ptr(), *o, _status_word(dev).data_ptr())
    _call(name, dev, packed, stream, (seq_lens, block_table, free_pages))
    return torch.split(buf, [T, T, B + 1, B, 2])


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
    return PageStep(*_tables_call("chia_page_tables", seq_lens, new_lens, block_table, free_pages,
                                  free_state, page_size, max_tokens, True))


def release_pages(done: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
                  free_pages: torch.Tensor, free_state: torch.Tensor, *,
                  page_size: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Give the pages of the requests with ``done[b] != 0`` (int32) back: they
    are written to the ring's tail. Returns the new ``seq_lens`` (0 for those
    requests) and ``free_state``."""
    return _tables_call("chia_release_pages", seq_lens, done, block_table, free_pages, free_state,
                        page_size, 0, False)[3:]


def cache_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
                 v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Write the tokens ``k, v`` ``[T, H_kv, D]`` (bf16 or fp16) to ``slots``
    ``[T]`` (int32; -1: skipped) of the cache, in place.

    The tokens of one page are adjacent rows, as ``page_tables`` lays them out.
    Scales are powers of two, the smallest that hold the page's largest finite
    value. Tokens that hold a page's first slot begin the page anew; others
    keep its scale or, where they need a larger one, have the values that the
    page holds expressed in theirs.
    """
    ct, shape, dev = _check_cache(k_cache, v_cache, k_scale, v_scale)
    _on_gpu("k", k, 3)
    _on_gpu("v", v, 3)
    T = k.shape[0]
    want = (T, shape[1], shape[3])
    dt = _TYPES.get(k.dtype)
    if dt is None or v.dtype is not k.dtype:
        raise ValueError(f"k, v must share a type, bf16 or fp16; got {k.dtype}, {v.dtype}")
    if k.shape != want or v.shape != want or k.device != dev or v.device != dev:
        raise ValueError(f"k, v must be {want} on {dev}, got {tuple(k.shape)}, {tuple(v.shape)}")
    _int32("slots", slots, (T,), dev)
    if T == 0:
        return
    k, v = _prep(k.detach()), _prep(v.detach())
    packed = _pack_append(
        N.PAGED_ABI_VERSION, dt, ct, shape[3], shape[1], shape[2], T, shape[0], k.data_ptr(),
        v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
        _status_word(dev).data_ptr())
    _call("chia_cache_append", dev, packed, _stream(dev.index), (k, k_cache))


def _workspace(dev: torch.device, stream: int) -> torch.Tensor:
    """Workspace of ``paged_attention`` for one (device, stream): as large as
    any call needs. A call that a CUDA graph captures gets one of its own,
    zero-filled within the graph: the graph may be replayed beside calls on the
    stream that captured it."""
    key = (dev.index, stream)
    t = _workspaces.get(key)
    capturing = torch.cuda.is_current_stream_capturing()
    if t is None or capturing:
        n = _workspace_bytes.get(dev.index)
        if n is None:
            with torch.cuda.device(dev):  # head_dim 128, few and many rows a K/V head
                n = max(N.load().chia_paged_attn_workspace_bytes(_pack_paged(
                    N.PAGED_ABI_VERSION, 0, 0, 128, 0, 0, 1, 1, 16, q, 1, 1, 1, 1, 1, *([256] * 2),
                    *([0] * 4), *([256] * 6), 0, 0, 0, 1.0, 1.0, 0.0, 1.0, -1, -1, 0, 0, 1, 0, 0, 0,
                    0)) for q in (16, 1024))
            _workspace_bytes[dev.index] = n
        t = torch.zeros(n, dtype=torch.uint8, device=dev)
        if not capturing:
            _workspaces[key] = t
    return t


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, cu_q: Optional[torch.Tensor] = None, *,
                    max_q: Optional[int] = None, norm: str = "softmax", mod: str = "none",
                    mask: Mask = CAUSAL, scale: Optional[float] = None, softcap: float = 30.0,
                    head_param: Optional[Union[torch.Tensor, Sequence[float]]] = None,
                    sig_bias: float = 0.0, out_scale: float = 1.0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    wait_limit_ns: int = 0):
    """``attention`` of a step's queries over the paged cache.

    ``q`` ``[T, H, D]`` (bf16 or fp16), request ``b``'s queries in rows
    ``[cu_q[b], cu_q[b + 1])`` (``None``: ``T / B`` each); its keys are the
    first ``seq_lens[b]`` tokens of the pages in ``block_table[b]``, its
    queries their last ones: query ``i`` of ``n`` has position ``seq_lens[b] -
    n + i``, and ``mask`` applies to positions. ``norm``, ``mod``, ``mask``,
    ``scale``, ``softcap``, ``head_param``, ``sig_bias``, ``out_scale``,
    ``wait_limit_ns`` as in ``attention``; ``H % H_kv == 0``. ``max_q``: the
    most queries of any request, as far as the host knows (``None``: ``T -
    B + 1``, or ``T / B`` without ``cu_q``); it chooses the schedule, never the result. A
    row that sees no key is zero. ``return_lse``: also the natural log-sum-exp,
    fp32 ``[T, H]`` (softmax only). Forward only.
    """
    ct, shape, dev = _check_cache(k_cache, v_cache, k_scale, v_scale)
    _on_gpu("q", q, 3)
    T, H, D = q.shape
    dt = _TYPES.get(q.dtype)
    if dt is None:
        raise ValueError(f"dtype {q.dtype} unsupported (bf16 or fp16)")
    if D != shape[3] or H < 1 or H % shape[1] or q.device != dev:
        raise ValueError(f"q {tuple(q.shape)} on {q.device} does not fit a cache "
                         f"{tuple(shape)} on {dev}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise ValueError("paged_attention has no backward pass")
    if norm not in _NORMS or mod not in _MODS:
        raise ValueError(f"unknown norm/mod {norm!r}/{mod!r}")
    if return_lse and norm != "softmax":
        raise ValueError("return_lse needs norm='softmax'")
    if norm != "softmax" and mod != "none":
        raise ValueError(f"mod {mod!r} needs norm='softmax'")
    if wait_limit_ns < 0:
        raise ValueError("wait_limit_ns must be >= 0")
    mask.validate()
    _on_gpu("block_table", block_table, 2)
    B, W = block_table.shape
    if B < 1 or W < 1:
        raise ValueError("empty block_table")
    _int32("block_table", block_table, (B, W), dev)
    _int32("seq_lens", seq_lens, (B,), dev)
    if B > 1 and block_table.stride(0) < W:
        raise ValueError("the rows of block_table must not overlap")
    if cu_q is not None:
        _int32("cu_q", cu_q, (B + 1,), dev)
    elif T % B:
        raise ValueError(f"{T} queries for {B} requests need cu_q")
    if max_q is None:
        max_q = max(1, T // B if cu_q is None else T - B + 1)
    elif max_q < 1:
        raise ValueError("max_q must be >= 1")
    q = _prep(q)
    if out is None:
        o = q.new_empty(q.shape)
    else:
        o = out
        if o.shape != q.shape or o.dtype is not q.dtype or o.device != dev:
            raise ValueError("out must match q in shape, dtype and device")
        if o.stride(-1) != 1 or any(s % 8 for s in o.stride()[:-1]) or o.data_ptr() % 16:
            raise ValueError("out must have unit last stride and 16-byte aligned rows")
    hp = None
    if mod in ("alibi", "temp"):
        hp = (_cached_default(mod, H, dev) if head_param is None
              else _param_tensor(head_param, H, dev))
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    if T:
        stream = _stream(dev.index)
        ws = _workspace(dev, stream)
        packed = _pack_paged(
            N.PAGED_ABI_VERSION, dt, ct, D, _NORMS[norm], _MODS[mod], H, shape[1], shape[2],
            min(max_q, T), B, T, shape[0], W, max(block_table.stride(0), W), q.data_ptr(),
            o.data_ptr(), *q.stride()[:2], *o.stride()[:2], k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            0 if cu_q is None else cu_q.data_ptr(), 0 if lse is None else lse.data_ptr(),
            0 if hp is None else hp.data_ptr(), 1.0 / math.sqrt(D) if scale is None else scale,
            softcap, sig_bias, out_scale, mask.left, mask.right, mask.block, mask.prefix,
            mask.dilation, _status_word(dev).data_ptr(), ws.data_ptr(), ws.numel(), wait_limit_ns)
        _call("chia_paged_attn", dev, packed, stream, (q, k_cache, block_table))
    return (o, lse) if return_lse else o
