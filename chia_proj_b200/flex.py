"""A ``flex_attention``-compatible frontend.

The reference benchmarks eight of its ten operators through PyTorch's
``flex_attention`` as ``score_mod`` / ``mask_mod`` callables
(JoshiP-commits/CHIA_proj ``extra_bench.py:85-99``; called as
``flex_attention(q, k, v, score_mod=..., block_mask=create_block_mask(...))``
at ``extra_bench.py:130-137``). This module accepts the same callables with
the same call signatures and runs them on the library's sm_100a kernels:

* ``create_block_mask(mask_mod, B, H, Q_LEN, KV_LEN, device=...)``
  evaluates ``mask_mod`` on the index grid and fits it to the library's mask
  model (``Mask``: window left / right, block, prefix, dilation), checking
  the fit element by element on the evaluated grid;
* ``flex_attention(query, key, value, score_mod=None, block_mask=None,
  scale=None, enable_gqa=False, return_lse=False)`` identifies ``score_mod``
  by evaluating it on probe scores and indices: identity, a per-head
  multiplier (temperature), an additive per-head slope times ``kv - q``
  (ALiBi) or ``cap * tanh(s / cap)`` (softcap).

Callables that fit none of these (a mask that depends on the batch or head,
a score_mod mixing two modifications, ...) raise ``NotExpressible``; like
the reference (``extra_bench.py:96-99``), sigmoid and ReLU attention are not
expressible here, because flex normalises with softmax -- they have their
own operators.

Evaluation happens once per block mask. A score_mod is evaluated once per
(heads, device) and again when a plain value that it depends on has changed;
one that depends on tensors, or on what cannot be listed, is evaluated in each
call, which waits for the GPU. Callables must be written with broadcasting
torch operations, as flex requires.
"""

from __future__ import annotations

import builtins
import collections
import dis
import functools
import math
import types
import weakref
from dataclasses import dataclass
from typing import Callable, Optional, Tuple

import torch

from .ops import Mask, attention

__all__ = ["NotExpressible", "BlockMask", "create_block_mask", "flex_attention",
           "fit_mask", "identify_score_mod"]

# Largest number of (query, key) entries evaluated densely; larger masks are
# evaluated on a sample of rows (all of the first and last rows, and a stride).
DENSE_LIMIT = 1 << 24


class NotExpressible(ValueError):
    """The callable has no exact counterpart in the library's kernels."""


# ---------------------------------------------------------------- masks
def _mask_dense(m: Mask, rows: torch.Tensor, kv_len: int) -> torch.Tensor:
    """The visibility rule of ``Mask`` (``include/chia_attn.h``) on rows x keys."""
    i = rows.view(-1, 1)
    j = torch.arange(kv_len, device=rows.device).view(1, -1)
    band = torch.ones(i.shape[0], kv_len, dtype=torch.bool, device=rows.device)
    if m.left >= 0:
        band &= (i - j) <= m.left
    if m.right >= 0:
        band &= (j - i) <= m.right
    if m.block > 0:
        band &= torch.div(i, m.block, rounding_mode="floor") == \
            torch.div(j, m.block, rounding_mode="floor")
    if m.dilation > 1:
        band &= torch.remainder(i - j, m.dilation) == 0
    return band | (j < m.prefix)


def _sample_rows(q_len: int, kv_len: int) -> torch.Tensor:
    if q_len * kv_len <= DENSE_LIMIT:
        return torch.arange(q_len)
    n = max(64, DENSE_LIMIT // kv_len)
    head = torch.arange(min(q_len, n // 4))
    tail = torch.arange(max(0, q_len - n // 4), q_len)
    mid = torch.linspace(0, q_len - 1, n // 2).round().long()
    return torch.unique(torch.cat([head, tail, mid]))


def fit_mask(vis: torch.Tensor, rows: torch.Tensor, kv_len: int) -> Mask:
    """The simplest ``Mask`` whose visibility equals ``vis`` (rows x keys, for
    the query indices ``rows``) exactly; raises ``NotExpressible``."""
    vis = vis.to(torch.bool).cpu()
    rows = rows.cpu()
    n_rows = vis.shape[0]
    # an always-visible prefix: the leading keys every row sees
    full_cols = vis.all(0)
    p_max = int(full_cols.long().cumprod(0).sum().item()) if n_rows else 0
    j = torch.arange(kv_len)
    for prefix in ([0, p_max] if p_max else [0]):
        v2 = vis.clone()
        v2[:, :prefix] = False
        has = v2.any(1)
        if not has.any():
            cand = [Mask(left=-1, right=-1, prefix=prefix)] if prefix else []
        else:
            r = rows[has]
            lo = torch.where(v2[has], j.view(1, -1), kv_len).min(1).values
            hi = torch.where(v2[has], j.view(1, -1), -1).max(1).values
            # dilation: gcd of the gaps between consecutive visible keys of a row
            nz = v2[has].nonzero()
            same_row = nz[1:, 0] == nz[:-1, 0]
            gaps = torch.unique((nz[1:, 1] - nz[:-1, 1])[same_row]).tolist()
            dil = 0
            for gap in gaps:
                dil = math.gcd(dil, int(gap))
            dil = max(dil, 1)
            left_opts = [-1]
            lmax = int((r - lo).max().item())
            if lmax >= 0:
                left_opts.append(lmax)
            right_opts = [-1]
            rmax = int((hi - r).max().item())
            if rmax >= 0:
                right_opts.append(rmax)
            block_opts = [0]
            starts = (lo == r) & (r > 0)
            if starts.any():
                bsz = int(r[starts].min().item())
                if bsz > 0:
                    block_opts.append(bsz)
            cand = [Mask(left=lft, right=rgt, block=blk, prefix=prefix, dilation=dil)
                    for blk in block_opts for lft in left_opts for rgt in right_opts]
        for m in cand:
            try:
                m.validate()
            except ValueError:
                continue
            if torch.equal(_mask_dense(m, rows, kv_len), vis):
                return m
    raise NotExpressible("mask_mod matches no window / block / prefix / dilation mask "
                         "of the library")


@dataclass
class BlockMask:
    """Result of ``create_block_mask``: the fitted mask and the shape it was
    made for (the counterpart of flex's ``BlockMask``)."""

    mask: Mask
    q_len: int
    kv_len: int
    BLOCK_SIZE: Tuple[int, int] = (128, 128)

    @property
    def shape(self):
        return (self.q_len, self.kv_len)


def create_block_mask(mask_mod: Callable, B: Optional[int], H: Optional[int], Q_LEN: int,
                      KV_LEN: int, device="cuda", BLOCK_SIZE=128, _compile=False) -> BlockMask:
    """Same signature as ``torch.nn.attention.flex_attention.create_block_mask``.

    ``mask_mod(b, h, q_idx, kv_idx) -> bool tensor`` is evaluated on the index
    grid (on ``device``, so callables that capture device tensors work) for
    batch and head 0, and for the last batch and head when ``B`` / ``H`` are
    given (a mask that differs between them is not expressible)."""
    rows = _sample_rows(Q_LEN, KV_LEN)
    dev = torch.device(device) if not isinstance(device, torch.device) else device
    if dev.type == "cuda" and not torch.cuda.is_available():
        dev = torch.device("cpu")
    qi = rows.to(dev).view(-1, 1)
    kj = torch.arange(KV_LEN, device=dev).view(1, -1)

    def ev(b, h):
        z = torch.zeros((), dtype=torch.long, device=dev)
        out = mask_mod(z + b, z + h, qi, kj)
        return torch.broadcast_to(torch.as_tensor(out, device=dev), (qi.shape[0], KV_LEN))

    vis = ev(0, 0)
    for b, h in (((B or 1) - 1, 0), (0, (H or 1) - 1)):
        if (b, h) != (0, 0) and not torch.equal(ev(b, h), vis):
            raise NotExpressible("mask_mod depends on the batch or head index")
    bs = (BLOCK_SIZE, BLOCK_SIZE) if isinstance(BLOCK_SIZE, int) else tuple(BLOCK_SIZE)
    return BlockMask(fit_mask(vis, rows, KV_LEN), Q_LEN, KV_LEN, bs)


# ------------------------------------------------------------ score mods
@dataclass(frozen=True)
class ScoreMod:
    """An identified score_mod: ``mod`` of ``attention()`` and its parameters."""

    mod: str                                # none, temp, alibi, softcap
    head_param: Optional[torch.Tensor] = None  # [H] temperatures or slopes
    softcap: float = 30.0


# Probe scores, the last one for the saturation value of a softcap, and (query, key) positions.
_SCORES = (-7.0, -1.5, -0.25, 0.0, 0.5, 2.0, 9.0, 1e6)
_POSITIONS = ((0, 0), (5, 2), (3, 11), (40, 17), (100, 100))


@functools.lru_cache(maxsize=64)
def _probes(H: int, device: str) -> Tuple[torch.Tensor, ...]:
    shape = (len(_SCORES), H, len(_POSITIONS))
    pos = torch.tensor(_POSITIONS)
    hh = torch.arange(H).view(1, -1, 1).expand(shape)
    probes = (torch.tensor(_SCORES).view(-1, 1, 1).expand(shape), torch.zeros_like(hh), hh, pos[:, 0].expand(shape),
              pos[:, 1].expand(shape))
    return tuple(p.contiguous().to(device) for p in probes)  # (copies that are waited for: any stream may use them)


def _evaluate(score_mod: Callable, H: int, device) -> torch.Tensor:
    """``score_mod`` on the probes: fp32 on the host, ``[scores, H, positions]``."""
    probes = [p.clone() for p in _probes(H, str(device))]  # (a callable may write to its arguments)
    with torch.no_grad():
        F = torch.as_tensor(score_mod(*probes), device=device).float()
        return torch.broadcast_to(F, probes[0].shape).cpu()


def _fit_score_mod(values: torch.Tensor) -> ScoreMod:
    """The modification that has these values on the probes; raises ``NotExpressible``."""
    H = values.shape[1]
    X, _, _, qi, kj = _probes(H, "cpu")
    F, Xf, rel = values[:-1], X[:-1], (kj - qi)[:-1].float()
    tol = lambda a, c: bool(torch.allclose(a, c, rtol=1e-4, atol=1e-4))
    if tol(F, Xf):
        return ScoreMod("none")
    # temperature: F = t_h * s, t_h independent of the position
    t = F[_SCORES.index(2.0)] / 2.0  # [H, P]
    th = t[:, 0]
    if tol(F, Xf * th.view(1, -1, 1)) and tol(t, th.view(-1, 1).expand_as(t)):
        return ScoreMod("temp", head_param=th.clone())
    # ALiBi: F = s + slope_h * (kv - q)
    d = F - Xf
    nz = rel[0, 0] != 0
    slope = (d[0][:, nz] / rel[0][:, nz])[:, 0]
    if tol(d, slope.view(1, -1, 1) * rel):
        return ScoreMod("alibi", head_param=slope.clone())
    # softcap: F = c tanh(s / c), c the saturation value
    c = float(values[-1, 0, 0])
    if math.isfinite(c) and c > 0 and tol(F, c * torch.tanh(Xf / c)):
        return ScoreMod("softcap", softcap=c)
    raise NotExpressible("score_mod is not the identity, a per-head temperature, "
                         "an ALiBi slope or a tanh softcap")


def identify_score_mod(score_mod: Optional[Callable], H: int, device) -> ScoreMod:
    """Identify ``score_mod(score, b, h, q_idx, kv_idx)`` by evaluating it."""
    if score_mod is None:
        return ScoreMod("none")
    return _fit_score_mod(_evaluate(score_mod, H, device))


# ---- what a callable's values depend on, as far as that can be listed
class _Unlisted(Exception):
    pass


_PLAIN = frozenset([bool, int, float, complex, str, bytes, type(None), torch.dtype, torch.device])
_BUILTINS = frozenset([abs, bool, divmod, enumerate, float, int, isinstance, len, list, max, min, pow, range, reversed, round,
                       sum, tuple, zip])
# what a class may define beside names of its own: nothing that runs where no name stands
_DUNDERS = frozenset("""__annotate__ __annotate_func__ __annotations__ __annotations_cache__ __call__ __dataclass_fields__
    __dataclass_params__ __delattr__ __dict__ __doc__ __eq__ __firstlineno__ __hash__ __init__ __match_args__ __module__
    __post_init__ __qualname__ __replace__ __repr__ __setattr__ __static_attributes__ __weakref__""".split())
_MOST_LEAVES = 4096  # listing more takes longer than evaluating


@functools.lru_cache(maxsize=1024)
def _global_names(code: types.CodeType) -> Optional[Tuple[str, ...]]:
    """The global names in a function's code and in what is defined within it; None: it may look up others."""
    names, todo = set(), [code]
    while todo:
        c = todo.pop()
        todo += [x for x in c.co_consts if isinstance(x, types.CodeType)]
        for i in dis.get_instructions(c):
            if i.opname == "LOAD_GLOBAL":
                names.add(i.argval)
            elif i.opname.startswith(("IMPORT_", "LOAD_NAME", "LOAD_BUILD_CLASS", "LOAD_FROM_DICT_OR_GLOBALS")):
                return None
    return tuple(sorted(names))


def _is_torch(name) -> bool:
    return isinstance(name, str) and (name == "torch" or name.startswith("torch."))


def _list(x, out: list, seen: set) -> None:
    """Append to ``out`` what ``x`` is made of: pairs of an object (the same one next time) and a value (an equal one).
    Nothing that could refer to a callable is held, so that nothing here keeps one alive."""
    t = type(x)
    if t in _PLAIN:
        out.append((t, repr(x)))
        return
    if id(x) in seen:
        return
    seen.add(id(x))
    if len(out) > _MOST_LEAVES:
        raise _Unlisted
    if t is torch.Tensor or t is torch.nn.Parameter:
        if x.is_inference() or vars(x):
            raise _Unlisted
        out.append((weakref.ref(x), x._version))
    elif t is tuple or t is list:
        out.append((t, len(x)))
        for y in x:
            _list(y, out, seen)
    elif t is set or t is frozenset:
        if not all(type(y) in _PLAIN for y in x):
            raise _Unlisted
        out.append((t, sorted(map(repr, x))))
    elif t is dict or t is collections.OrderedDict:
        out.append((t, len(x)))
        for k, y in x.items():
            if type(k) not in _PLAIN:
                raise _Unlisted
            out.append((t, repr(k)))
            _list(y, out, seen)
    elif t is types.ModuleType:
        if not _is_torch(x.__name__) and x is not math:
            raise _Unlisted
        out.append((x, None))
    elif t is types.FunctionType:
        if _is_torch(x.__module__):
            out.append((x, None))
            return
        out.append((x.__code__, None))
        names = _global_names(x.__code__)
        if names is None:
            raise _Unlisted
        for c in x.__closure__ or ():
            try:
                c = c.cell_contents
            except ValueError:
                raise _Unlisted from None
            _list(c, out, seen)
        for d in (x.__defaults__, x.__kwdefaults__, vars(x)):
            if d:
                _list(d, out, seen)
        for n in names:
            if n not in x.__globals__ and not hasattr(builtins, n):
                raise _Unlisted
            _list(x.__globals__[n] if n in x.__globals__ else getattr(builtins, n), out, seen)
    elif t is types.MethodType:
        _list(x.__func__, out, seen)
        _list(x.__self__, out, seen)
    elif t is functools.partial:
        for y in (x.func, x.args, x.keywords):
            _list(y, out, seen)
    elif t is types.BuiltinFunctionType or t is type:
        if not (x in _BUILTINS or getattr(math, x.__name__, None) is x or getattr(torch, x.__name__, None) is x):
            raise _Unlisted
        out.append((x, None))
    else:
        _list_object(x, t, out, seen)


def _list_object(x, t: type, out: list, seen: set) -> None:
    """An object of a class written in Python: its attributes and its classes' own, methods among them."""
    if type(t) is not type:
        raise _Unlisted
    out.append((type, t.__qualname__))
    for c in t.__mro__[:-1]:
        if c is torch.nn.Module:  # (looks up attributes in the object's own dicts)
            continue
        own = vars(c)
        if not c.__flags__ & 1 << 9 or not all(n in _DUNDERS for n in own if n.startswith("__") and n.endswith("__")):
            raise _Unlisted
        for n, y in own.items():
            if n.startswith("__") and n.endswith("__") and n != "__call__":
                continue
            for z in ((y.fget,) if type(y) is property else (y.__func__,) if type(y) in (staticmethod, classmethod) else (y,)):
                _list(z, out, seen)
    _list(vars(x), out, seen)


def _dependencies(score_mod: Callable) -> Optional[list]:
    out = []
    try:
        _list(score_mod, out, set())
    except (_Unlisted, RecursionError):
        return None
    return out


def _same(a: Optional[list], b: Optional[list]) -> bool:
    return a is not None and b is not None and len(a) == len(b) and all(x[0] is y[0] and x[1] == y[1] for x, y in zip(a, b))


# What a callable was identified as, as long as it lives (its address alone names nothing: another
# callable may have it next), and as long as what it depends on is as it was. A bound method's stands with
# its object, since the method itself is a new object in each call.
_score_cache: "weakref.WeakKeyDictionary" = weakref.WeakKeyDictionary()


@dataclass
class _Kept:
    depends: Optional[list]
    tensors: bool  # are among them
    values: torch.Tensor  # on the probes
    mod: ScoreMod


def _score_of(score_mod: Optional[Callable], H: int, device) -> ScoreMod:
    """Plain values that a callable depends on are compared; where tensors are among them (which may change unseen: through
    ``data``, by a graph's replay), or where not all can be listed, it is evaluated again (a call takes 34
    and 134 us of the host's time, 25 without a score_mod). While a CUDA graph is captured nothing can be read back, so
    tensors are compared by identity and version there, and what cannot be listed counts as unchanged."""
    if score_mod is None:
        return ScoreMod("none")
    method = type(score_mod) is types.MethodType
    key = (getattr(score_mod.__func__, "__code__", None) if method else None, H, str(device))
    try:
        kept = _score_cache.setdefault(score_mod.__self__ if method else score_mod, {})
    except TypeError:  # neither hashed nor referred to weakly
        kept = {}
    depends, old = _dependencies(score_mod), kept.get(key)
    same = old is not None and _same(depends, old.depends)
    if same and not old.tensors:
        return old.mod
    if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
        if same or (old is not None and depends is None and old.depends is None):
            return old.mod
        raise RuntimeError("a score_mod is identified by evaluating it, which a CUDA graph cannot capture: call flex_attention "
                           "with it once before the capture, and after any change of what it depends on")
    values = _evaluate(score_mod, H, device)
    if old is not None and torch.equal(values, old.values):
        mod = old.mod
    else:
        mod = _fit_score_mod(values)
    tensors = depends is not None and any(type(x) is weakref.ref for x, _ in depends)
    kept[key] = _Kept(depends, tensors, values, mod)
    return mod


def flex_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                   score_mod: Optional[Callable] = None, block_mask: Optional[BlockMask] = None,
                   scale: Optional[float] = None, enable_gqa: bool = False,
                   return_lse: bool = False, kernel_options=None):
    """Same call as ``torch.nn.attention.flex_attention.flex_attention``, run
    on the library's kernels. ``block_mask=None`` means every key is visible
    (flex's default). Returns ``out`` or ``(out, lse)`` with the natural
    log-sum-exp when ``return_lse``."""
    B, H, Sq, D = query.shape
    Hkv, Skv = key.shape[1], key.shape[2]
    if Hkv != H and not enable_gqa:
        raise ValueError("query and key head counts differ: pass enable_gqa=True")
    if block_mask is None:
        mask = Mask(left=-1, right=-1)
    else:
        if block_mask.q_len != Sq or block_mask.kv_len != Skv:
            raise ValueError(f"block_mask was made for {block_mask.shape}, "
                             f"inputs are {(Sq, Skv)}")
        mask = block_mask.mask
    sm = _score_of(score_mod, H, query.device)
    kw = {}
    if sm.mod == "softcap":
        kw["softcap"] = sm.softcap
    if sm.mod in ("temp", "alibi"):
        kw["head_param"] = sm.head_param
    return attention(query, key, value, mod=sm.mod, mask=mask, scale=scale,
                     return_lse=return_lse, **kw)
