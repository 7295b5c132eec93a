"""Norm of queries and keys, head by head, with the rotation to their positions in the same pass
(``include/chia_rope.h``); forward and backward.

It stands between the projections and ``attention`` (``[B, H, S, D]``) or ``cache_append`` and ``paged_attention``
(``[T, H, D]``). All computation happens in ``libchia_attn.so`` on the current CUDA stream; there is no CPU or PyTorch
fallback.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _native as N

__all__ = ["rope_frequencies", "qk_norm_rope", "qk_norm_rope_backward"]


def rope_frequencies(rot_dim: int, *, base: float = 10000.0, inv_freq: Optional[Sequence[float]] = None,
                     device: Union[str, torch.device] = "cuda") -> torch.Tensor:
    """The frequencies of ``qk_norm_rope`` for ``rot_dim`` channels (a multiple of 8): pair ``i`` turns by ``base ** (-2 i
    / rot_dim)`` radians a position, or by ``inv_freq[i]`` (scaled frequencies of long contexts).

    int64 ``[rot_dim / 2]``: turns a position, in units of ``2**-64``. Whole numbers, so that the angle of a far position
    loses nothing to the reduction by whole turns.
    """
    if rot_dim < 0 or rot_dim % 8 != 0:
        raise ValueError("rot_dim must be a multiple of 8")
    if inv_freq is None:
        if not base > 0:
            raise ValueError("base must be positive")
        inv_freq = [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
    elif isinstance(inv_freq, torch.Tensor):
        inv_freq = inv_freq.detach().double().cpu().tolist()
    if len(inv_freq) != rot_dim // 2:
        raise ValueError(f"inv_freq must have {rot_dim // 2} entries, got {len(inv_freq)}")
    if not all(math.isfinite(f) for f in inv_freq):
        raise ValueError("inv_freq must be finite")
    turns = [round(math.fmod(f / (2.0 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64 for f in inv_freq]
    return torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=device)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 freqs: torch.Tensor, positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 interleaved: bool = False, weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each row ``x`` of ``q`` and ``k`` over its channels as ``x / sqrt(mean(x^2) + eps) * (weight + weight_offset)``,
    its first ``2 * len(freqs)`` channels then turned to its position.

    ``q`` ``[T, H, D]``, ``k`` ``[T, H_kv, D]`` with ``positions`` ``[T]``, or ``[B, H, S, D]``, ``[B, H_kv, S, D]`` with
    ``[S]`` or ``[B, S]`` (int32; ``None``: 0, 1, ...); bf16, fp16 or fp32, ``D`` 64 or 128. Views of a fused projection
    are taken as they are (strides that are multiples of 8 elements, unit last stride); outputs have their order of
    dimensions. ``q_weight``, ``k_weight`` ``[D]`` (bf16, fp16 or fp32; ``None``: ones, without the offset; the rows are
    normed all the same). Pair ``i`` is
    channels ``i`` and ``i + rot / 2``, or neighbours with ``interleaved``. ``freqs``: ``rope_frequencies``; an empty one
    turns nothing. Computed in 32 bits and rounded once. Differentiable in ``q``, ``k`` and the weights, once
    (a second derivative is an error); only the inputs are kept for the backward pass.
    """
    r = N.binding().qk_norm_rope(q, k, q_weight, k_weight, freqs, positions, eps, interleaved, weight_offset)
    if type(r) is int:
        N.check(r, f"chia_qk_norm_rope(q={tuple(q.shape)}, k={tuple(k.shape)})")
    return r


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], freqs: torch.Tensor,
                          positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6, interleaved: bool = False,
                          weight_offset: float = 0.0, weight_grads: Tuple[bool, bool] = (True, True)):
    """Gradients ``(dq, dk, dq_weight, dk_weight)`` of ``qk_norm_rope`` from those of its outputs and from its inputs.
    ``weight_grads``: which of the weights' are wanted (``None`` in the place of one that is not, or that has no weight);
    they are summed in 32 bits in an order that is the same in every call."""
    r = N.binding().qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, freqs, positions, eps, interleaved,
                                     weight_offset, *weight_grads)
    if type(r) is int:
        N.check(r, f"chia_qk_norm_rope_bwd(q={tuple(q.shape)}, k={tuple(k.shape)})")
    return r
