"""Rotary positions with several axes (time, height and width of a video, two axes of an image, one of a text), in front of the attention of attention.py and of the
cache of paged_cache.py.  No counterpart in the reference's operations, whose models turn queries and keys outside of them.  bf16 and fp32; the arithmetic runs in
csrc/rotary.h, and there is no other path: what the kernels do not take raises."""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .attention import _autocast, _plain_only


@torch.compiler.disable
def axial_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, axes: Sequence[int], *, base: float = 10000.0,
                 frequencies: Optional[Sequence[float]] = None, interleaved: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q: [b, l, hq, d], k: [b, l, hkv, d] or None (bf16 or fp32, d even and at most 256); or [b, hq, d] and [b, hkv, d], one token each -> the same, turned.

    axes: how many channels of a head belong to each axis, even numbers, together at most d; the first axes[0] channels (with halves: pairs) are axis 0's, and so
    on; channels that remain go through as they are.  Pair i of an axis of n channels turns by the angle positions[..., axis] * base ** (-2 i / n):

        (x, y) -> (x cos - y sin, x sin + y cos)

    interleaved: a pair is two neighbouring channels; else the pairs' first channels are the first half of sum(axes) and their second ones the second half.
    positions: [l, axes], the same for every sequence, or [b, l, axes] ([b, axes] for one token each), int32, int64 or fp32, without a gradient.  Angles are formed in fp64.
    frequencies: an angle per unit of position for each of the sum(axes) / 2 pairs, in place of base's.

    Differentiable in q and k, once.  Under autocast they are cast to its type.  While a stream is captured, leaves that a graph made on the default stream still holds are
    refused."""
    name = "axial_rotary"
    _plain_only(name, q, k, positions)
    if q.dim() not in (3, 4) or (k is not None and k.dim() != q.dim()):
        raise ValueError(f"{name}: q and k must both have 4 dimensions, or 3 for one token each")
    given = list(axes)
    axes = [int(n) for n in given]
    if not axes or axes != given or min(axes) <= 0 or any(n % 2 for n in axes) or sum(axes) > q.shape[-1]:
        raise ValueError(f"{name}: axes must be positive even numbers of channels that fit a head of {q.shape[-1]}, got {given}")
    if not (0.0 < base < math.inf):
        raise ValueError(f"{name}: base must be positive and finite, got {base}")
    given, frequencies = frequencies is not None, [] if frequencies is None else [float(f) for f in frequencies]
    if given and (len(frequencies) != sum(axes) // 2 or not all(math.isfinite(f) for f in frequencies)):
        raise ValueError(f"{name}: frequencies must be {sum(axes) // 2} finite numbers, one for each pair")
    if torch.is_grad_enabled() and positions.requires_grad:
        raise RuntimeError(f"{name}: positions have no gradient; detach them")
    q, k = (_autocast(q) + (None,)) if k is None else _autocast(q, k)
    res = _lib.host().axial_rotary(q, k, positions, axes, float(base), frequencies, bool(interleaved))
    return (res[0], None) if k is None else (res[0], res[1])
