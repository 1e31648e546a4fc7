"""Softmax attention beside layers.sliding_window_attention: over packed documents, with prefixes, capped scores, a distance bias and
grouped heads, for whole sequences (differentiable) and for single tokens against a cache.  No counterpart in the reference, whose causal
layer asks for a plain causal window (causal_lact_with_sliding_window_attn.py:371-375).  bf16 and fp32, heads of 64 and 128; the arithmetic
runs in csrc/masked_attention.h and csrc/attention_step.h, and there is no other path: what the kernels do not take raises."""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad as fwad

from . import _lib

_SMALLEST, _LARGEST = 2.0 ** -149, (2.0 - 2.0 ** -23) * 2.0 ** 127      # of fp32


_PLAIN = {torch.Tensor, nn.Parameter}


def _plain_only(name: str, *ts: Optional[torch.Tensor]) -> None:
    """The kernels read memory: what needs to see tensor operations (function transforms, tracing, forward mode, subclasses) is refused."""
    ts = [t for t in ts if t is not None]
    types = set(map(type, ts))
    if not types <= _PLAIN and not all(isinstance(t, torch.Tensor) for t in ts):
        raise TypeError(f"{name} takes tensors")
    if not types <= _PLAIN or torch._C._are_functorch_transforms_active() or torch._C._is_tracing() or any(map(torch._C._functorch.is_legacy_batchedtensor, ts)):
        raise NotImplementedError(f"{name} takes plain tensors: no function transforms, tracing, tensor subclasses or batches of gradients")
    if fwad._current_level >= 0 and any(fwad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError(f"{name} has no forward-mode derivative (jvp)")


def _autocast(*ts: torch.Tensor):
    """What autocast makes of the operands."""
    if not (ts[0].is_cuda and torch.is_autocast_enabled("cuda")):
        return ts
    dtype = torch.get_autocast_dtype("cuda")
    return tuple(t.to(dtype) if t.is_floating_point() else t for t in ts)


def _dims(name: str, n: int, **ts: Optional[torch.Tensor]) -> None:
    for what, t in ts.items():
        if t is not None and t.dim() != n:
            raise ValueError(f"{name}: {what} must have {n} dimensions, got {tuple(t.shape)}")


def _options(name, d, window, score_cap, scale, slopes):
    if window is not None and (int(window) != window or window < 1):
        raise ValueError(f"{name}: window must be a positive number of tokens or None, got {window}")
    # (the kernels take both in fp32, where a smaller one would be 0, and a cap of 0 none)
    if score_cap is not None and not (_SMALLEST <= float(score_cap) <= _LARGEST):
        raise ValueError(f"{name}: score_cap must be positive and a number of fp32, or None, got {score_cap}")
    if scale is not None and not (_SMALLEST <= float(scale) <= _LARGEST):
        raise ValueError(f"{name}: scale must be positive and a number of fp32, or None, got {scale}")
    if slopes is not None and torch.is_grad_enabled() and slopes.requires_grad:
        raise RuntimeError(f"{name}: distance_slopes have no gradient; detach them")
    return (1 << 30 if window is None else int(window), 1.0 / math.sqrt(d) if scale is None else float(scale),
            0.0 if score_cap is None else float(score_cap))


@torch.compiler.disable
def masked_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, *, score_cap: Optional[float] = None,
                            distance_slopes: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None,
                            prefixes: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """q: [b, l, hq, d], k, v: [b, l, hkv, d] (bf16 or fp32, d = 64 or 128, hkv a divisor of hq: query heads h * hq / hkv ... share key head
    h) -> [b, l, hq, d], the softmax over the keys j that query i sees of

        s_ij = f(scale q_i . k_j) - distance_slopes[h] |i - j|,    f(x) = score_cap tanh(x / score_cap), or x

    times v.  Query i sees key j of its own document when j > i - window and (j <= i or j is in the document's prefix).

    window: tokens that a query looks back on, its own included; None: all.   score_cap, scale: positive numbers of fp32; scale 1 / sqrt(d) if None.
    distance_slopes: [hq], without a gradient.
    documents: [b, n + 1] int32 (int64 is converted): document i of a sequence is its tokens [documents[:, i], documents[:, i + 1]).  The bounds do not
    fall; equal ones are empty documents.  Tokens in front of the first and behind the last bound are in none: their output and their
    gradients are 0, and nothing of them reaches another token, whatever they hold.  The bounds are not checked (they stay on the device);
    what lies outside the sequence is cut off.  None: the whole sequence is one document.
    prefixes: [b, n] ([b, 1] without documents): how many of a document's first tokens all of its tokens see, in both directions; a prefix as
    long as the document makes its attention bidirectional.  (A plain causal window of bf16 and equal heads is sliding_window_attention's as well, whose kernels are up to a
    tenth faster there.)
    What is not finite makes NaN of the heads of all tokens that see it, in every element (a key whose score is -infinity, or infinite under a cap, only of gradients).

    Differentiable in q, k and v, once.  Scores are numbers of fp32.  The gradients use a row's log2 of its sum of 2^scores in fp32: they have lost 2^-24 of its size, and all digits
    at scores past 2^20.  Under autocast the operands are cast to its type.  While a stream is captured, leaves that a graph made on the default stream still
    holds are refused."""
    name = "masked_window_attention"
    _plain_only(name, q, k, v, distance_slopes, documents, prefixes)
    _dims(name, 4, q=q, k=k, v=v)
    _dims(name, 2, documents=documents, prefixes=prefixes)
    q, k, v = _autocast(q, k, v)
    window, scale, cap = _options(name, q.shape[3], window, score_cap, scale, distance_slopes)
    if documents is not None and documents.shape[1] < 2:
        raise ValueError(f"{name}: documents must hold at least two bounds, got {tuple(documents.shape)}")
    if q.is_cuda and 0 in q.shape[:2] and q.shape[:2] == k.shape[:2] == v.shape[:2]:
        return q + (k.sum() + v.sum())      # nothing to attend to; empty sums keep every operand in the graph
    return _lib.host().masked_attention(q, k, v, window, scale, cap, distance_slopes, documents, prefixes)


@torch.compiler.disable
def window_attention_step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, window: Optional[int] = None, *,
                          score_cap: Optional[float] = None, distance_slopes: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """masked_window_attention for the newest token of every sequence: q [b, hq, d], k_cache, v_cache [b, n, hkv, d] -> [b, hq, d].

    lengths: [b] int32 (int64 is converted), on the device: the first lengths[i] entries of sequence i's cache are its tokens, the last of them
    the one that q belongs to (its key and value are in the cache already).  0 (a sequence that takes no part): output 0.  Entries past the length
    are not read.  Lengths outside 0 .. n are cut to it.  The caches may have any strides between sequences, tokens and heads ([b, hkv, n, d]
    transposed, a part of a longer cache) with d contiguous and rows on 16-byte boundaries.  For inference: under torch.no_grad(), or with operands
    that need no gradient."""
    name = "window_attention_step"
    _plain_only(name, q, k_cache, v_cache, lengths, distance_slopes)
    _dims(name, 3, q=q)
    _dims(name, 4, k_cache=k_cache, v_cache=v_cache)
    q, = _autocast(q)
    window, scale, cap = _options(name, q.shape[2], window, score_cap, scale, distance_slopes)
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError(f"{name} is for inference: call it under torch.no_grad()")
    return _lib.host().attention_step(q, k_cache, v_cache, lengths, window, scale, cap, distance_slopes)
