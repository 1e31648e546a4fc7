"""Linear attention whose state decays: the linear counterpart of the fast weights (ttt_operation.py), as a memory beside the attention of
attention.py or as a baseline for the operation.  No counterpart in the reference.  bf16 and fp32, key and value sizes of 64 and 128; the arithmetic runs in
csrc/linear_attention.h, and there is no other path: what the kernels do not take raises."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .attention import _autocast, _dims, _plain_only


def _scale(name, scale, d):
    if scale is None:
        return 1.0 / math.sqrt(d)
    if not math.isfinite(scale):
        raise ValueError(f"{name}: scale must be finite, got {scale}")
    return float(scale)


@torch.compiler.disable
def decayed_linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, state: Optional[torch.Tensor] = None,
                             scale: Optional[float] = None, return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q, k: [b, l, h, dk], v: [b, l, h, dv] (bf16 or fp32, dk, dv = 64 or 128) -> [b, l, h, dv]:

        S_t = exp(log_decay_t) S_(t-1) + k_t v_t^T,    out_t = scale S_t^T q_t

    log_decay: [h], a constant per head, or [b, l, h], one per token; at most 0 in use.  -infinity forgets the state (the first token of
    a document); anything below -200 counts as that.
    state: [b, h, dk, dv] fp32, S in front of the first token; None: zero.   return_state: also return S behind the last token, fp32.
    scale: 1 / sqrt(dk) if None.

    Differentiable in q, k, v, log_decay and state, once.  Under autocast q, k and v are cast to its type.  While a stream is captured, leaves that a
    graph made on the default stream still holds are refused."""
    name = "decayed_linear_attention"
    _plain_only(name, q, k, v, log_decay, state)
    _dims(name, 4, q=q, k=k, v=v, state=state)
    if log_decay.dim() not in (1, 3):
        raise ValueError(f"{name}: log_decay must be [h] or [b, l, h], got {tuple(log_decay.shape)}")
    q, k, v = _autocast(q, k, v)
    s = _scale(name, scale, q.shape[3])
    if q.is_cuda and 0 in q.shape[:2] and q.shape[:3] == k.shape[:3] == v.shape[:3]:
        out = v + (q.sum() + k.sum() + log_decay.sum())      # (empty: the sums keep every operand in the graph)
        last = state if state is not None else torch.zeros(q.shape[0], q.shape[2], q.shape[3], v.shape[3], device=q.device)
        return (out, last.float().clone()) if return_state else out
    res = _lib.host().linear_attention(q, k, v, log_decay, state, s, bool(return_state))
    return (res[0], res[1]) if return_state else res[0]


@torch.compiler.disable
def decayed_linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                                  state_out: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decayed_linear_attention for one token of every sequence: q, k [b, h, dk], v [b, h, dv], log_decay [h] or [b, h], state [b, h, dk, dv] ->
    (out [b, h, dv], the new state, fp32).  state_out: where the new state goes; it may be `state` itself (then nothing is
    allocated for it), but must not overlap it otherwise; for autograd it is an operation in place.  For inference: under torch.no_grad(), or with operands
    (and a state_out) that need no gradient."""
    name = "decayed_linear_attention_step"
    _plain_only(name, q, k, v, log_decay, state, state_out)
    _dims(name, 3, q=q, k=k, v=v)
    _dims(name, 4, state=state, state_out=state_out)
    if log_decay.dim() not in (1, 2):
        raise ValueError(f"{name}: log_decay must be [h] or [b, h], got {tuple(log_decay.shape)}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, state, state_out)):
        raise RuntimeError(f"{name} is for inference: call it under torch.no_grad()")
    out, new = _lib.host().linear_attention_step(q, k, v, log_decay, state, state_out, _scale(name, scale, q.shape[2]))
    return out, new
