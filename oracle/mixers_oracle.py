"""The token mixers (lact_amd.attention, lact_amd.linear_attention) in float64 on the CPU, from their definitions, with bounds of what a
kernel's roundings can add up to.  Test infrastructure only."""
from __future__ import annotations

import math

import torch


def visible(l, window=None, documents=None, prefixes=None):
    """[b or 1, l, l]: whether query i sees key j."""
    i, j = torch.arange(l)[:, None], torch.arange(l)[None, :]
    near = j > i - (l if window is None else window)
    bounds = [[0, l]] if documents is None and prefixes is None else [[0, l]] * len(prefixes) if documents is None else documents.tolist()
    out = torch.zeros(len(bounds), l, l, dtype=torch.bool)
    for b, row in enumerate(bounds):
        for n, (s, e) in enumerate(zip(row, row[1:])):
            p = s + (0 if prefixes is None else int(prefixes[b][n]))
            inside = (i >= s) & (i < e) & (j >= s) & (j < e)
            out[b] |= inside & near & ((j <= i) | (j < p))
    return out


def _bent(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def attention(q, k, v, window=None, score_cap=None, distance_slopes=None, documents=None, prefixes=None, scale=None, grad=None, p_err=0.0, out_err=0.0):
    """(out, dq, dk, dv) of [b, l, h, d] in float64, and elementwise bounds of the errors of a kernel that has a relative error of p_err in its probabilities
    and in the gradients of its scores, and of out_err in what it stores.  grad None: (out, bound)."""
    q, k, v = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    b, hq, l, d = q.shape
    group = hq // k.shape[1]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    scale = d ** -0.5 if scale is None else scale
    raw = q @ k.transpose(2, 3) * scale
    s = _bent(raw, score_cap)
    slope = 1 - (s / score_cap) ** 2 if score_cap else torch.ones_like(s)
    if distance_slopes is not None:
        far = (torch.arange(l)[:, None] - torch.arange(l)[None, :]).abs().double()
        s = s - distance_slopes.double()[:, None, None] * far
    seen = visible(l, window, documents, prefixes)[:, None].expand(b, hq, l, l)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ v
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    heads = lambda t: t.reshape(b, -1, group, l, d).sum(2).transpose(1, 2)  # noqa: E731
    weight = p @ v.abs()
    o_bound = p_err * weight + out_err * out.abs()
    if grad is None:
        return back(out), back(o_bound)
    g = grad.detach().double().transpose(1, 2)
    dp = g @ v.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    ds = torch.where(seen, p * (dp - delta) * slope, torch.zeros_like(p))
    dq, dk, dv = ds @ k * scale, ds.transpose(2, 3) @ q * scale, p.transpose(2, 3) @ g
    # The sum of dout * out is formed from the stored output; its error, and those of the fp32 sums of d products in it and in dp, are in every
    # score's gradient.
    delta_err = (g.abs() * o_bound).sum(-1, keepdim=True)
    sums = d * 2.0 ** -24 * (g.abs() @ v.abs().transpose(2, 3) + (g.abs() * out.abs()).sum(-1, keepdim=True))
    ds_err = p * slope * (p_err * (dp - delta).abs() + delta_err + sums)
    bounds = [o_bound, ds_err @ k.abs() * scale + out_err * dq.abs(), ds_err.transpose(2, 3) @ q.abs() * scale, p_err * p.transpose(2, 3) @ g.abs()]
    dk, dv = heads(dk), heads(dv)
    return (back(out), back(dq), dk, dv), (back(bounds[0]), back(bounds[1]), heads(bounds[2]) + out_err * dk.abs(), heads(bounds[3]) + out_err * dv.abs())


def attention_step(q, k, v, lengths, window=None, score_cap=None, distance_slopes=None, scale=None, p_err=0.0, out_err=0.0):
    """(out [b, hq, d], bound) of one token against caches [b, n, hkv, d]."""
    b, hq, d = q.shape
    group = hq // k.shape[2]
    out, bound = torch.zeros(b, hq, d, dtype=torch.float64), torch.zeros(b, hq, d, dtype=torch.float64)
    for i in range(b):
        n = max(0, min(int(lengths[i]), k.shape[1]))
        first = 0 if window is None else max(0, n - window)
        if n == 0:
            continue
        for h in range(hq):
            kk, vv = k[i, first:n, h // group].double(), v[i, first:n, h // group].double()
            s = _bent(kk @ q[i, h].double() * (d ** -0.5 if scale is None else scale), score_cap)
            if distance_slopes is not None:
                s = s - float(distance_slopes[h]) * torch.arange(n - 1 - first, -1, -1).double()
            p = torch.softmax(s, 0)
            out[i, h] = p @ vv
            bound[i, h] = p_err * (p @ vv.abs()) + out_err * out[i, h].abs()
    return out, bound


def linear(q, k, v, log_decay, state=None, scale=None):
    """(out, last state) of [b, l, h, d] in float64, token by token; differentiable."""
    b, l, h, dk = q.shape
    scale = dk ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    g = log_decay.double()
    g = g.expand(b, l, h) if g.dim() == 1 else g
    s = torch.zeros(b, h, dk, v.shape[-1], dtype=torch.float64) if state is None else state.double()
    outs = []
    for t in range(l):
        s = torch.exp(g[:, t])[..., None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append(scale * (q[:, t, :, None, :] @ s)[..., 0, :])
    return torch.stack(outs, 1), s
