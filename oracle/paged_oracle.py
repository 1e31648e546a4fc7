"""The paged cache and rotary positions (lact_amd.paged_cache, lact_amd.rotary) in float64 on the CPU, from their definitions.  Test infrastructure only."""
from __future__ import annotations

import math

import torch


def e4m3_values():
    """What the 256 codes stand for."""
    c = torch.arange(256)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.pow(torch.tensor(2.0, dtype=torch.float64), (e - 7).double()))
    v[(c & 127) == 127] = math.nan
    return torch.where(c >= 128, -v, v)


def to_8_bits(x):
    """(codes, exponents) of rows [..., d]: uint8 and uint8."""
    x = x.double()
    finite = torch.where(torch.isfinite(x), x, torch.zeros(()).double())
    top = finite.abs().amax(-1)
    exponent = torch.zeros(top.shape, dtype=torch.int64)
    for e in range(255):      # the smallest that holds the row
        exponent += (top > 448.0 * 2.0 ** (e - 127)).long()
    y = finite * torch.pow(torch.tensor(2.0, dtype=torch.float64), (127 - exponent).double())[..., None]
    table = e4m3_values()[:127]
    # nearest, ties to the even code
    near = torch.searchsorted(table, y.abs().contiguous())
    low, high = (near - 1).clamp(min=0), near.clamp(max=126)
    dl, dh = y.abs() - table[low], table[high] - y.abs()
    code = torch.where((dl < dh) | ((dl == dh) & (low % 2 == 0)), low, high)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 127))
    sign = torch.signbit(x).long() * 128
    return (code + sign).to(torch.uint8), exponent.to(torch.uint8)


def held(pages, exponents):
    """The numbers of pages: [pages, heads, size, d], float64."""
    if exponents is None:
        return pages.double()
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), exponents.view(torch.uint8).double() - 127)
    scale = torch.where(exponents.view(torch.uint8) == 255, math.nan, scale)
    return e4m3_values()[pages.view(torch.uint8).long()] * scale[..., None]


def page_of(table, pages, size, seq, place):
    if place < 0 or place >= table.shape[1] * size:
        return -1
    p = int(table[seq, place // size])
    return p if 0 <= p < pages else -1


def tokens(numbers, table, starts, lengths, n):
    """[b, n, heads, d] of the places starts[s] + i, zeros from lengths[s] on and where there is no page; and whether there was one."""
    pages, heads, size, d = numbers.shape
    out, there = torch.zeros(len(table), n, heads, d, dtype=torch.float64), torch.zeros(len(table), n, dtype=torch.bool)
    for s in range(len(table)):
        for i in range(n):
            place = int(starts[s]) + i
            p = page_of(table, pages, size, s, place) if place < int(lengths[s]) else -1
            if p >= 0:
                out[s, i], there[s, i] = numbers[p, :, place % size], True
    return out, there


def step(q, k, v, table, lengths, window=None, score_cap=None, distance_slopes=None, scale=None, p_err=0.0, out_err=0.0):
    """(out [b, hq, d], bound) of one token with numbers of pages k, v [pages, hkv, size, d]: see mixers_oracle.attention_step."""
    b, hq, d = q.shape
    size, wide = k.shape[2], table.shape[1]
    group = hq // k.shape[1]
    out, bound = torch.zeros(b, hq, d, dtype=torch.float64), torch.zeros(b, hq, d, dtype=torch.float64)
    for i in range(b):
        n = max(0, min(int(lengths[i]), wide * size))
        first = 0 if window is None else max(0, n - window)
        at = [(j, page_of(table, k.shape[0], size, i, j)) for j in range(first, n)]
        at = [(j, p) for j, p in at if p >= 0]
        if not at:
            continue
        j, p = torch.tensor(at).T
        kk, vv = k[p, :, j % size], v[p, :, j % size]
        for h in range(hq):
            s = kk[:, h // group] @ q[i, h].double() * (d ** -0.5 if scale is None else scale)
            if score_cap:
                s = score_cap * torch.tanh(s / score_cap)
            if distance_slopes is not None:
                s = s - float(distance_slopes[h]) * (n - 1 - j).double()
            w = torch.softmax(s, 0)
            out[i, h] = w @ vv[:, h // group]
            bound[i, h] = p_err * (w @ vv[:, h // group].abs()) + out_err * out[i, h].abs()
    return out, bound


def angles(positions, axes, base=10000.0, frequencies=None):
    """[..., pairs] of positions [..., axes]."""
    at, parts = 0, []
    for a, n in enumerate(axes):
        f = [base ** (-2.0 * i / n) for i in range(n // 2)] if frequencies is None else list(frequencies[at:at + n // 2])
        parts.append(positions[..., a, None].double() * torch.tensor(f, dtype=torch.float64))
        at += n // 2
    return torch.cat(parts, -1)


def rotary(x, angle, interleaved=True):
    """x [..., heads, d] turned by angle [..., pairs], float64; differentiable."""
    x = x.double()
    n = angle.shape[-1]
    cos, sin = angle.cos()[..., None, :], angle.sin()[..., None, :]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    c, s = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((c, s), -1).flatten(-2) if interleaved else torch.cat((c, s), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)
