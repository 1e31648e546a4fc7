"""Serving from a paged cache, and positions with several axes, as cases that can be timed and compared.

  step     paged_attention_step: softmax attention of one new token of every sequence with keys and values that lie in pages, in 8 bits too
  store    paged_cache_write: the keys and values of new tokens into their places in the pages
  through  paged_cache_write into pages of 8 bits, and paged_cache_read of the same tokens
  read     paged_cache_read: tokens of every sequence out of the pages as one tensor
  rotary   axial_rotary: queries and keys turned by angles of several axes; training steps and single tokens

Pages are [pages, heads, page size, head size].  Pages of 8 bits hold e4m3 numbers, and every row of them an exponent (e8m0): the smallest
with which the row's largest magnitude is at most 448.  Table entries of -1 are no page.

`own` chooses between the framework's calls and their plain forms: elementary tensor operations in fp32, with angles in fp64, rounded once at
the end.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST_BYTES = 9.0e8


def listed():
    return [
        # One sequence with a long cache: the next token of a long document.
        dict(name="step long document", path="step", b=1, capacity=131072, hq=32, hkv=8, d=128, page=64, pages="bf16", window=0, cap=0.0, slopes=False,
             layout=1, dtype="bf16"),
        # Serving: the next tokens of a batch of sequences of very different lengths in 8 bits, small pages, capped scores and a distance bias.
        dict(name="step ragged batch 8 bits", path="step", b=32, capacity=8192, hq=32, hkv=8, d=128, page=16, pages="e4m3", window=0, cap=30.0,
             slopes=True, layout=2, dtype="bf16"),
        # The smallest step: one short sequence, a head of its own for every query head, full precision.
        dict(name="step short fp32", path="step", b=1, capacity=512, hq=12, hkv=12, d=64, page=16, pages="fp32", window=256, cap=0.0, slopes=False,
             layout=3, dtype="fp32"),
        # A full server: many long sequences in 8 bits, five query heads to a key head.
        dict(name="step full server 8 bits", path="step", b=64, capacity=16384, hq=40, hkv=8, d=128, page=48, pages="e4m3", window=0, cap=0.0,
             slopes=False, layout=4, dtype="bf16"),
        # A ragged batch of prompts of the causal layer's 12 heads into the pages as they are.
        dict(name="write ragged prompts", path="store", b=8, l=2048, hkv=12, d=128, page=64, pages="bf16", ragged=True, before=500, layout=5, dtype="bf16"),
        # A long prompt of odd length quantised into the cache, and read back as the next part of the prompt sees it.
        dict(name="prompt through 8 bits", path="through", b=1, l=16381, hkv=8, d=128, page=64, pages="e4m3", ragged=False, before=0, layout=6, dtype="bf16"),
        # Serving: one new token of 64 sequences, quantised, and read back.
        dict(name="new tokens through 8 bits", path="through", b=64, l=1, hkv=8, d=128, page=16, pages="e4m3", ragged=False, before=2000, layout=7,
             dtype="bf16"),
        # Long sequences out of the 8-bit cache, to go on with as a dense one.
        dict(name="read long 8 bits", path="read", b=4, tokens=16384, hkv=8, d=128, page=32, pages="e4m3", behind=0, layout=8, dtype="bf16"),
        # The last tokens of two sequences in full precision, as a window needs them.
        dict(name="read window fp32", path="read", b=2, tokens=300, hkv=4, d=64, page=16, pages="fp32", behind=700, layout=9, dtype="fp32"),
        # A video of 16 frames of 30 x 52 patches, 12 heads of 128, time, height and width: training step.
        dict(name="rotary video train", path="rotary", b=1, grid="16x30x52", hq=12, hkv=12, d=128, axes="44,42,42", interleaved=True, train=True, far=0,
             layout=10, dtype="bf16"),
        # Two images of odd size, grouped heads of 64, a quarter of each head without a position, full precision: training step.
        dict(name="rotary image train fp32", path="rotary", b=2, grid="37x41", hq=16, hkv=4, d=64, axes="24,24", interleaved=False, train=True, far=0,
             layout=11, dtype="fp32"),
        # Serving: one new token of 32 sequences, far positions.
        dict(name="rotary single tokens", path="rotary", b=32, grid="1", hq=32, hkv=8, d=128, axes="64,32,32", interleaved=True, train=False, far=1 << 20,
             layout=12, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= LARGEST_BYTES and _held(case) <= 1.08e9:
            return case


def _draw(rng):
    path = rng.choice(("step", "step", "step", "store", "through", "read", "rotary", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    layout = rng.randrange(1 << 30)
    d = rng.choice((64, 128))
    hkv = _spread(rng, 1, 16)
    group = rng.choice((1, 1, 2, 3, 4, 5, 8, 16))
    page = rng.choice((16, 16, 32, 48, 64, 80, 128, 256))
    pages = rng.choice((dtype, "e4m3"))
    if path == "step":
        return dict(path=path, b=_spread(rng, 1, 64), capacity=_spread(rng, 1, 65536), hq=hkv * group, hkv=hkv, d=d, page=page, pages=pages,
                    window=rng.choice((0, 0, _spread(rng, 1, 4096))), cap=rng.choice((0.0, 0.0, 30.0)), slopes=rng.random() < 0.4, layout=layout,
                    dtype=dtype)
    if path in ("store", "through"):
        return dict(path=path, b=_spread(rng, 1, 64), l=_spread(rng, 1, 16384), hkv=hkv, d=d, page=page, pages="e4m3" if path == "through" else dtype,
                    ragged=rng.random() < 0.5, before=rng.choice((0, _spread(rng, 1, 4000))), layout=layout, dtype=dtype)
    if path == "read":
        return dict(path=path, b=_spread(rng, 1, 16), tokens=_spread(rng, 1, 16384), hkv=hkv, d=d, page=page, pages=pages,
                    behind=rng.choice((0, _spread(rng, 1, 4000))), layout=layout, dtype=dtype)
    grid = rng.choice(([_spread(rng, 1, 16384)], [_spread(rng, 1, 100), _spread(rng, 1, 100)], [_spread(rng, 1, 32), _spread(rng, 1, 40), _spread(rng, 1, 40)]))
    axes = rng.choice({1: ((d,), (d // 2,)), 2: ((d // 2, d // 2), (d // 4, d // 4), (d // 2, d // 4)),
                       3: ((d - 4 * (d // 6), 2 * (d // 6), 2 * (d // 6)), (d // 2, d // 4, d // 4))}[len(grid)])
    axes = [a - a % 2 for a in axes]
    return dict(path=path, b=_spread(rng, 1, 16), grid="x".join(map(str, grid)), hq=hkv * group, hkv=hkv, d=d, axes=",".join(map(str, axes)),
                interleaved=rng.random() < 0.6, train=rng.random() < 0.6, far=rng.choice((0, _spread(rng, 1, 1 << 22))), layout=layout, dtype=dtype)


def _held(case):
    """Elements that the plain form holds of one operand."""
    if case["path"] == "step":
        return case["b"] * case["capacity"] * case["hkv"] * case["d"]
    if case["path"] == "rotary":
        return case["b"] * _tokens(case) * case["hq"] * case["d"]
    return case["b"] * (case.get("l") or case["tokens"]) * case["hkv"] * case["d"]


def _tokens(case):
    return math.prod(int(n) for n in case["grid"].split("x"))


def _lengths(case):
    """Step: tokens of every sequence, the new one among them; a single one has them all, of several some have none."""
    rng = random.Random(case["layout"])
    if case["b"] == 1:
        return [case["capacity"]]
    return [rng.randint(0, case["capacity"]) if i % 8 else _spread(rng, 1, case["capacity"]) for i in range(case["b"])]


def _spans(case):
    """Write and read: for every sequence where its tokens begin in the cache, and how many there are."""
    rng = random.Random(case["layout"])
    if case["path"] == "read":
        starts = [rng.randint(0, case["behind"]) for _ in range(case["b"])]
        return starts, [rng.randint(0, case["tokens"]) if i else case["tokens"] for i in range(case["b"])]
    starts = [rng.randint(0, case["before"]) for _ in range(case["b"])]
    return starts, [rng.randint(0, case["l"]) if case["ragged"] and i else case["l"] for i in range(case["b"])]


def _pool(case, ends, gen, dev, fill):
    """Pages for sequences that reach to `ends`, in no order, and a few that belong to nobody."""
    page, hkv, d = case["page"], case["hkv"], case["d"]
    need = [-(-n // page) for n in ends]
    wide = max(1, -(-case["capacity"] // page) if case["path"] == "step" else max(need))
    count = sum(need) + 3
    order = torch.randperm(count, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(ends), wide), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (count, hkv, page, d)
    got = {"page_table": table}
    for n in ("k", "v"):
        if case["pages"] == "e4m3":
            # numbers of all sizes, and an exponent for every row with which they are about 1
            codes = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16).mul_(100).clamp_(-448, 448) if fill else torch.zeros(shape, device=dev)
            got[n] = codes.to(torch.float8_e4m3fn)
            got[n + "_scale"] = torch.randint(118, 122, shape[:3], generator=gen, device=dev, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        else:
            got[n] = torch.randn(shape, generator=gen, device=dev, dtype=DTYPES[case["pages"]]) if fill else torch.zeros(shape, dtype=DTYPES[case["pages"]], device=dev)
            got[n + "_scale"] = None
    return got


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _prepare_step(case, gen, dev, dtype):
    lengths = _lengths(case)
    state = dict(q=torch.randn(case["b"], case["hq"], case["d"], generator=gen, device=dev).to(dtype), lengths=_int32(lengths, dev),
                 window=case["window"] or None, score_cap=case["cap"] or None, slopes=None, **_pool(case, lengths, gen, dev, True))
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / case["hq"]) for i in range(case["hq"])], device=dev)
    return state


def _prepare_write(case, gen, dev, dtype):
    starts, counts = _spans(case)
    b, l, hkv, d = (case[n] for n in ("b", "l", "hkv", "d"))
    # the keys' and values' part of one packed projection
    packed = torch.randn(b, l, 2 * hkv * d, generator=gen, device=dev).to(dtype)
    new_k, new_v = (t.reshape(b, l, hkv, d) for t in packed.split(hkv * d, dim=-1))
    ends = [s + n for s, n in zip(starts, counts)]
    return dict(new_k=new_k, new_v=new_v, starts=_int32(starts, dev), counts=_int32(counts, dev) if case["ragged"] else None, ends=_int32(ends, dev),
                **_pool(case, ends, gen, dev, False))


def _prepare_read(case, gen, dev, dtype):
    starts, counts = _spans(case)
    ends = [s + n for s, n in zip(starts, counts)]
    return dict(starts=_int32(starts, dev), lengths=_int32(ends, dev), dtype=dtype, **_pool(case, ends, gen, dev, True))


def _prepare_rotary(case, gen, dev, dtype):
    b, l, hq, hkv, d = case["b"], _tokens(case), case["hq"], case["hkv"], case["d"]
    packed = torch.randn(b, l, (hq + hkv) * d, generator=gen, device=dev).to(dtype)
    q, k = (t.reshape(b, l, -1, d) for t in packed.split((hq * d, hkv * d), dim=-1))
    axes = tuple(int(a) for a in case["axes"].split(","))
    sizes = [int(n) for n in case["grid"].split("x")]
    sizes = [1] * (len(axes) - len(sizes)) + sizes
    place = torch.stack(torch.meshgrid(*(torch.arange(n, device=dev, dtype=torch.int32) for n in sizes), indexing="ij"), -1).reshape(l, len(axes))
    if case["far"]:      # every sequence from a place of its own
        place = place[None] + torch.randint(0, case["far"], (b, 1, len(axes)), generator=gen, device=dev, dtype=torch.int32)
    state = dict(q=q, k=k, positions=place, axes=axes, interleaved=case["interleaved"])
    if case["train"]:
        q.requires_grad_(True)
        k.requires_grad_(True)
        state["grads"] = [torch.randn(t.shape, generator=gen, device=dev).to(dtype) for t in (q, k)]
    return state


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    make = {"step": _prepare_step, "store": _prepare_write, "through": _prepare_write, "read": _prepare_read, "rotary": _prepare_rotary}
    return dict(case=case, **make[case["path"]](case, gen, dev, DTYPES[case["dtype"]]))


def run(state):
    path = state["case"]["path"]
    if path == "rotary":
        with torch.set_grad_enabled(state["case"]["train"]):
            q, k = _rotary(state)
        if not state["case"]["train"]:
            return [q, k]
        return [q, k, *torch.autograd.grad([q, k], [state["q"], state["k"]], state["grads"])]
    with torch.no_grad():
        if path == "step":
            return _step(state)
        if path == "read":
            return list(_read(state, state["lengths"], state["case"]["tokens"], state["dtype"]))
        _write(state)
        if path == "store":
            return [state["k"], state["v"]]
        return list(_read(state, state["ends"], state["case"]["l"], state["new_k"].dtype))


# ---- the calls, and their plain forms

def _cache(s):
    from lact_amd import PagedCache
    return PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])


def _gathered(pages, scale, table):
    """The pages of every sequence behind one another: [b, heads, places, d], fp32."""
    at = table.long().clamp(min=0)
    rows = pages.view(torch.uint8)[at].view(pages.dtype).float() if scale is not None else pages[at].float()
    if scale is not None:
        rows = rows * torch.exp2(scale.view(torch.uint8)[at].float() - 127.0)[..., None]
    b, n, h, p, d = rows.shape
    return rows.transpose(1, 2).reshape(b, h, n * p, d)


def _on_pages(s):
    return (s["page_table"] >= 0).repeat_interleave(s["case"]["page"], 1)


def _step(s):
    if own:
        from lact_amd import paged_attention_step
        return paged_attention_step(s["q"], _cache(s), s["page_table"], s["lengths"], s["window"], score_cap=s["score_cap"], distance_slopes=s["slopes"])
    k, v = (_gathered(s[n], s[n + "_scale"], s["page_table"]) for n in ("k", "v"))
    q = s["q"].float()
    b, hq, d = q.shape
    hkv, n = k.shape[1:3]
    scores = (q.reshape(b, hkv, hq // hkv, d) @ k.transpose(2, 3)).reshape(b, hq, n) / math.sqrt(d)
    if s["score_cap"]:
        scores = s["score_cap"] * torch.tanh(scores / s["score_cap"])
    back = s["lengths"].long()[:, None] - 1 - torch.arange(n, device=q.device)[None]      # how far behind the new token
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None] * back[:, None].float()
    seen = (back >= 0) & _on_pages(s)
    if s["window"]:
        seen = seen & (back < s["window"])
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return (p.reshape(b, hkv, hq // hkv, n) @ v).reshape(b, hq, d).to(s["q"].dtype)


def _write(s):
    if own:
        from lact_amd import paged_cache_write
        paged_cache_write(_cache(s), s["new_k"], s["new_v"], s["page_table"], s["starts"], s["counts"])
        return
    b, l = s["new_k"].shape[:2]
    p = s["case"]["page"]
    i = torch.arange(l, device=s["new_k"].device)[None]
    place = s["starts"].long()[:, None] + i
    page = s["page_table"].long().gather(1, (place // p).clamp(max=s["page_table"].shape[1] - 1))
    if s["counts"] is not None:
        taken = i < s["counts"][:, None]
        page, place = page[taken], place[taken]
    _put(s, "k", s["new_k"] if s["counts"] is None else s["new_k"][taken], page, place % p)
    _put(s, "v", s["new_v"] if s["counts"] is None else s["new_v"][taken], page, place % p)


def _put(s, name, rows, page, at):
    rows = rows.reshape(-1, *rows.shape[-2:]).float()                                      # [tokens, heads, d]
    page, at = page.reshape(-1), at.reshape(-1)
    if s[name + "_scale"] is None:
        s[name].transpose(1, 2)[page, at] = rows.to(s[name].dtype)
        return
    part, exponent = torch.frexp(rows.abs().amax(-1))                                      # part in [0.5, 1): 448 is 0.875 * 2^9
    exponent = (exponent - 9 + (part > 0.875)).clamp(min=-127)
    codes = (rows * torch.exp2(-exponent.float())[..., None]).to(torch.float8_e4m3fn)
    s[name].view(torch.uint8).transpose(1, 2)[page, at] = codes.view(torch.uint8)
    s[name + "_scale"].view(torch.uint8).transpose(1, 2)[page, at] = (exponent + 127).to(torch.uint8)


def _read(s, lengths, tokens, dtype):
    if own:
        from lact_amd import paged_cache_read
        return paged_cache_read(_cache(s), s["page_table"], lengths, tokens, s["starts"], dtype=dtype)
    place = s["starts"].long()[:, None] + torch.arange(tokens, device=lengths.device)[None]
    there = place < lengths[:, None]
    p, wide = s["case"]["page"], s["page_table"].shape[1]
    page = s["page_table"].long().gather(1, (place // p).clamp(max=wide - 1))
    there = there & (page >= 0)
    return (_taken(s, "k", page.clamp(min=0), place % p, there).to(dtype), _taken(s, "v", page.clamp(min=0), place % p, there).to(dtype))


def _taken(s, name, page, at, there):
    if s[name + "_scale"] is None:
        rows = s[name].transpose(1, 2)[page, at].float()
    else:
        rows = s[name].view(torch.uint8).transpose(1, 2)[page, at].view(torch.float8_e4m3fn).float()
        rows = rows * torch.exp2(s[name + "_scale"].view(torch.uint8).transpose(1, 2)[page, at].float() - 127.0)[..., None]
    return torch.where(there[..., None, None], rows, 0.0)


def _rotary(s):
    if own:
        from lact_amd import axial_rotary
        return axial_rotary(s["q"], s["k"], s["positions"], s["axes"], interleaved=s["interleaved"])
    dev = s["q"].device
    sizes = torch.tensor(s["axes"], device=dev, dtype=torch.float64)
    axis = torch.repeat_interleave(torch.arange(len(s["axes"]), device=dev), sizes.long() // 2)
    within = torch.arange(axis.numel(), device=dev) - (sizes.long() // 2).cumsum(0)[axis] + (sizes.long() // 2)[axis]
    angle = s["positions"].double()[..., axis] * 10000.0 ** (-2.0 * within / sizes[axis])   # [.., l, pairs]
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    return _turned(s["q"], cos, sin, s["interleaved"]), _turned(s["k"], cos, sin, s["interleaved"])


def _turned(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    y, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :pairs], y[..., pairs:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y.to(x.dtype), rest), -1)


# ---- what a pass cannot do without

def work(case):
    act = 2 if case["dtype"] == "bf16" else 4
    if case["path"] == "rotary":
        rows = case["b"] * _tokens(case) * (case["hq"] + case["hkv"])
        turned = sum(int(a) for a in case["axes"].split(","))
        times = 2 if case["train"] else 1
        return {"bytes": times * (2 * rows * case["d"] * act + 4 * _tokens(case) * case["axes"].count(",") + 4 * _tokens(case)), "flops": times * 3 * rows * turned}
    held = {"bf16": 2, "fp32": 4, "e4m3": 1}[case["pages"]]
    row = case["d"] * held + (held == 1)                                                   # of a key or a value
    if case["path"] == "step":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        return {"bytes": 2 * seen * case["hkv"] * row + 4 * seen // case["page"] + 2 * case["b"] * case["hq"] * case["d"] * act,
                "flops": 4 * seen * case["hq"] * case["d"]}
    tokens = sum(_spans(case)[1])
    whole = case["b"] * (case["tokens"] if case["path"] == "read" else case["l"])          # of the tensor that is read back, zeros among them
    new, kept, back = (2 * n * case["hkv"] * size for n, size in ((tokens, case["d"] * act), (tokens, row), (whole, case["d"] * act)))
    return {"bytes": {"store": new + kept, "through": new + 2 * kept + back, "read": kept + back}[case["path"]], "flops": 2 * tokens * case["hkv"] * case["d"]}


# ---- the definitions in 64 bits, sequence by sequence

def _rows64(s, name, i, first, last):
    """Tokens [first, last) of sequence i: [tokens, heads, d]."""
    p = s["case"]["page"]
    at = torch.arange(first, last, device=s["page_table"].device)
    page = s["page_table"][i].long()[at // p]
    if s[name + "_scale"] is None:
        return s[name][page, :, at % p].double()
    code = s[name].view(torch.uint8)[page, :, at % p].view(torch.float8_e4m3fn).double()
    return torch.ldexp(code, s[name + "_scale"].view(torch.uint8)[page, :, at % p].int()[..., None] - 127)


def _exact_step(case, s):
    b, hq, d = s["q"].shape
    hkv = case["hkv"]
    group = hq // hkv
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(_lengths(case)):
        first = max(0, n - (case["window"] or n))
        if n == 0:
            continue
        back = torch.arange(n - 1 - first, -1, -1, device=out.device, dtype=torch.float64)
        k, v = (_rows64(s, x, i, first, n) for x in ("k", "v"))
        for h in range(hkv):
            own_heads = slice(h * group, (h + 1) * group)
            x = s["q"][i, own_heads].double() @ k[:, h].T * (1 / math.sqrt(d))
            if case["cap"]:
                x = torch.tanh(x * (1 / case["cap"])) * case["cap"]
            if case["slopes"]:
                x = x - s["slopes"][own_heads, None].double() * back
            out[i, own_heads] = torch.softmax(x, -1) @ v[:, h]
    return out


def _through_8_bits(x):
    """Every row's e4m3 numbers, times its power of two."""
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -127)
    for _ in range(256):                                                                   # the smallest power of two that holds the row
        scale = torch.where(top > 448 * scale, scale * 2, scale)
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _exact_write(case, s):
    starts, counts = _spans(case)
    if case["path"] == "through":
        res = []
        for n in ("new_k", "new_v"):
            x = _through_8_bits(s[n].double())
            for i, c in enumerate(counts):
                x[i, c:] = 0
            res.append(x)
        return res
    k, v = s["k"].double(), s["v"].double()
    for i, (first, n) in enumerate(zip(starts, counts)):
        at = torch.arange(first, first + n, device=k.device)
        page = s["page_table"][i].long()[at // case["page"]]
        k[page, :, at % case["page"]] = s["new_k"][i, :n].double()
        v[page, :, at % case["page"]] = s["new_v"][i, :n].double()
    return [k, v]


def _exact_read(case, s):
    res = [torch.zeros(case["b"], case["tokens"], case["hkv"], case["d"], dtype=torch.float64, device=s["k"].device) for _ in range(2)]
    for i, (first, n) in enumerate(zip(*_spans(case))):
        for x, name in zip(res, ("k", "v")):
            x[i, :n] = _rows64(s, name, i, first, first + n)
    return res


def _exact_rotary(case, s):
    axes = s["axes"]
    angles = [s["positions"][..., a, None].double() * torch.exp(torch.arange(n // 2, device=s["q"].device, dtype=torch.float64) * (-2 * math.log(10000.0) / n))
              for a, n in enumerate(axes)]
    angle = torch.cat(angles, -1)[..., None, :]
    turn = torch.polar(torch.ones_like(angle), angle)
    pairs = turn.shape[-1]

    def turned(x, by):
        y = x.detach().double().clone()
        if case["interleaved"]:
            z = torch.complex(y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) * by
            y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :pairs], y[..., pairs:2 * pairs]) * by
            y[..., :pairs], y[..., pairs:2 * pairs] = z.real, z.imag
        return y

    res = [turned(s["q"], turn), turned(s["k"], turn)]
    return res + [turned(g, turn.conj()) for g in s["grads"]] if case["train"] else res


def exact(case, seed):
    s = prepare(case, seed)
    make = {"step": _exact_step, "store": _exact_write, "through": _exact_write, "read": _exact_read, "rotary": _exact_rotary}
    with torch.no_grad():
        return make[case["path"]](case, s)
