"""The token mixers beside the test-time-training operation, as cases that can be timed and compared.

  attention       masked_window_attention: softmax attention inside a window, over packed documents with prefixes that all of a
                  document's tokens see, scores capped by a tanh and lowered with the distance; training steps and prompts
  attention_step  window_attention_step: the same for one new token of every sequence against its cache of keys and values
  linear          decayed_linear_attention: linear attention whose state decays by a factor per head, or per head and token; training
                  steps and prompts
  linear_step     decayed_linear_attention_step: the same for one new token of every sequence

`own` chooses between the framework's calls and their plain forms: elementary tensor operations in fp32, with the sums of log
decays in fp64, rounded once at the end.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
LARGEST_FLOPS = 5.6e11
LARGEST_BYTES = 6.0e8
LARGEST_SCORES = 2.2e9


def listed():
    return [
        # The causal layer's attention (12 heads of 128, window 2048) on packed documents, training step.
        dict(name="packed documents train", path="attention", b=2, l=4096, hq=12, hkv=12, d=128, window=2048, cap=0.0, slopes=False, docs=7,
             prefix=False, pad=0, layout=1, train=True, dtype="bf16"),
        # A long prompt of odd length whose instruction part is read in both directions, grouped heads, capped scores: one forward.
        dict(name="prefix prompt grouped heads", path="attention", b=1, l=8191, hq=32, hkv=8, d=128, window=0, cap=30.0, slopes=False, docs=1,
             prefix=True, pad=0, layout=2, train=False, dtype="bf16"),
        # A padded batch of short sequences, heads of 64 with a distance bias, training step.
        dict(name="padded batch distance bias", path="attention", b=3, l=1021, hq=16, hkv=4, d=64, window=0, cap=0.0, slopes=True, docs=1,
             prefix=False, pad=200, layout=3, train=True, dtype="bf16"),
        # Everything at once in full precision, a training step at the size of a test.
        dict(name="all masks fp32 train", path="attention", b=1, l=300, hq=4, hkv=2, d=64, window=100, cap=20.0, slopes=True, docs=3, prefix=True,
             pad=9, layout=4, train=True, dtype="fp32"),
        # One sequence with a long cache: the next token of a long document.
        dict(name="step long cache", path="attention_step", b=1, capacity=131072, hq=32, hkv=8, d=128, window=0, cap=0.0, slopes=False, layout=5,
             dtype="bf16"),
        # Serving: the next tokens of a batch of sequences of very different lengths.
        dict(name="step ragged batch", path="attention_step", b=32, capacity=8192, hq=32, hkv=8, d=128, window=0, cap=30.0, slopes=True, layout=6,
             dtype="bf16"),
        # The smallest step: one short sequence with a head of its own for every query head, full precision.
        dict(name="step short fp32", path="attention_step", b=1, capacity=512, hq=12, hkv=12, d=64, window=256, cap=0.0, slopes=False, layout=7,
             dtype="fp32"),
        # Training step with a decay for every token that is learned, at the width of the causal layer.
        dict(name="linear train gated", path="linear", b=4, l=4096, h=12, dk=128, dv=128, gated=True, state=False, train=True, dtype="bf16"),
        # A long prompt that continues from a state and hands its own on, constant decays.
        dict(name="linear prompt with state", path="linear", b=1, l=16381, h=16, dk=64, dv=128, gated=False, state=True, train=False, dtype="bf16"),
        # Full precision training of a small model, the state's gradient included.
        dict(name="linear train fp32", path="linear", b=2, l=333, h=4, dk=64, dv=64, gated=True, state=True, train=True, dtype="fp32"),
        # Serving: one token of 64 sequences.
        dict(name="linear step batch", path="linear_step", b=64, h=16, dk=128, dv=128, gated=True, dtype="bf16"),
        # The smallest step of all: one sequence.
        dict(name="linear step single fp32", path="linear_step", b=1, h=12, dk=64, dv=128, gated=False, dtype="fp32"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        # the plain form holds whole score matrices
        if case["path"] == "attention" and case["b"] * case["hq"] * case["l"] ** 2 > LARGEST_SCORES:
            continue
        # a 32-bit product costs some 16 times one of bf16
        if w["flops"] * (16 if case["dtype"] == "fp32" else 1) <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES:
            return case


def _draw(rng):
    path = rng.choice(("attention", "attention", "attention_step", "linear", "linear", "linear_step"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    layout = rng.randrange(1 << 30)
    if path == "attention":
        l = _spread(rng, 1, 8192)
        group = rng.choice((1, 1, 2, 3, 4, 8))
        docs = rng.choice((1, 1, _spread(rng, 1, 40)))
        return dict(path=path, b=_spread(rng, 1, 8), l=l, hq=_spread(rng, 1, 16) * group, hkv=0, group=group, d=rng.choice((64, 128)),
                    window=rng.choice((0, _spread(rng, 1, 4096))), cap=rng.choice((0.0, 0.0, 20.0, 50.0)), slopes=rng.random() < 0.4, docs=docs,
                    prefix=rng.random() < 0.4, pad=rng.choice((0, 0, rng.randint(0, l // 2))), layout=layout, train=rng.random() < 0.6,
                    dtype=dtype)
    if path == "attention_step":
        group = rng.choice((1, 2, 3, 4, 7, 8, 16))
        return dict(path=path, b=_spread(rng, 1, 64), capacity=_spread(rng, 1, 65536), hq=_spread(rng, 1, 16) * group, hkv=0, group=group,
                    d=rng.choice((64, 128)), window=rng.choice((0, 0, _spread(rng, 1, 4096))), cap=rng.choice((0.0, 0.0, 30.0)),
                    slopes=rng.random() < 0.4, layout=layout, dtype=dtype)
    dk, dv = rng.choice((64, 128)), rng.choice((64, 128))
    if path == "linear":
        return dict(path=path, b=_spread(rng, 1, 8), l=_spread(rng, 1, 16384), h=_spread(rng, 1, 24), dk=dk, dv=dv, gated=rng.random() < 0.5,
                    state=rng.random() < 0.5, train=rng.random() < 0.6, dtype=dtype)
    return dict(path=path, b=_spread(rng, 1, 128), h=_spread(rng, 1, 32), dk=dk, dv=dv, gated=rng.random() < 0.5, dtype=dtype)


def _kv_heads(case):
    return case["hkv"] or case["hq"] // case["group"]


def _documents(case):
    """Where the documents of every sequence begin and end, and how many of each one's first tokens all of it sees."""
    rng = random.Random(case["layout"])
    bounds, prefixes = [], []
    for _ in range(case["b"]):
        pad = rng.randint(0, case["pad"])
        left = rng.randint(0, pad) if case["pad"] else 0          # padded on the left, on the right, or on both sides
        end = max(left, case["l"] - (pad - left))
        cuts = sorted(rng.randint(left, end) for _ in range(case["docs"] - 1))
        row = [left] + cuts + [end]
        bounds.append(row)
        prefixes.append([rng.randint(0, (e - s + 1) // 2) for s, e in zip(row, row[1:])])
    return bounds, prefixes


def _lengths(case):
    rng = random.Random(case["layout"])
    if case["b"] == 1:
        return [case["capacity"]]
    return [rng.randint(0, case["capacity"]) if i % 8 else _spread(rng, 1, case["capacity"]) for i in range(case["b"])]


def _pairs(case):
    """How many (query, key) pairs the mask leaves, over the batch."""
    n = 0
    w = case["window"] or case["l"]
    for row, pre in zip(*_documents(case)):
        for s, e, p in zip(row, row[1:], pre):
            m = e - s
            c = min(w, m)
            n += c * (c + 1) // 2 + (m - c) * c
            if case["prefix"]:
                n += p * (p - 1) // 2
    return n


def _prepare_attention(case, rand, dev, dtype):
    b, l, hq, hkv, d = case["b"], case["l"], case["hq"], _kv_heads(case), case["d"]
    # one packed projection, whose parts the attention takes as views
    packed = rand(b, l, (hq + 2 * hkv) * d).to(dtype)
    q, k, v = (t.reshape(b, l, -1, d) for t in packed.split((hq * d, hkv * d, hkv * d), dim=-1))
    state = dict(case=case, q=q, k=k, v=v, window=case["window"] or None, score_cap=case["cap"] or None, slopes=None, documents=None, prefixes=None)
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], device=dev)
    if case["docs"] > 1 or case["pad"] or case["prefix"]:
        bounds, prefixes = _documents(case)
        state["documents"] = torch.tensor(bounds, dtype=torch.int32, device=dev)
        if case["prefix"]:
            state["prefixes"] = torch.tensor(prefixes, dtype=torch.int32, device=dev)
    if case["train"]:
        for n in ("q", "k", "v"):
            state[n].requires_grad_(True)
        state["grad"] = rand(b, l, hq, d).to(dtype)
    return state


def _prepare_step(case, rand, dev, dtype):
    b, n, hq, hkv, d = case["b"], case["capacity"], case["hq"], _kv_heads(case), case["d"]
    state = dict(case=case, q=rand(b, hq, d).to(dtype), k=rand(b, n, hkv, d, dtype=dtype), v=rand(b, n, hkv, d, dtype=dtype),
                 lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=dev), window=case["window"] or None,
                 score_cap=case["cap"] or None, slopes=None)
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], device=dev)
    return state


def _decays(case, rand, dev, shape):
    """Log decays: gates as a sigmoid makes them, from nearly nothing forgotten to most of it; or one constant for every head."""
    if case["gated"]:
        return torch.nn.functional.logsigmoid(rand(*shape) * 1.5 + 4.0)
    return torch.tensor([math.log1p(-2.0 ** (-4.0 - 6.0 * i / case["h"])) for i in range(case["h"])], device=dev)


def _prepare_linear(case, rand, dev, dtype):
    b, l, h, dk, dv = (case[n] for n in ("b", "l", "h", "dk", "dv"))
    # queries and keys as the layers make them: of unit length
    unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
    state = dict(case=case, q=unit(rand(b, l, h, dk)).to(dtype), k=unit(rand(b, l, h, dk)).to(dtype), v=rand(b, l, h, dv).to(dtype),
                 log_decay=_decays(case, rand, dev, (b, l, h)), state=rand(b, h, dk, dv) if case["state"] else None)
    if case["train"]:
        for n in ("q", "k", "v", "log_decay", "state"):
            if state[n] is not None:
                state[n].requires_grad_(True)
        state["grad"] = rand(b, l, h, dv).to(dtype)
        if case["state"]:
            state["state_grad"] = rand(b, h, dk, dv) * 0.1
    return state


def _prepare_linear_step(case, rand, dev, dtype):
    b, h, dk, dv = (case[n] for n in ("b", "h", "dk", "dv"))
    unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
    state = rand(b, h, dk, dv)
    return dict(case=case, q=unit(rand(b, h, dk)).to(dtype), k=unit(rand(b, h, dk)).to(dtype), v=rand(b, h, dv).to(dtype),
                log_decay=_decays(case, rand, dev, (b, h)), state=state, state_out=torch.empty_like(state))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev = torch.device("cuda", torch.cuda.current_device())

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    make = {"attention": _prepare_attention, "attention_step": _prepare_step, "linear": _prepare_linear, "linear_step": _prepare_linear_step}
    return make[case["path"]](case, rand, dev, DTYPES[case["dtype"]])


def run(state):
    path = state["case"]["path"]
    if path == "attention":
        with torch.set_grad_enabled(state["case"]["train"]):
            out = _attention(state)
        if not state["case"]["train"]:
            return out
        return [out, *torch.autograd.grad(out, [state["q"], state["k"], state["v"]], state["grad"])]
    if path == "linear":
        with torch.set_grad_enabled(state["case"]["train"]):
            out, last = _linear(state)
        if not state["case"]["train"]:
            return [out, last]
        ins = [state[n] for n in ("q", "k", "v", "log_decay", "state") if state[n] is not None]
        outs, grads = ([out, last], [state["grad"], state["state_grad"]]) if state["state"] is not None else ([out], [state["grad"]])
        return [out, last, *torch.autograd.grad(outs, ins, grads)]
    with torch.no_grad():
        return _attention_step(state) if path == "attention_step" else list(_linear_step(state))


# ---- the calls, and their plain forms

def _attention(s):
    if own:
        from lact_amd import masked_window_attention
        return masked_window_attention(s["q"], s["k"], s["v"], s["window"], score_cap=s["score_cap"], distance_slopes=s["slopes"],
                                       documents=s["documents"], prefixes=s["prefixes"])
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))                      # [b, h, l, d]
    b, hq, l, d = q.shape
    group = hq // k.shape[1]
    scores = (q.reshape(b, -1, group * l, d) @ k.transpose(2, 3)).reshape(b, hq, l, l) / math.sqrt(d)
    if s["score_cap"]:
        scores = s["score_cap"] * torch.tanh(scores / s["score_cap"])
    pos = torch.arange(l, device=q.device)
    ahead = pos[None, :] - pos[:, None]                                                    # key's place minus query's
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None, None] * ahead.abs().float()
    seen = ahead[None] <= 0
    if s["documents"] is not None:
        bounds = s["documents"].long()
        which = (pos[None, :, None] >= bounds[:, None, :]).sum(-1) - 1                     # document of every token; -1 and n: none
        inside = (which >= 0) & (which < bounds.shape[1] - 1)
        at = which.clamp(0, bounds.shape[1] - 2)
        if s["prefixes"] is not None:
            seen = seen | (pos[None, None, :] < (bounds.gather(1, at) + s["prefixes"].long().gather(1, at))[:, :, None])
        seen = seen & (which[:, :, None] == which[:, None, :]) & inside[:, :, None]
    if s["window"]:
        seen = seen & (ahead > -s["window"])[None]
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.detach().amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = (p.reshape(b, -1, group * l, l) @ v).reshape(b, hq, l, d)
    return out.transpose(1, 2).to(s["q"].dtype)


def _attention_step(s):
    if own:
        from lact_amd import window_attention_step
        return window_attention_step(s["q"], s["k"], s["v"], s["lengths"], s["window"], score_cap=s["score_cap"], distance_slopes=s["slopes"])
    q, k, v = s["q"].float(), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    b, hq, d = q.shape
    hkv, n = k.shape[1:3]
    scores = (q.reshape(b, hkv, hq // hkv, d) @ k.transpose(2, 3)).reshape(b, hq, n) / math.sqrt(d)
    if s["score_cap"]:
        scores = s["score_cap"] * torch.tanh(scores / s["score_cap"])
    back = s["lengths"].long()[:, None] - 1 - torch.arange(n, device=q.device)[None]      # how far behind the new token
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None] * back[:, None].float()
    seen = back >= 0
    if s["window"]:
        seen = seen & (back < s["window"])
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return (p.reshape(b, hkv, hq // hkv, n) @ v).reshape(b, hq, d).to(s["q"].dtype)


CHUNK = 64


def _linear(s):
    if own:
        from lact_amd import decayed_linear_attention
        return decayed_linear_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], return_state=True)
    b, l, h, dk = s["q"].shape
    dv = s["v"].shape[-1]
    n = -(-l // CHUNK)
    fill = n * CHUNK - l
    chunks = lambda t: torch.nn.functional.pad(t, (0, 0, 0, fill)).reshape(b, h, n, CHUNK, -1)  # noqa: E731
    q, k, v = (chunks(s[x].float().transpose(1, 2)) for x in ("q", "k", "v"))             # [b, h, n, CHUNK, d]
    g = s["log_decay"].double()
    g = (g.expand(b, l, h) if g.dim() == 1 else g).transpose(1, 2)[..., None]
    g = chunks(g)[..., 0].cumsum(-1)                                                      # from the chunk's start, this token's included
    whole = g[..., -1]                                                                    # [b, h, n]
    tri = torch.ones(CHUNK, CHUNK, device=q.device, dtype=torch.bool).tril()
    pair = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~tri, -math.inf)).float()
    q = q * dk ** -0.5
    inside = ((q @ k.transpose(-1, -2)) * pair) @ v
    added = (k * torch.exp(whole[..., None] - g).float()[..., None]).transpose(-1, -2) @ v     # [b, h, n, dk, dv]
    # the state in front of chunk i: what every earlier one added, and the initial one, decayed by the chunks between
    start = s["state"] if s["state"] is not None else torch.zeros(b, h, dk, dv, device=q.device)
    added = torch.cat((start[:, :, None], added), 2)
    total = torch.nn.functional.pad(whole.cumsum(-1), (1, 0))                             # decay up to the chunk, [b, h, n + 1]
    tri = torch.ones(n + 1, n + 1, device=q.device, dtype=torch.bool).tril()
    between = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~tri, -math.inf)).float()
    states = (between @ added.reshape(b, h, n + 1, dk * dv)).reshape(b, h, n + 1, dk, dv)
    out = inside + (q * torch.exp(g).float()[..., None]) @ states[:, :, :n]
    return out.reshape(b, h, n * CHUNK, dv)[:, :, :l].transpose(1, 2).to(s["q"].dtype), states[:, :, n]


def _linear_step(s):
    if own:
        from lact_amd import decayed_linear_attention_step
        return decayed_linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], state_out=s["state_out"])
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    decay = torch.exp(s["log_decay"])
    new = torch.add(decay[..., None, None] * s["state"], k[..., :, None] * v[..., None, :], out=s["state_out"])
    out = (q[..., None, :] @ new)[..., 0, :] * q.shape[-1] ** -0.5
    return out.to(s["q"].dtype), new


# ---- what a pass cannot do without

def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["path"] == "attention":
        q, kv = (case["b"] * case["l"] * n * case["d"] * size for n in (case["hq"], _kv_heads(case)))
        pairs = _pairs(case) * case["hq"]
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * case["d"]}
        # forward, then q, k, v, the output and its gradient read and three gradients written
        return {"bytes": (2 * q + 2 * kv) + (4 * q + 4 * kv), "flops": 14 * pairs * case["d"]}
    if case["path"] == "attention_step":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        return {"bytes": 2 * seen * _kv_heads(case) * case["d"] * size + 2 * case["b"] * case["hq"] * case["d"] * size,
                "flops": 4 * seen * case["hq"] * case["d"]}
    b, h, dk, dv = (case[n] for n in ("b", "h", "dk", "dv"))
    if case["path"] == "linear_step":
        return {"bytes": 8 * b * h * dk * dv + b * h * 2 * (dk + dv) * size, "flops": 5 * b * h * dk * dv}
    tokens = b * case["l"] * h
    states = 4 * b * h * dk * dv
    gates = 4 * (tokens if case["gated"] else h)
    # the recurrence: k v^T added to the decayed state, the state times q
    forward = {"bytes": 2 * tokens * (dk + dv) * size + gates + (2 if case["state"] else 1) * states, "flops": 4 * tokens * dk * dv}
    if not case["train"]:
        return forward
    return {"bytes": forward["bytes"] + tokens * (4 * dk + 3 * dv) * size + 2 * gates + (3 * states if case["state"] else 0), "flops": 3 * forward["flops"]}


# ---- the definitions in 64 bits, head by head

def _exact_attention(case, s):
    b, l, hq, d = s["q"].shape
    group = hq // s["k"].shape[2]
    dev = s["q"].device
    bounds, prefixes = _documents(case)
    if s["documents"] is None:
        bounds, prefixes = [[0, l]] * b, [[0]] * b
    outs = torch.zeros(b, l, hq, d, dtype=torch.float64, device=dev)
    grads = [torch.zeros(s[n].shape, dtype=torch.float64, device=dev) for n in ("q", "k", "v")]
    for i in range(b):
        for h in range(hq):
            for start, end, pre in zip(bounds[i], bounds[i][1:], prefixes[i]):
                if end <= start:
                    continue
                q, k, v = (s[n].detach()[i, start:end, x].double().requires_grad_(case["train"]) for n, x in (("q", h), ("k", h // group), ("v", h // group)))
                x = q @ k.T * (1 / math.sqrt(d))
                if case["cap"]:
                    x = torch.tanh(x * (1 / case["cap"])) * case["cap"]
                place = torch.arange(end - start, device=dev, dtype=torch.float64)
                far = place[:, None] - place[None, :]
                if case["slopes"]:
                    x = x - float(s["slopes"][h]) * far.abs()
                hidden = far < 0
                if case["prefix"]:
                    hidden &= place[None, :] >= pre
                if case["window"]:
                    hidden |= far >= case["window"]
                o = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
                outs[i, start:end, h] = o.detach()
                if case["train"]:
                    for acc, y, at in zip(grads, torch.autograd.grad(o, (q, k, v), s["grad"][i, start:end, h].double()), (h, h // group, h // group)):
                        acc[i, start:end, at] += y
    return [outs, *grads] if case["train"] else outs


def _exact_attention_step(case, s):
    b, hq, d = s["q"].shape
    group = hq // s["k"].shape[2]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(_lengths(case)):
        first = max(0, n - (case["window"] or n))
        if n == 0:
            continue
        back = torch.arange(n - 1 - first, -1, -1, device=out.device, dtype=torch.float64)
        for kv in range(s["k"].shape[2]):
            k, v = (s[x][i, first:n, kv].double() for x in ("k", "v"))
            x = s["q"][i, kv * group:(kv + 1) * group].double() @ k.T * (1 / math.sqrt(d))
            if case["cap"]:
                x = torch.tanh(x * (1 / case["cap"])) * case["cap"]
            if case["slopes"]:
                x = x - s["slopes"][kv * group:(kv + 1) * group, None].double() * back
            out[i, kv * group:(kv + 1) * group] = torch.softmax(x, -1) @ v
    return out


def _exact_linear(case, s):
    b, l, h, dk = s["q"].shape
    dv = s["v"].shape[-1]
    dev = s["q"].device
    out = torch.zeros(b, l, h, dv, dtype=torch.float64, device=dev)
    last = torch.zeros(b, h, dk, dv, dtype=torch.float64, device=dev)
    names = [n for n in ("q", "k", "v", "log_decay", "state") if s[n] is not None]
    grads = {n: torch.zeros(s[n].shape, dtype=torch.float64, device=dev) for n in names}
    later = torch.ones(l, l, dtype=torch.bool, device=dev).triu(1)
    for i in range(b):
        for j in range(h):
            at = {"q": (i, slice(None), j), "k": (i, slice(None), j), "v": (i, slice(None), j), "log_decay": (i, slice(None), j) if case["gated"] else (j,),
                  "state": (i, j)}
            x = {n: s[n].detach()[at[n]].double().requires_grad_(case["train"]) for n in names}
            run_ = (x["log_decay"] if case["gated"] else x["log_decay"].expand(l)).cumsum(0)
            w = torch.exp((run_[:, None] - run_[None, :]).masked_fill(later, -math.inf))
            o = (x["q"] @ x["k"].T * w) @ x["v"]
            z = (x["k"] * torch.exp(run_[-1] - run_)[:, None]).T @ x["v"]
            if "state" in x:
                o = o + torch.exp(run_)[:, None] * (x["q"] @ x["state"])
                z = z + torch.exp(run_[-1]) * x["state"]
            o = o * (1 / math.sqrt(dk))
            out[i, :, j], last[i, j] = o.detach(), z.detach()
            if case["train"]:
                ys, gs = ([o, z], [s["grad"][i, :, j].double(), s["state_grad"][i, j].double()]) if "state" in x else ([o], [s["grad"][i, :, j].double()])
                for n, y in zip(names, torch.autograd.grad(ys, [x[n] for n in names], gs)):
                    grads[n][at[n]] += y
    return [out, last, *(grads[n] for n in names)] if case["train"] else [out, last]


def _exact_linear_step(case, s):
    q, k, v, z = (s[n].double() for n in ("q", "k", "v", "state"))
    new = torch.exp(s["log_decay"].double())[..., None, None] * z + torch.einsum("bhk,bhv->bhkv", k, v)
    return [torch.einsum("bhk,bhkv->bhv", q, new) * (1 / math.sqrt(q.shape[-1])), new]


def exact(case, seed):
    if case["path"] == "attention" and case["b"] * case["hq"] * case["docs"] > 3000:
        return None                                                                       # half a minute of single documents
    s = prepare(case, seed)
    if case["path"] == "attention":
        return _exact_attention(case, s)
    with torch.set_grad_enabled(case["path"] == "linear"):
        return {"attention_step": _exact_attention_step, "linear": _exact_linear, "linear_step": _exact_linear_step}[case["path"]](case, s)
