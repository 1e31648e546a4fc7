"""decayed_linear_attention and its step (csrc/linear_attention.h) against the recurrence in float64, output, state and gradients."""
import pytest
import torch
import torch.nn.functional as F

from oracle import mixers_oracle as MO
from oracle.lact_oracle import rel_l2

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


def make(b, l, h, dk, dv, dtype, gates, state=True, seed=1):
    g = torch.Generator().manual_seed(seed)
    unit = lambda t: F.normalize(t, dim=-1)  # noqa: E731
    x = dict(q=unit(torch.randn(b, l, h, dk, generator=g)).to(dtype), k=unit(torch.randn(b, l, h, dk, generator=g)).to(dtype),
             v=torch.randn(b, l, h, dv, generator=g).to(dtype))
    if gates == "head":
        x["log_decay"] = -torch.rand(h, generator=g) * 0.2
    elif gates == "strong":
        x["log_decay"] = -torch.rand(b, l, h, generator=g) * 8.0
    elif gates == "none":
        x["log_decay"] = torch.zeros(h)
    else:
        x["log_decay"] = F.logsigmoid(torch.randn(b, l, h, generator=g) * 1.5 + 3.0)
    if state:
        x["state"] = torch.randn(b, h, dk, dv, generator=g)
    go = torch.randn(b, l, h, dv, generator=g).to(dtype)
    gs = torch.randn(b, h, dk, dv, generator=g) * 0.3
    return x, go, gs


def on_gpu(x):
    return {n: t.to("cuda").requires_grad_(True) for n, t in x.items()}


def check(b, l, h, dk, dv, dtype, gates, state=True, scale=None):
    """bf16: weights of pairs and, in the sums that only rounded results depend on, the state are rounded to bf16 (2^-8 at most, 2^-9.8 in the mean square), results
    once more: a relative 2-norm under 2^-8 * 1.5.  Everything in fp32, the states and the gradients of decays and state among it, comes from products
    of 24 bits: sums of up to 64 + dk + l / 64 terms with cancellation, 2^-24 * 200."""
    import lact_amd
    print("[gpu-test] linear attention", b, l, h, dk, dv, dtype, gates, state, flush=True)
    x, go, gs = make(b, l, h, dk, dv, dtype, gates, state)
    dev = on_gpu(x)
    st = dev.get("state")
    out, last = lact_amd.decayed_linear_attention(dev["q"], dev["k"], dev["v"], dev["log_decay"], state=st, scale=scale, return_state=True)
    grads = torch.autograd.grad([out, last], list(dev.values()), [go.to("cuda"), gs.to("cuda")])
    ref_in = {n: t.double().requires_grad_(True) for n, t in x.items()}
    ref, ref_last = MO.linear(ref_in["q"], ref_in["k"], ref_in["v"], ref_in["log_decay"], ref_in.get("state"), scale)
    ref_grads = torch.autograd.grad([ref, ref_last], list(ref_in.values()), [go.double(), gs.double()])
    for name, a, r in zip(["out", "last"] + ["d" + n for n in x], [out, last, *grads], [ref, ref_last, *ref_grads]):
        bound = 1.5 * 2.0 ** -8 if a.dtype == torch.bfloat16 else 200 * 2.0 ** -24
        e = rel_l2(a, r)
        print(f"[gpu-test]   {name}: {e:.2e}", flush=True)
        assert a.shape == r.shape and bool(torch.isfinite(a).all()) and e < bound, (name, e)


@BOTH
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_sizes(dk, dv, dtype):
    check(2, 150, 3, dk, dv, dtype, "token")


@BOTH
@pytest.mark.parametrize("l", [1, 2, 63, 64, 65, 127, 129, 700])
def test_lengths(l, dtype):
    check(1, l, 2, 64, 64, dtype, "token")


@BOTH
@pytest.mark.parametrize("gates", ["head", "strong", "none"])
def test_decays(gates, dtype):
    check(2, 200, 2, 64, 128, dtype, gates)
    check(1, 130, 2, 128, 64, dtype, gates, state=False)


@BOTH
def test_many_heads_walk_alone(dtype):
    """As many heads as compute units: a block walks the whole sequence."""
    check(16, 140, 16, 64, 64, dtype, "token", scale=1.0)


@BOTH
def test_without_the_last_state(dtype):
    import lact_amd
    x, go, _ = make(2, 210, 3, 64, 64, dtype, "head", state=False)
    dev = on_gpu(x)
    out = lact_amd.decayed_linear_attention(dev["q"], dev["k"], dev["v"], dev["log_decay"])
    grads = torch.autograd.grad(out, list(dev.values()), go.to("cuda"))
    ref_in = {n: t.double().requires_grad_(True) for n, t in x.items()}
    ref, _ = MO.linear(*ref_in.values())
    for a, r in zip([out, *grads], [ref, *torch.autograd.grad(ref, list(ref_in.values()), go.double())]):
        assert rel_l2(a, r) < (1.5 * 2.0 ** -8 if a.dtype == torch.bfloat16 else 200 * 2.0 ** -24)


@BOTH
def test_forgetting_everything_is_a_new_document(dtype):
    """A log decay of -infinity at a token gives what a sequence that begins there gives."""
    import lact_amd
    b, l, h, d, cuts = 1, 300, 2, 64, [0, 37, 64, 65, 200]
    x, go, _ = make(b, l, h, d, d, dtype, "token", state=False)
    for c in cuts:
        x["log_decay"][:, c] = -float("inf")
    dev = on_gpu(x)
    out, last = lact_amd.decayed_linear_attention(**{n: dev[n] for n in ("q", "k", "v", "log_decay")}, state=torch.randn(b, h, d, d, device="cuda"), return_state=True)
    grads = torch.autograd.grad(out, list(dev.values()), go.to("cuda"))
    tol = 2.0 ** -7 if dtype == torch.bfloat16 else 200 * 2.0 ** -24
    for s, e in zip(cuts, cuts[1:] + [l]):
        part = {n: t[:, s:e].clone() for n, t in x.items()}
        part["log_decay"][:, 0] = 0.0
        part = {n: t.double().requires_grad_(True) for n, t in part.items()}
        ref, ref_last = MO.linear(*part.values())
        assert rel_l2(out[:, s:e], ref) < tol
        for n, a, r in zip(x, grads, torch.autograd.grad(ref, list(part.values()), go[:, s:e].double())):
            if n != "log_decay":
                assert rel_l2(a[:, s:e], r) < tol, n
    assert rel_l2(last, ref_last) < 200 * 2.0 ** -24
    dg = grads[-1]
    assert bool(torch.isfinite(dg).all()) and not dg[:, cuts].any()


@BOTH
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_later_tokens_reach_nothing(value, dtype):
    import lact_amd
    b, l, h, d, at = 1, 200, 2, 64, 100
    x, _, _ = make(b, l, h, d, d, dtype, "token")
    dev = {n: t.to("cuda") for n, t in x.items()}
    ref = lact_amd.decayed_linear_attention(**dev)
    for n in ("q", "k", "v"):
        spoilt = dict(dev)
        spoilt[n] = dev[n].clone()
        spoilt[n][0, at, 0, 5] = value
        out = lact_amd.decayed_linear_attention(**spoilt)
        # a chunk whose values are not all finite is summed in another order
        assert rel_l2(out[:, :at], ref[:, :at]) < (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20) and torch.equal(out[:, :, 1], ref[:, :, 1]), n
        assert not bool(torch.isfinite(out[0, at, 0]).all()), n


def test_views_and_broadcast_decays():
    import lact_amd
    x, go, _ = make(2, 100, 3, 64, 64, torch.bfloat16, "token", state=False)
    q, k, v, g = (x[n].to("cuda") for n in ("q", "k", "v", "log_decay"))
    ref = lact_amd.decayed_linear_attention(q, k, v, g)
    packed = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    views = [t.reshape(2, 100, 3, 64) for t in packed.split(192, -1)]
    assert torch.equal(lact_amd.decayed_linear_attention(*views, g), ref)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(lact_amd.decayed_linear_attention(*turned, g.transpose(0, 1).contiguous().transpose(0, 1)), ref)
    # one gate for all heads: its gradient is the sum over them
    shared = g[:, :, :1].clone().requires_grad_(True)
    out = lact_amd.decayed_linear_attention(q, k, v, shared.expand(2, 100, 3))
    got, = torch.autograd.grad(out, shared, go.to("cuda"))
    ref_in = x["log_decay"][:, :, :1].double().requires_grad_(True)
    r, = torch.autograd.grad(MO.linear(x["q"], x["k"], x["v"], ref_in.expand(2, 100, 3))[0], ref_in, go.double())
    assert rel_l2(got, r) < 200 * 2.0 ** -24


def test_empty_sequences_keep_the_state():
    import lact_amd
    s = torch.randn(2, 3, 64, 128, device="cuda")
    q, k = (torch.empty(2, 0, 3, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    out, last = lact_amd.decayed_linear_attention(q, k, torch.empty(2, 0, 3, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(3, device="cuda"), state=s, return_state=True)
    assert out.shape == (2, 0, 3, 128) and torch.equal(last, s)


def test_gradient_against_differences():
    import lact_amd
    x, go, gs = make(1, 90, 2, 64, 64, torch.float32, "token", seed=4)
    dev = on_gpu(x)
    f = lambda d: lact_amd.decayed_linear_attention(**d, return_state=True)  # noqa: E731
    value = lambda r: (r[0].double() * go.double().to("cuda")).sum() + (r[1].double() * gs.double().to("cuda")).sum()  # noqa: E731
    grads = dict(zip(dev, torch.autograd.grad(f(dev), list(dev.values()), [go.to("cuda"), gs.to("cuda")])))
    g = torch.Generator().manual_seed(6)
    for n in dev:
        step = torch.randn(x[n].shape, generator=g).to("cuda")
        h = 2.0 ** -8
        up, down = ({m: (t.detach() + s * h * step if m == n else t.detach()) for m, t in dev.items()} for s in (1, -1))
        diff, exact = (value(f(up)) - value(f(down))) / (2 * h), (grads[n].double() * step.double()).sum()
        scale = (grads[n].double() * step.double()).abs().sum()
        # second order in h for the decays, which meet along a path; fp32 outputs over 2 h for the others
        assert abs(diff - exact) < 2e-3 * scale, (n, float(diff), float(exact))


def test_captured_training_step():
    import lact_amd
    x, go, gs = make(2, 300, 2, 64, 128, torch.bfloat16, "token")
    static = {n: t.to("cuda") for n, t in x.items()}
    go, gs = go.to("cuda"), gs.to("cuda")

    def step(x):
        leaves = {n: t.detach().requires_grad_(True) for n, t in x.items()}
        res = lact_amd.decayed_linear_attention(**leaves, return_state=True)
        return [t.detach() for t in res] + list(torch.autograd.grad(res, list(leaves.values()), [go, gs]))

    step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(static)
    for i in range(3):
        fresh, _, _ = make(2, 300, 2, 64, 128, torch.bfloat16, "token", seed=20 + i)
        fresh = {n: t.to("cuda") for n, t in fresh.items()}
        for n in static:
            static[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(res, step(fresh)):
            assert torch.equal(a, r), i


def test_capture_refuses_leaves_that_an_eager_graph_holds():
    import lact_amd
    x, go, _ = make(1, 100, 2, 64, 64, torch.bfloat16, "token", state=False)
    leaves = {n: t.to("cuda").requires_grad_(n == "log_decay") for n, t in x.items() if t is not None}
    out = lact_amd.decayed_linear_attention(**leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"), torch.cuda.graph(graph):
        lact_amd.decayed_linear_attention(**leaves)
    assert torch.equal(out, lact_amd.decayed_linear_attention(**leaves))


@BOTH
@pytest.mark.parametrize("l", [1, 130])
def test_nothing_in_front_has_no_gradient_of_its_decay(l, dtype):
    """Without a state in front, the first token's decay has nothing to act on."""
    import lact_amd
    x, go, gs = make(2, l, 2, 64, 128, dtype, "token", state=False)
    x = {n: t.to("cuda").requires_grad_(True) for n, t in x.items() if t is not None}
    res = lact_amd.decayed_linear_attention(**x, return_state=True)
    dg, = torch.autograd.grad(res, x["log_decay"], [go.to("cuda"), torch.randn(2, 2, 64, 128, device="cuda")])
    assert not dg[:, 0].any() and (l == 1 or bool(dg[:, 1:].all()))


def test_empty_sequences_keep_every_operand_in_the_graph():
    import lact_amd
    q = torch.zeros(2, 0, 3, 64, device="cuda", requires_grad=True)
    g, s = torch.zeros(3, device="cuda", requires_grad=True), torch.randn(2, 3, 64, 64, device="cuda", requires_grad=True)
    out, last = lact_amd.decayed_linear_attention(q, q, q, g, state=s, return_state=True)
    assert out.shape == (2, 0, 3, 64) and torch.equal(last, s)
    dq, dg, ds = torch.autograd.grad((out, last), (q, g, s), (torch.zeros_like(out), torch.ones_like(last)))
    assert dq.shape == q.shape and not dg.any() and bool((ds == 1).all())


# ---- single tokens

@BOTH
@pytest.mark.parametrize("b,h,dk,dv,gates", [(1, 1, 64, 64, "head"), (3, 5, 64, 128, "token"), (2, 3, 128, 64, "token"), (4, 2, 128, 128, "head")])
def test_step(b, h, dk, dv, gates, dtype):
    import lact_amd
    print("[gpu-test] linear attention step", b, h, dk, dv, gates, dtype, flush=True)
    x, _, _ = make(b, 1, h, dk, dv, dtype, gates)
    ref, ref_last = MO.linear(**x)
    one = {n: (t[:, 0] if n in ("q", "k", "v") or t.dim() == 3 else t).to("cuda") for n, t in x.items()}
    kept = one["state"].clone()
    out, last = lact_amd.decayed_linear_attention_step(**one)
    tol = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -19      # the output rounded once; sums of dk terms
    assert out.dtype == dtype and rel_l2(out, ref[:, 0]) < tol and rel_l2(last, ref_last) < 2.0 ** -21 and torch.equal(one["state"], kept)
    into = torch.empty_like(kept)
    out2, last2 = lact_amd.decayed_linear_attention_step(**one, state_out=into)
    assert last2 is into or last2.data_ptr() == into.data_ptr()
    out3, last3 = lact_amd.decayed_linear_attention_step(**one, state_out=one["state"])      # in place
    assert torch.equal(out, out2) and torch.equal(out, out3) and torch.equal(last, into) and torch.equal(one["state"], last)


def test_step_forgets_and_lets_views_in():
    import lact_amd
    x, _, _ = make(2, 1, 3, 64, 64, torch.float32, "token")
    one = {n: (t[:, 0] if n != "state" else t).to("cuda") for n, t in x.items()}
    one["log_decay"][0] = -float("inf")
    out, last = lact_amd.decayed_linear_attention_step(**one)
    assert torch.equal(last[0], one["k"][0, :, :, None] * one["v"][0, :, None, :])
    turned = {n: t.transpose(0, 1).contiguous().transpose(0, 1) for n, t in one.items()}
    out2, last2 = lact_amd.decayed_linear_attention_step(**turned)
    assert torch.equal(out, out2) and torch.equal(last, last2)


def test_prompt_and_tokens_agree():
    """A prompt, then token after token in place, is the attention over all of it; beside it the softmax attention does the same: a layer of both."""
    import lact_amd
    b, l, h, d, prompt, window = 2, 150, 4, 64, 130, 40
    x, _, _ = make(b, l, h, d, d, torch.float32, "token", state=False)
    q, k, v, g = (x[n].to("cuda") for n in ("q", "k", "v", "log_decay"))
    both = lambda q, k, v, g: lact_amd.decayed_linear_attention(q, k, v, g) + lact_amd.masked_window_attention(q, k, v, window)  # noqa: E731
    whole = both(q, k, v, g)
    head = [t[:, :prompt] for t in (q, k, v, g)]
    first, state = lact_amd.decayed_linear_attention(*head, return_state=True)
    outs = [first + lact_amd.masked_window_attention(*head[:3], window)]
    kc, vc = (torch.zeros(b, l, h, d, device="cuda") for _ in range(2))
    kc[:, :prompt], vc[:, :prompt] = k[:, :prompt], v[:, :prompt]
    for t in range(prompt, l):
        kc[:, t], vc[:, t] = k[:, t], v[:, t]
        a, state = lact_amd.decayed_linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], state, state_out=state)
        outs.append((a + lact_amd.window_attention_step(q[:, t], kc, vc, torch.full((b,), t + 1, device="cuda"), window))[:, None])
    assert rel_l2(torch.cat(outs, 1), whole) < 200 * 2.0 ** -24


def test_captured_steps_in_place():
    import lact_amd
    x, _, _ = make(3, 1, 4, 128, 128, torch.bfloat16, "token")
    one = {n: (t[:, 0] if n != "state" else t).to("cuda") for n, t in x.items()}
    eager = one["state"].clone()
    lact_amd.decayed_linear_attention_step(**one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = lact_amd.decayed_linear_attention_step(**one, state_out=one["state"])
    one["state"].copy_(eager)
    for i in range(4):
        one["v"].copy_(torch.randn_like(one["v"].float()))
        ref, eager = lact_amd.decayed_linear_attention_step(**{**one, "state": eager})
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(one["state"], eager), i


def test_refusals_on_the_gpu():
    import lact_amd
    f = lact_amd.decayed_linear_attention
    q = torch.zeros(1, 8, 2, 64, device="cuda", dtype=torch.bfloat16)
    g = torch.zeros(2, device="cuda")
    for bad, error in ((dict(k=q.float()), TypeError), (dict(v=q[:, :7]), ValueError), (dict(k=torch.cat([q, q], -1)), ValueError), (dict(log_decay=torch.zeros(3, device="cuda")), ValueError),
                       (dict(log_decay=torch.zeros(1, 8, 1, device="cuda")), ValueError), (dict(log_decay=g.cpu()), RuntimeError),
                       (dict(state=torch.zeros(1, 2, 64, 128, device="cuda")), ValueError)):
        with pytest.raises(error):
            f(**{**dict(q=q, k=q, v=q, log_decay=g), **bad})
    with pytest.raises(TypeError):
        f(q.half(), q.half(), q.half(), g)
    wide = torch.zeros(1, 8, 2, 96, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="64 or 128"):
        f(wide, wide, q, g)
    step = lact_amd.decayed_linear_attention_step
    one, s = q[:, 0], torch.zeros(2, 2, 64, 64, device="cuda")
    with pytest.raises(RuntimeError):                 # overlapping, but not the same
        step(one, one, one, g, s.view(-1)[:8192].view(1, 2, 64, 64), state_out=s.view(-1)[4096:12288].view(1, 2, 64, 64))
    with pytest.raises(TypeError):
        step(one, one, one, g, s[:1], state_out=s[1:].bfloat16())
    with pytest.raises(ValueError):
        step(one, one, one, g, s[:1], state_out=s[1:].transpose(2, 3))
    leaf = q.clone().requires_grad_(True)
    first, = torch.autograd.grad(f(leaf, q, q, g).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), leaf)


def test_steps_in_place_are_seen_by_autograd():
    """The states that a sequence call keeps for its backward, stepped in place in front of it: the backward refuses, as behind any operation in place."""
    import lact_amd
    x, go, gs = make(1, 100, 2, 64, 64, torch.bfloat16, "token")
    go, gs = go.to("cuda"), gs.to("cuda")
    dev = {n: t.to("cuda").requires_grad_(n != "state") for n, t in x.items()}
    one = [dev[n].detach()[:, 0] for n in ("q", "k", "v", "log_decay")]
    for which in ("last", "state", "neither"):
        out, last = lact_amd.decayed_linear_attention(**dev, return_state=True)
        before = last._version, dev["state"]._version
        with torch.no_grad():
            target = {"last": last, "state": dev["state"], "neither": torch.empty_like(last)}[which]
            _, new = lact_amd.decayed_linear_attention_step(*one, target if which != "neither" else last, state_out=target)
        assert new is target or new.data_ptr() == target.data_ptr()
        assert (last._version > before[0], dev["state"]._version > before[1]) == (which == "last", which == "state")
        if which == "neither":
            torch.autograd.grad([out, last], dev["q"], [go, gs])
        else:
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad([out, last], dev["q"], [go, gs])
    with torch.inference_mode():
        state = torch.zeros(1, 2, 64, 64, device="cuda")
        lact_amd.decayed_linear_attention_step(*one, state, state_out=state)
    with torch.no_grad():      # a state made for inference, which no graph can keep
        lact_amd.decayed_linear_attention_step(*one, state, state_out=state)
    leaf = torch.zeros(1, 2, 64, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="inference"):
        lact_amd.decayed_linear_attention_step(*one, state.clone(), state_out=leaf)
    with torch.no_grad():
        lact_amd.decayed_linear_attention_step(*one, state.clone(), state_out=leaf)
    assert leaf.any()


@BOTH
@pytest.mark.parametrize("gates", ["token", "head"])
@pytest.mark.parametrize("b,l,h,d", [(2, 1100, 130, 64), (2, 1100, 130, 128), (1, 3000, 100, 64)])
def test_long_walks(b, l, h, d, gates, dtype):
    """260 heads: more than segments are made for, so that a block walks all 18 chunks of its head; 100 heads: five segments of ten chunks, seven in the last.  The decays'
    gradient is carried over eight chunks at a time.  Some of the heads, which do not depend on each other, are compared."""
    import lact_amd
    print("[gpu-test] linear attention, long walks", b, l, h, d, gates, dtype, flush=True)
    some = [0, h // 2 - 1, h - 1]
    x, go, gs = make(b, l, h, d, d, dtype, gates)
    dev = on_gpu(x)
    out, last = lact_amd.decayed_linear_attention(dev["q"], dev["k"], dev["v"], dev["log_decay"], state=dev["state"], return_state=True)
    grads = torch.autograd.grad([out, last], list(dev.values()), [go.to("cuda"), gs.to("cuda")])
    at = {"state": 1, "log_decay": x["log_decay"].dim() - 1}
    part = lambda t, n: t.index_select(at.get(n, 2), torch.tensor(some, device=t.device))  # noqa: E731
    ref_in = {n: part(t, n).double().requires_grad_(True) for n, t in x.items()}
    ref, ref_last = MO.linear(*ref_in.values())
    ref_grads = torch.autograd.grad([ref, ref_last], list(ref_in.values()), [part(go, "q").double(), part(gs, "state").double()])
    for name, a, r in zip(["q", "state"] + list(x), [out, last, *grads], [ref, ref_last, *ref_grads]):
        bound = 1.5 * 2.0 ** -8 if a.dtype == torch.bfloat16 else 200 * 2.0 ** -24      # as in check()
        e = rel_l2(part(a, name), r)
        print(f"[gpu-test]   {name}: {e:.2e}", flush=True)
        assert bool(torch.isfinite(a).all()) and e < bound, (name, e)
