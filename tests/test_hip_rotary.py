"""axial_rotary (csrc/rotary.h) against its definition in float64, forwards and backwards: one to three axes, pairs side by side and in halves, channels without a position, sizes and
strides that vectors do not fit."""
import math

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
BOTH = pytest.mark.parametrize("dtype", [BF16, F32])
PAIRS = pytest.mark.parametrize("interleaved", [True, False])


def turn_error():
    """Of a cosine or a sine.  The rest of an angle is at most half a quarter turn: rounded to fp32 (2^-25 quarters for numbers up to 1/2), times pi / 2, which is rounded, and the product
    as well: pi / 2 * 2^-25 + pi / 4 * 2 * 2^-24 of the angle, whose sine and cosine move by no more; five steps of their series, each off by 2^-24 of what it adds to at most 1, and the
    terms left out, 2e-9."""
    return (math.pi / 4 + math.pi / 2 + 5) * 2.0 ** -24 + 2e-9


def bound(x, angle, interleaved, dtype):
    """Of each output: the turn's error times the pair's magnitudes, three roundings of products and their sum, and what is stored."""
    n = angle.shape[-1]
    x = x.double().abs()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    e = (a + b) * (turn_error() + 3 * 2.0 ** -24)
    e = torch.stack((e, e), -1).flatten(-2) if interleaved else torch.cat((e, e), -1)
    return torch.cat((e, torch.zeros_like(x[..., 2 * n:])), -1)


def near(got, ref, e, dtype, name):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), name
    worst = ((got - ref).abs() / (e + (ref.abs() + e) * HALF[dtype] + 1e-40)).max() if got.numel() else 0.0
    print(f"[gpu-test]   {name}: {float(worst):.3f} of the bound", flush=True)
    assert worst <= 1.0, (name, float(worst))


def check(q, k, positions, axes, interleaved, dtype, dev=lambda t: t.to("cuda"), **kw):
    import lact_amd
    print("[gpu-test] rotary", tuple(q.shape), None if k is None else tuple(k.shape), tuple(positions.shape), axes, interleaved, dtype, flush=True)
    angle = PO.angles(positions, axes, **kw)
    if q.dim() == 4 and positions.dim() == 2:
        angle = angle[None]
    xs = [t for t in (q, k) if t is not None]
    on = [dev(t).requires_grad_(True) for t in xs]
    out = lact_amd.axial_rotary(on[0], on[1] if k is not None else None, positions.to("cuda"), axes, interleaved=interleaved, **kw)
    assert (out[1] is None) == (k is None)
    out = [t for t in out if t is not None]
    g = [torch.randn(t.shape, generator=torch.Generator().manual_seed(8 + i)).to(dtype) for i, t in enumerate(xs)]
    grads = torch.autograd.grad(out, on, [t.to("cuda") for t in g])
    for name, x, y, go, gx in zip("qk", xs, out, g, grads):
        assert y.dtype == gx.dtype == dtype and y.is_contiguous()
        near(y, PO.rotary(x, angle, interleaved), bound(x, angle, interleaved, dtype), dtype, name)
        near(gx, PO.rotary(go, -angle, interleaved), bound(go, angle, interleaved, dtype), dtype, "d" + name)
        rest = 2 * angle.shape[-1]
        assert torch.equal(y[..., rest:].cpu(), x[..., rest:]) and torch.equal(gx[..., rest:].cpu(), go[..., rest:])
    return out, grads


def make(b, l, hq, hkv, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(b, l, hq, d, generator=g).to(dtype), torch.randn(b, l, hkv, d, generator=g).to(dtype)


def grid(*sizes):
    return torch.stack(torch.meshgrid(*(torch.arange(n, dtype=torch.int32) for n in sizes), indexing="ij"), -1).reshape(-1, len(sizes))


@BOTH
@PAIRS
@pytest.mark.parametrize("b,sizes,hq,hkv,d,axes", [
    (1, (1,), 1, 1, 64, (64,)), (2, (3, 4, 5), 4, 2, 128, (44, 42, 42)), (1, (2, 3, 7), 3, 3, 128, (64, 32, 32)), (2, (37,), 2, 1, 64, (32,)), (1, (9, 11), 5, 1, 64, (24, 24)),
    (3, (2, 2), 2, 2, 256, (128, 128)), (1, (300,), 40, 8, 128, (128,)),
    (2, (5, 3), 3, 1, 66, (34, 30)), (1, (4, 4, 4), 2, 1, 10, (2, 4, 2)), (2, (7,), 3, 2, 2, (2,)), (1, (6, 5), 2, 1, 96, (20, 22)), (1, (5,), 1, 1, 250, (6,))])
def test_turns(b, sizes, hq, hkv, d, axes, interleaved, dtype):
    check(*make(b, math.prod(sizes), hq, hkv, d, dtype), grid(*sizes), axes, interleaved, dtype)


@BOTH
@PAIRS
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_far_positions_of_every_type(kind, interleaved, dtype):
    """Positions to 2^24 (whole numbers of 64 bits beyond, fp32 between whole numbers), one for each sequence and token, negative ones too.  The oracle's own angles are off by
    2^-53 of themselves: 2^24 by 2e-9."""
    g = torch.Generator().manual_seed(3)
    b, l = 2, 40
    positions = torch.randint(-2 ** 24, 2 ** 24, (b, l, 2), generator=g)
    positions[0, :4, 0] = torch.tensor([2 ** 24, -2 ** 24, 0, 1])
    if kind == torch.float32:
        positions = positions / 64
    check(*make(b, l, 3, 2, 64, dtype), positions.to(kind), (40, 24), interleaved, dtype)


@BOTH
@PAIRS
def test_frequencies_and_bases(interleaved, dtype):
    q, k = make(2, 21, 3, 1, 64, dtype)
    check(q, k, grid(3, 7), (32, 16), interleaved, dtype, base=500000.0)
    check(q, k, grid(3, 7), (32, 16), interleaved, dtype, frequencies=[0.0, 3.5, -1.25] * 8)
    check(q, k, grid(3, 7), (32, 16), interleaved, dtype, base=1.0)


@BOTH
@PAIRS
def test_one_token_each(interleaved, dtype):
    import lact_amd
    q, k = make(5, 1, 6, 2, 128, dtype)
    positions = torch.randint(0, 5000, (5, 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    out, _ = check(q[:, 0], k[:, 0], positions, (64, 32, 32), interleaved, dtype)
    many = lact_amd.axial_rotary(q.to("cuda"), k.to("cuda"), positions[:, None].to("cuda"), (64, 32, 32), interleaved=interleaved)
    assert all(torch.equal(a, m[:, 0]) for a, m in zip(out, many))


@BOTH
@PAIRS
def test_queries_alone_and_gradients_of_one(interleaved, dtype):
    import lact_amd
    q, k = make(2, 12, 3, 2, 64, dtype)
    check(q, None, grid(3, 4), (32, 32), interleaved, dtype)
    x, y = q.to("cuda").requires_grad_(True), k.to("cuda").requires_grad_(True)
    p = grid(3, 4).to("cuda")
    a, b = lact_amd.axial_rotary(x, y, p, (32, 32), interleaved=interleaved)
    whole = torch.autograd.grad([a, b], [x, y], [a.detach(), b.detach()], retain_graph=True)
    assert torch.equal(torch.autograd.grad(b, y, b.detach(), retain_graph=True)[0], whole[1])
    assert torch.equal(torch.autograd.grad(a, x, a.detach(), retain_graph=True)[0], whole[0])
    got = torch.autograd.grad(a, [x, y], a.detach(), allow_unused=True)
    assert torch.equal(got[0], whole[0]) and got[1] is None
    z = q.to("cuda").requires_grad_(True)
    a, b = lact_amd.axial_rotary(z, y.detach(), p, (32, 32), interleaved=interleaved)
    assert torch.equal(torch.autograd.grad([a, b], z, [a.detach(), b.detach()])[0], whole[0])


@BOTH
@PAIRS
def test_views_strides_and_broadcast(interleaved, dtype):
    """Parts of a packed projection, heads in front of tokens, off the alignment of vectors, every other channel, shared over the batch; gradients that are one number everywhere."""
    import lact_amd
    b, l, d, axes = 2, 15, 64, (32, 16)
    p = grid(3, 5)
    q, k = make(b, l, 3, 2, d, dtype)

    def packed(t):
        room = torch.zeros(b, l, t.shape[2] * d + 8, dtype=dtype, device="cuda")
        room[..., 8:] = t.flatten(2).to("cuda")
        return room[..., 8:].unflatten(2, (-1, d)).detach()

    def unaligned(t):
        room = torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")
        room[1:] = t.flatten().to("cuda")
        return room[1:].view(t.shape).detach()

    def apart(t):
        return torch.stack((t, t), -1).to("cuda")[..., 0].detach()

    plain, _ = check(q, k, p, axes, interleaved, dtype)
    for dev in (packed, unaligned, apart, lambda t: t.to("cuda").transpose(1, 2).contiguous().transpose(1, 2).detach()):
        got, _ = check(q, k, p, axes, interleaved, dtype, dev)
        assert all(torch.equal(a, r) for a, r in zip(got, plain))
    one = q[:1].to("cuda").requires_grad_(True)
    out, _ = lact_amd.axial_rotary(one.expand(b, l, 3, d), None, p.to("cuda"), axes, interleaved=interleaved)
    wide = torch.autograd.grad(out.sum(), one)[0]                   # (a gradient with strides of 0, to an input with one)
    each = q[:1].to("cuda").requires_grad_(True)
    out, _ = lact_amd.axial_rotary(each, None, p.to("cuda"), axes, interleaved=interleaved)
    ref = torch.autograd.grad(out, each, torch.ones_like(out))[0]
    assert torch.equal(wide, ref + ref)


@PAIRS
def test_gradient_against_differences(interleaved):
    """The operation is linear: the difference of two outputs is the output of the difference, and <g, f(x)> = <f'(g), x>."""
    import lact_amd
    q, k = make(1, 20, 2, 1, 64, F32)
    p, axes = grid(4, 5).to("cuda"), (32, 24)
    x = q.to("cuda").requires_grad_(True)
    f = lambda t: lact_amd.axial_rotary(t, None, p, axes, interleaved=interleaved)[0]  # noqa: E731
    g = torch.randn_like(x)
    grad, = torch.autograd.grad(f(x), x, g)
    step = torch.randn_like(x)
    with torch.no_grad():
        there = ((f(x + step / 16).double() - f(x - step / 16).double()) * 8 * g.double()).sum()
    along = (grad.double() * step.double()).sum()
    # every output is off by at most 12 2^-24 of its pair's magnitudes (|x| + |step| / 16 < 6), eightfold, at random signs among 2560
    assert abs(float(there - along)) < 8 * 2 * 12 * 2.0 ** -24 * 12 * 2560 ** 0.5 * 6, (float(there), float(along))


@BOTH
@PAIRS
def test_what_is_not_finite_stays_in_its_pair(interleaved, dtype):
    import lact_amd
    q, _ = make(1, 6, 2, 1, 64, dtype)
    p = grid(6)
    ref = lact_amd.axial_rotary(q.to("cuda"), None, p.to("cuda"), (48,), interleaved=interleaved)[0]
    for at in (5, 30, 48, 63):
        x = q.clone()
        x[0, 4, 1, at] = math.inf
        out = lact_amd.axial_rotary(x.to("cuda"), None, p.to("cuda"), (48,), interleaved=interleaved)[0]
        pair = {at} if at >= 48 else {at, at ^ 1} if interleaved else {at, (at + 24) % 48}
        changed = {int(i) for i in (out != ref).nonzero()[:, 3]}
        assert changed == pair and bool((~torch.isfinite(out[0, 4, 1, sorted(pair)])).all())
    assert float(out[0, 4, 1, 63]) == math.inf


@BOTH
def test_captured_training_step(dtype):
    """Forward and backward, captured once and replayed, eager calls in between."""
    import lact_amd
    q, k = (t.to("cuda") for t in make(2, 24, 4, 2, 128, dtype))
    p = grid(2, 3, 4).to("cuda")
    g = [torch.randn_like(t.float()).to(dtype) for t in (q, k)]

    def step():
        x, y = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        out = lact_amd.axial_rotary(x, y, p, (64, 32, 32))
        return [*(t.detach() for t in out), *torch.autograd.grad(out, [x, y], g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for t in (q, k, *g):
            t.copy_(torch.randn_like(t.float()))
        p += 5
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r) for a, r in zip(out, step())), i


def test_capture_refuses_leaves_that_an_eager_graph_holds():
    import lact_amd
    q = torch.randn(1, 8, 2, 64, device="cuda", requires_grad=True)
    p = grid(8).to("cuda")
    kept = lact_amd.axial_rotary(q, None, p, (64,))[0]      # lives on
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured call"):
            lact_amd.axial_rotary(q, None, p, (64,))
        out = lact_amd.axial_rotary(q.detach(), None, p, (64,))[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, kept)


def test_many_heads_and_tokens():
    """Blocks with several heads each, queries and keys in one."""
    import lact_amd
    q, k = (torch.randn(2, 3000, h, 128, device="cuda", dtype=BF16) for h in (24, 5))
    p = grid(10, 15, 20).to("cuda")
    for interleaved in (True, False):
        a, b = lact_amd.axial_rotary(q, k, p, (44, 42, 42), interleaved=interleaved)
        for t in (0, 1499, 2999):
            c, d = lact_amd.axial_rotary(q[:, t], k[:, t], p[t].expand(2, 3), (44, 42, 42), interleaved=interleaved)
            assert torch.equal(a[:, t], c) and torch.equal(b[:, t], d)


def test_autocast_empty_calls_and_refusals():
    import lact_amd
    f = lact_amd.axial_rotary
    q, k = (t.to("cuda") for t in make(2, 6, 4, 2, 64, F32))
    p = grid(2, 3).to("cuda")
    with torch.autocast("cuda", BF16):
        out = f(q, k, p, (32, 32))
    assert all(torch.equal(a, b) for a, b in zip(out, f(q.bfloat16(), k.bfloat16(), p, (32, 32))))
    assert f(q[:, :0], k[:, :0], p[:0], (32, 32))[0].shape == (2, 0, 4, 64) and f(q[:0], None, p, (32, 32))[1] is None
    for bad, error in ((dict(k=k.bfloat16()), TypeError), (dict(q=q.half(), k=k.half()), TypeError), (dict(k=k[:, :5]), ValueError), (dict(k=k.cpu()), RuntimeError),
                       (dict(positions=p[:5]), ValueError), (dict(positions=p[None]), ValueError), (dict(positions=p[:, :1]), ValueError), (dict(positions=p.cpu()), RuntimeError),
                       (dict(positions=p.double()), TypeError), (dict(positions=p.bool()), TypeError), (dict(q=q[..., :63], k=k[..., :63], axes=(32, 30)), RuntimeError),
                       (dict(q=q.repeat(1, 1, 1, 5), k=k.repeat(1, 1, 1, 5)), RuntimeError)):
        with pytest.raises(error):
            f(**{**dict(q=q, k=k, positions=p, axes=(32, 32)), **bad})
    x = q.clone().requires_grad_(True)
    y = f(x, None, p, (32, 32))[0]
    first, = torch.autograd.grad(y, x, y, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


@pytest.mark.parametrize("shape", [(0, 6), (2, 0), (0, 0), (0,)])
def test_calls_without_tokens_are_checked(shape):
    """What other calls refuse is refused where there is nothing to turn as well; keys of another batch among it, which would come back as they are."""
    import lact_amd
    f = lact_amd.axial_rotary
    q, k = (torch.zeros(*shape, h, 64, device="cuda", dtype=BF16, requires_grad=True) for h in (4, 2))
    p = torch.zeros(*shape, 2, dtype=torch.int32, device="cuda")
    a, b = f(q, k, p, (32, 32))
    assert a.shape == q.shape and b.shape == k.shape and a.dtype == b.dtype == BF16
    assert all(g.shape == t.shape for g, t in zip(torch.autograd.grad([a, b], [q, k], [a, b]), (q, k)))
    assert f(q, None, p, (32, 32))[1] is None
    more = torch.ones(*(n + 3 for n in shape), 2, 64, device="cuda", dtype=BF16)
    for bad, error in ((dict(k=more), ValueError), (dict(k=k.float()), TypeError), (dict(q=q.half(), k=k.half()), TypeError), (dict(k=k.cpu()), RuntimeError),
                       (dict(positions=p[..., :1]), ValueError), (dict(positions=p.double()), TypeError), (dict(positions=p.cpu()), RuntimeError), (dict(q=q.cpu(), k=k.cpu(), positions=p.cpu()), RuntimeError)):
        with pytest.raises(error):
            f(**{**dict(q=q, k=k, positions=p, axes=(32, 32)), **bad})
