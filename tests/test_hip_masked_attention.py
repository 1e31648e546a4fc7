"""masked_window_attention and window_attention_step (csrc/masked_attention.h, csrc/attention_step.h) against their definition in float64:
every mask, at the edges of the 32-row waves, 64-row tiles and 128 / 256-row blocks, output and gradients."""
import pytest
import torch

from oracle import mixers_oracle as MO

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def errors(dtype, l, d, size=8.0):
    """Relative errors of a probability and of a stored value.  bf16: probabilities are rounded for the product (2^-8), scores are summed in fp32.
    fp32: the sums of d and of l terms, and the exponential of a score of `size` off by the roundings of its d terms."""
    fp32 = (2 * d + l + 16 * size + 64) * 2.0 ** -24
    return (HALF[dtype] if dtype == torch.bfloat16 else 0.0) + fp32, HALF[dtype]


def near(got, ref, bound, name):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), name
    worst = ((got - ref).abs() / (bound + 1e-7)).max() if got.numel() else 0.0
    print(f"[gpu-test]   {name}: {float(worst):.3f} of the bound", flush=True)
    assert worst <= 1.0, (name, float(worst))


def make(b, l, hq, hkv, d, dtype, seed=3, growth=1.0):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(b, l, (hq + 2 * hkv) * d, generator=g)
    packed[..., hq * d:(hq + hkv) * d] *= torch.linspace(1.0, growth, max(l, 1))[None, :, None]
    go = torch.randn(b, l, hq, d, generator=g).to(dtype)
    return packed.to(dtype), go


def parts(packed, hq, hkv, d):
    b, l = packed.shape[:2]
    return [t.reshape(b, l, -1, d) for t in packed.split((hq * d, hkv * d, hkv * d), -1)]


def ints(rows, dtype=torch.int32):
    return None if rows is None else torch.tensor(rows, dtype=dtype)


def check(b, l, hq, hkv, d, dtype, window=None, cap=None, slopes=False, documents=None, prefixes=None, growth=1.0, scale=None):
    import lact_amd
    print("[gpu-test] masked attention", b, l, hq, hkv, d, dtype, window, cap, slopes, documents, prefixes, flush=True)
    packed, go = make(b, l, hq, hkv, d, dtype, growth=growth)
    sl = 2.0 ** -torch.arange(1, hq + 1).float() if slopes else None
    docs, pre = ints(documents), ints(prefixes)
    dev = lambda t: None if t is None else t.to("cuda")  # noqa: E731
    x = packed.to("cuda").requires_grad_(True)
    out = lact_amd.masked_window_attention(*parts(x, hq, hkv, d), window, score_cap=cap, distance_slopes=dev(sl), documents=dev(docs), prefixes=dev(pre), scale=scale)
    gx, = torch.autograd.grad(out, x, go.to("cuda"))
    p_err, out_err = errors(dtype, l, d, 8.0 * growth + (l if slopes else 0))
    ref, bound = MO.attention(*parts(packed, hq, hkv, d), window, cap, sl, docs, pre, scale, go, p_err, out_err)
    assert out.dtype == dtype
    for name, a, r, e in zip(("out", "dq", "dk", "dv"), [out, *parts(gx, hq, hkv, d)], ref, bound):
        near(a, r, e, name)
    seen = MO.visible(l, window, docs, pre).any(-1)
    for i in range(b):
        assert not out[i][~seen[i if len(seen) > 1 else 0].to("cuda")].any()
    return out, gx


BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@BOTH
@pytest.mark.parametrize("b,l,hq,hkv,d,window", [
    (1, 1, 1, 1, 64, None), (2, 5, 2, 1, 128, 2), (1, 64, 1, 1, 128, 64), (2, 129, 3, 3, 128, 33), (1, 257, 4, 2, 64, 65), (2, 333, 6, 2, 128, 200),
    (1, 300, 5, 5, 64, None), (1, 70, 2, 2, 64, 1)])
def test_causal_windows(b, l, hq, hkv, d, window, dtype):
    check(b, l, hq, hkv, d, dtype, window)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("documents,prefixes,window", [
    ([[0, 40, 41, 41, 150, 200]], None, None),                      # one token, none, and an edge inside a tile
    ([[3, 64, 128, 190]], None, 50),                                # padded on both sides, edges on tiles
    ([[0, 200]], [[200]], None),                                    # all of it a prefix: bidirectional
    ([[0, 90, 200]], [[0, 70]], 30),                                # a prefix wider than the window
    ([[0, 0, 0]], None, None),                                      # no token in any document
    ([[0, 1, 2, 3, 64, 65, 199, 200]], [[1, 0, 1, 61, 1, 2, 1]], 64),
    (None, [[33]], 70)])
def test_documents_and_prefixes(documents, prefixes, window, d, dtype):
    check(1, 200, 4, 2, d, dtype, window, documents=documents, prefixes=prefixes)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
def test_keys_gradients_in_splits(d, dtype):
    """Few key heads: the queries are walked in parts, which end inside heads and tiles."""
    check(1, 700, 8, 1, d, dtype, 300, 30.0, True, documents=[[3, 250, 690]], prefixes=[[50, 100]])


@BOTH
def test_documents_of_a_batch_differ(dtype):
    check(3, 150, 2, 1, 64, dtype, None, documents=[[0, 150, 150], [20, 30, 100], [0, 75, 150]], prefixes=[[10, 0], [10, 3], [0, 75]])


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,slopes,scale", [(20.0, False, None), (None, True, None), (2.0, True, 0.3)])
def test_capped_scores_and_distance(cap, slopes, scale, d, dtype):
    check(2, 170, 4, 4, d, dtype, 100, cap, slopes, documents=[[0, 60, 170], [5, 100, 165]], prefixes=[[20, 0], [0, 33]], scale=scale)


@pytest.mark.parametrize("b,l,hq,hkv,d,window", [(2, 1030, 26, 26, 128, 256), (1, 1100, 64, 64, 64, 300), (2, 520, 64, 16, 128, None)])
def test_many_blocks(b, l, hq, hkv, d, window):
    check(b, l, hq, hkv, d, torch.bfloat16, window, documents=[[0, 200, l - 3]] * b)


@BOTH
@pytest.mark.parametrize("cap,slopes", [(None, False), (25.0, False), (None, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_many_heads(d, cap, slopes, dtype):
    """More blocks of 128 queries than the compute units hold at once, of few tokens: a wave has its queries for itself."""
    check(2, 140, 160, 32, d, dtype, 90, cap, slopes, documents=[[0, 70, 70, 140], [3, 50, 100, 130]], prefixes=[[20, 0, 0], [0, 9, 30]])


@BOTH
@pytest.mark.parametrize("growth", [40.0, 300.0])
def test_scores_that_grow_along_the_sequence(growth, dtype):
    """The rows' maxima follow by far more than exp2 reaches."""
    check(1, 515, 3, 3, 128, dtype, 190, growth=growth)


@BOTH
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_what_is_masked_reaches_nothing(bad, dtype):
    """Padding and another document hold values that are not finite, or the type's lowest: the outputs and gradients of the rest are those without."""
    import lact_amd
    print("[gpu-test] masked attention, masked places hold", bad, dtype, flush=True)
    b, l, hq, hkv, d = 1, 230, 4, 2, 128
    value = torch.finfo(dtype).min if bad == "lowest" else bad
    docs = torch.tensor([[10, 100, 140, 200]], dtype=torch.int32, device="cuda")
    spoilt = torch.zeros(l, dtype=torch.bool)
    spoilt[:10] = spoilt[100:140] = spoilt[200:] = True
    packed, go = make(b, l, hq, hkv, d, dtype)
    results = []
    for spoil in (False, True):
        x, g = packed.clone(), go.clone()
        if spoil:
            x[:, spoilt], g[:, spoilt] = value, value
        x = x.to("cuda").requires_grad_(True)
        out = lact_amd.masked_window_attention(*parts(x, hq, hkv, d), None, score_cap=30.0, documents=docs, prefixes=torch.tensor([[30, 0, 0]], device="cuda"))
        gx, = torch.autograd.grad(out, x, g.to("cuda"))
        results.append((out.detach().cpu(), gx.cpu()))
    for clean, other in zip(*results):
        assert torch.equal(clean[:, ~spoilt], other[:, ~spoilt])
    alone = torch.zeros(l, dtype=torch.bool)
    alone[:10] = alone[200:] = True            # in no document
    assert not results[1][0][:, alone].any() and not results[1][1][:, alone].any()


@BOTH
def test_future_values_reach_nothing_and_seen_ones_do(dtype):
    import lact_amd
    b, l, h, d = 1, 100, 2, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(b, l, h, d, generator=g).to(dtype).to("cuda") for _ in range(3))
    ref = lact_amd.masked_window_attention(q, k, v)
    v2, k2 = v.clone(), k.clone()
    v2[0, 70, 0, 3] = float("nan")
    out = lact_amd.masked_window_attention(q, k2, v2)
    assert torch.equal(out[:, :70], ref[:, :70]) and torch.equal(out[:, :, 1], ref[:, :, 1])
    assert bool(torch.isnan(out[0, 70:, 0, 3]).all())
    k2[0, 70, 0, 3] = float("nan")
    out = lact_amd.masked_window_attention(q, k2, v)
    assert torch.equal(out[:, :70], ref[:, :70]) and bool(torch.isnan(out[0, 70:, 0]).all())


@BOTH
@pytest.mark.parametrize("cap", [None, 25.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (36, 36)])
def test_values_that_are_not_finite_in_every_tile(hq, hkv, d, cap, dtype):
    """One token of every 64: the tokens whose windows hold it are NaN, in all of its heads, and the others what they are without."""
    import lact_amd
    print("[gpu-test] masked attention, a NaN in every tile", hq, d, cap, dtype, flush=True)
    l, window = 1500, 9
    packed, go = make(1, l, hq, hkv, d, dtype)
    at = torch.arange(5, l, 61)
    hit = torch.zeros(l, dtype=torch.bool)
    for i in range(window):
        hit[(at + i).clamp(max=l - 1)] = True
    docs = torch.tensor([[0, l]], dtype=torch.int32, device="cuda")
    results = []
    for spoil in (False, True):
        x = packed.clone()
        if spoil:
            x[:, at, hq * d:] = float("nan")         # keys and values
        x = x.to("cuda").requires_grad_(True)
        out = lact_amd.masked_window_attention(*parts(x, hq, hkv, d), window, score_cap=cap, documents=docs)
        gx, = torch.autograd.grad(out, x, go.to("cuda"))
        results.append((out.detach().cpu(), gx.cpu()))
    (ref, gref), (out, gx) = results
    assert bool(torch.isnan(out[:, hit]).all()) and torch.equal(out[:, ~hit], ref[:, ~hit])
    q = slice(0, hq * d)
    assert bool(torch.isnan(gx[:, hit, q]).all()) and torch.equal(gx[:, ~hit, q], gref[:, ~hit, q])
    reached = torch.zeros(l, dtype=torch.bool)       # keys that a query with a NaN sees
    for i in range(window):
        reached[(torch.nonzero(hit)[:, 0] - i).clamp(min=0)] = True
    assert bool(torch.isnan(gx[:, reached, hq * d:]).all()) and torch.equal(gx[:, ~reached, hq * d:], gref[:, ~reached, hq * d:])


@BOTH
@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_a_single_key_has_no_gradient_of_scores(d, cap, slopes, dtype):
    """A window of one token, and documents of one: the softmax is constant, dq and dk are 0 and dv is the output's gradient."""
    import lact_amd
    print("[gpu-test] masked attention, one key", d, cap, slopes, dtype, flush=True)
    l, h = 200, 3
    packed, go = make(1, l, h, h, d, dtype)
    sl = torch.tensor([0.5, 0.25, 0.1], device="cuda") if slopes else None
    bounds = [0] + list(range(1, 65)) + [130, 131, 162, 163, 200]      # single tokens, and longer documents that start with one
    for window, docs in ((1, None), (1, bounds), (None, bounds)):
        x = packed.to("cuda").requires_grad_(True)
        documents = None if docs is None else torch.tensor([docs], dtype=torch.int32, device="cuda")
        out = lact_amd.masked_window_attention(*parts(x, h, h, d), window, score_cap=cap, distance_slopes=sl, documents=documents)
        g, = torch.autograd.grad(out, x, go.to("cuda"))
        q, k, v = (t[0] for t in parts(g, h, h, d))
        single = torch.ones(l, dtype=torch.bool)
        if window is None:
            single[64:] = False
            single[[130, 162]] = True
            assert bool(k[64:130].any())
            single[64] = single[131] = single[163] = False
        alone = single.to("cuda")
        assert not q[alone].any()
        only = alone if window == 1 else torch.arange(l, device="cuda") < 64      # keys that nobody else sees either
        assert not k[only].any()
        tol = torch.finfo(dtype).eps * 4      # p / sum, rounded to the type, and the gradient
        ref = go.to("cuda")[0, only].float()
        assert float((v[only].float() - ref).abs().max()) <= tol * float(ref.abs().max())


@BOTH
def test_scores_far_below_zero(dtype):
    """Scores of -1e36 and below are ordinary ones to the softmax: the largest of them has the weight."""
    import lact_amd
    l, h, d = 70, 2, 64
    q, k = torch.full((1, l, h, d), -1e18), torch.full((1, l, h, d), 1e18)
    k[:, 1:] *= 4.0
    v = torch.randn(1, l, h, d, generator=torch.Generator().manual_seed(2))
    q, k, v = (t.to(dtype).to("cuda") for t in (q, k, v))
    out = lact_amd.masked_window_attention(q, k, v)
    assert torch.equal(out, v[:, :1].expand_as(out))
    lengths = torch.tensor([l], dtype=torch.int32, device="cuda")
    assert torch.equal(lact_amd.window_attention_step(q[:, -1], k, v, lengths), v[:, 0])


@BOTH
def test_bounds_that_are_not_in_order_stay_inside(dtype):
    """Nobody checks the bounds: whatever they hold, no read leaves the sequence and no token outside is attended to."""
    import lact_amd
    b, l, h, d = 2, 90, 2, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(b, l, h, d, generator=g).to(dtype).to("cuda").requires_grad_(True) for _ in range(3))
    docs = torch.tensor([[50, -7, 400, 20], [2 ** 31 - 1, 0, -2 ** 31, 90]], dtype=torch.int32, device="cuda")
    pre = torch.tensor([[1000, -5, 2 ** 31 - 1]] * 2, dtype=torch.int32, device="cuda")
    out = lact_amd.masked_window_attention(q, k, v, documents=docs, prefixes=pre)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert all(bool(torch.isfinite(t).all()) for t in (out, *grads))


def test_views_strides_and_alignment():
    """Operands that the kernels do not read as they lie give what their copies give."""
    import lact_amd
    b, l, h, d = 2, 77, 3, 64
    g = torch.Generator().manual_seed(1)
    base = [torch.randn(b, h, l, d, generator=g).bfloat16().to("cuda") for _ in range(3)]
    q, k, v = (t.transpose(1, 2) for t in base)                      # heads outside tokens
    ref = lact_amd.masked_window_attention(*(t.contiguous() for t in (q, k, v)), 40)
    assert torch.equal(lact_amd.masked_window_attention(q, k, v, 40), ref)
    odd = torch.empty(b * l * h * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(b, l, h, d)
    odd.copy_(k)
    assert odd.data_ptr() % 16 and torch.equal(lact_amd.masked_window_attention(q, odd, v, 40), ref)
    one = v[:, :, :1]
    wide = lact_amd.masked_window_attention(q, k[:, :, :1].expand(b, l, 1, d), one.expand(b, l, 1, d), 40)
    assert torch.equal(wide, lact_amd.masked_window_attention(q, k[:, :, :1].contiguous(), one.contiguous(), 40))
    same = lact_amd.masked_window_attention(q[:1].expand(2, l, h, d), k[:1].expand(2, l, h, d), v[:1].expand(2, l, h, d), 40)
    assert torch.equal(same[0], same[1]) and torch.equal(same[0], ref[0])


def test_empty_sequences_and_batches():
    import lact_amd
    for b, l in ((0, 5), (2, 0)):
        q, k, v = (torch.randn(b, l, n, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for n in (4, 2, 2))
        out = lact_amd.masked_window_attention(q, k, v)
        assert out.shape == q.shape and all(t.shape == x.shape for t, x in zip(torch.autograd.grad(out, (q, k, v), torch.empty_like(out)), (q, k, v)))


def test_gradient_against_differences():
    import lact_amd
    b, l, hq, hkv, d = 1, 40, 2, 1, 64
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(b, l, n, d, generator=g).to("cuda") for n in (hq, hkv, hkv))
    w = torch.randn(b, l, hq, d, generator=g).double().to("cuda")
    docs, sl = torch.tensor([[0, 17, 38]], device="cuda"), torch.tensor([0.1, 0.02], device="cuda")
    f = lambda *a: lact_amd.masked_window_attention(*a, 20, score_cap=5.0, distance_slopes=sl, documents=docs)  # noqa: E731
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(f(*x), x, w.float())
    for i in range(3):
        step = torch.randn(x[i].shape, generator=g).to("cuda")
        h = 2.0 ** -7
        moved = [[t + (s * h * step if j == i else 0) for j, t in enumerate((q, k, v))] for s in (1, -1)]
        diff = ((f(*moved[0]).double() - f(*moved[1]).double()) * w).sum() / (2 * h)
        exact = (grads[i].double() * step.double()).sum()
        # the third derivative times h^2 / 6, and fp32 outputs off by 2^-20 over 2 h
        scale = (grads[i].double().abs() * step.double().abs()).sum()
        assert abs(diff - exact) < 2e-3 * scale, (i, float(diff), float(exact))


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_captured_training_step(dtype):
    """Forward and backward captured into one graph and replayed with other inputs, eager work between the replays."""
    import lact_amd
    b, l, hq, hkv, d = 2, 200, 4, 2, 64
    docs = torch.tensor([[0, 90, 200], [10, 20, 190]], dtype=torch.int32, device="cuda")
    x = torch.randn(b, l, (hq + 2 * hkv) * d, device="cuda").to(dtype)
    go = torch.randn(b, l, hq, d, device="cuda").to(dtype)

    def step(x):
        leaf = x.detach().requires_grad_(True)
        out = lact_amd.masked_window_attention(*parts(leaf, hq, hkv, d), 64, documents=docs)
        return out.detach(), torch.autograd.grad(out, leaf, go)[0]

    step(x)
    torch.cuda.synchronize()
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(static)
    for i in range(3):
        fresh = torch.randn_like(x)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(res, step(fresh)):
            assert torch.equal(a, r), i


def test_capture_refuses_leaves_that_an_eager_graph_holds():
    """Their nodes belong to the default stream, which a captured backward would wait for.  Without the eager graph the same leaves are captured."""
    import lact_amd
    leaf = torch.randn(1, 70, 6, 64, device="cuda").bfloat16().requires_grad_(True)
    go = torch.randn(1, 70, 2, 64, device="cuda").bfloat16()
    f = lambda: lact_amd.masked_window_attention(leaf[:, :, :2], leaf[:, :, 2:4], leaf[:, :, 4:], 20)  # noqa: E731
    out = f()
    ref, = torch.autograd.grad(out, leaf, go, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"), torch.cuda.graph(graph):
        f()
    with torch.no_grad():
        assert torch.equal(f(), out)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(f(), leaf, go)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g, ref)


def test_other_streams_give_the_same():
    import lact_amd
    q, k, v = (torch.randn(1, 300, n, 128, device="cuda").bfloat16() for n in (8, 2, 2))
    ref = lact_amd.masked_window_attention(q, k, v, 77)
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    ref1 = lact_amd.window_attention_step(q[:, -1], k, v, lengths, 77)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append((lact_amd.masked_window_attention(q, k, v, 77), lact_amd.window_attention_step(q[:, -1], k, v, lengths, 77)))
    torch.cuda.synchronize()
    for a, c in outs:
        assert torch.equal(a, ref) and torch.equal(c, ref1)


# ---- single tokens

def check_step(b, n, hq, hkv, d, dtype, lengths, window=None, cap=None, slopes=False, layout="tokens"):
    import lact_amd
    print("[gpu-test] attention step", b, n, hq, hkv, d, dtype, lengths, window, cap, slopes, layout, flush=True)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(b, hq, d, generator=g).to(dtype)
    k, v = (torch.randn(b, n, hkv, d, generator=g).to(dtype) for _ in range(2))
    sl = 2.0 ** -torch.arange(1, hq + 1).float() if slopes else None
    kc, vc = (t.to("cuda") for t in (k, v))
    for i, m in enumerate(lengths):                                  # what lies behind the lengths is not read
        kc[i, max(0, min(m, n)):] = float("nan")
        vc[i, max(0, min(m, n)):] = float("nan")
    if layout == "heads":
        kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kc, vc))
    out = lact_amd.window_attention_step(q.to("cuda"), kc, vc, torch.tensor(lengths, device="cuda"), window, score_cap=cap,
                                         distance_slopes=None if sl is None else sl.to("cuda"))
    p_err, out_err = errors(dtype, n, d, 8.0 + (n if slopes else 0))
    ref, bound = MO.attention_step(q, k, v, lengths, window, cap, sl, None, p_err, out_err)
    assert out.dtype == dtype
    near(out, ref, bound, "out")


@BOTH
@pytest.mark.parametrize("b,n,hq,hkv,d,lengths,window", [
    (1, 1, 1, 1, 64, [1], None), (1, 300, 12, 12, 64, [300], 256), (3, 200, 4, 2, 128, [0, 1, 200], None), (2, 500, 7, 1, 128, [33, 499], 1),
    (5, 129, 8, 8, 64, [-3, 128, 129, 1000, 32], 100), (2, 3000, 32, 4, 128, [2999, 31], None), (1, 4100, 40, 1, 64, [4097], None),
    (70, 40, 2, 1, 64, [i % 41 for i in range(70)], 33)])
def test_step(b, n, hq, hkv, d, lengths, window, dtype):
    check_step(b, n, hq, hkv, d, dtype, lengths, window)


@BOTH
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_step_with_cap_and_distance(layout, dtype):
    check_step(3, 700, 8, 2, 128, dtype, [700, 5, 333], 400, 20.0, True, layout)
    check_step(2, 150, 4, 4, 64, dtype, [150, 64], None, 2.0, True, layout)


def test_step_of_many_parts_is_joined():
    """One long sequence over all compute units, and one block's share over many short ones."""
    check_step(1, 20000, 2, 1, 128, torch.bfloat16, [19999])
    check_step(600, 9, 4, 4, 64, torch.bfloat16, [i % 10 for i in range(600)])


def test_step_of_a_cache_past_32_bits():
    """The last sequence's cache lies more than 2^32 bytes behind the tensor's start, and its tokens more than 2^31 elements apart."""
    import lact_amd
    print("[gpu-test] attention step, far cache", flush=True)
    b, n, hkv, d = 2, 70000, 256, 128
    k = torch.zeros(b, n, hkv, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(b, hkv, d, generator=g).bfloat16()
    kk, vv = (torch.randn(6, 2, d, generator=g).bfloat16() for _ in range(2))
    lengths = [n, n - 3]
    for i in range(b):
        k[i, lengths[i] - 6:lengths[i], -2:], v[i, lengths[i] - 6:lengths[i], -2:] = kk.to("cuda"), vv.to("cuda")
    out = lact_amd.window_attention_step(q.to("cuda"), k, v, torch.tensor(lengths, device="cuda"), 6)
    p_err, out_err = errors(torch.bfloat16, 6, d)
    for i in range(b):
        ref, bound = MO.attention_step(q[i:i + 1, -2:], kk[None], vv[None], [6], None, None, None, None, p_err, out_err)
        near(out[i:i + 1, -2:], ref, bound, f"sequence {i}")
    assert not out[:, :-2].any()


def test_prompt_and_tokens_agree():
    """A prompt through the attention, then token after token through the step, is the attention over all of it."""
    import lact_amd
    b, l, hq, hkv, d, prompt, window = 2, 90, 4, 2, 64, 70, 50
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(b, l, n, d, generator=g).to("cuda") for n in (hq, hkv, hkv))
    sl = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    opts = dict(score_cap=10.0, distance_slopes=sl)
    whole = lact_amd.masked_window_attention(q, k, v, window, **opts)
    kc, vc = (torch.full((b, 128, hkv, d), float("nan"), device="cuda") for _ in range(2))
    kc[:, :prompt], vc[:, :prompt] = k[:, :prompt], v[:, :prompt]
    outs = [lact_amd.masked_window_attention(q[:, :prompt], k[:, :prompt], v[:, :prompt], window, **opts)]
    for t in range(prompt, l):
        kc[:, t], vc[:, t] = k[:, t], v[:, t]
        lengths = torch.full((b,), t + 1, dtype=torch.int32, device="cuda")
        outs.append(lact_amd.window_attention_step(q[:, t], kc, vc, lengths, window, **opts)[:, None])
    # both sides sum up to 50 probabilities in fp32, in another order
    assert float((torch.cat(outs, 1) - whole).abs().max()) < (2 * d + 2 * l + 128) * 2.0 ** -24 * float(v.abs().max()) * 2


def test_captured_steps():
    """A step captured once and replayed while the sequences grow."""
    import lact_amd
    b, n, hq, hkv, d = 3, 400, 8, 2, 128
    q, k, v = (torch.randn(*s, device="cuda").bfloat16() for s in ((b, hq, d), (b, n, hkv, d), (b, n, hkv, d)))
    lengths = torch.tensor([1, 100, 250], dtype=torch.int32, device="cuda")
    lact_amd.window_attention_step(q, k, v, lengths, 300)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lact_amd.window_attention_step(q, k, v, lengths, 300)
    for i in range(4):
        q.copy_(torch.randn_like(q.float()))
        lengths += 37
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lact_amd.window_attention_step(q, k, v, lengths, 300)), i


def test_refusals_on_the_gpu():
    import lact_amd
    f = lact_amd.masked_window_attention
    q, k = torch.zeros(2, 8, 4, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 8, 2, 64, device="cuda", dtype=torch.bfloat16)
    for bad, error in ((dict(k=k.float()), TypeError), (dict(v=k[:, :7]), ValueError), (dict(k=q), ValueError), (dict(distance_slopes=torch.zeros(2, device="cuda")), ValueError),
                       (dict(distance_slopes=torch.zeros(4)), RuntimeError), (dict(documents=torch.zeros(1, 2, device="cuda", dtype=torch.int32)), ValueError),
                       (dict(documents=torch.zeros(2, 2, device="cuda")), TypeError), (dict(prefixes=torch.zeros(2, 2, device="cuda", dtype=torch.int32)), ValueError),
                       (dict(documents=torch.zeros(2, 2, dtype=torch.int32)), RuntimeError)):
        with pytest.raises(error):
            f(**{**dict(q=q, k=k, v=k), **bad})
    with pytest.raises(TypeError):
        f(q.half(), k.half(), k.half())
    with pytest.raises(RuntimeError, match="divide"):
        f(q[:, :, :3], k, k)
    wide = torch.zeros(1, 8, 2, 96, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="64 or 128"):
        f(wide, wide, wide)
    leaf = q.clone().requires_grad_(True)
    first, = torch.autograd.grad(f(leaf, k, k).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.float().sum(), leaf)
    step, n = lact_amd.window_attention_step, torch.ones(2, dtype=torch.int32, device="cuda")
    for bad, error in ((dict(lengths=n.float()), TypeError), (dict(lengths=n[:1]), ValueError), (dict(v_cache=k[:, :7]), ValueError), (dict(lengths=n.cpu()), RuntimeError),
                       (dict(k_cache=torch.zeros(2, 8, 2, 128, device="cuda", dtype=torch.bfloat16)[..., ::2]), ValueError),
                       (dict(k_cache=torch.zeros(2 * 8 * 2 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 8, 2, 64)), ValueError)):
        with pytest.raises(error):
            step(**{**dict(q=q[:, 0], k_cache=k, v_cache=k, lengths=n), **bad})
    assert not step(q[:, 0], k[:, :0], k[:, :0], n).any()


def test_autocast_casts_the_operands():
    import lact_amd
    x = torch.randn(1, 40, 2, 64, device="cuda", requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16):
        out = lact_amd.masked_window_attention(x, x, x, 9)
    g, = torch.autograd.grad(out.float().sum(), x)
    b = x.detach().bfloat16()
    assert out.dtype == torch.bfloat16 and g.dtype == torch.float32 and torch.equal(out, lact_amd.masked_window_attention(b, b, b, 9))
    with torch.autocast("cuda", torch.float16), pytest.raises(TypeError):
        lact_amd.masked_window_attention(x, x, x)


@BOTH
def test_wide_integers_are_cut_to_the_sequence(dtype):
    """Bounds, prefixes and lengths past 32 bits lie outside the sequence like any others."""
    import lact_amd
    b, l, h, d = 3, 150, 2, 64
    packed, go = make(b, l, h, h, d, dtype)
    far = 2 ** 63 - 1
    wide = torch.tensor([[0, 40, 2 ** 40], [10, 2 ** 32 + 60, far], [-far - 1, 2 ** 31, far]])
    plain = torch.tensor([[0, 40, l], [10, l, l], [0, l, l]])
    wide_pre, plain_pre = torch.tensor([[far, 2 ** 32 + 1], [-far - 1, 5], [2 ** 32, 0]]), torch.tensor([[l, l], [0, 5], [l, 0]])
    results = []
    for docs, pre in ((wide, wide_pre), (plain.int(), plain_pre.int())):
        x = packed.to("cuda").requires_grad_(True)
        out = lact_amd.masked_window_attention(*parts(x, h, h, d), 70, documents=docs.to("cuda"), prefixes=pre.to("cuda"))
        results.append((out.detach(), *torch.autograd.grad(out, x, go.to("cuda"))))
    assert all(torch.equal(a, r) for a, r in zip(*results))
    assert bool(results[0][0].any(-1).sum() == b * l * h - 10 * h)
    q, k, v = (t.to("cuda") for t in parts(packed, h, h, d))
    step = lambda *n: lact_amd.window_attention_step(q[:, 0], k, v, torch.tensor(n, device="cuda"), 40)  # noqa: E731
    assert torch.equal(step(far, 2 ** 31, 2 ** 32 + 5), step(l, l, l)) and not step(-far - 1, -2 ** 32 + 9, -2 ** 31).any()


def capped_errors(dtype, l, d, size, cap):
    """bf16, caps up to 256 / log2(e): the exponential, 1 + it and its reciprocal are off by 2^-23, 2^-24 and 2^-23 of themselves, which the cap multiplies: in
    units of cap log2(e) by 1/2, 1/2 and 1 of 2^-23, and the last sum by 2^-24 of it."""
    p_err, out_err = errors(dtype, l, d, size)
    return p_err + (2.5 * 2.0 ** -23 * cap if dtype == torch.bfloat16 and cap * 1.4427 <= 256 else 0.0), out_err


@BOTH
@pytest.mark.parametrize("hq", [3, 200])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [150.0, 2000.0, 1e5, 1e7, 1e30, 3e38])
def test_large_caps(cap, d, hq, dtype):
    """A cap far above the scores leaves them as they are."""
    import lact_amd
    print("[gpu-test] masked attention, large cap", cap, d, hq, dtype, flush=True)
    l = 140
    packed, go = make(1, l, hq, hq, d, dtype)
    x = packed.to("cuda").requires_grad_(True)
    out = lact_amd.masked_window_attention(*parts(x, hq, hq, d), 90, score_cap=cap)
    gx, = torch.autograd.grad(out, x, go.to("cuda"))
    ref, bound = MO.attention(*parts(packed, hq, hq, d), 90, cap, None, None, None, None, go, *capped_errors(dtype, l, d, 8.0, cap))
    for name, a, r, e in zip(("out", "dq", "dk", "dv"), [out, *parts(gx, hq, hq, d)], ref, bound):
        near(a, r, e, name)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [150.0, 2500.0])
def test_large_caps_that_bend_scores(cap, d, dtype):
    """Keys that grow along the sequence: scores from nothing to beyond the cap."""
    import lact_amd
    print("[gpu-test] masked attention, scores about a large cap", cap, d, dtype, flush=True)
    l, h = 300, 3
    growth = cap / 8
    packed, go = make(1, l, h, h, d, dtype, growth=growth)
    x = packed.to("cuda").requires_grad_(True)
    out = lact_amd.masked_window_attention(*parts(x, h, h, d), 190, score_cap=cap)
    gx, = torch.autograd.grad(out, x, go.to("cuda"))
    ref, bound = MO.attention(*parts(packed, h, h, d), 190, cap, None, None, None, None, go, *capped_errors(dtype, l, d, 8.0 * growth, cap))
    for name, a, r, e in zip(("out", "dq", "dk", "dv"), [out, *parts(gx, h, h, d)], ref, bound):
        near(a, r, e, name)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [150.0, 1e5, 1e7, 3e38])
def test_step_with_large_caps(cap, d, dtype):
    import lact_amd
    print("[gpu-test] attention step, large cap", cap, d, dtype, flush=True)
    b, n, hq, hkv, lengths = 2, 300, 4, 2, [300, 77]
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(*s, generator=g).to(dtype) for s in ((b, hq, d), (b, n, hkv, d), (b, n, hkv, d)))
    out = lact_amd.window_attention_step(*(t.to("cuda") for t in (q, k, v)), torch.tensor(lengths, device="cuda"), score_cap=cap)
    near(out, *MO.attention_step(q, k, v, lengths, None, cap, None, None, *capped_errors(dtype, n, d, 8.0, cap)), "out")


@BOTH
def test_the_smallest_caps_leave_equal_weights(dtype):
    """A cap of 1e-40: scores are nothing but their sign's, and a score of 0 is 0."""
    import lact_amd
    l, h, d = 100, 2, 64
    packed, _ = make(1, l, h, h, d, dtype)
    packed[:, ::3, :h * d] = 0.0
    q, k, v = parts(packed, h, h, d)
    out = lact_amd.masked_window_attention(*(t.to("cuda") for t in (q, k, v)), score_cap=1e-40)
    near(out, *MO.attention(q, k, v, None, 1e-40, None, None, None, None, None, *errors(dtype, l, d)), "out")
    lengths = torch.tensor([l], device="cuda")
    one = lact_amd.window_attention_step(q[:, 3].to("cuda"), k.to("cuda"), v.to("cuda"), lengths, score_cap=1e-40)
    near(one, *MO.attention_step(q[:, 3], k, v, [l], None, 1e-40, None, None, *errors(dtype, l, d)), "step")


@BOTH
@pytest.mark.parametrize("hq", [3, 200])
@pytest.mark.parametrize("size", [1e30, 1e-30])
@pytest.mark.parametrize("cap,sign", [(12.0, 1.0), (30.0, 1.0), (60.0, 1.0), (30.0, -1.0), (60.0, -1.0)])
def test_large_and_small_values_under_scores_at_their_cap(cap, sign, size, hq, dtype):
    """All scores at the cap, or at its negative: the outputs are means of the values, whose sums stay far from the ends of what fp32 holds.  Values of 1e30 times 140
    terms and the 2^8 that a row's largest probability may reach: 2^115; values of 1e-30 times a probability of 1 or more: 2^-100."""
    import lact_amd
    print("[gpu-test] masked attention, values and caps", cap, sign, size, hq, dtype, flush=True)
    l, d = 140, 64
    q, k = torch.full((1, l, hq, d), 16.0), torch.full((1, l, hq, d), 16.0 * sign)
    v = torch.randn(1, l, hq, d, generator=torch.Generator().manual_seed(3)) * size
    q, k, v = (t.to(dtype) for t in (q, k, v))
    out = lact_amd.masked_window_attention(*(t.to("cuda") for t in (q, k, v)), score_cap=cap)
    ref, bound = MO.attention(q, k, v, None, cap, None, None, None, None, None, *errors(dtype, l, d, cap))
    near(out.double() / size, ref / size, bound / size, "out")


@BOTH
@pytest.mark.parametrize("h", [2, 200])
@pytest.mark.parametrize("lead,step,rise", [((2048.0, 16384.0, 0.0, 0.0, 0.0), 4.0, 0.0), ((-2048.0, 16384.0, 0.0, 0.0, 0.0), 4.0, 0.0),
                                            ((354.0, 16384.0, 256.0, 57.0, 12.0), 0.5, 0.0), ((354.0, 16384.0, 256.0, 57.0, 12.0), 0.5, 48.0),
                                            ((-354.0, 16384.0, -256.0, 57.0, -12.0), 0.5, 48.0)])
def test_far_scores_that_nearly_tie(lead, step, rise, h, dtype):
    """Scores about 2^22 (and about 2^20 / log2(e), where rows begin to subtract their maximum ahead of the product) that differ by some units: whichever
    waves share a row and wherever its maximum moves to, what its keys weigh comes from the differences.  Every product and sum of a score is a whole number of
    steps of fp32, and so exact."""
    import lact_amd
    print("[gpu-test] masked attention, far scores", lead, rise, h, dtype, flush=True)
    l, d = 140, 64
    g = torch.Generator().manual_seed(4)
    q, k = torch.zeros(1, l, h, d), torch.zeros(1, l, h, d)
    q[..., 0], k[..., 0], q[..., 1], k[..., 1], q[..., 2] = lead[0], lead[1], lead[2], lead[3], 1.0
    k[..., 2] = lead[4] + step * torch.randint(-8, 9, (1, l, h), generator=g)
    k[:, :64, :, 2] -= rise / 2
    k[:, 64:, :, 2] += rise / 2
    v = torch.randn(1, l, h, d, generator=g)
    q, k, v = (t.to(dtype) for t in (q, k, v))
    out = lact_amd.masked_window_attention(*(t.to("cuda") for t in (q, k, v)))
    near(out, *MO.attention(q, k, v, None, None, None, None, None, None, None, *errors(dtype, l, d)), "out")


@BOTH
@pytest.mark.parametrize("cap", [20.0, 1e4])
def test_keys_of_infinity_under_a_cap(cap, dtype):
    """Their scores are the cap or its negative, as those of very large keys are: outputs are finite, gradients of the queries that see them NaN."""
    import lact_amd
    l, h, d = 90, 2, 64
    packed, go = make(1, l, h, h, d, dtype)
    results = []
    for value in (1e30, float("inf")):
        x = packed.clone()
        x[:, 40, h * d:2 * h * d:d] = value           # one element of a key in every head
        x = x.to("cuda").requires_grad_(True)
        out = lact_amd.masked_window_attention(*parts(x, h, h, d), 30, score_cap=cap)
        results.append((out.detach(), torch.autograd.grad(out, x, go.to("cuda"))[0]))
    (ref, gref), (out, g) = results
    assert bool(torch.isfinite(out).all()) and torch.equal(out, ref)
    q = slice(0, h * d)
    assert bool(torch.isnan(g[:, 40:70, q]).all()) and torch.equal(g[:, :40], gref[:, :40]) and torch.equal(g[:, 70:, q], gref[:, 70:, q])


@pytest.mark.parametrize("h", [2, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_scores_past_their_cap_in_fp32(d, h):
    """What is left of a gradient behind scores of 8 to 12 under a cap of 2, 1e-3 to 2e-5, keeps its digits.  The scores are one product each, and exact; the derivative's
    exponent of up to 12 is off by two roundings, as the scores' of this size are allowed to be."""
    import lact_amd
    print("[gpu-test] masked attention, gradients past the cap", d, h, flush=True)
    l = 140
    packed, go = make(1, l, h, h, d, torch.float32)
    q, k, _ = parts(packed, h, h, d)
    q[:], q[..., 0] = 0.0, 1.0
    g = torch.Generator().manual_seed(1)
    k[..., 0] = torch.randint(64, 97, (1, l, h), generator=g) / 8 * (2 * torch.randint(0, 2, (1, l, h), generator=g) - 1)
    packed = torch.cat([q.flatten(2), k.flatten(2), packed[..., 2 * h * d:]], -1)
    x = packed.to("cuda").requires_grad_(True)
    out = lact_amd.masked_window_attention(*parts(x, h, h, d), 90, score_cap=2.0, scale=1.0)
    gx, = torch.autograd.grad(out, x, go.to("cuda"))
    ref, bound = MO.attention(*parts(packed, h, h, d), 90, 2.0, None, None, None, 1.0, go, *errors(torch.float32, l, d))
    for name, a, r, e in zip(("out", "dq", "dk", "dv"), [out, *parts(gx, h, h, d)], ref, bound):
        near(a, r, e, name)
