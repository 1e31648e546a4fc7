"""Host side of the token mixers: what the entry points of lact_amd.attention and lact_amd.linear_attention refuse, in Python and at the C
ABI, before anything is launched; and the oracle against independent forms."""
import ctypes
import math

import pytest
import torch

import lact_amd
from lact_amd import _lib
from oracle import mixers_oracle as MO


def lib_error():
    return _lib.lib().lact_last_error().decode()


def attention_desc(**kw):
    d = _lib.AttentionDesc(0, 2, 100, 4, 2, 64, 100, 0, 0.125, 0.0, 256, 128, 128, 256, 25600, 12800, 12800, 25600, None, None, None)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


P = ctypes.c_void_p(1 << 20)      # never read


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=2), "act_dtype"), (dict(B=0), "positive"), (dict(L=-1), "positive"), (dict(HK=3), "divide"), (dict(D=96), "64 or 128"), (dict(window=0), "positive"),
    (dict(L=(1 << 24) + 1), "too large"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(score_cap=-1.0), "cap"), (dict(score_cap=math.inf), "cap"),
    (dict(q_ld=252), "aligned"), (dict(q_ld=192), "hold all heads"), (dict(k_ld=1 << 24), "too large"), (dict(v_bs=12801), "aligned"), (dict(n_documents=2), "documents"),
    (dict(n_documents=-1), "documents")])
def test_attention_arguments(change, message):
    d = attention_desc(**change)
    assert _lib.lib().lact_masked_attention_forward(ctypes.byref(d), P, P, P, P, P, P, None) < 0
    assert message in lib_error()


def test_attention_pointers():
    L, d = _lib.lib(), attention_desc()
    for i in range(5):
        args = [P] * 6
        args[i] = None
        assert L.lact_masked_attention_forward(ctypes.byref(d), *args, None) < 0 and "null pointer" in lib_error()
    assert L.lact_masked_attention_forward(ctypes.byref(d), ctypes.c_void_p((1 << 20) + 2), *[P] * 5, None) < 0 and "aligned" in lib_error()
    assert L.lact_masked_attention_forward(None, *[P] * 6, None) < 0 and "descriptor" in lib_error()
    d = attention_desc(n_documents=1)
    assert L.lact_attention_ranges_bytes(ctypes.byref(d)) == 2 * 100 * 16 and L.lact_attention_ranges_bytes(ctypes.byref(attention_desc())) == 0
    assert L.lact_masked_attention_forward(ctypes.byref(d), *[P] * 5, None, None) < 0 and "ranges" in lib_error()
    assert L.lact_masked_attention_backward(ctypes.byref(attention_desc(do_ld=8)), *[P] * 12, None) < 0 and "dout" in lib_error()


def test_attention_workspace():
    """Few blocks of 128 keys: the sums of dk and dv over the queries come in splits of their own."""
    L = _lib.lib()
    size = lambda **kw: L.lact_masked_attention_workspace_bytes(ctypes.byref(attention_desc(**kw)))  # noqa: E731
    assert size() == 0                                                     # four tiles of queries for one split
    assert size(L=1024, window=1024) == 2 * 8 * 2 * 1024 * 2 * 64 * 4      # 2 heads x 16 tiles
    assert size(L=1 << 20, window=1 << 20) == 0 and size(D=32) == 0


def step_desc(**kw):
    d = _lib.AttentionStepDesc(0, 2, 500, 8, 2, 128, 500, 0.1, 0.0, 1024, 256, 128000, 128, 256, 128000, 128, None)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=7), "act_dtype"), (dict(N=0), "positive"), (dict(H=9), "divide"), (dict(D=80), "64 or 128"), (dict(window=-3), "positive"), (dict(scale=-1.0), "scale"),
    (dict(score_cap=math.nan), "cap"), (dict(k_ld=100), "aligned"), (dict(v_hs=4), "aligned"), (dict(k_bs=-8), "strides"), (dict(k_ld=1 << 24), "strides"),
    (dict(N=1 << 25), "too large")])
def test_attention_step_arguments(change, message):
    L, d = _lib.lib(), step_desc(**change)
    assert L.lact_attention_step_workspace_bytes(ctypes.byref(d)) == 0
    assert L.lact_attention_step(ctypes.byref(d), P, P, P, P, P, P, None) < 0 and message in lib_error()


def test_attention_step_workspace():
    """Two parts for every block of at most one per compute unit: rows of the grouped heads, their sums, maximum and row sum."""
    L = _lib.lib()
    assert L.lact_attention_step_workspace_bytes(ctypes.byref(step_desc())) == 2 * 16 * 4 * 130 * 4      # 2 sequences x 2 heads x 4 steps of 128 keys
    assert L.lact_attention_step_workspace_bytes(ctypes.byref(step_desc(N=1 << 20, window=1 << 20))) == 2 * 256 * 4 * 130 * 4
    for i in range(6):
        args = [P] * 6
        args[i] = None
        assert L.lact_attention_step(ctypes.byref(step_desc()), *args, None) < 0 and "null pointer" in lib_error()


def linear_desc(**kw):
    d = _lib.LinearDesc(0, 2, 1000, 3, 64, 128, 1, 0.125, 192, 192, 384, 384, 192000, 192000, 384000, 384000)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=-1), "act_dtype"), (dict(l=0), "positive"), (dict(h=0), "positive"), (dict(dk=32), "64 or 128"), (dict(dv=96), "64 or 128"), (dict(scale=math.inf), "scale"),
    (dict(b=1 << 20, h=2), "too large"), (dict(q_ld=190), "aligned"), (dict(v_ld=376), "hold all heads"), (dict(k_ld=1 << 24), "too large")])
def test_linear_arguments(change, message):
    L, d = _lib.lib(), linear_desc(**change)
    assert L.lact_linear_attention_forward(ctypes.byref(d), P, P, P, P, P, P, P, P, None) < 0 and message in lib_error()
    assert L.lact_linear_attention_backward(ctypes.byref(d), *[P] * 15, None) < 0 and message in lib_error()


def test_linear_buffers_and_pointers():
    L = _lib.lib()
    a, s = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.lact_linear_attention_sizes(ctypes.byref(linear_desc()), ctypes.byref(a), ctypes.byref(s)) == 0
    assert a.value > 0 and s.value > 0
    # enough heads to fill the chip: no segments, no states, the tokens' weights alone
    assert L.lact_linear_attention_sizes(ctypes.byref(linear_desc(b=172)), ctypes.byref(a), None) == 0 and a.value == 172 * 3 * 1024 * 16
    for i in (0, 1, 2, 3, 5):      # state, last and states may be absent or are asked for by name
        args = [P] * 8
        args[i] = None
        assert L.lact_linear_attention_forward(ctypes.byref(linear_desc()), *args, None) < 0 and "null pointer" in lib_error()
    assert L.lact_linear_attention_forward(ctypes.byref(linear_desc()), *[P] * 7, None, None) < 0 and "states" in lib_error()
    assert L.lact_linear_attention_forward(ctypes.byref(linear_desc()), P, P, P, P, ctypes.c_void_p(8), P, P, P, None) < 0 and "aligned" in lib_error()
    args = [P] * 15
    args[5] = None                 # the last state, with its gradient and the decays' wanted
    assert L.lact_linear_attention_backward(ctypes.byref(linear_desc()), *args, None) < 0 and "last state" in lib_error()
    step = lambda *a: L.lact_linear_attention_step(*a)  # noqa: E731
    assert step(0, 1, 1, 64, 48, 1, 0.1, P, 64, P, 64, P, 48, P, P, P, P, None) < 0 and "64 or 128" in lib_error()
    assert step(0, 1, 1, 64, 64, 1, 0.1, P, 64, P, 64, P, 60, P, P, P, P, None) < 0 and "aligned" in lib_error()
    assert step(0, 1, 1, 64, 64, 1, 0.1, P, 64, P, 64, P, 64, P, P, None, P, None) < 0 and "null pointer" in lib_error()


def test_python_refusals():
    q, k, v = torch.zeros(1, 8, 4, 64), torch.zeros(1, 8, 2, 64), torch.zeros(1, 8, 2, 64)
    f = lact_amd.masked_window_attention
    for kw in (dict(window=0), dict(window=2.5), dict(score_cap=0.0), dict(score_cap=-1), dict(score_cap=math.nan), dict(scale=0), dict(scale=math.inf),
               dict(documents=torch.zeros(1, 1, dtype=torch.int32)), dict(documents=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            f(q, k, v, **kw)
    with pytest.raises(ValueError):
        f(q[0], k, v)
    with pytest.raises(RuntimeError, match="no gradient"):
        f(q, k, v, distance_slopes=torch.ones(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="MI355X"):
        f(q, k, v)
    with pytest.raises(TypeError):
        f(q, k, [1.0])
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda t: f(t, k, v))(q[None])
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(q, q), k, v)
    g = lact_amd.window_attention_step
    with pytest.raises(RuntimeError, match="inference"):
        g(q[:, 0].requires_grad_(), k, v, torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="MI355X"):
        g(torch.zeros(1, 4, 64), k, v, torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        g(torch.zeros(1, 4, 64), k, v, torch.ones(1, dtype=torch.int32), 0)
    h = lact_amd.decayed_linear_attention
    for bad in (torch.zeros(1, 8), torch.zeros(1, 8, 2, 64)):
        with pytest.raises(ValueError):
            h(k, k, v, bad)
    with pytest.raises(ValueError):
        h(k, k, v, torch.zeros(2), scale=math.nan)
    with pytest.raises(RuntimeError, match="MI355X"):
        h(k, k, v, torch.zeros(2))
    s = lact_amd.decayed_linear_attention_step
    with pytest.raises(RuntimeError, match="inference"):
        s(k[:, 0], k[:, 0], v[:, 0], torch.zeros(2), torch.zeros(1, 2, 64, 64, requires_grad=True))
    with pytest.raises(RuntimeError, match="MI355X"):
        s(k[:, 0], k[:, 0], v[:, 0], torch.zeros(2), torch.zeros(1, 2, 64, 64))


def test_oracle_attention_gradients_are_autograds():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 30, n, 8, generator=g, dtype=torch.double, requires_grad=True) for n in (4, 2, 2))
    docs, pre, sl = torch.tensor([[0, 10, 10, 28], [2, 5, 20, 30]]), torch.tensor([[3, 0, 5], [0, 9, 0]]), torch.tensor([0.1, 0.2, 0.3, 0.4]).double()
    kk, vv = (t.repeat_interleave(2, 2) for t in (k, v))
    s = 3 * torch.tanh(torch.einsum("bihd,bjhd->bhij", q, kk) / math.sqrt(8) / 3)
    s = s - sl[:, None, None] * (torch.arange(30)[:, None] - torch.arange(30)).abs()
    m = MO.visible(30, 7, docs, pre)[:, None]
    p = torch.where(m.any(-1, keepdim=True), torch.softmax(s.masked_fill(~m, -1e300), -1), torch.zeros(())) * m
    out = torch.einsum("bhij,bjhd->bihd", p, vv)
    go = torch.randn(out.shape, generator=g, dtype=torch.double)
    ref, _ = MO.attention(q, k, v, 7, 3.0, sl, docs, pre, None, go)
    for a, r in zip(ref, (out, *torch.autograd.grad(out, (q, k, v), go))):
        assert float((a - r).abs().max()) < 1e-13
    one, _ = MO.attention_step(q[:, 20], k, v, [21, 21], 7, 3.0, sl)
    whole, _ = MO.attention(q, k, v, 7, 3.0, sl)
    assert float((one - whole[:, 20]).abs().max()) < 1e-13


def test_oracle_recurrence_is_the_quadratic_form():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 20, 2, 8, generator=g, dtype=torch.double) for _ in range(3))
    d = -torch.rand(1, 20, 2, generator=g, dtype=torch.double)
    s = torch.randn(1, 2, 8, 8, generator=g, dtype=torch.double)
    out, last = MO.linear(q, k, v, d, s)
    run = d.cumsum(1)
    w = torch.exp(run[:, :, None] - run[:, None]) * torch.ones(20, 20).tril()[None, :, :, None]
    ref = (torch.einsum("bihd,bjhd,bijh,bjhe->bihe", q, k, w, v) + torch.einsum("bih,bihd,bhde->bihe", run.exp(), q, s)) / math.sqrt(8)
    assert float((out - ref).abs().max()) < 1e-12
    assert float((last - (torch.einsum("bjhd,bjh,bjhe->bhde", k, (run[:, -1:] - run).exp(), v) + run[:, -1].exp()[..., None, None] * s)).abs().max()) < 1e-12


def test_step_refuses_a_state_out_that_needs_a_gradient():
    k, s = torch.zeros(1, 2, 64), torch.zeros(1, 2, 64, 64)
    with pytest.raises(RuntimeError, match="inference"):
        lact_amd.decayed_linear_attention_step(k, k, k, torch.zeros(2), s, state_out=s.clone().requires_grad_(True))


@pytest.mark.parametrize("value", [1e-50, 1e39, -1e-50, 5e-324])
def test_caps_and_scales_that_fp32_does_not_hold(value):
    """The kernels take them in fp32, where these would be 0 (no cap at all) or infinite."""
    q = torch.zeros(1, 8, 2, 64)
    for kw in (dict(score_cap=value), dict(scale=value)):
        with pytest.raises(ValueError):
            lact_amd.masked_window_attention(q, q, q, **kw)
        with pytest.raises(ValueError):
            lact_amd.window_attention_step(q[:, 0], q, q, torch.ones(1, dtype=torch.int32), **kw)
    with pytest.raises(RuntimeError, match="MI355X"):
        lact_amd.masked_window_attention(q, q, q, score_cap=3e38, scale=1e-40)
