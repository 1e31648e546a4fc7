"""Host side of the paged cache and of rotary positions: what their entry points refuse, in Python and at the C ABI, before anything is launched; and the oracle against independent
forms."""
import ctypes
import math
import random

import pytest
import torch

import lact_amd
from lact_amd import _lib
from oracle import mixers_oracle as MO
from oracle import paged_oracle as PO


def lib_error():
    return _lib.lib().lact_last_error().decode()


P = ctypes.c_void_p(1 << 20)      # never read


def cache_desc(**kw):
    """20 pages of 32 places, 2 heads of 64, bf16."""
    d = _lib.PagedCacheDesc(0, 20, 32, 2, 64, 6, 4096, 4096, 64, 64, P, P, P, P)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


CACHE_REFUSALS = [
    (dict(dtype=1), "act_dtype or"), (dict(dtype=3), "act_dtype or"), (dict(pages=0), "positive"), (dict(page_size=0), "positive"), (dict(HK=-1), "positive"), (dict(width=0), "positive"),
    (dict(D=96), "64 or 128"), (dict(page_size=24), "multiple of 16"), (dict(page_size=8), "multiple of 16"), (dict(width=1 << 20), "too many"), (dict(k_page=4092), "aligned"),
    (dict(v_page=4088), "overlap"), (dict(k_page=-4096), "overlap"), (dict(k=ctypes.c_void_p((1 << 20) + 8)), "aligned"), (dict(v=None), "null pointer"),
    (dict(dtype=2, k_exponents=None), "null pointer"), (dict(dtype=2, ke_page=72), "aligned"), (dict(dtype=2, ve_page=48), "overlap"),
    (dict(dtype=2, v_exponents=ctypes.c_void_p((1 << 20) + 4)), "aligned")]


@pytest.mark.parametrize("change,message", CACHE_REFUSALS)
def test_cache_arguments(change, message):
    L, c = _lib.lib(), ctypes.byref(cache_desc(**change))
    assert L.lact_paged_cache_write(c, 0, 3, 5, P, 128, 640, P, 128, 640, P, P, P, None) < 0 and message in lib_error()
    assert L.lact_paged_cache_read(c, 0, 3, 5, P, P, P, P, P, None) < 0 and message in lib_error()
    d = ctypes.byref(step_desc())
    assert L.lact_paged_attention_step_workspace_bytes(c, d, P, ctypes.byref(ctypes.c_size_t())) < 0 and message in lib_error()
    assert L.lact_paged_attention_step(c, d, P, P, P, P, P, None) < 0 and message in lib_error()


def test_write_and_read_arguments():
    L, c = _lib.lib(), ctypes.byref(cache_desc())
    write = lambda *a: L.lact_paged_cache_write(c, *a, None)  # noqa: E731
    good = [0, 3, 5, P, 128, 640, P, 128, 640, P, P, P]
    for at, bad, message in ((0, 5, "act_dtype"), (1, 0, "positive"), (2, -1, "positive"), (2, 1 << 30, "too many"), (3, None, "null pointer"), (4, 100, "aligned"), (5, -640, "aligned"),
                             (6, ctypes.c_void_p((1 << 20) + 2), "aligned"), (8, 4, "aligned"), (9, None, "null pointer")):
        assert write(*good[:at], bad, *good[at + 1:]) < 0 and message in lib_error(), at
    good = [0, 3, 5, P, P, P, P, P]
    for at, bad, message in ((1, -3, "positive"), (3, None, "null pointer"), (5, None, "null pointer"), (6, None, "null pointer"), (7, ctypes.c_void_p((1 << 20) + 8), "aligned")):
        assert L.lact_paged_cache_read(c, *good[:at], bad, *good[at + 1:], None) < 0 and message in lib_error(), at
    assert L.lact_paged_cache_write(None, 0, 3, 5, P, 128, 640, P, 128, 640, P, P, P, None) < 0 and "descriptor" in lib_error()


def test_writes_must_not_overlap():
    """Keys, values and exponents apart, or parts of the same pages of one pool; the tokens and whole numbers elsewhere."""
    L, at = _lib.lib(), lambda n: ctypes.c_void_p((1 << 24) + n)  # noqa: E731
    page = 2 * 32 * 64
    apart = dict(k=at(0), v=at(20 * page), k_exponents=at(40 * page), v_exponents=at(40 * page + 20 * 64))
    record = dict(k_page=2 * page + 128, v_page=2 * page + 128, ke_page=2 * page + 128, ve_page=2 * page + 128, k=at(0), v=at(page), k_exponents=at(2 * page), v_exponents=at(2 * page + 64))
    far = ctypes.c_void_p((1 << 24) - (1 << 16))

    def refused(**kw):
        rc = L.lact_paged_cache_write(ctypes.byref(cache_desc(dtype=2, **{k: v for k, v in kw.items() if k not in ("tokens", "table", "starts")})), 0, 1, 1,
                                      kw.get("tokens", far), 128, 128, far, 128, 128, kw.get("table", far), kw.get("starts", far), None, None)
        assert rc < 0
        return lib_error()

    for layout in (apart, record):
        for change in (dict(v=at(0)), dict(v=at(page - 16)), dict(k_exponents=at(16)), dict(v_exponents=layout["k_exponents"])):
            assert "must not overlap" in refused(**{**layout, **change}), change
        for change in (dict(tokens=at(32)), dict(table=at(20 * page)), dict(starts=layout["k_exponents"])):
            assert "must not lie in the cache" in refused(**{**layout, **change}), change
    assert "must not overlap" in refused(**{**record, "v_page": 2 * page + 256})


def write_of(c):
    """What a write of one token says whose table lies in the keys, so that no call gets past the checks: that of the pages among themselves comes first."""
    far = ctypes.c_void_p(1 << 10)
    assert _lib.lib().lact_paged_cache_write(ctypes.byref(c), 0, 1, 1, far, c.HK * c.D, c.HK * c.D, far, c.HK * c.D, c.HK * c.D, ctypes.c_void_p(c.k), far, None, None) < 0
    return "apart" if "must not lie in the cache" in lib_error() else "overlap" if "must not overlap" in lib_error() else lib_error()


@pytest.mark.parametrize("heads,size,d", [(2, 32, 64), (3, 32, 64), (12, 64, 128), (6, 64, 128), (8, 48, 64), (8, 80, 128), (5, 16, 64)])
@pytest.mark.parametrize("values_first", [False, True])
@pytest.mark.parametrize("dtype", [0, 2])
def test_pages_of_one_pool(dtype, values_first, heads, size, d):
    """Keys and values of a page behind one another, their exponents behind them or in a pool of their own: apart, whatever a page's length, also where the values' pages begin some pages further
    on or back.  16 bytes off and they overlap."""
    rows = heads * size
    page, item = rows * d * (1 if dtype == 2 else 2), (1 if dtype == 2 else 2)
    for record, e_record in ((2 * page, 2 * rows), (2 * page + 2 * rows, 2 * page + 2 * rows)):
        for shift in (0, 3 * record, -3 * record):
            parts = [1 << 32, (1 << 32) + page]
            exps = [1 << 33, (1 << 33) + rows] if record == 2 * page else [(1 << 32) + 2 * page, (1 << 32) + 2 * page + rows]
            k, v = parts[::-1] if values_first else parts
            ke, ve = exps[::-1] if values_first else exps
            kw = dict(dtype=dtype, pages=20, page_size=size, HK=heads, D=d, k_page=record // item, v_page=record // item, ke_page=e_record, ve_page=e_record, k=k, v=v + shift,
                      k_exponents=ke, v_exponents=ve + shift // record * e_record)
            assert write_of(cache_desc(**kw)) == "apart", (record, shift)
            nearer = 16 if values_first else -16
            assert write_of(cache_desc(**{**kw, "v": v + shift + nearer})) == "overlap", (record, shift)
            if dtype == 2:
                assert write_of(cache_desc(**{**kw, "v_exponents": kw["v_exponents"] + nearer})) == "overlap", (record, shift)


def test_overlaps_of_pages_are_those_of_their_bytes():
    """Keys and values the same distance from page to page, at any distance from each other, against all pages one by one."""
    g, seen = random.Random(1), set()
    length = 16 * 64 * 2
    for _ in range(3000):
        pages, stride = g.randint(1, 5), length + 16 * g.choice((0, 1, g.randint(0, 300)))
        k = (1 << 24) + 16 * g.randint(0, 999)
        v = k + g.randint(-6, 6) * stride + g.choice((length, -length, stride - length, 16 * g.randint(0, stride // 16)))
        at = [range(x, x + pages * stride, stride) for x in (k, v)]
        overlap = any(abs(x - y) < length for x in at[0] for y in at[1])
        seen.add(overlap)
        got = write_of(cache_desc(pages=pages, page_size=16, HK=1, k_page=stride // 2, v_page=stride // 2, k=k, v=v))
        assert got == ("overlap" if overlap else "apart"), (pages, stride, v - k)
    assert seen == {True, False}


def step_desc(**kw):
    d = _lib.PagedStepDesc(0, 3, 8, 100, 0.125, 0.0, 512, None)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=2), "act_dtype"), (dict(B=0), "positive"), (dict(H=0), "positive"), (dict(H=7), "divide"), (dict(window=0), "positive"), (dict(B=1 << 18), "too large"),
    (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(score_cap=-1.0), "cap"), (dict(score_cap=math.inf), "cap"), (dict(q_bs=510), "aligned"), (dict(q_bs=-512), "aligned")])
def test_step_arguments(change, message):
    L, c, d = _lib.lib(), ctypes.byref(cache_desc()), ctypes.byref(step_desc(**change))
    assert L.lact_paged_attention_step_workspace_bytes(c, d, P, ctypes.byref(ctypes.c_size_t())) < 0 and message in lib_error()
    assert L.lact_paged_attention_step(c, d, P, P, P, P, P, None) < 0 and message in lib_error()


def test_step_pointers_and_workspace():
    L, c = _lib.lib(), cache_desc(width=40)
    for i in range(5):
        args = [P] * 5
        args[i] = None
        assert L.lact_paged_attention_step(ctypes.byref(c), ctypes.byref(step_desc(window=1280)), *args, None) < 0 and "null pointer" in lib_error()
    assert L.lact_paged_attention_step(ctypes.byref(c), ctypes.byref(step_desc()), ctypes.c_void_p((1 << 20) + 2), P, P, P, P, None) < 0 and "aligned" in lib_error()
    assert L.lact_paged_attention_step(ctypes.byref(c), None, P, P, P, P, P, None) < 0 and "descriptor" in lib_error()

    def size(**kw):
        n = ctypes.c_size_t(7)
        assert L.lact_paged_attention_step_workspace_bytes(ctypes.byref(c), ctypes.byref(step_desc(**kw)), P, ctypes.byref(n)) == 0
        return n.value
    assert L.lact_paged_attention_step_workspace_bytes(ctypes.byref(c), ctypes.byref(step_desc()), P, None) < 0 and "null pointer" in lib_error()
    # two parts a block, of 4 query heads to a key head: 3 sequences x 2 heads x 10 steps of 128 places; none where every item has a block of its own
    assert size(window=1 << 30) == 2 * 60 * 4 * 66 * 4 and size() == 0
    c = cache_desc(pages=1 << 20, width=1 << 18)
    assert size(window=1 << 30) == 2 * 512 * 4 * 66 * 4      # two blocks to a compute unit
    c.D, c.k_page, c.v_page = 128, 8192, 8192
    assert size(window=1 << 30, q_bs=1024) == 2 * 256 * 4 * 130 * 4      # one
    c.dtype = 2
    assert size(window=1 << 30, q_bs=1024) == 2 * 512 * 4 * 130 * 4


def rotary_desc(**kw):
    f, a = (ctypes.c_double * 32)(*[0.5] * 32), (ctypes.c_int32 * 32)(*[i % 2 for i in range(32)])
    d = _lib.RotaryDesc(0, 2, 10, 4, 2, 64, 32, 2, 1, 0, 0, 2560, 256, 64, 1280, 128, 64, 20, 2, f, a)
    for n, v in kw.items():
        setattr(d, n, v)
    d._keep = (f, a)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=2), "act_dtype"), (dict(B=0), "positive"), (dict(L=0), "positive"), (dict(H=0), "positive"), (dict(HK=-1), "positive"), (dict(D=65), "even"), (dict(D=258), "256"),
    (dict(D=62), "fit"), (dict(pairs=0), "fit"), (dict(n_axes=0), "axes"), (dict(n_axes=1), "out of range"), (dict(position_type=3), "positions"), (dict(H=65535), "too many"),
    (dict(B=1 << 16, L=1 << 16), "too many"), (dict(frequencies=(ctypes.c_double * 32)(*[math.nan] * 32)), "out of range"),
    (dict(axis_of_pair=(ctypes.c_int32 * 32)(*[-1] * 32)), "out of range")])
def test_rotary_arguments(change, message):
    d = rotary_desc(**change)
    assert _lib.lib().lact_axial_rotary(ctypes.byref(d), P, P, P, P, P, None) < 0 and message in lib_error()


def test_rotary_pointers():
    L = _lib.lib()
    for i in range(5):
        args = [P] * 5
        args[i] = None
        assert L.lact_axial_rotary(ctypes.byref(rotary_desc()), *args, None) < 0 and "null pointer" in lib_error()
    assert L.lact_axial_rotary(None, P, P, P, P, P, None) < 0 and "descriptor" in lib_error()
    d = rotary_desc(frequencies=None)
    assert L.lact_axial_rotary(ctypes.byref(d), P, P, P, P, P, None) < 0 and "null pointer" in lib_error()


def test_python_refusals():
    cache = lact_amd.PagedCache.empty(4, 2, 16, 64, device="cpu")
    eight = lact_amd.PagedCache.empty(4, 2, 16, 64, dtype=torch.float8_e4m3fn, device="cpu")
    assert cache.k_scale is None and eight.v_scale.dtype == torch.float8_e8m0fnu and eight.k_scale.shape == (4, 2, 16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, k = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    step, write, read = lact_amd.paged_attention_step, lact_amd.paged_cache_write, lact_amd.paged_cache_read
    for bad, error in ((dict(cache=tuple(cache)), TypeError), (dict(q=q[0]), ValueError), (dict(page_table=table[0]), ValueError), (dict(window=0), ValueError), (dict(score_cap=0.0), ValueError),
                       (dict(scale=1e-50), ValueError), (dict(lengths=[1]), TypeError), (dict(cache=cache._replace(k=cache.k[0])), ValueError),
                       (dict(cache=eight._replace(k_scale=eight.k_scale[0])), ValueError), (dict(distance_slopes=torch.ones(4, requires_grad=True)), RuntimeError),
                       (dict(q=q.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(error):
            step(**{**dict(q=q, cache=cache, page_table=table, lengths=n), **bad})
    with pytest.raises(RuntimeError, match="MI355X"):
        step(q, cache, table, n)
    for bad, error in ((dict(k=k[0]), ValueError), (dict(k=k[0], v=k), ValueError), (dict(k=k[0, 0], v=k[0, 0]), ValueError), (dict(starts=table), ValueError), (dict(counts=table), ValueError),
                       (dict(cache=None), TypeError), (dict(v=k.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(error):
            write(**{**dict(cache=cache, k=k, v=k, page_table=table), **bad})
    with pytest.raises(RuntimeError, match="MI355X"):
        write(cache, k, k, table)
    for bad, error in ((dict(tokens=-1), ValueError), (dict(tokens=2.5), ValueError), (dict(lengths=table), ValueError), (dict(dtype="bf16"), TypeError)):
        with pytest.raises(error):
            read(**{**dict(cache=cache, page_table=table, lengths=n, tokens=3), **bad})
    with pytest.raises(RuntimeError, match="MI355X"):
        read(cache, table, n, 3)
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda t: step(t, cache, table, n))(q[None])
    f, x, p = lact_amd.axial_rotary, torch.zeros(1, 6, 2, 64), torch.zeros(6, 2, dtype=torch.int32)
    for bad, error in ((dict(axes=()), ValueError), (dict(axes=(32, 33)), ValueError), (dict(axes=(32, 0)), ValueError), (dict(axes=(64, 2)), ValueError), (dict(base=0.0), ValueError),
                       (dict(base=math.inf), ValueError), (dict(frequencies=[]), ValueError), (dict(frequencies=[1.0] * 31), ValueError), (dict(frequencies=[math.nan] * 32), ValueError),
                       (dict(q=x[0, 0]), ValueError), (dict(k=x[0]), ValueError), (dict(positions=p.float().requires_grad_()), RuntimeError), (dict(positions=[1]), TypeError)):
        with pytest.raises(error):
            f(**{**dict(q=x, k=x, positions=p, axes=(32, 32)), **bad})
    with pytest.raises(RuntimeError, match="MI355X"):
        f(x, x, p, (32, 32))
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        f(torch.autograd.forward_ad.make_dual(x, x), None, p, (32, 32))


@pytest.mark.parametrize("part", ["k", "v"])
def test_caches_without_keys_or_values(part):
    cache = lact_amd.PagedCache.empty(4, 2, 16, 64, device="cpu")._replace(**{part: None})
    table, n, q = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: lact_amd.paged_attention_step(q, cache, table, n), lambda: lact_amd.paged_cache_write(cache, q, q, table), lambda: lact_amd.paged_cache_read(cache, table, n, 3)):
        with pytest.raises(TypeError, match="keys and values"):
            call()


@pytest.mark.parametrize("axes", [(32.5, 32), (32, 31.999), (2.25,), (32, -2.5)])
def test_axes_are_whole_numbers(axes):
    x, p = torch.zeros(1, 6, 2, 64), torch.zeros(6, len(axes), dtype=torch.int32)
    with pytest.raises(ValueError, match="even numbers"):
        lact_amd.axial_rotary(x, x, p, axes)
    with pytest.raises(RuntimeError, match="MI355X"):
        lact_amd.axial_rotary(x, x, p, (float(2 * int(n / 2) if n > 0 else 2) for n in axes))      # (what is whole may come in any type)


def test_oracle_of_8_bits_is_torchs():
    """The codes' values, and rounding, against torch's own type where a row's scale is 1."""
    codes = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(torch.nan_to_num(PO.e4m3_values(), 7777.0), torch.nan_to_num(codes.view(torch.float8_e4m3fn).double(), 7777.0))
    x = torch.randn(2000, 64, generator=torch.Generator().manual_seed(0)) * 60
    x[:, 0] = 300.0                                                     # between 224 and 448: an exponent of 0
    x = x.clamp(-448, 448)
    code, e = PO.to_8_bits(x)
    assert torch.equal(code, x.to(torch.float8_e4m3fn).view(torch.uint8)) and bool((e == 127).all())
    _, e = PO.to_8_bits(torch.tensor([[448.0, 1.0], [448.5, 1.0], [224.0, 0.0], [0.0, 0.0], [2.0 ** -149, 0.0], [3e38, 0.0]]))
    assert e.tolist() == [127, 128, 126, 0, 0, 247]                      # (448 * 2^119 = 2.98e38)


def test_oracle_of_pages_is_the_dense_one():
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 48, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    table = torch.tensor([[3, 0, 5], [1, 2, 4]])
    pages = [torch.zeros(6, 2, 16, 8, dtype=torch.float64) for _ in range(2)]
    for s in range(2):
        for j in range(48):
            for t, x in zip(pages, (k, v)):
                t[table[s, j // 16], :, j % 16] = x[s, j]
    for t, x in zip(pages, (k, v)):
        got, there = PO.tokens(t, table, [0, 0], [48, 30], 48)
        assert torch.equal(got[0], x[0]) and torch.equal(got[1, :30], x[1, :30]) and not got[1, 30:].any() and int(there.sum()) == 78
    q = torch.randn(2, 4, 8, generator=g, dtype=torch.float64)
    sl = torch.tensor([0.1, 0.2, 0.3, 0.4])
    for a, r in zip(PO.step(q, *pages, table, [41, 17], 20, 3.0, sl, None, 1.0, 1.0), MO.attention_step(q, k, v, [41, 17], 20, 3.0, sl, None, 1.0, 1.0)):
        assert float((a - r).abs().max()) < 1e-13


def test_oracle_of_turns_is_multiplication_of_complex_numbers():
    x = torch.randn(3, 5, 2, 12, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    p = torch.randint(0, 50, (5, 2), generator=torch.Generator().manual_seed(1))
    a = PO.angles(p, (4, 6), 100.0)
    want = torch.tensor([[p_[0], p_[0] * 100.0 ** -0.5, p_[1], p_[1] * 100.0 ** (-2 / 6), p_[1] * 100.0 ** (-4 / 6)] for p_ in p.double().tolist()], dtype=torch.float64)
    assert float((a - want).abs().max()) < 1e-12
    turn = torch.polar(torch.ones_like(a), a)[:, None]
    y = torch.view_as_real(torch.view_as_complex(x[..., :10].reshape(3, 5, 2, 5, 2)) * turn).flatten(-2)
    assert float((PO.rotary(x, a) - torch.cat((y, x[..., 10:]), -1)).abs().max()) < 1e-13
    z = torch.complex(x[..., :5], x[..., 5:10]) * turn
    assert float((PO.rotary(x, a, False) - torch.cat((z.real, z.imag, x[..., 10:]), -1)).abs().max()) < 1e-13
