"""The paged cache (csrc/paged_cache.h, csrc/paged_attention.h) against its definition in float64: what is written and read bit by bit, the attention of single tokens at the
edges of its pieces of 16 places, tiles of 32, steps and pages."""
import math

import pytest
import torch

from oracle import mixers_oracle as MO
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

E4M3, E8M0, BF16, F32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
KINDS = pytest.mark.parametrize("dtype,held", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])


def errors(dtype, held, l, d, size=8.0):
    """Relative errors of a probability and of a stored value.  bf16: probabilities are rounded for the product (2^-8), scores are summed in fp32.  fp32: the sums of d and
    of l terms, three times as many with pages of 8 bits, and the exponential of a score of `size` off by the roundings of its d terms."""
    times = 3 if (dtype, held) == (F32, E4M3) else 1
    fp32 = (times * (2 * d + l) + 16 * size + 64) * 2.0 ** -24
    return (HALF[dtype] if dtype == BF16 else 0.0) + fp32, HALF[dtype]


def near(got, ref, bound, name):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), name
    worst = ((got - ref).abs() / (bound + 1e-7)).max() if got.numel() else 0.0
    print(f"[gpu-test]   {name}: {float(worst):.3f} of the bound", flush=True)
    assert worst <= 1.0, (name, float(worst))


def random_cache(pages, hkv, size, d, held, seed=1, spread=4):
    """A cache on the CPU: (k, v, k_scale, v_scale)."""
    g = torch.Generator().manual_seed(seed)
    if held != E4M3:
        return [torch.randn(pages, hkv, size, d, generator=g).to(held) for _ in range(2)] + [None, None]
    k, v = ((torch.randn(pages, hkv, size, d, generator=g) * 100).clamp(-448, 448).to(E4M3) for _ in range(2))
    return [k, v] + [torch.randint(121 - spread // 2, 121 + spread // 2, (pages, hkv, size), generator=g).to(torch.uint8).view(E8M0) for _ in range(2)]


def cuda(cache):
    import lact_amd
    return lact_amd.PagedCache(*(t if t is None else t.to("cuda") for t in cache))


def numbers(cache):
    return PO.held(cache[0], cache[2]), PO.held(cache[1], cache[3])


def tables(lengths, size, wide, seed=2, extra=2):
    """A table of pages in no order for sequences of these lengths, -1 behind them, and how many pages there are."""
    need = [-(-max(0, min(n, wide * size)) // size) for n in lengths]
    count = sum(need) + extra
    order = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), wide), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        for j in range(n):
            table[i, j] = order.pop()
    return table, count


def check_step(lengths, wide, size, hq, hkv, d, dtype, held, window=None, cap=None, slopes=False, scale=None, table=None, cache=None, seed=3):
    import lact_amd
    print("[gpu-test] paged step", lengths if len(lengths) < 20 else len(lengths), wide, size, hq, hkv, d, dtype, held, window, cap, slopes, flush=True)
    made, count = tables(lengths, size, wide)
    table = made if table is None else table
    cache = random_cache(count, hkv, size, d, held) if cache is None else cache
    q = torch.randn(len(lengths), hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype)
    sl = 2.0 ** -torch.arange(1, hq + 1).float() if slopes else None
    out = lact_amd.paged_attention_step(q.to("cuda"), cuda(cache), table.to("cuda"), torch.tensor(lengths, device="cuda"), window, score_cap=cap,
                                        distance_slopes=None if sl is None else sl.to("cuda"), scale=scale)
    l = min(max(lengths), wide * size) if lengths else 0
    ref, bound = PO.step(q, *numbers(cache), table, lengths, window, cap, sl, scale, *errors(dtype, held, max(1, l), d, 8.0 + (l if slopes else 0)))
    assert out.dtype == dtype
    near(out, ref, bound, "out")
    return out


# ---- the attention

@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,wide,size,hq,hkv,window", [
    ([1], 1, 16, 1, 1, None), ([16], 2, 16, 2, 1, None), ([17, 0, 15], 3, 16, 4, 2, None), ([33, 31, 32], 2, 32, 3, 3, None), ([100], 3, 48, 8, 1, 33),
    ([300, 129, 2, 0, 128], 20, 16, 6, 2, 200), ([511], 2, 256, 5, 1, None), ([700, 650], 9, 80, 40, 1, 37), ([260], 5, 64, 70, 2, None), ([257], 17, 16, 2, 2, 1)])
def test_step(lengths, wide, size, hq, hkv, window, d, dtype, held):
    check_step(lengths, wide, size, hq, hkv, d, dtype, held, window)


@KINDS
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 32, 33, 48, 127, 129])
def test_windows_that_begin_anywhere_in_a_piece(window, dtype, held):
    check_step([130, 131, 144, 160, 97], 12, 16, 2, 1, 64, dtype, held, window)


@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,slopes,scale", [(20.0, False, None), (None, True, None), (2.0, True, 0.3), (1e5, False, None)])
def test_step_with_cap_and_distance(cap, slopes, scale, d, dtype, held):
    check_step([170, 64, 3], 6, 32, 4, 2, d, dtype, held, 100, cap, slopes, scale)


@KINDS
def test_lengths_outside_the_table(dtype, held):
    """Negative lengths are none, longer ones end with the table, in 64 bits as well."""
    out = check_step([-5, 10 ** 9, 96, -2 ** 31, 2 ** 40], 3, 32, 2, 1, 64, dtype, held, 50, table=torch.tensor([[0, 1, 2]] * 5), cache=random_cache(4, 1, 32, 64, held))
    assert not out[0].any() and not out[3].any() and torch.equal(out[1].cpu()[0], out[1].cpu()[0])


@KINDS
@pytest.mark.parametrize("wide", [3, 50])
def test_lengths_past_the_table_are_its_end(wide, dtype, held):
    """The same query of every sequence, over the same pages: longer lengths, in 32 bits and past them, are the table's places bit by bit, and negative ones none."""
    import lact_amd
    size, ends = 32, wide * 32
    lengths = torch.tensor([ends, ends + 1, 10 ** 9, 2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 32 + 7, -1, -2 ** 31, -2 ** 40, -2 ** 32 + 7], device="cuda")
    cache = cuda(random_cache(wide, 1, size, 64, held))
    table = torch.randperm(wide, generator=torch.Generator().manual_seed(2)).expand(len(lengths), wide).to("cuda")
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(3)).to(dtype).to("cuda")
    for window in (None, 50):
        for n, t in ((lengths, table), (lengths.clamp(-2 ** 31, 2 ** 31 - 1).int(), table.int())):
            one = lambda i: lact_amd.paged_attention_step(q, cache, t[i:i + 1], n[i:i + 1], window)  # noqa: E731
            ref = one(0)
            assert bool(ref.any())
            for i in range(1, len(lengths)):
                assert torch.equal(one(i), ref if i < 7 else torch.zeros_like(ref)), (window, i)


@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("table,lengths,window", [
    ([[0, -1, 2, -1, 4, -1]], [96], None),                                # every other page
    ([[-1, -1, -1, -1, -1, -1]], [90], None),                             # none
    ([[-1, -1, 5, 6, 7, 1]], [91], 40),                                   # those that the window has left are gone
    ([[9, 10, 2 ** 31 - 1, -2 ** 31, 3, 4]], [85], None),                 # out of range
    ([[3, 4, 5, 6, 7, -1]], [90], None),                                  # the new token itself
    ([[3, 3, 3, 3, 3, 3], [3, 4, 3, 4, 3, 4]], [90, 96], None)])          # the same page again and again, and shared
def test_places_without_a_page(table, lengths, window, d, dtype, held):
    table = torch.tensor(table, dtype=torch.int32)
    out = check_step(lengths, 6, 16, 4, 2, d, dtype, held, window, table=table, cache=random_cache(8, 2, 16, d, held))
    if not (table >= 0).any():
        assert not out.any()


@KINDS
@pytest.mark.parametrize("wide", [4, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_reaches_nothing(d, wide, dtype, held):
    """Places past the length, in front of the window and on other pages hold NaN and infinities, exponents of NaN beside them."""
    import lact_amd
    print("[gpu-test] paged step, unseen", d, dtype, held, flush=True)
    size, lengths, window = 48, [100, 55, 1, 96], 37
    table, count = tables(lengths, size, wide)
    cache = random_cache(count, 2, size, d, held)
    q = torch.randn(len(lengths), 4, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    step = lambda c: lact_amd.paged_attention_step(q.to("cuda"), cuda(c), table.to("cuda"), torch.tensor(lengths, device="cuda"), window)  # noqa: E731
    seen = torch.zeros(count, size, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for j in range(max(0, n - window), n):
            seen[table[s, j // size], j % size] = True
    ref = step(cache)
    for bad in (math.nan, math.inf, -math.inf):
        spoilt = []
        for t in cache[:2]:
            f = t.float()
            f[~seen[:, None].expand(f.shape[:3])] = bad
            spoilt.append(f.to(t.dtype))
        for t in cache[2:]:
            spoilt.append(t if t is None else torch.where(seen[:, None].expand(t.shape), t.view(torch.uint8), torch.tensor(255, dtype=torch.uint8)).view(E8M0))
        assert torch.equal(step(spoilt), ref), bad


@KINDS
def test_seen_values_that_are_not_finite_are_seen(dtype, held):
    import lact_amd
    cache = random_cache(6, 2, 16, 64, held)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]])
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    for which in (0, 1):
        c = [t if t is None else t.clone() for t in cache]
        f = c[which].float()
        f[4, 1, 3, 7] = math.nan
        c[which] = f.to(held)
        out = lact_amd.paged_attention_step(q.to("cuda"), cuda(c), table.to("cuda"), torch.tensor([40, 40], device="cuda"))
        bad = torch.isnan(out).cpu()
        assert not bad[0].any() and not bad[1, :2].any()
        assert bool(bad[1, 2:].all() if which == 0 else bad[1, 2:, 7].all())


@pytest.mark.parametrize("held", [BF16, E4M3])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,size,hq,hkv,cap,slopes", [([700, 33, 1], 16, 4, 2, None, False), ([3000, 2600], 48, 5, 1, None, False), ([1500, 900], 16, 20, 1, 20.0, False), ([800], 16, 2, 1, None, True)])
def test_weights_keep_their_bits(lengths, size, hq, hkv, cap, slopes, d, held):
    """bf16 queries: what is stored is rounded to bf16, nothing in front of it.  The second part of a weight is at most 2^-7 of it, and off by 2^-8 of itself; the rest is fp32's, with three times as many
    terms as one part has, and twice the exponent's error where a distance adds to the score."""
    import lact_amd
    print("[gpu-test] paged step, weights", lengths, size, hq, hkv, d, held, cap, slopes, flush=True)
    table, count = tables(lengths, size, 4096 // size)
    cache = random_cache(count, hkv, size, d, held)
    q = torch.randn(len(lengths), hq, d, generator=torch.Generator().manual_seed(3)).to(BF16)
    sl = 2.0 ** -torch.arange(4, hq + 4).float() if slopes else None
    out = lact_amd.paged_attention_step(q.to("cuda"), cuda(cache), table.to("cuda"), torch.tensor(lengths, device="cuda"), score_cap=cap, distance_slopes=None if sl is None else sl.to("cuda"))
    p_err, _ = errors(F32, E4M3, max(lengths), d, 8.0 + (max(lengths) if slopes else 0))
    ref, bound = PO.step(q, *numbers(cache), table, lengths, None, cap, sl, None, 2.0 ** -15 + p_err, HALF[BF16])
    near(out, ref, bound, "out")


@KINDS
def test_step_of_many_parts_is_joined(dtype, held):
    check_step([i * 7 % 190 for i in range(600)], 12, 16, 4, 4, 64, dtype, held)


@KINDS
def test_step_of_a_long_sequence(dtype, held):
    """More pieces than the waves look up at once, in every block: one head of 70000 places, which a sequence of others splits in odd shares."""
    check_step([70000, 333, 4000], 70016 // 16, 16, 3, 1, 64, dtype, held)


@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,size,hq,hkv,window,cap,slopes", [
    ([0, 1500, 1, 0, 700, 16, 1100], 16, 5, 1, None, None, False),               # shares that begin and end anywhere, in front of a first step too
    ([1300, 20, 1290], 48, 17, 1, None, None, False), ([900, 1500], 16, 33, 1, 1200, None, True),      # more query heads to a key head than 16, and than 32
    ([1500, 0, 1400], 80, 32, 2, 1111, 20.0, False), ([0, 0, 0], 16, 2, 2, None, None, False), ([1], 16, 1, 1, None, None, False),
    ([1040, 0, 1030, 16, 17, 1200] * 20, 16, 4, 4, None, None, False),           # more sequences than a wave looks at at once
    ([i * 37 % 1500 if i % 3 else 0 for i in range(150)], 32, 6, 2, None, None, False)])
def test_shares_of_long_tables(lengths, size, hq, hkv, window, cap, slopes, d, dtype, held):
    """Tables wide enough that the work is cut into shares and joined."""
    check_step(lengths, 4096 // size, size, hq, hkv, d, dtype, held, window, cap, slopes)


@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq", [15, 16, 17, 31, 32, 33, 48, 49, 65])
def test_query_heads_of_one_key_head(hq, d, dtype, held):
    check_step([150, 77], 10, 16, hq, 1, d, dtype, held)


@KINDS
def test_places_without_a_page_in_shares(dtype, held):
    """Holes of a page and of long runs, in sequences that several blocks share; a sequence of holes alone."""
    g = torch.Generator().manual_seed(3)
    wide, size = 140, 16
    table = torch.randint(0, 60, (3, wide), generator=g, dtype=torch.int32)
    table[0, ::3] = -1
    table[1, 20:115] = 60
    table[2] = -1
    check_step([2200, 2111, 2240], wide, size, 4, 2, 64, dtype, held, table=table, cache=random_cache(60, 2, size, 64, held))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("wide", [4, 100])
def test_exponents_of_all_sizes(wide, dtype):
    """Keys that are small and large against each other, values whose powers of two differ by a hundred."""
    lengths, size, hkv, d = [60, 33], 16, 2, 64
    table, count = tables(lengths, size, wide)
    cache = random_cache(count, hkv, size, d, E4M3)
    g = torch.Generator().manual_seed(5)
    cache[2] = torch.randint(90, 122, cache[2].shape, generator=g).to(torch.uint8).view(E8M0)
    cache[3] = torch.randint(50, 150, cache[3].shape, generator=g).to(torch.uint8).view(E8M0)
    check_step(lengths, wide, size, 4, hkv, d, dtype, E4M3, table=table, cache=cache)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wide", [4, 100])
def test_a_seen_exponent_of_255_is_nan(wide, d, dtype):
    """The exponent that stands for NaN, beside numbers that are large, small and 0: of a key all its head's outputs are NaN, of a value as well; everybody else's stay."""
    import lact_amd
    print("[gpu-test] paged step, exponents of NaN", wide, d, dtype, flush=True)
    lengths, size = [60, 33], 16
    table, count = tables(lengths, size, wide)
    cache = random_cache(count, 2, size, d, E4M3)
    for t in cache[:2]:
        t.view(torch.uint8)[:, :, 5] = torch.tensor([0, 1, 0x80, 0x7e], dtype=torch.uint8).repeat(d // 4)
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    step = lambda c: lact_amd.paged_attention_step(q.to("cuda"), cuda(c), table.to("cuda"), torch.tensor(lengths, device="cuda")).cpu()  # noqa: E731
    ref = step(cache)
    for which in (2, 3):
        for place in (5, 31, 59):
            c = [t.clone() for t in cache]
            c[which].view(torch.uint8)[table[0, place // size], 1, place % size] = 255
            out = step(c)
            want, _ = PO.step(q, *numbers(c), table, lengths)
            assert torch.equal(torch.isnan(out), torch.isnan(want)) and bool(torch.isnan(out[0, 2:]).all()), (which, place)
            assert torch.equal(out[1], ref[1]) and torch.equal(out[0, :2], ref[0, :2])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wide,window", [(4, None), (4, 20), (100, None)])
def test_seen_values_that_are_infinite(wide, window, d, dtype):
    """Infinities of one sign among the values that are seen make that infinity, of both signs NaN, in the first and last places that are seen as anywhere else, beside places that are not."""
    import lact_amd
    lengths, size = [60, 33], 16
    print("[gpu-test] paged step, infinities", wide, window, d, dtype, flush=True)
    table, count = tables(lengths, size, wide)
    cache = random_cache(count, 2, size, d, dtype)
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(3)).to(dtype)
    for seq, places in ((0, (59,)), (0, (44,)), (0, (40, 47)), (1, (32,)), (1, (13,)), (1, (31, 32, 14))):
        c = [t if t is None else t.clone() for t in cache]
        for i, place in enumerate(places):
            c[1][table[seq, place // size], 1, place % size, 3 + i:9] = math.inf if i < 2 else -math.inf
        out = lact_amd.paged_attention_step(q.to("cuda"), cuda(c), table.to("cuda"), torch.tensor(lengths, device="cuda"), window).cpu().double()
        ref, bound = PO.step(q, *numbers(c), table, lengths, window, None, None, None, *errors(dtype, dtype, 60, d))
        assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(torch.isinf(out), torch.isinf(ref)) and bool((out[torch.isinf(ref)] == ref[torch.isinf(ref)]).all()), (seq, places)
        finite = torch.isfinite(ref)
        near(out[finite], ref[finite], bound[finite], f"{seq} {places}")


@KINDS
@pytest.mark.parametrize("wide", [32, 200])
def test_large_values_within_the_bound(wide, dtype, held):
    """500 places of values up to 2^109, in 8 bits of rows that hold as much, whose scores rise slowly: the running maximum lags behind them by up to 2^8."""
    import lact_amd
    size, d, n = 16, 64, 500
    table, count = tables([n], size, wide)
    cache = random_cache(count, 1, size, d, held)
    q = torch.full((1, 2, d), 0.25, dtype=dtype)
    for j in range(n):
        cache[0][table[0, j // size], 0, j % size] = 0.01 * j if held != E4M3 else torch.ones(d).to(held)
    if held == E4M3:
        for x, e in ((2, 0), (3, 100)):
            cache[x] = torch.full(cache[x].shape, 127 + e, dtype=torch.uint8).view(E8M0)
    else:
        cache[1] = ((torch.rand(cache[1].shape, generator=torch.Generator().manual_seed(8)) * 2 - 1) * 2.0 ** 109).to(held)
    out = lact_amd.paged_attention_step(q.to("cuda"), cuda(cache), table.to("cuda"), torch.tensor([n], device="cuda"))
    ref, bound = PO.step(q, *numbers(cache), table, [n], None, None, None, None, *errors(dtype, held, n, d, 16.0))
    near(out, ref, bound, "out")


@KINDS
def test_queries_and_tables_with_strides(dtype, held):
    import lact_amd
    lengths, size, hkv, d = [70, 33], 32, 2, 64
    table, count = tables(lengths, size, 3)
    cache = cuda(random_cache(count, hkv, size, d, held))
    q = torch.randn(4, 8, d, device="cuda").to(dtype)
    n = torch.tensor(lengths, device="cuda")
    wide = torch.stack((table, table + 1), -1).to("cuda")
    ref = lact_amd.paged_attention_step(q[::2, 1::2].contiguous(), cache, table.to("cuda"), n.int())
    assert torch.equal(lact_amd.paged_attention_step(q[::2, 1::2], cache, wide[..., 0], torch.stack((n, n), 1)[:, 1]), ref)
    odd = torch.cat((torch.zeros(1, device="cuda", dtype=dtype), q[::2, 1::2].flatten()))[1:].view(2, 4, d)
    assert torch.equal(lact_amd.paged_attention_step(odd, cache, table.long().to("cuda"), n), ref)


def test_long_share_of_one_block():
    """Batches of pages one after the other in the same wave: many heads, so that a block's share of 20000 places is longer than 64 pieces a wave."""
    import lact_amd
    n, size, hkv, d = 20000, 16, 300, 64
    print("[gpu-test] paged step, long shares", flush=True)
    wide = -(-n // size)
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(wide, hkv, size, d, generator=g, device="cuda", dtype=BF16)
    v = torch.randn(wide, hkv, size, d, generator=g, device="cuda", dtype=BF16)
    q = torch.randn(1, hkv, d, generator=g, device="cuda", dtype=BF16)
    table = torch.randperm(wide, generator=g, device="cuda").to(torch.int32)[None]
    table[0, 700] = -1
    out = lact_amd.paged_attention_step(q, lact_amd.PagedCache(k, v), table, torch.tensor([n - 3], device="cuda"))
    for h in (0, 7, 150, 299):
        one = [k[:, h:h + 1].cpu(), v[:, h:h + 1].cpu(), None, None]
        ref, bound = PO.step(q[:, h:h + 1].cpu(), *numbers(one), table.cpu(), [n - 3], None, None, None, None, *errors(BF16, BF16, n, d))
        near(out[:, h:h + 1], ref, bound, f"head {h}")


@pytest.mark.parametrize("held", [BF16, E4M3])
def test_pools_past_32_bits(held):
    """The last pages lie more than 2^32 bytes behind the first."""
    import lact_amd
    print("[gpu-test] paged cache, far pages", held, flush=True)
    size, hkv, d = 256, 8, 128
    pages = (2 ** 32 // (size * hkv * d * (1 if held == E4M3 else 2))) + 9
    cache = lact_amd.PagedCache.empty(pages, hkv, size, d, dtype=held)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, 600, hkv, d, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(1, 2 * hkv, d, generator=g).to(BF16)
    lact_amd.paged_cache_write(cache, k.to("cuda"), v.to("cuda"), table)
    out = lact_amd.paged_attention_step(q.to("cuda"), cache, table, torch.tensor([600], device="cuda"))
    near_cache = lact_amd.PagedCache.empty(3, hkv, size, d, dtype=held)
    near_table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    lact_amd.paged_cache_write(near_cache, k.to("cuda"), v.to("cuda"), near_table)
    assert torch.equal(out, lact_amd.paged_attention_step(q.to("cuda"), near_cache, near_table, torch.tensor([600], device="cuda")))
    n = torch.tensor([600], device="cuda")
    for a, b in zip(lact_amd.paged_cache_read(cache, table, n, 600), lact_amd.paged_cache_read(near_cache, near_table, n, 600)):
        assert torch.equal(a, b)


@KINDS
def test_keys_and_values_in_one_pool(dtype, held):
    """[pages, 2, heads, size, d]: pages further apart than they are long."""
    import lact_amd
    size, hkv, d, lengths = 32, 2, 64, [70, 33]
    table, count = tables(lengths, size, 3)
    cache = random_cache(count, hkv, size, d, held)
    join = lambda a, b: torch.stack((a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b), 1).to("cuda")  # noqa: E731
    pool = join(cache[0], cache[1])
    views = [pool[:, 0].view(held), pool[:, 1].view(held), None, None]
    if held == E4M3:
        exps = join(cache[2], cache[3])
        views[2:] = [exps[:, 0].view(E8M0), exps[:, 1].view(E8M0)]
    views = lact_amd.PagedCache(*views)
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(3)).to(dtype).to("cuda")
    n = torch.tensor(lengths, device="cuda")
    apart = cuda(cache)
    assert torch.equal(lact_amd.paged_attention_step(q, views, table.to("cuda"), n), lact_amd.paged_attention_step(q, apart, table.to("cuda"), n))
    new = [torch.randn(2, 20, hkv, d, generator=torch.Generator().manual_seed(i)).to(dtype).to("cuda") for i in (7, 8)]
    for c in (views, apart):
        lact_amd.paged_cache_write(c, *new, table.to("cuda"), torch.tensor([11, 5], device="cuda"))
    for a, b in zip(views, apart):
        assert a is None or torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))
    kw = dict(dtype=dtype) if held == E4M3 else {}
    for a, b in zip(lact_amd.paged_cache_read(views, table.to("cuda"), n, 80, **kw), lact_amd.paged_cache_read(apart, table.to("cuda"), n, 80, **kw)):
        assert torch.equal(a, b)


@KINDS
@pytest.mark.parametrize("hkv,size", [(3, 32), (12, 16), (2, 48), (3, 80)])
def test_pools_of_any_page_length(hkv, size, dtype, held):
    """One record a page: keys, values, their exponents and room behind them, from which the tokens come; and [pages, 2, ...]."""
    import lact_amd
    d, lengths, l = 64, [2 * size + 6, size + 1], 20
    print("[gpu-test] paged cache, records", hkv, size, dtype, held, flush=True)
    table, count = tables(lengths, size, 3)
    plain = random_cache(count, hkv, size, d, held)
    tail = 2 * 2 * l * hkv * d * dtype.itemsize                                      # of one page's room
    parts = [t.reshape(count, -1).view(torch.uint8) for t in plain if t is not None]
    pool = torch.cat((*parts, torch.zeros(count, tail, dtype=torch.uint8)), 1).to("cuda")
    ends = torch.tensor([p.shape[1] for p in parts]).cumsum(0).tolist()
    part = lambda i: pool[:, ends[i] - parts[i].shape[1]:ends[i]]  # noqa: E731
    record = lact_amd.PagedCache(*(None if t is None else part(i).view(t.dtype).unflatten(1, t.shape[1:]) for i, t in enumerate(plain)))
    codes = torch.stack(parts[:2], 1).to("cuda")
    exps = torch.stack(parts[2:], 1).to("cuda") if held == E4M3 else None
    both = lact_amd.PagedCache(*(codes[:, i].view(held).unflatten(1, plain[0].shape[1:]) for i in range(2)),
                               *(None if exps is None else exps[:, i].view(E8M0).unflatten(1, plain[2].shape[1:]) for i in range(2)))
    apart = cuda(plain)
    assert record.k.data_ptr() == pool.data_ptr() and record.v.stride(0) * held.itemsize == pool.stride(0) and both.v.data_ptr() == codes[:, 1].data_ptr()
    room = pool[1, ends[-1]:].view(dtype).view(2, 2, l, hkv, d)
    room.copy_(torch.randn(2, 2, l, hkv, d, generator=torch.Generator().manual_seed(5)))
    new, starts, n = room.clone(), torch.tensor([size - 5, 1], device="cuda"), torch.tensor(lengths, device="cuda")
    q = torch.randn(2, 2 * hkv, d, generator=torch.Generator().manual_seed(3)).to(dtype).to("cuda")
    table = table.to("cuda")
    lact_amd.paged_cache_write(apart, *new, table, starts)
    ref = lact_amd.paged_attention_step(q, apart, table, n)
    for cache, tokens in ((record, room), (both, new)):
        lact_amd.paged_cache_write(cache, *tokens, table, starts)
        for a, b in zip(cache, apart):
            assert a is None or torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(lact_amd.paged_attention_step(q, cache, table, n), ref)
        for a, b in zip(lact_amd.paged_cache_read(cache, table, n, 3 * size, dtype=dtype), lact_amd.paged_cache_read(apart, table, n, 3 * size, dtype=dtype)):
            assert torch.equal(a, b)
    assert torch.equal(room, new)
    for name in ("v", "v_scale") if held == E4M3 else ("v",):
        t = getattr(record, name)
        off = t.storage_offset() - 16 // t.element_size()
        bad = record._replace(**{name: t.as_strided(t.shape, t.stride(), off)})
        with pytest.raises(RuntimeError, match="must not overlap"):
            lact_amd.paged_cache_write(bad, *new, table, starts)
    with pytest.raises(RuntimeError, match="must not lie in the cache"):
        lact_amd.paged_cache_write(record, pool[1, ends[-1] - 16:ends[-1] - 16 + tail // 2].view(dtype).view(2, l, hkv, d)[:1], new[1][:1], table[:1], starts[:1])


# ---- writing and reading

def places_written(table, pages, size, starts, counts, l):
    for s in range(len(table)):
        for i in range(min(l, counts[s])):
            p = PO.page_of(table, pages, size, s, starts[s] + i)
            if p >= 0:
                yield s, i, p, (starts[s] + i) % size


@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,l,hkv,size,starts,counts", [
    (1, 1, 1, 16, None, None), (2, 33, 3, 16, [5, 0], None), (3, 70, 2, 32, [0, 31, 90], [70, 0, 13]), (2, 40, 1, 48, [-7, 130], [40, 2 ** 31 - 1]),
    (5, 1, 4, 64, [0, 63, 64, 191, 192], [1, 1, 0, 1, 1]), (1, 300, 2, 16, [2 ** 31 - 100], None), (3, 130, 1, 32, [3, 77, -20], [100, 130, 64]),
    (2, 64, 2, 48, [15, 0], None)])
def test_write_puts_tokens_into_their_places(b, l, hkv, size, starts, counts, d, dtype, held):
    """Bit by bit, and nothing else changes."""
    import lact_amd
    print("[gpu-test] paged write", b, l, hkv, size, starts, counts, d, dtype, held, flush=True)
    wide = 6
    pages = b * wide + 2
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:b * wide].reshape(b, wide).to(torch.int32)
    table[0, 2] = -1
    table[b - 1, 3] = pages
    cache = random_cache(pages, hkv, size, d, held)
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(b, l, hkv, d, generator=g).to(dtype) * torch.exp2(torch.randint(-20, 20, (b, l, hkv, 1), generator=g).float()).to(dtype) for _ in range(2))
    dev = lambda t: None if t is None else torch.tensor(t, device="cuda")  # noqa: E731
    on = cuda(cache)
    lact_amd.paged_cache_write(on, k.to("cuda"), v.to("cuda"), table.to("cuda"), dev(starts), dev(counts))
    want = [t if t is None else t.view(torch.uint8).clone() if held == E4M3 else t.clone() for t in cache]
    new = [PO.to_8_bits(t) for t in (k, v)] if held == E4M3 else [(k, None), (v, None)]
    for s, i, p, r in places_written(table, pages, size, starts or [0] * b, counts or [l] * b, l):
        for x in range(2):
            want[x][p, :, r] = new[x][0][s, i]
            if held == E4M3:
                want[2 + x][p, :, r] = new[x][1][s, i]
    for name, a, r in zip(("k", "v", "k_scale", "v_scale"), on, want):
        if r is not None:
            a = a.cpu().view(torch.uint8) if held == E4M3 else a.cpu()
            assert torch.equal(a, r), (name, int((a != r).sum()))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rounding_to_8_bits(dtype):
    """Every number and midpoint of e4m3, with rows whose largest magnitude lies on, just below and just above every border of the exponent; zeros, the smallest and largest
    numbers, and what is not finite."""
    import lact_amd
    d = 64
    values = PO.e4m3_values()[:127]
    points = torch.cat((values, (values[1:] + values[:-1]) / 2)).float()
    points = torch.cat((points, torch.nextafter(points, torch.tensor(1e9)), torch.nextafter(points, torch.tensor(-1.0))))
    points = torch.cat((points, -points))
    points = torch.cat((points, points.new_zeros(-len(points) % (d - 1)))).reshape(-1, d - 1)
    rows = []
    for top in (448.0, 447.0, 256.0, 449.0):
        rows.append(torch.cat((points.clamp(-top, top), torch.full((len(points), 1), top)), 1))
    rows = torch.cat(rows)
    scales = torch.exp2(torch.randint(-110, 110, (len(rows), 1), generator=torch.Generator().manual_seed(1)).float())
    more = torch.zeros(10, d)
    more[1, 5] = 2.0 ** -149
    more[2, 5], more[2, 6] = 2.0 ** -126, -2.0 ** -130
    more[3] = 3e38
    more[4, 3], more[4, 7] = math.inf, 1.5
    more[5, 3], more[5, 7] = math.nan, -2.5
    more[6] = -math.inf
    more[7, 0] = -0.0
    more[8, 0], more[8, 1] = 2.0 ** -119, 2.0 ** -120
    more[9, 0], more[9, 1] = 448 * 2.0 ** -127, 449 * 2.0 ** -130
    rows = torch.cat((rows * scales, rows, more)).to(dtype)
    n, size = len(rows), 16
    cache = lact_amd.PagedCache.empty(-(-n // size), 1, size, d, dtype=E4M3)
    table = torch.arange(cache.k.shape[0], device="cuda")[None]
    lact_amd.paged_cache_write(cache, rows[None, :, None].to("cuda"), rows.flip(0)[None, :, None].to("cuda"), table)
    code, exponent = PO.to_8_bits(rows)
    nan = (code & 127) == 127
    for got, exp, c, e, is_nan in ((cache.k, cache.k_scale, code, exponent, nan), (cache.v, cache.v_scale, code.flip(0), exponent.flip(0), nan.flip(0))):
        got, exp = got.cpu().view(torch.uint8).reshape(-1, d)[:n], exp.cpu().view(torch.uint8).reshape(-1)[:n]
        assert torch.equal(exp, e)
        assert torch.equal(got[~is_nan], c[~is_nan]) and bool(((got[is_nan] & 127) == 127).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_reading_every_number_of_8_bits(dtype):
    """256 codes under 256 exponents."""
    import lact_amd
    d, size = 128, 256
    codes = torch.arange(256, dtype=torch.uint8).reshape(2, 1, d).expand(2, size, d)[None].contiguous().view(E4M3)
    exps = torch.arange(256, dtype=torch.uint8).expand(1, 2, size).contiguous().view(E8M0)
    cache = cuda((codes, codes, exps, exps))
    k, v = lact_amd.paged_cache_read(cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([size], device="cuda"), size, dtype=dtype)
    want = PO.held(codes, exps)[0].transpose(0, 1).float().to(dtype)[None]      # (exact in fp32, but past its ends)
    for t in (k, v):
        t = t.cpu()
        assert torch.equal(torch.isnan(t), torch.isnan(want)) and torch.equal(t[~torch.isnan(t)], want[~torch.isnan(want)])


def test_the_smallest_numbers_of_8_bits():
    """Under exponents of 0 to 3 the codes 0 to 8 are multiples of 2^-136 to 2^-133: fp32 has them all, bf16 those of 2^-133, and others to nearest, ties to even."""
    import lact_amd
    d, size = 64, 16
    codes = (torch.arange(d, dtype=torch.uint8) % 9).expand(1, 1, size, d).contiguous().view(E4M3)
    exps = (torch.arange(size, dtype=torch.uint8) % 4).expand(1, 1, size).contiguous().view(E8M0)
    table, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([size], device="cuda")
    want = (torch.arange(d) % 9)[None] * 2 ** (torch.arange(size) % 4)[:, None]                # in 2^-136
    for dtype, w in ((F32, want.double() * 2.0 ** -136), (BF16, torch.round(want.double() / 8) * 2.0 ** -133)):
        for t in lact_amd.paged_cache_read(cuda((codes, codes, exps, exps)), table, n, size, dtype=dtype):
            assert torch.equal(t[0, :, 0].double().cpu(), w), dtype
    small = torch.full((1, 1, d), 5 * 2.0 ** -133)                                             # written, its row's exponent is 0
    cache = lact_amd.PagedCache.empty(1, 1, size, d, dtype=E4M3)
    lact_amd.paged_cache_write(cache, small.to("cuda"), small.to("cuda"), table)
    assert int(cache.k_scale.view(torch.uint8)[0, 0, 0]) == 0
    for dtype in (F32, BF16):
        assert bool((lact_amd.paged_cache_read(cache, table, n, 1, dtype=dtype)[1].double() == 5 * 2.0 ** -133).all())


@KINDS
@pytest.mark.parametrize("hkv", [1, 2, 3])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("starts,lengths,tokens", [(None, [100, 33, 0], 100), ([10, 0, 96], [90, 200, 97], 64), ([-5, 2 ** 31 - 1, 100], [50, 2 ** 31 - 1, 100], 70), ([3, 4, 5], [7, 4, 6], 1)])
def test_read(starts, lengths, tokens, d, hkv, dtype, held):
    import lact_amd
    print("[gpu-test] paged read", starts, lengths, tokens, d, hkv, dtype, held, flush=True)
    size = 32
    table = torch.tensor([[0, 5, -1, 2], [7, 7, 1, 9], [3, 4, 10, 6]], dtype=torch.int32)
    cache = random_cache(10, hkv, size, d, held)
    dev = lambda t: None if t is None else torch.tensor(t, device="cuda")  # noqa: E731
    got = lact_amd.paged_cache_read(cuda(cache), table.to("cuda"), dev(lengths), tokens, dev(starts), dtype=dtype)
    for a, n in zip(got, numbers(cache)):
        want, _ = PO.tokens(n, table, starts or [0] * 3, lengths, tokens)
        assert a.dtype == dtype and torch.equal(a.double().cpu(), want)      # (what 8 bits hold is exact in bf16)


def test_default_types_of_what_is_read():
    import lact_amd
    table, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for held, want in ((BF16, BF16), (F32, F32), (E4M3, BF16)):
        assert lact_amd.paged_cache_read(cuda(random_cache(1, 1, 16, 64, held)), table, n, 1)[0].dtype == want


@KINDS
def test_views_strides_and_one_token(dtype, held):
    """Tokens as parts of a packed projection, with strides of their own, off their alignment, without a dimension for one token."""
    import lact_amd
    b, l, hkv, d, size = 2, 19, 3, 64, 16
    g = torch.Generator().manual_seed(2)
    packed = torch.randn(b, l, 2 * hkv * d + 8, generator=g).to(dtype).to("cuda")
    k, v = (t.reshape(b, l, hkv, d) for t in packed[..., :2 * hkv * d].split(hkv * d, -1))
    odd = torch.randn(b * l * hkv * d + 1, generator=g).to(dtype).to("cuda")[1:].view(b, l, hkv, d)
    turned = torch.randn(b, hkv, l, d, generator=g).to(dtype).to("cuda").transpose(1, 2)
    shared = torch.randn(1, l, hkv, d, generator=g).to(dtype).to("cuda").expand(b, l, hkv, d)
    table = torch.randperm(6, generator=g).reshape(b, 3).to("cuda")
    starts = torch.tensor([3, 20], device="cuda")
    for a, c in ((k, v), (odd, turned), (shared, k)):
        one, two, three = (lact_amd.PagedCache(*(None if t is None else t.view(torch.uint8).zero_().view(t.dtype) for t in lact_amd.PagedCache.empty(6, hkv, size, d, dtype=held)))
                           for _ in range(3))
        lact_amd.paged_cache_write(one, a, c, table, starts)
        lact_amd.paged_cache_write(two, a.contiguous(), c.contiguous(), table, starts)
        for i in range(l):
            lact_amd.paged_cache_write(three, a[:, i], c[:, i], table, starts + i)
        for x, y, z in zip(one, two, three):
            assert x is None or (torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and torch.equal(x.view(torch.uint8), z.view(torch.uint8)))


# ---- together, and what a caller may do

@KINDS
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_and_tokens_agree(d, dtype, held):
    """Positions, a prompt through the attention and into the cache, then token after token: the attention over all of what the cache holds."""
    import lact_amd
    print("[gpu-test] prompt and tokens", d, dtype, held, flush=True)
    b, l, hq, hkv, prompt, window, size = 2, 90, 4, 2, 70, 50, 16
    axes = (d // 2, d // 4, d // 4)
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(b, l, n, d, generator=g).to(dtype).to("cuda") for n in (hq, hkv, hkv))
    places = torch.stack((torch.arange(l) // 30, torch.arange(l) // 6 % 5, torch.arange(l) % 6), -1).to(torch.int32).to("cuda")
    sl = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    opts = dict(score_cap=10.0, distance_slopes=sl)
    cache = lact_amd.PagedCache.empty(14, hkv, size, d, dtype=held)
    for t in cache:
        if t is not None:
            t.view(torch.uint8).fill_(255)                     # NaN in all types
    table = torch.randperm(14, generator=g)[:12].reshape(b, 6).to("cuda")
    with torch.no_grad():
        qp, kp = lact_amd.axial_rotary(q[:, :prompt], k[:, :prompt], places[:prompt], axes)
        lact_amd.paged_cache_write(cache, kp, v[:, :prompt], table)
        full = torch.full((b,), prompt, dtype=torch.int32, device="cuda")
        kc, vc = lact_amd.paged_cache_read(cache, table, full, prompt, dtype=dtype)
        outs = [lact_amd.masked_window_attention(qp, kc, vc, window, **opts)]
        for t in range(prompt, l):
            q1, k1 = lact_amd.axial_rotary(q[:, t], k[:, t], places[t].expand(b, 3), axes)
            n = torch.full((b,), t, dtype=torch.int32, device="cuda")
            lact_amd.paged_cache_write(cache, k1, v[:, t], table, n)
            outs.append(lact_amd.paged_attention_step(q1, cache, table, n + 1, window, **opts)[:, None])
        qr, kr = lact_amd.axial_rotary(q, k, places, axes)
        full += l - prompt
        kc, vc = lact_amd.paged_cache_read(cache, table, full, l, dtype=dtype)
    for a, r in ((kc, kr), (vc, v)):
        if held == E4M3:
            code, e = PO.to_8_bits(r.cpu())
            assert torch.equal(a.double().cpu(), PO.held(code, e))
        else:
            assert torch.equal(a, r)
    ref, bound = MO.attention(qr.cpu(), kc.cpu(), vc.cpu(), window, 10.0, sl.cpu(), None, None, None, None, *errors(dtype, held, l, d, 8.0 + l))
    near(torch.cat(outs, 1), ref, bound, "out")


@KINDS
@pytest.mark.parametrize("wide", [8, 100])
def test_captured_tokens(wide, dtype, held):
    """Positions, writing and attention captured once and replayed while the sequences grow and their tables change; eager calls and other work in between."""
    import lact_amd
    b, hq, hkv, d, size = 3, 4, 2, 64, 16
    q, k, v = (torch.randn(b, n, d, device="cuda").to(dtype) for n in (hq, hkv, hkv))
    caches = [lact_amd.PagedCache(*(None if t is None else t.view(torch.uint8).zero_().view(t.dtype) for t in lact_amd.PagedCache.empty(b * wide, hkv, size, d, dtype=held)))
              for _ in range(2)]
    table = torch.randperm(b * wide, device="cuda").reshape(b, wide).to(torch.int32)
    lengths = torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")
    places = torch.zeros(b, 2, dtype=torch.int32, device="cuda")

    def token(cache):
        q1, k1 = lact_amd.axial_rotary(q, k, places, (32, 32))
        lact_amd.paged_cache_write(cache, k1, v, table, lengths)
        return lact_amd.paged_attention_step(q1, cache, table, lengths + 1, 60)

    with torch.no_grad():
        token(caches[0])
        token(caches[1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = token(caches[0])
        for i in range(6):
            for t in (q, k, v):
                t.copy_(torch.randn_like(t.float()))
            places += 3
            if i == 3:
                table[1] = torch.flip(table[1], (0,))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, token(caches[1])), i
            for x, y in zip(*caches):
                assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            lengths += 1


@KINDS
def test_other_streams_give_the_same(dtype, held):
    """Calls on two streams at once, with workspaces of their own."""
    import lact_amd
    lengths, size, hkv, d = [900, 64, 1300], 32, 2, 128
    table, count = tables(lengths, size, 41)
    cache = cuda(random_cache(count, hkv, size, d, held))
    table, n = table.to("cuda"), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(3, 8, d, device="cuda").to(dtype) for _ in range(2)]
    refs = [lact_amd.paged_attention_step(q, cache, table, n) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(lact_amd.paged_attention_step(qs[i], cache, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, refs[i]) for i in range(2) for o in outs[i])


def test_writing_raises_the_version():
    import lact_amd
    cache = lact_amd.PagedCache.empty(2, 1, 16, 64, dtype=E4M3)
    before = [t._version for t in cache]
    x = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    lact_amd.paged_cache_write(cache, x, x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    assert [t._version for t in cache] == [n + 1 for n in before]
    with torch.inference_mode():
        kept = lact_amd.PagedCache.empty(2, 1, 16, 64)
        lact_amd.paged_cache_write(kept, x, x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))


def test_nothing_to_do():
    import lact_amd
    cache = lact_amd.PagedCache.empty(2, 2, 16, 64)
    none = lact_amd.PagedCache.empty(0, 2, 16, 64)
    table, n = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(3, 4, 64, device="cuda", dtype=BF16), torch.zeros(3, 5, 2, 64, device="cuda", dtype=BF16)
    for c, t in ((none, table), (cache, table[:, :0])):
        assert not lact_amd.paged_attention_step(q, c, t, n).any()
        assert not any(x.any() for x in lact_amd.paged_cache_read(c, t, n, 5))
        lact_amd.paged_cache_write(c, k, k, t)
    lact_amd.paged_cache_write(cache, k[:, :0], k[:, :0], table)
    lact_amd.paged_cache_write(cache, k[:0], k[:0], table[:0])
    assert lact_amd.paged_attention_step(q[:0], cache, table[:0], n[:0]).shape == (0, 4, 64)
    assert lact_amd.paged_cache_read(cache, table, n, 0)[1].shape == (3, 0, 2, 64)


def test_refusals_on_the_gpu():
    import lact_amd
    cache = lact_amd.PagedCache.empty(4, 2, 16, 64)
    eight = lact_amd.PagedCache.empty(4, 2, 16, 64, dtype=E4M3)
    table, n = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(3, 4, 64, device="cuda", dtype=BF16), torch.zeros(3, 5, 2, 64, device="cuda", dtype=BF16)
    odd = torch.zeros(4 * 2 * 16 * 64 + 1, device="cuda", dtype=BF16)[1:].view(4, 2, 16, 64)
    wide = torch.zeros(4, 2, 16, 128, device="cuda", dtype=BF16)
    of = lambda c, **kw: c._replace(**kw)  # noqa: E731
    for f, good, bad in (
            (lact_amd.paged_attention_step, dict(q=q, cache=cache, page_table=table, lengths=n), [
                (dict(q=q.float()), TypeError), (dict(q=q.half()), TypeError), (dict(q=q[..., :32]), ValueError), (dict(q=q[:, :3]), RuntimeError),
                (dict(page_table=table[:2]), ValueError), (dict(page_table=table.float()), TypeError), (dict(page_table=table.cpu()), RuntimeError), (dict(lengths=n[:1]), ValueError),
                (dict(lengths=n.float()), TypeError), (dict(cache=of(cache, v=cache.v[:3])), ValueError), (dict(cache=of(cache, v=cache.v.float())), TypeError),
                (dict(cache=of(cache, k=cache.k.cpu())), RuntimeError), (dict(cache=of(cache, k=odd)), ValueError), (dict(cache=of(cache, k=wide[..., ::2])), ValueError),
                (dict(cache=of(cache, k_scale=eight.k_scale)), ValueError), (dict(cache=of(eight, v_scale=None)), ValueError), (dict(cache=of(eight, k_scale=eight.k_scale[:, :1])), ValueError),
                (dict(cache=of(eight, k_scale=eight.k_scale.view(torch.uint8))), TypeError), (dict(distance_slopes=torch.zeros(3, device="cuda")), ValueError),
                (dict(cache=lact_amd.PagedCache.empty(4, 2, 24, 64)), RuntimeError), (dict(cache=lact_amd.PagedCache.empty(4, 2, 16, 96), q=torch.zeros(3, 4, 96, device="cuda", dtype=BF16)), RuntimeError),
                (dict(cache=of(cache, k=cache.k[:1].expand(4, 2, 16, 64))), RuntimeError)]),
            (lact_amd.paged_cache_write, dict(cache=cache, k=k, v=k, page_table=table), [
                (dict(k=k.float()), TypeError), (dict(k=k[..., :1, :]), ValueError), (dict(v=k[:, :4]), ValueError), (dict(starts=n[:2]), ValueError), (dict(counts=n.cpu()), RuntimeError),
                (dict(starts=n.float()), TypeError), (dict(cache=of(cache, v=cache.k)), RuntimeError), (dict(k=cache.k.flatten()[:3 * 5 * 128].view(3, 5, 2, 64)), RuntimeError),
                (dict(page_table=table[:, 0]), ValueError)]),
            (lact_amd.paged_cache_read, dict(cache=cache, page_table=table, lengths=n, tokens=5), [
                (dict(dtype=F32), TypeError), (dict(cache=eight, dtype=torch.float16), TypeError), (dict(lengths=n[:2]), ValueError), (dict(starts=n.cpu()), RuntimeError)])):
        f(**good)
        for kw, error in bad:
            with pytest.raises(error):
                f(**{**good, **kw})
                print(f.__name__, {x: getattr(y, "shape", y) for x, y in kw.items()}, flush=True)
    for c in (cache, eight):
        leaf = of(c, k=c.k.float().requires_grad_(True))
        with pytest.raises(RuntimeError, match="inference"):
            lact_amd.paged_attention_step(q.float(), leaf, table, n)


@pytest.mark.parametrize("given", [BF16, F32])
@pytest.mark.parametrize("held", [BF16, F32, E4M3])
def test_autocast_takes_what_the_pages_hold(held, given):
    """Under autocast tokens and queries of either type go with pages of any: cast to the pages' type; 8 bits take tokens as they are, and queries of autocast's type."""
    import lact_amd
    size, hkv, d = 16, 2, 64
    table, starts = torch.tensor([[0, 1], [2, 3]], device="cuda"), torch.tensor([0, 9], device="cuda")
    k, v, q = (torch.randn(2, *n, d, device="cuda").to(given) for n in ((20, hkv), (20, hkv), (4,)))
    n = torch.tensor([20, 29], device="cuda")
    empty = lambda: lact_amd.PagedCache(*(None if t is None else t.view(torch.uint8).zero_().view(t.dtype) for t in lact_amd.PagedCache.empty(4, hkv, size, d, dtype=held)))  # noqa: E731
    write = given if held == E4M3 else held
    ask = BF16 if held == E4M3 else held
    with torch.autocast("cuda", BF16):
        one = empty()
        lact_amd.paged_cache_write(one, k, v, table, starts)
        lact_amd.paged_cache_write(one, k[:, 0], v[:, 0], table, n)
        out = lact_amd.paged_attention_step(q, one, table, n + 1)
        back = lact_amd.paged_cache_read(one, table, n, 30)
    two = empty()
    lact_amd.paged_cache_write(two, k.to(write), v.to(write), table, starts)
    lact_amd.paged_cache_write(two, k[:, 0].to(write), v[:, 0].to(write), table, n)
    ref = lact_amd.paged_attention_step(q.to(ask), two, table, n + 1)
    for a, b in ((out, ref), *zip(back, lact_amd.paged_cache_read(two, table, n, 30)), *zip(one, two)):
        assert a is None or (a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8)))
    if held != E4M3:
        assert out.dtype == held
        other = F32 if held == BF16 else BF16
        with pytest.raises(TypeError):      # and nothing is cast without it
            lact_amd.paged_attention_step(q.to(other), two, table, n)
        with pytest.raises(TypeError):
            lact_amd.paged_cache_write(two, k.to(other), v.to(other), table, starts)
