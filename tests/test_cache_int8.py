"""The cache in 8 bits: what is written into it, exactly; attention over it, against the formula in
64 bits over the values that it holds, with the bounds of tests/_attention64.py; and a cache of any
type read back.

The bounds hold as they are. A key n times its scale is exact in 64 bits; here q is in three bf16
parts (2^-25 of it) and n exact, the sum's products as many as for other caches, and the scale adds
one rounding, u |s|, where the bound counts two for the second factor's parts. The same for a weight
times its scale of V, of which the bound's m + 5 terms count five that are not additions."""
import ctypes as C
import math

import pytest

import ehip as E
from _attention64 import packed, within
from _hip import print_case

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU test ran without a visible GPU")
    return E.Backend()


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def quantised(x):
    """(codes, scales) on the CPU: the scale in 32 bits, the quotient in 64."""
    import torch
    x = x.detach().cpu()
    top = x.abs().amax(-1)
    scale = (top.numpy() / top.new_tensor(127.0).numpy())
    scale = torch.from_numpy(scale.copy() if hasattr(scale, "copy") else scale)
    fine = torch.isfinite(x).all(-1)
    scale = torch.where(torch.isinf(scale * 127) & fine,
                        torch.nextafter(scale, torch.zeros_like(scale)), scale)
    scale = torch.where(fine, scale, torch.full_like(scale, math.nan))
    safe = torch.where((scale > 0) & fine, scale, torch.ones_like(scale)).double()
    n = torch.round(torch.where(fine[..., None], x, torch.zeros_like(x)).double() / safe[..., None])
    n = torch.where((scale > 0)[..., None], n.clamp(-127, 127), torch.zeros_like(n))
    return n.to(torch.int8), scale


def pools(pages, page, kv, d, kind="int8", fill=0):
    """Empty (k_pages, v_pages, scales) that hold `fill` where nothing was written."""
    import torch
    dtype = getattr(torch, kind)
    made = [torch.full((pages, page, kv, d), fill, dtype=dtype, device="cuda") for _ in range(2)]
    scales = None
    if kind == "int8":
        scales = tuple(torch.full((pages, kv, page), float(fill), device="cuda") for _ in range(2))
    return (*made, scales)


def table_of(lengths, page, gen, spare=2, extra=1):
    import torch
    each = [-(-n // page) for n in lengths]
    count = sum(each) + spare
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), max(each + [0]) + extra, dtype=torch.int32, device="cuda")
    at = 0
    for s, m in enumerate(each):
        table[s, :m] = order[at:at + m]
        at += m
    return table, count


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return ints(out)


def held(pool, scales, table, lengths):
    """The values of each sequence's positions in 64 bits on the CPU."""
    import torch
    x = pool.cpu().double()
    if scales is not None:
        x = x * scales.cpu().double().transpose(1, 2)[..., None]
    x = x.reshape(-1, *x.shape[2:])
    page = pool.shape[1]
    out = []
    for s, n in enumerate(lengths):
        p = torch.arange(n)
        out.append(x[table[s].cpu().long()[p // page] * page + p % page])
    return out


def fill(hip, lengths, kv, d, page, seed=0, spread=1.0, kind="int8"):
    """A cache into which sequences of these lengths were written."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table, count = table_of(lengths, page, gen)
    kp, vp, scales = pools(count, page, kv, d, kind)
    n = sum(lengths)
    k, v = (torch.randn(n, kv, d, generator=gen, device="cuda") * spread for _ in range(2))
    hip.cache_append(k, v, kp, vp, table, ints([0] * len(lengths)), offsets(lengths), scales=scales)
    return kp, vp, scales, table, k, v


# ------------------------------------------------------------------- append

@gpu
@pytest.mark.parametrize("kv,d,page", [(1, 1, 1), (3, 2, 4), (2, 5, 16), (1, 16, 8), (2, 17, 16),
                                       (2, 24, 16), (5, 31, 3), (8, 32, 16), (3, 33, 7), (2, 63, 16),
                                       (16, 64, 16), (1, 77, 16), (4, 96, 100), (8, 128, 32),
                                       (40, 127, 2)])
def test_append_is_exact(hip, kv, d, page):
    import torch
    print_case("append8", kv, d, page)
    lengths = [0, 1, 37, 5, 2 * page, 64]
    kp, vp, scales, table, k, v = fill(hip, lengths, kv, d, page, seed=d)
    for pool, sc, x in ((kp, scales[0], k), (vp, scales[1], v)):
        codes, scale = quantised(x)
        at = 0
        for s, n in enumerate(lengths):
            for p in range(0, n, max(1, n // 9)):
                where = int(table[s, p // page]), p % page
                assert torch.equal(pool[where].cpu(), codes[at + p])
                assert torch.equal(sc[where[0], :, where[1]].cpu(), scale[at + p])
            at += n
        whole = held(pool, None, table, lengths)
        assert torch.equal(torch.cat(whole), codes.double())
    used = sum(lengths) * kv
    assert int((scales[0] != 0).sum()) == used and int((scales[1] != 0).sum()) == used


@gpu
def test_append_where_it_is_hard(hip):
    """Ties, quotients next to a half, scales of few bits, subnormal and largest values, zeros."""
    import torch
    print_case("append8 hard")
    gen = torch.Generator().manual_seed(1)
    rows = [torch.arange(-64, 64).float(),                       # scale 64 / 127
            torch.arange(-63.5, 64.5, 1.0) * 2 - 1,              # scale 1 (127): whole numbers
            (torch.arange(-64, 64).float() + 0.5) * 127 / 63.5 / 2,
            torch.cat([torch.tensor([127.0]), torch.arange(127) - 63.5]),        # ties
            torch.cat([torch.tensor([381.0]), 3 * (torch.arange(127) - 63.5)]),  # ties, scale 3
            torch.zeros(128),
            torch.full((128,), 2.0 ** -149),
            torch.cat([torch.tensor([2.0 ** -149 * 200]), torch.arange(127) * 2.0 ** -149]),
            torch.cat([torch.tensor([2.0 ** -130]), torch.randn(127, generator=gen) * 2.0 ** -132]),
            torch.cat([torch.tensor([3.0e-37]), torch.rand(127, generator=gen) * 3e-37]),
            torch.cat([torch.tensor([3.4028234e38]), (torch.rand(127, generator=gen) - .5) * 6e38]),
            torch.cat([torch.tensor([3.4028234e38]), (torch.rand(127, generator=gen) - .5) * 3e38]),
            torch.randn(128, generator=gen).bfloat16().float(),
            torch.randn(128, generator=gen).half().float()]
    # Neighbours of halves of random scales.
    for _ in range(20):
        top = torch.rand(1, generator=gen) + 0.5
        scale = (top.double() / 127).float()
        near = ((torch.arange(63).double() + 0.5) * scale.double()).float()
        rows.append(torch.cat([top, near, -torch.nextafter(near, top.expand(63)),
                               torch.zeros(1)]))
    x = torch.stack([r.float() for r in rows])[:, None].cuda()
    n = x.shape[0]
    kp, vp, scales = pools(3, 16, 1, 128)
    hip.cache_append(x, -x, kp, vp, ints([[0, 1, 2]]), ints([0]), ints([0, n]), scales=scales)
    codes, scale = quantised(x)
    got = kp.reshape(-1, 1, 128)[:n].cpu()
    for i in range(n):
        assert torch.equal(got[i], codes[i]), (i, (got[i] != codes[i]).nonzero()[:3])
    # 6e38 is an infinity in fp32, so that row's scale is NaN.
    assert int(torch.isnan(scale).sum()) == 1
    got = scales[0].transpose(1, 2).reshape(-1, 1)[:n].cpu()
    assert torch.equal(torch.nan_to_num(got, nan=-1.0), torch.nan_to_num(scale, nan=-1.0))
    assert torch.equal(vp.reshape(-1, 1, 128)[:n].cpu(), -codes)
    # And so what is read back is at most half a scale off, or clipped where the scale rounded.
    k, _ = hip.cache_read(kp, vp, ints([[0, 1, 2]]), ints([0]), ints([0, n]), n, scales=scales)
    off = (k.cpu().double() - x.cpu().double()).abs().amax(-1)
    normal = scale > 2.0 ** -126
    # Half a scale, and the product's rounding in 32 bits: 2^-24 of at most 127 scales.
    assert bool((off[normal] <= (0.5 + 127 * 2.0 ** -24) * scale.double()[normal]).all())


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_heads_that_are_not_finite(hip, bad):
    import torch
    print_case("append8 not finite", bad)
    x = torch.randn(4, 3, 40, device="cuda")
    y = x.clone()
    y[1, 2, 39], y[3, 0, 0] = bad, bad
    kp, vp, scales = pools(2, 4, 3, 40)
    hip.cache_append(y, x, kp, vp, ints([[1]]), ints([0]), ints([0, 4]), scales=scales)
    k, v = hip.cache_read(kp, vp, ints([[1]]), ints([0]), ints([0, 4]), 4, scales=scales)
    hit = torch.isnan(k)
    assert bool(hit[1, 2].all()) and bool(hit[3, 0].all()) and int(hit.sum()) == 80
    codes, scale = quantised(y)
    want = torch.where(torch.isnan(scale)[..., None], torch.full_like(codes.float(), math.nan),
                       codes.float() * scale[..., None])
    assert torch.equal(torch.nan_to_num(k.cpu(), nan=9.), torch.nan_to_num(want, nan=9.))
    assert bool(torch.isfinite(v).all())


@gpu
def test_append_places_and_refused_places(hip):
    """Positions from a start on, one token each without offsets, tokens that have no place or no
    sequence: not stored, and nothing else is touched."""
    import torch
    print_case("append8 places")
    x = torch.randn(3, 2, 8, device="cuda")
    table = ints([[2, 0], [3, 9], [1, -1]])
    kp, vp, scales = pools(4, 4, 2, 8, fill=7)
    hip.cache_append(x, x, kp, vp, table, ints([5, 3, 6]), scales=scales)
    codes, scale = quantised(x)
    want, wscale = torch.full((4, 4, 2, 8), 7, dtype=torch.int8), torch.full((4, 2, 4), 7.0)
    want[0, 1], want[3, 3] = codes[0], codes[1]
    wscale[0, :, 1], wscale[3, :, 3] = scale[0], scale[1]
    assert torch.equal(kp.cpu(), want) and torch.equal(vp.cpu(), want)
    assert torch.equal(scales[0].cpu(), wscale) and torch.equal(scales[1].cpu(), wscale)
    hip.cache_append(x, x, kp, vp, table, ints([-1, 8, 2 ** 31 - 1]), scales=scales)
    hip.cache_append(x, x, kp, vp, table, ints([4, 0, 0]), ints([1, 1, 1, 1]), scales=scales)
    assert torch.equal(kp.cpu(), want) and torch.equal(scales[1].cpu(), wscale)


# --------------------------------------------------------------------- read

KINDS = ["float32", "bfloat16", "int8"]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,d,page", [(1, 1, 1), (2, 24, 16), (8, 128, 32), (3, 33, 7), (1, 100, 5),
                                       (5, 6, 3)])
def test_read_gives_what_is_held(hip, kv, d, page, kind):
    import torch
    print_case("read", kv, d, page, kind)
    lengths = [3, 0, 70, 1, 2 * page]
    kp, vp, scales, table, k, v = fill(hip, lengths, kv, d, page, seed=d, kind=kind)
    n = sum(lengths)
    got = hip.cache_read(kp, vp, table, ints([0] * 5), offsets(lengths), n, scales=scales)
    for x, pool, sc in zip(got, (kp, vp), scales or (None, None)):
        # One product in 32 bits, or none.
        assert torch.equal(x.cpu(), torch.cat(held(pool, sc, table, lengths)).float())
    if kind == "float32":
        assert torch.equal(got[0], k) and torch.equal(got[1], v)
    # From a position on, and one for each sequence.
    part = hip.cache_read(kp, vp, table, ints([1, 0, 64, 0, page]), ints([0, 2, 2, 8, 9, 9 + page]),
                          9 + page, scales=scales)
    for x, y in zip(part, got):
        assert torch.equal(x, torch.cat([y[1:3], y[67:73], y[73:74], y[74 + page:74 + 2 * page]]))
    rows = [0, 4]
    one = hip.cache_read(kp, vp, table[rows], ints([2, 1 if page > 0 else 0]), scales=scales)
    assert torch.equal(one[0][0], got[0][2]) and torch.equal(one[1][1], got[1][74 + 1])


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_read_of_places_that_are_none(hip, kind):
    """NaN in place of a read out of bounds; rows of no sequence stay; strided outputs."""
    import torch
    print_case("read places", kind)
    lengths = [20, 20]
    kp, vp, scales, table, k, v = fill(hip, lengths, 2, 12, 8, seed=3, kind=kind)
    want, _ = hip.cache_read(kp, vp, table, ints([0, 0]), ints([0, 20, 40]), 40, scales=scales)
    table = table.clone()
    table[0, 1], table[1, 2] = kp.shape[0], -7
    out = torch.full((50, 5, 12), 5.0, device="cuda")
    hip.cache_read(kp, vp, table, ints([-2, 14]), ints([1, 21, 45]), 50, scales=scales,
                   out=(out[:, :2], out[:, 3:]))
    assert bool((out[:, 2] == 5.0).all())
    assert bool((out[0] == 5.0).all()) and bool((out[45:] == 5.0).all())
    assert bool(torch.isnan(out[1:3, :2]).all()) and torch.equal(out[3:11, :2], want[:8])
    assert bool(torch.isnan(out[11:19, :2]).all()) and torch.equal(out[19:21, :2], want[16:18])
    assert torch.equal(out[21:23, :2], want[34:36])
    assert bool(torch.isnan(out[23:31, :2]).all())              # the page -7
    assert bool(torch.isnan(out[23 + 16:45, :2]).all())          # past the table


# ---------------------------------------------------------------- attention

def reference(q, k, v, lengths, scale):
    import torch
    return packed(q, torch.cat(k), torch.cat(v), [1] * len(lengths), lengths, scale, False)


def check(hip, lengths, heads, kv, d, page, seed=0, longest=None, scale=None, spread=1.0):
    import torch
    print_case("paged8", lengths, heads, kv, d, page, seed)
    kp, vp, scales, table, _, _ = fill(hip, lengths, kv, d, page, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(len(lengths), heads, d, generator=gen, device="cuda") * spread
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths), longest=longest, scale=scale,
                                   scales=scales)
    k, v = held(kp, scales[0], table, lengths), held(vp, scales[1], table, lengths)
    value, bound = reference(q, k, v, lengths, d ** -0.5 if scale is None else scale)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")
    return kp, vp, scales, table, q, out, lse


@gpu
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 64), (4, 4, 24), (8, 2, 128), (5, 1, 33),
                                        (16, 1, 128), (24, 2, 64), (6, 3, 80), (17, 1, 64),
                                        (40, 2, 128), (33, 1, 32)])
def test_lengths_and_heads(hip, heads, kv, d):
    check(hip, [0, 1, 2, 15, 16, 17, 64, 200, 3], heads, kv, d, 16, seed=heads)


@gpu
@pytest.mark.parametrize("page", [1, 3, 8, 16, 64, 100, 512])
def test_page_sizes(hip, page):
    check(hip, [1, page, page + 1, 3 * page - 1, 130], 4, 2, 64, page, seed=page)


@gpu
@pytest.mark.parametrize("d", [1, 2, 5, 7, 8, 9, 15, 16, 31, 32, 40, 48, 63, 65, 72, 77, 96, 100,
                               112, 120, 121, 127])
def test_head_dims(hip, d):
    check(hip, [37, 5, 130], 6, 2, d, 8, seed=d)


@gpu
@pytest.mark.parametrize("lengths", [[3000], [5000, 1, 0, 2049], [1023, 1024, 1025, 4096]])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_that_are_split(hip, lengths, d):
    check(hip, lengths, 4, 2, d, 16, seed=len(lengths))


@gpu
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 3.0), (0.125, 40.0)])
def test_scales_and_sharp_rows(hip, scale, spread):
    check(hip, [700, 33], 4, 2, 64, 16, seed=4, scale=scale, spread=spread)


@gpu
def test_bad_pages_and_lengths_make_their_row_nan(hip):
    import torch
    lengths = [70, 40, 90, 33, 20, 64]
    kp, vp, scales, table, q, want, want_lse = check(hip, lengths, 4, 2, 64, 16, seed=7, longest=96)
    table = table.clone()
    table[0, 4], table[1, 0] = kp.shape[0], -1
    bad = list(lengths)
    bad[2], bad[3], bad[5] = 97, -1, 2 ** 31 - 1
    out, lse = hip.attention_paged(q, kp, vp, table, ints(bad), longest=96, scales=scales)
    for s in range(6):
        if s == 4:
            assert torch.equal(out[s], want[s]) and torch.equal(lse[s], want_lse[s])
        else:
            assert bool(torch.isnan(out[s]).all()) and bool(torch.isnan(lse[s]).all())


@gpu
@pytest.mark.parametrize("d", [64, 77])
def test_positions_past_the_length_do_not_reach_a_row(hip, d):
    """Nor do their scales, whatever they hold."""
    import torch
    lengths = [20, 33, 5]
    kp, vp, scales, table, q, want, _ = check(hip, lengths, 4, 2, d, 16, seed=8)
    used = torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lengths):
        for p in range(n):
            used[table[s, p // 16].long(), p % 16] = True
    kp[~used], vp[~used] = 127, -128
    for sc in scales:
        sc.transpose(1, 2)[~used] = math.nan
    out, _ = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_scales_that_are_not_finite(hip, which, d):
    """A NaN scale of K makes its key head's heads NaN, one of V their outputs and not lse; an
    infinity in q its head."""
    import torch
    lengths = [300, 40]
    kp, vp, scales, table, q, want, want_lse = check(hip, lengths, 6, 2, d, 16, seed=10)
    page = int(table[0, 3])
    if which == "q":
        q[0, 1, 5] = math.inf
    else:
        scales[0 if which == "k" else 1][page, 0, 2] = math.nan
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    hit = slice(1, 2) if which == "q" else slice(0, 3)
    assert bool(torch.isnan(out[0, hit]).all())
    assert bool(torch.isnan(lse[0, hit]).all()) == (which != "v")
    if which == "v":
        value = packed(q, torch.cat(held(kp, scales[0], table, lengths)),
                       torch.cat(held(kp, scales[0], table, lengths)), [1, 1], lengths, d ** -0.5,
                       False)
        within(lse, value[0]["lse"], value[1]["lse"], "lse")
    rest = [h for h in range(6) if h not in range(6)[hit]]
    assert torch.equal(out[0, rest], want[0, rest]) and torch.equal(out[1], want[1])
    assert torch.equal(lse[0, rest], want_lse[0, rest])


@gpu
@pytest.mark.parametrize("power", [-70, -80, 100])
def test_small_and_large_values(hip, power):
    """A weight times its scale runs on 2^-24 of it, in parts of at least 2^-133: with codes of up
    to 127, 2^-126 of a position, 2^-102 in what it stands for, and as much for the sums."""
    import torch
    print_case("paged8 range", power)
    lengths = [300, 7]
    kp, vp, scales, table, _, _ = fill(hip, lengths, 2, 64, 16, seed=9)
    scales[1].mul_(2.0 ** power)
    q = torch.randn(2, 4, 64, device="cuda")
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    value, bound = reference(q, held(kp, scales[0], table, lengths),
                             held(vp, scales[1], table, lengths), lengths, 0.125)
    for s, n in enumerate(lengths):
        within(out[s], value["out"][s], bound["out"][s] + n * 2.0 ** -100, "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("d", [24, 64, 100, 128])
@pytest.mark.parametrize("power", [100, 113, 118, 120, 122, 126])
def test_large_queries_and_small_scales(hip, power, d):
    """Queries times the whole numbers alone are past fp32, the scores are not. The scales are taken as
    they are held, of few bits where they are subnormal; powers of two add no rounding."""
    import torch
    print_case("paged8 large q", power, d)
    lengths = [300, 7]
    kp, vp, scales, table, _, _ = fill(hip, lengths, 2, d, 16, seed=9)
    scales[0].mul_(2.0 ** -power)
    gen = torch.Generator(device="cuda").manual_seed(power)
    q = torch.randn(2, 4, d, generator=gen, device="cuda") * 2.0 ** power
    q[1, 0].abs_()
    kp[:, :, 0].abs_()
    q[0, 0] = -q[0, 0].abs()  # sums far below zero alone
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    value, bound = reference(q, held(kp, scales[0], table, lengths),
                             held(vp, scales[1], table, lengths), lengths, d ** -0.5)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("heads,kv,d", [(4, 4, 64), (8, 2, 128), (3, 1, 33)])
def test_many_sequences(hip, heads, kv, d):
    """More than a wave has lanes, of uneven lengths, some empty."""
    check(hip, [(37 * i) % 90 if i % 7 else 0 for i in range(200)] + [3000] + [1] * 70, heads, kv, d,
          16, seed=15)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_scales_and_outputs_in_one_tensor(hip, kind):
    """A pair may be a tensor of two."""
    import torch
    print_case("cache pairs", kind)
    lengths = [20, 3]
    kp, vp, scales, table, k, v = fill(hip, lengths, 2, 32, 8, seed=17, kind=kind)
    want = hip.cache_read(kp, vp, table, ints([0, 0]), offsets(lengths), 23, scales=scales)
    both = torch.empty(2, 23, 2, 32, device="cuda")
    got = hip.cache_read(kp, vp, table, ints([0, 0]), offsets(lengths), 23,
                         scales=None if scales is None else torch.stack(scales), out=both)
    assert torch.equal(both[0], want[0]) and torch.equal(both[1], want[1])
    assert got[0].data_ptr() == both.data_ptr()


@gpu
def test_a_cache_past_32_bit_offsets(hip):
    """Written, read back and attended to at the end of pools of 2^31 values and more: the same bits
    as in small ones."""
    import torch
    print_case("paged8 large")
    pages, page, kv, d, lengths = 16400, 128, 8, 128, [300, 1, 40]
    kp, vp, scales, table, k, v = fill(hip, lengths, kv, d, page, seed=16)
    q = torch.randn(3, 16, d, device="cuda")
    want = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    held_k, held_v = hip.cache_read(kp, vp, table, ints([0] * 3), offsets(lengths), 341,
                                    scales=scales)
    kp, vp, scales = pools(pages, page, kv, d)
    assert kp.numel() > 2 ** 31
    table = (pages - 1 - table).to(torch.int32)
    hip.cache_append(k, v, kp, vp, table, ints([0] * 3), offsets(lengths), scales=scales)
    got = hip.cache_read(kp, vp, table, ints([0] * 3), offsets(lengths), 341, scales=scales)
    assert torch.equal(got[0], held_k) and torch.equal(got[1], held_v)
    out = hip.attention_paged(q, kp, vp, table, ints(lengths), scales=scales)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    del kp, vp
    torch.cuda.empty_cache()


@gpu
def test_strides_and_outputs(hip):
    import torch
    lengths = [100, 17]
    kp, vp, scales, table, q, want, want_lse = check(hip, lengths, 4, 2, 40, 16, seed=11)
    rows = torch.full((2, 9, 40), 5.0, device="cuda")
    rows[:, 4:8] = q
    into = torch.full((2, 6, 40), 5.0, device="cuda")
    out, lse = hip.attention_paged(rows[:, 4:8], kp, vp, table, ints(lengths), scales=scales,
                                   out=into[:, 1:5])
    assert torch.equal(into[:, 1:5], want) and torch.equal(lse, want_lse)
    assert bool((into[:, 0] == 5.0).all()) and bool((into[:, 5] == 5.0).all())


@gpu
def test_pools_at_any_address(hip):
    """Pools that begin at an odd byte of a larger one."""
    import torch
    lengths = [100, 17]
    kp, vp, scales, table, q, want, _ = check(hip, lengths, 4, 2, 40, 16, seed=13)
    shifted = []
    for pool in (kp, vp):
        flat = torch.zeros(pool.numel() + 3, dtype=torch.int8, device="cuda")
        flat[3:] = pool.reshape(-1)
        shifted.append(flat[3:].view(pool.shape))
    out, _ = hip.attention_paged(q, *shifted, table, ints(lengths), scales=scales)
    assert torch.equal(out, want)
    got = hip.cache_read(*shifted, table, ints([0, 0]), offsets(lengths), 117, scales=scales)
    same = hip.cache_read(kp, vp, table, ints([0, 0]), offsets(lengths), 117, scales=scales)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    x = torch.randn(117, 2, 40, device="cuda")
    for to in (shifted, (kp, vp)):
        hip.cache_append(x, x, *to, table, ints([0, 0]), offsets(lengths), scales=scales)
    assert torch.equal(shifted[0], kp) and torch.equal(shifted[1], vp)


@gpu
def test_a_prompt_in_pieces(hip):
    """Each piece is written and all that is held read back for packed attention, whose last row is
    then what attention over the cache gives."""
    import torch
    print_case("pieces in 8 bits")
    gen = torch.Generator(device="cuda").manual_seed(14)
    pieces = [[5, 0, 40], [1, 17, 3], [30, 2, 1]]
    total = [sum(p[s] for p in pieces) for s in range(3)]
    table, count = table_of(total, 16, gen)
    kp, vp, scales = pools(count, 16, 2, 64)
    before = [0, 0, 0]
    for new in pieces:
        n = sum(new)
        q, k, v = (torch.randn(n, h, 64, generator=gen, device="cuda") for h in (4, 2, 2))
        hip.cache_append(k, v, kp, vp, table, ints(before), offsets(new), scales=scales)
        upto = [a + b for a, b in zip(before, new)]
        rows = hip.cache_read(kp, vp, table, ints([0] * 3), offsets(upto), sum(upto), scales=scales)
        out, lse = hip.attention_packed(q, *rows, offsets(new), offsets(upto))
        kh, vh = (held(p, sc, table, upto) for p, sc in zip((kp, vp), scales))
        value, bound = packed(q, torch.cat(kh), torch.cat(vh), new, upto, 0.125, True)
        # The rows read back are products in 32 bits, one rounding more of K and of V.
        within(out, value["out"], 2 * bound["out"], "out")
        last = [i for s, i in enumerate(offsets(new).tolist()[1:]) if new[s]]
        have = [s for s in range(3) if new[s]]
        one, _ = hip.attention_paged(q[[i - 1 for i in last]], kp, vp, table[have],
                                     ints([upto[s] for s in have]), scales=scales)
        at = [i - 1 for i in last]
        within(one, value["out"][at], bound["out"][at], "paged")
        before = upto


@gpu
def test_same_bits_each_time_on_other_streams_and_in_a_graph(hip):
    import torch
    lengths = [4000, 130, 1, 0]
    kp, vp, scales, table, q, want, want_lse = check(hip, lengths, 8, 2, 64, 16, seed=12)
    n = ints(lengths)
    new = torch.randn(4, 2, 64, device="cuda")
    at = ints([3999, 129, 0, 0])

    def step():
        hip.cache_append(new, new, kp, vp, table, at, scales=scales)
        return (*hip.cache_read(kp, vp, table, at, scales=scales),
                *hip.attention_paged(q, kp, vp, table, n, scales=scales))

    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(hip.attention_paged(q, kp, vp, table, n, scales=scales))
    torch.cuda.synchronize()
    for o, l in got:
        assert torch.equal(o, want) and torch.equal(l, want_lse)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        new.copy_(torch.randn(4, 2, 64, device="cuda"))
        at.copy_(ints([3990 + i, 5 * i, 0, 0]))
        n.copy_(ints([4000 - i, 100 + i, 1, 0]))
        eager = step()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager))


# ----------------------------------------------------------------- refusals

def cache(**changes):
    d = dict(k_pages=64, v_pages=64, type=2, pages=4, page_size=16, kv_heads=2, head_dim=64,
             table=64, ld_table=4, table_width=4, sequences=3, k_scales=64, v_scales=64)
    d.update(changes)
    return E.Cache(*[d[n] for n, _ in E.Cache._fields_])


REFUSED = [dict(type=3), dict(type=-1), dict(k_scales=None), dict(v_scales=None),
           dict(head_dim=129), dict(k_pages=None)]


@pytest.mark.parametrize("changes", REFUSED)
def test_refused_caches(changes):
    """The query answers without a device."""
    lib = E.load_library()
    assert lib.ehip_attention_paged_workspace(C.byref(cache(**changes)), 4, 64) == -1
    assert b"attention_paged" in lib.ehip_last_error()


def test_scales_are_of_the_cache_in_8_bits_alone():
    lib = E.load_library()
    for kind in (0, 1):
        c = cache(type=kind, k_scales=None, v_scales=None)
        assert lib.ehip_attention_paged_workspace(C.byref(c), 4, 64) > 0
    assert lib.ehip_attention_paged_workspace(C.byref(cache(pages=0, k_scales=None)), 4, 64) > 0


@gpu
def test_refused_calls(hip):
    import torch
    print_case("cache8 refused")
    lib = hip.lib
    for changes in REFUSED + [dict(sequences=-1), dict(page_size=0), dict(ld_table=3)]:
        c = cache(**changes)
        assert lib.ehip_cache_append_f32(C.byref(c), 64, 1 << 20, 64, 1 << 20, 64, 64, 5, None) == 1
        assert lib.ehip_cache_read_f32(C.byref(c), 64, 64, 5, 64, 1 << 20, 64, 1 << 20, None) == 1
    c = cache()
    read = lambda starts=64, cu=64, n=5, k=64, lk=128, v=64, lv=128: lib.ehip_cache_read_f32(
        C.byref(c), starts, cu, n, k, lk, v, lv, None)
    assert read(starts=None) == 1 and read(k=None) == 1 and read(v=None) == 1
    assert read(lk=127) == 1 and read(lv=127) == 1 and read(n=-1) == 1 and read(cu=None) == 1
    assert read(n=1 << 30) == 1 and read(n=0) == 0
    kp, vp, scales, table, k, v = fill(hip, [5, 6], 2, 8, 4)
    z, cu = ints([0, 0]), ints([0, 5, 11])
    with pytest.raises(ValueError):
        hip.cache_append(k, v, kp, vp, table, z, cu)
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, cu, 11)
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, cu, scales=scales)
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, None, 11, scales=scales)
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, cu, 11, scales=(scales[0].double(), scales[1]))
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, cu, 11, scales=(scales[0][:1], scales[1]))
    with pytest.raises(ValueError):
        hip.cache_read(kp, vp, table, z, cu, 11, scales=scales, out=(k[:10], v))
    with pytest.raises(ValueError):
        hip.cache_read(kp.float(), vp.float(), table, z, cu, 11, scales=scales)
    with pytest.raises(ValueError):
        hip.attention_paged(k[:2], kp, vp, table, z)
