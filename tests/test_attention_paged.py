"""The paged cache: writing tokens into it and attention of one new token over it, against the
formula in 64 bits with bounds from arithmetic (tests/_attention64.py), and what they refuse."""
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


def make(lengths, kv, d, page, dtype, seed=0, spare=2, extra=1):
    """(k_pages, v_pages, table, k, v): pools whose pages hold random keys and values in a random
    order, a table with `extra` columns more than are needed (naming page 0), and the same rows
    per sequence as lists."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    each = [-(-n // page) for n in lengths]
    pages = sum(each) + spare
    pools = [torch.randn(pages, page, kv, d, generator=gen, device="cuda").to(dtype)
             for _ in range(2)]
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), max(each) + extra, dtype=torch.int32, device="cuda")
    k, v, at = [], [], 0
    for s, (n, m) in enumerate(zip(lengths, each)):
        table[s, :m] = order[at:at + m]
        which = order[at:at + m].long()
        for pool, rows in zip(pools, (k, v)):
            rows.append(pool[which].reshape(-1, kv, d)[:n].float())
        at += m
    return (*pools, table, k, v)


def reference(q, k, v, lengths, scale):
    import torch
    return packed(q, torch.cat(k), torch.cat(v), [1] * len(lengths), lengths, scale, False)


def check(hip, lengths, heads, kv, d, page, dtype, seed=0, longest=None, scale=None, spread=1.0):
    import torch
    print_case("paged", lengths, heads, kv, d, page, dtype, seed)
    kp, vp, table, k, v = make(lengths, kv, d, page, dtype, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(len(lengths), heads, d, generator=gen, device="cuda") * spread
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths), longest=longest, scale=scale)
    value, bound = reference(q, k, v, lengths, d ** -0.5 if scale is None else scale)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")
    return kp, vp, table, q, out, lse


def types():
    import torch
    return [torch.float32, torch.bfloat16]


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 64), (4, 4, 24), (8, 2, 128), (5, 1, 33),
                                        (16, 1, 128), (24, 2, 64), (6, 3, 80)])
def test_lengths_and_heads(hip, dtype, heads, kv, d):
    check(hip, [0, 1, 2, 15, 16, 17, 64, 200, 3], heads, kv, d, 16, dtype, seed=heads)


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("page", [1, 3, 8, 16, 64, 100, 512])
def test_page_sizes(hip, dtype, page):
    check(hip, [1, page, page + 1, 3 * page - 1, 130], 4, 2, 64, page, dtype, seed=page)


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("d", [1, 2, 5, 8, 16, 31, 32, 40, 63, 65, 72, 96, 100, 127])
def test_head_dims(hip, dtype, d):
    check(hip, [37, 5], 6, 2, d, 8, dtype, seed=d)


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("lengths", [[3000], [5000, 1, 0, 2049], [1023, 1024, 1025, 4096]])
def test_lengths_that_are_split(hip, dtype, lengths):
    check(hip, lengths, 4, 2, 64, 16, dtype, seed=len(lengths))


@gpu
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 3.0), (0.125, 40.0)])
def test_scales_and_sharp_rows(hip, scale, spread):
    import torch
    check(hip, [700, 33], 4, 2, 64, 16, torch.float32, seed=4, scale=scale, spread=spread)


@gpu
def test_batches_and_bounds_on_the_length(hip):
    """The same rows whatever `longest` says; the sequences' lengths are what counts."""
    import torch
    lengths = [(37 * i) % 300 for i in range(150)]
    for longest in (None, 299, 5000):
        check(hip, lengths, 2, 1, 32, 32, torch.float32, seed=5, longest=longest)


@gpu
def test_as_the_packed_attention_of_one_query(hip):
    import torch
    print_case("paged against packed")
    lengths = [50, 1, 333]
    kp, vp, table, q, out, lse = check(hip, lengths, 8, 2, 64, 16, torch.float32, seed=6)
    _, _, _, k, v = make(lengths, 2, 64, 16, torch.float32, seed=6)
    cu = ints([0, 1, 2, 3])
    ck = ints([0, 50, 51, 384])
    other, lse2 = hip.attention_packed(q, torch.cat(k), torch.cat(v), cu, ck)
    value, bound = reference(q, k, v, lengths, 0.125)
    within(out, other.cpu().double(), 2 * bound["out"], "out")
    within(lse, lse2.cpu().double(), 2 * bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("dtype", types())
def test_bad_pages_and_lengths_make_their_row_nan(hip, dtype):
    """A page outside the pool, or a length below zero, past `longest` or past the table: that
    sequence's row is NaN, the others are as they were, and nothing else is read."""
    import torch
    print_case("paged bad", dtype)
    lengths = [70, 40, 90, 33, 20, 64]
    kp, vp, table, k, v = make(lengths, 2, 64, 16, dtype, seed=7)
    q = torch.randn(6, 4, 64, device="cuda")
    want, want_lse = hip.attention_paged(q, kp, vp, table, ints(lengths), longest=96)
    table = table.clone()
    table[0, 4] = kp.shape[0]  # the page of positions 64 to 69
    table[1, 0] = -1
    bad = list(lengths)
    bad[2], bad[3], bad[5] = 97, -1, 2 ** 31 - 1
    out, lse = hip.attention_paged(q, kp, vp, table, ints(bad), longest=96)
    for s in range(6):
        if s == 4:
            assert torch.equal(out[s], want[s]) and torch.equal(lse[s], want_lse[s])
        else:
            assert bool(torch.isnan(out[s]).all()) and bool(torch.isnan(lse[s]).all())
    # Past the table, with a `longest` that would allow it.
    wide = table.shape[1] * 16
    out, _ = hip.attention_paged(q, kp, vp, table, ints([20, 20, wide + 1, 20, 20, 20]),
                                 longest=10 ** 6)
    assert bool(torch.isnan(out[2]).all()) and not bool(torch.isnan(out[4]).any())
    # A bad page that the length does not reach is not looked at.
    out, _ = hip.attention_paged(q, kp, vp, table, ints([64, 0, 90, 33, 20, 64]))
    assert not bool(torch.isnan(out).any())


@gpu
def test_positions_past_the_length_do_not_reach_a_row(hip):
    import torch
    print_case("paged unseen")
    lengths = [20, 33, 5]
    kp, vp, table, k, v = make(lengths, 2, 64, 16, torch.float32, seed=8)
    q = torch.randn(3, 4, 64, device="cuda")
    want, _ = hip.attention_paged(q, kp, vp, table, ints(lengths))
    used = torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(lengths):
        for p in range(n):
            used[table[s, p // 16].long(), p % 16] = True
    kp[~used], vp[~used] = math.nan, math.inf
    out, _ = hip.attention_paged(q, kp, vp, table, ints(lengths))
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("size", [1e-38, 1e30, 2e38])
def test_values_near_the_ends_of_the_range(hip, size):
    import torch
    print_case("paged range", size)
    lengths = [300, 7]
    kp, vp, table, k, v = make(lengths, 2, 64, 16, torch.float32, seed=9)
    vp.clamp_(-1, 1).mul_(size)
    v = [x.clamp(-1, 1) * size for x in v]
    q = torch.randn(2, 4, 64, device="cuda")
    out, _ = hip.attention_paged(q, kp, vp, table, ints(lengths))
    value, bound = reference(q, k, v, lengths, 0.125)
    within(out, value["out"], bound["out"] + 2.0 ** -126, "out")


@gpu
def test_values_that_are_seen_and_not_finite(hip):
    import torch
    print_case("paged not finite")
    lengths = [300, 40]
    kp, vp, table, k, v = make(lengths, 1, 32, 16, torch.float32, seed=10)
    vp[table[0, 3].long(), 2, 0, 5] = math.inf
    vp[table[0, 9].long(), 2, 0, 6] = math.nan
    kp[table[1, 1].long(), 2, 0, 6] = math.nan
    q = torch.randn(2, 2, 32, device="cuda")
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths))
    assert bool((out[0, :, 5] == math.inf).all()) and bool(torch.isnan(out[0, :, 6]).all())
    assert bool(torch.isfinite(out[0, :, [0, 1, 31]]).all()) and bool(torch.isfinite(lse[0]).all())
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(lse[1]).all())


@gpu
def test_bf16_values_that_are_seen_and_not_finite(hip):
    """Blocks of the matrix instructions' kernel whose sums are not finite."""
    import torch
    print_case("paged bf16 not finite")
    lengths = [300, 40]
    kp, vp, table, k, v = make(lengths, 2, 64, 16, torch.bfloat16, seed=10)
    vp[table[0, 3].long(), 2, 0, 5] = math.inf
    vp[table[0, 9].long(), 2, 0, 6] = math.nan
    kp[table[1, 1].long(), 2, 0, 6] = math.nan
    q = torch.randn(2, 6, 64, device="cuda")
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths))
    assert bool((out[0, :3, 5] == math.inf).all()) and bool(torch.isnan(out[0, :3, 6]).all())
    assert bool(torch.isfinite(out[0, :3, [0, 1, 31, 63]]).all())
    assert bool(torch.isnan(out[1, :3]).all()) and bool(torch.isnan(lse[1, :3]).all())
    value, bound = reference(q[:, 3:], [x[:, 1:] for x in k], [x[:, 1:] for x in v], lengths,
                             64 ** -0.5)
    within(out[:, 3:], value["out"], bound["out"], "out")
    within(lse[:, 3:], value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_part_whose_scores_are_all_minus_infinity(hip, dtype):
    """Weight 0 beside the other parts' positions, whichever blocks the length is split over; alone
    no distribution, with lse = -inf."""
    import torch
    print_case("paged -inf scores", dtype)
    lengths = [385, 7, 300]
    kp, vp, table, k, v = make(lengths, 1, 64, 16, getattr(torch, dtype), seed=12)
    q = torch.rand(3, 4, 64, device="cuda") + 0.5
    kp[table[0, 24].long(), 0, 0, 9] = -math.inf              # the last tile's one position
    for p in range(256, 300):                                 # all of a tile
        kp[table[2, p // 16].long(), p % 16, 0, 3] = -math.inf
    for p in range(7):                                        # all of a sequence
        kp[table[1, 0].long(), p, 0, 0] = -math.inf
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths))
    value, bound = reference(q, [k[0][:384], k[1], k[2][:256]], [v[0][:384], v[1], v[2][:256]],
                             [384, 7, 256], 0.125)
    for s in (0, 2):
        within(out[s], value["out"][s], bound["out"][s], "out")
        within(lse[s], value["lse"][s], bound["lse"][s], "lse")
    assert bool(torch.isnan(out[1]).all()) and bool((lse[1] == -math.inf).all())


@gpu
def test_strides_and_outputs(hip):
    """q and out as columns of wider rows, a table that is part of a larger one."""
    import torch
    print_case("paged strides")
    lengths = [100, 17]
    kp, vp, table, q, want, want_lse = check(hip, lengths, 4, 2, 40, 16, torch.float32, seed=11)
    rows = torch.full((2, 9, 40), 5.0, device="cuda")
    rows[:, 4:8] = q
    into = torch.full((2, 6, 40), 5.0, device="cuda")
    big = torch.full((3, table.shape[1] + 4), -9, dtype=torch.int32, device="cuda")
    big[:2, :table.shape[1]] = table
    out, lse = hip.attention_paged(rows[:, 4:8], kp, vp, big[:2, :table.shape[1]], ints(lengths),
                                   out=into[:, 1:5])
    assert torch.equal(into[:, 1:5], want) and torch.equal(lse, want_lse)
    assert bool((into[:, 0] == 5.0).all()) and bool((into[:, 5] == 5.0).all())


@gpu
def test_same_bits_each_time_on_other_streams_and_in_a_graph(hip):
    import torch
    lengths = [4000, 130, 1, 0]
    kp, vp, table, q, want, want_lse = check(hip, lengths, 8, 2, 64, 16, torch.bfloat16, seed=12)
    n = ints(lengths)
    torch.cuda.synchronize()
    got = []
    for _ in range(2):  # two calls at once
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(hip.attention_paged(q, kp, vp, table, n))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = hip.attention_paged(q, kp, vp, table, n)
        graphs.append((graph, outs))
    for o, l in got:
        assert torch.equal(o, want) and torch.equal(l, want_lse)
    for step in range(3):
        q.copy_(torch.randn(4, 8, 64, device="cuda"))
        n.copy_(ints([4000 - step, 130 + step, 1 + step, step]))  # lengths stay on the device
        o, l = hip.attention_paged(q, kp, vp, table, n)
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert torch.equal(outs[0], o) and torch.equal(outs[1], l)


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("which,value", [("k", math.nan), ("k", math.inf), ("v", math.nan),
                                         ("v", math.inf), ("v", -math.inf)])
def test_a_value_that_is_not_finite_anywhere_in_a_length(hip, which, value, dtype):
    """One of the first, middle or last positions of lengths that are one part and several: its key
    head's heads are what the formula has, the others as ever."""
    import torch
    print_case("paged not finite anywhere", which, value, dtype)
    lengths = [3000, 130, 70]
    kp, vp, table, k, v = make(lengths, 2, 64, 16, dtype, seed=16)
    q = torch.rand(3, 10, 64, device="cuda") + 0.5  # a key of inf is a score of inf
    for at in ("first", "middle", "last"):
        kx, vx = kp.clone(), vp.clone()
        rows = {"k": [t.clone() for t in k], "v": [t.clone() for t in v]}
        for s, n in enumerate(lengths):
            p = {"first": 0, "middle": n // 2, "last": n - 1}[at]
            pool = kx if which == "k" else vx
            pool[table[s, p // 16].long(), p % 16, 0, 7] = value
            rows[which][s][p, 0, 7] = value
        out, lse = hip.attention_paged(q, kx, vx, table, ints(lengths))
        if which == "k":  # no distribution
            assert bool(torch.isnan(out[:, :5]).all()) and bool(torch.isnan(lse[:, :5]).all())
        heads = slice(5 if which == "k" else 0, 10)
        each = slice(1 if which == "k" else 0, 2)
        want, bound = reference(q[:, heads], [t[:, each] for t in rows["k"]],
                                [t[:, each] for t in rows["v"]], lengths, 0.125)
        within(out[:, heads], want["out"], bound["out"], "out")
        within(lse[:, heads], want["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("dtype", types())
def test_a_cache_that_is_not_finite_takes_no_longer(hip, dtype):
    """A NaN in each sequence's first key, or nothing else: value by value it took 33 times as long."""
    import torch
    print_case("paged time of NaN", dtype)
    lengths = [1024] * 64
    kp, vp, table, _, _ = make(lengths, 8, 128, 16, dtype, seed=17)
    q = torch.randn(64, 32, 128, device="cuda")
    n = ints(lengths)

    def took():
        """The least of five, in ms."""
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            hip.attention_paged(q, kp, vp, table, n)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    took()
    times = [took()]
    kp[table[:, 0].long(), 0] = math.nan
    times.append(took())
    kp.fill_(math.nan)
    vp.fill_(math.nan)
    times.append(took())
    print(times, flush=True)
    assert max(times) < 8 * times[0]


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("d", [33, 64])
@pytest.mark.parametrize("power", [-100, -104, -110])
def test_small_values(hip, power, dtype, d):
    """Sums run on 2^-24 of a weight, so fp32's least step is 2^-125 of what they stand for: besides
    the relative bound there is that for each of the at most four roundings a position (three part
    products and the running sum)."""
    import torch
    print_case("paged small values", power, dtype, d)
    lengths = [300, 7]
    kp, vp, table, k, v = make(lengths, 2, d, 16, torch.float32, seed=9)
    vp = ((torch.rand_like(vp) + 1) * vp.sign() * 2.0 ** (power - 1)).to(dtype)
    kp = kp.to(dtype)
    rows = [[pool[table[s, :-(-n // 16)].long()].reshape(-1, 2, d)[:n].float()
             for s, n in enumerate(lengths)] for pool in (kp, vp)]
    q = torch.randn(2, 4, d, device="cuda")
    out, lse = hip.attention_paged(q, kp, vp, table, ints(lengths))
    value, bound = reference(q, *rows, lengths, d ** -0.5)
    for s, n in enumerate(lengths):
        # In place of the reference's own allowance.
        bounds = bound["out"][s] - 1e-37 + n * 2.0 ** -123
        within(out[s], value["out"][s], bounds, "out")
    assert float((value["out"][1].abs() > 10 * bounds).double().mean()) > 0.9  # not zeros
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("heads,kv,d", [(17, 1, 64), (33, 1, 32), (40, 2, 128), (64, 2, 40)])
def test_groups_over_several_blocks(hip, dtype, heads, kv, d):
    """More query heads a key head than a block takes at a time."""
    check(hip, [200, 0, 1, 33, 700], heads, kv, d, 16, dtype, seed=heads)


@gpu
@pytest.mark.parametrize("d", [64, 100])
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 3.0), (0.125, 40.0)])
def test_scales_and_sharp_rows_in_bf16(hip, scale, spread, d):
    import torch
    check(hip, [700, 33], 4, 2, d, 16, torch.bfloat16, seed=4, scale=scale, spread=spread)


# ------------------------------------------------------------------- append

@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("kv,d,page", [(1, 1, 1), (2, 24, 16), (8, 128, 32), (3, 33, 7),
                                       (4, 64, 100)])
def test_append(hip, dtype, kv, d, page):
    """Every token lands in its place, rounded to the pool's type, and nothing else changes."""
    import torch
    print_case("append", dtype, kv, d, page)
    new, starts = [5, 0, 1, 40, 3], [0, 9, 31, 2, 100]
    total = [a + b for a, b in zip(new, starts)]
    kp, vp, table, _, _ = make(total, kv, d, page, dtype, seed=d)
    want_k, want_v = kp.clone(), vp.clone()
    tail = 6
    rows = torch.randn(sum(new) + tail, 2 * kv + 1, d, device="cuda")
    k, v = rows[:, :kv], rows[:, kv:2 * kv]
    cu = [0, 5, 5, 6, 46, 49]
    hip.cache_append(k, v, kp, vp, table, ints(starts), ints(cu))
    t = 0
    for s, n in enumerate(new):
        for i in range(n):
            p = starts[s] + i
            at = (int(table[s, p // page]), p % page)
            want_k[at], want_v[at] = k[t].to(dtype), v[t].to(dtype)
            t += 1
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


@gpu
@pytest.mark.parametrize("dtype", types())
@pytest.mark.parametrize("kv,d", [(1, 30), (2, 260), (9, 135), (10, 120)])
def test_append_to_many_sequences(hip, dtype, kv, d):
    """More sequences than a wave has lanes, and than its square, many of them without a token; rows
    of one wave and of four, in multiples of four values and not."""
    import torch
    print_case("append many", dtype, kv, d)
    page = 4
    for count in (65, 4200):
        new = [(7 * s) % 4 if s % 3 else 0 for s in range(count)]
        starts = [s % 9 for s in range(count)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        table = torch.randperm(count * 3, device="cuda").to(torch.int32).reshape(count, 3)
        kp = torch.zeros(count * 3, page, kv, d, dtype=dtype, device="cuda")
        vp = torch.zeros_like(kp)
        want_k, want_v = torch.zeros_like(kp), torch.zeros_like(kp)
        k, v = (torch.randn(cu[-1] + 2, kv, d, device="cuda") for _ in range(2))
        hip.cache_append(k, v, kp, vp, table, ints(starts), ints(cu))
        who = torch.repeat_interleave(torch.arange(count), torch.tensor(new))
        at = torch.arange(cu[-1]) - torch.tensor(cu)[who] + torch.tensor(starts)[who]
        row = table.cpu()[who, at // page].long() * page + at % page
        for want, x in ((want_k, k), (want_v, v)):
            want.view(-1, kv, d)[row.cuda()] = x[:cu[-1]].to(dtype)
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v), count


@gpu
@pytest.mark.parametrize("dtype", types())
def test_append_one_token_each(hip, dtype):
    import torch
    print_case("append one each", dtype)
    starts = [0, 16, 15, 99]
    kp, vp, table, _, _ = make([s + 1 for s in starts], 2, 64, 16, dtype, seed=3)
    want = kp.clone()
    k, v = torch.randn(4, 2, 64, device="cuda"), torch.randn(4, 2, 64, device="cuda")
    hip.cache_append(k, v, kp, vp, table, ints(starts))
    for s, p in enumerate(starts):
        want[int(table[s, p // 16]), p % 16] = k[s].to(dtype)
    assert torch.equal(kp, want)


@gpu
def test_append_special_values(hip):
    """Infinities, NaN, the ends of the range and ties to even on the way to bf16."""
    import torch
    print_case("append special")
    x = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 3.4028235e38, 1e-45, 1.00390625,
                      1.01171875, -1.00390625, 3.3895314e38, 1.17549435e-38], device="cuda")
    k = x.reshape(1, 1, 12).contiguous()
    kp = torch.zeros(1, 4, 1, 12, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    hip.cache_append(k, k, kp, vp, ints([[0]]), ints([2]))
    want = x.to(torch.bfloat16)
    got = kp[0, 2, 0]
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan].view(torch.int16), want[~nan].view(torch.int16))


@gpu
def test_append_out_of_the_table_is_not_stored(hip):
    import torch
    print_case("append bad")
    kp = torch.zeros(4, 16, 1, 8, device="cuda")
    vp = torch.zeros(4, 16, 1, 8, device="cuda")
    table = ints([[0, 1], [4, -1], [2, 3]])
    k = torch.ones(9, 1, 8, device="cuda")
    # Sequence 0: past its table row from its second token on; 1: pages outside the pool;
    # 2: negative positions first, then 0.
    hip.cache_append(k, k, kp, vp, table, ints([31, 10, -2]), ints([0, 3, 6, 9]))
    for pool in (kp, vp):
        assert bool((pool[1, 15] == 1).all()) and bool((pool[2, 0] == 1).all())
        assert int((pool != 0).sum()) == 2 * 8
    # Offsets that leave tokens out or run past the tokens.
    kp.zero_()
    hip.cache_append(k, k, kp, vp, table, ints([0, 0, 0]), ints([2, 3, 3, 2 ** 31 - 1]))
    assert int((kp != 0).sum()) == 8 * (1 + 6)


@gpu
@pytest.mark.parametrize("dtype", types())
def test_prompt_then_tokens_one_by_one(hip, dtype):
    """The operators together: a packed prompt's attention, its keys and values into the cache,
    then tokens one by one, each written and attended, the sequences sharing the pool; against
    the formula over all the tokens at once, with the keys and values that the cache holds."""
    import torch
    print_case("prompt and tokens", dtype)
    heads, kv, d, page, steps = 4, 2, 40, 16, 5
    prompt = [30, 1, 47]
    gen = torch.Generator(device="cuda").manual_seed(4)
    r = lambda n, h: torch.randn(n, h, d, generator=gen, device="cuda")
    kp = torch.zeros(12, page, kv, d, dtype=dtype, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.randperm(12, generator=gen, device="cuda").to(torch.int32).reshape(3, 4)
    cu = ints([0, 30, 31, 78])
    q, k, v = r(78, heads), r(78, kv), r(78, kv)
    out, _ = hip.attention_packed(q, k, v, cu)
    value, bound = packed(q, k, v, prompt, prompt, d ** -0.5, True)
    within(out, value["out"], bound["out"], "prompt")
    hip.cache_append(k, v, kp, vp, table, ints([0, 0, 0]), cu)
    held = [[t[a:b].to(dtype).float() for a, b in ((0, 30), (30, 31), (31, 78))] for t in (k, v)]
    lengths = ints(prompt)
    for step in range(steps):
        q, k, v = r(3, heads), r(3, kv), r(3, kv)
        hip.cache_append(k, v, kp, vp, table, lengths)
        lengths.add_(1)
        out, lse = hip.attention_paged(q, kp, vp, table, lengths, longest=52)
        for rows, t in zip(held, (k, v)):
            for s in range(3):
                rows[s] = torch.cat([rows[s], t[s:s + 1].to(dtype).float()])
        n = [x + step + 1 for x in prompt]
        value, bound = reference(q, *held, n, d ** -0.5)
        within(out, value["out"], bound["out"], f"token {step}")
        within(lse, value["lse"], bound["lse"], f"token {step}")


@gpu
def test_a_cache_past_32_bit_offsets(hip):
    """Pools of 2^31 values and more: the last page is read and written where it is."""
    import torch
    print_case("large cache")
    pages, page, kv, d = 16400, 128, 8, 128  # 2.15e9 values a pool
    kp = torch.zeros(pages, page, kv, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros(pages, page, kv, d, dtype=torch.bfloat16, device="cuda")
    assert kp.numel() > 2 ** 31
    table = ints([[pages - 1], [3]])
    k, v = torch.randn(2, kv, d, device="cuda"), torch.randn(2, kv, d, device="cuda")
    hip.cache_append(k, v, kp, vp, table, ints([127, 0]))
    assert torch.equal(kp[pages - 1, 127], k[0].bfloat16())
    assert torch.equal(vp[3, 0], v[1].bfloat16())
    q = torch.randn(2, kv, d, device="cuda")
    out, _ = hip.attention_paged(q, kp, vp, table, ints([128, 1]))
    rows = [torch.zeros(128, kv, d), v[1:].bfloat16().float().cpu()]
    keys = [torch.zeros(128, kv, d), k[1:].bfloat16().float().cpu()]
    keys[0][127], rows[0][127] = k[0].bfloat16().float().cpu(), v[0].bfloat16().float().cpu()
    value, bound = reference(q, keys, rows, [128, 1], d ** -0.5)
    within(out, value["out"], bound["out"], "out")
    del kp, vp
    torch.cuda.empty_cache()


# ----------------------------------------------------------------- refusals

def cache(**changes):
    fields = dict(k_pages=4096, v_pages=4096, type=0, pages=10, page_size=16, kv_heads=2,
                  head_dim=64, table=4096, ld_table=4, table_width=4, sequences=3)
    fields.update(changes)
    return E.Cache(**fields)


def test_refused_caches_and_sizes():
    """The checks that every call starts with, through the query that needs no device."""
    lib = E.load_library()
    size = lib.ehip_attention_paged_workspace
    assert size(C.byref(cache()), 4, 64) >= 0
    assert size(C.byref(cache(sequences=0, table=None)), 4, 64) == 0
    assert size(None, 4, 64) == -1
    for bad in (dict(type=2), dict(type=-1), dict(pages=-1), dict(page_size=0), dict(kv_heads=0),
                dict(head_dim=0), dict(head_dim=129), dict(ld_table=3), dict(table_width=-1),
                dict(sequences=-1), dict(k_pages=None), dict(v_pages=None), dict(table=None),
                dict(sequences=2 ** 24), dict(pages=2 ** 31), dict(page_size=2 ** 31)):
        assert size(C.byref(cache(**bad)), 4, 64) == -1, bad
        assert b"attention_paged" in lib.ehip_last_error()
    for heads, longest in ((3, 64), (0, 64), (-2, 64), (4, -1), (4, 2 ** 31), (2 ** 24, 64)):
        assert size(C.byref(cache()), heads, longest) == -1, (heads, longest)


def test_lengths_end_where_positions_leave_their_range():
    """2^30: positions are counted on past a length in 32 bits."""
    size = E.load_library().ehip_attention_paged_workspace
    assert size(C.byref(cache()), 4, 2 ** 30) >= 0
    assert size(C.byref(cache()), 4, 2 ** 30 + 1) == -1


@gpu
def test_calls_are_refused(hip):
    import torch
    print_case("paged refusals")
    kp, vp, table, _, _ = make([20, 5], 2, 16, 8, torch.float32)
    q = torch.zeros(2, 4, 16, device="cuda")
    n = ints([20, 5])
    hip.attention_paged(q, kp, vp, table, n)
    k = torch.zeros(2, 2, 16, device="cuda")
    launched = hip.launched()
    for args in ((q[:, :, :15], kp, vp, table, n), (q, kp.half(), vp.half(), table, n),
                 (q, kp, vp.bfloat16(), table, n), (q, kp, vp[1:], table, n),
                 (q, kp, vp, table.long(), n), (q, kp, vp, table, n[:1]),
                 (q[:1], kp, vp, table, n), (q, kp, vp, table, n.cpu()),
                 (q, kp[:, :, :, ::2], vp[:, :, :, ::2], table, n)):
        with pytest.raises(ValueError):
            hip.attention_paged(*args)
    with pytest.raises(RuntimeError, match="heads"):
        hip.attention_paged(torch.zeros(2, 3, 16, device="cuda"), kp, vp, table, n)
    for args in ((k[:1], k[:1], kp, vp, table, n), (k, k[:, :1], kp, vp, table, n),
                 (k, k, kp, vp, table, n[:1]), (k, k, kp, vp, table, n, n)):
        with pytest.raises(ValueError):
            hip.cache_append(*args)
    assert hip.launched() == launched
