"""Attention over packed sequences with grouped heads, forward and backward, against the formula in
64 bits with bounds from arithmetic (tests/_attention64.py), and what it refuses."""
import ctypes as C
import math

import pytest

import ehip as E
from _attention64 import packed, within
from _hip import print_case

gpu = pytest.mark.gpu

# (queries, keys) of each sequence.
LENGTHS = {
    "one": [(1, 1)],
    "mixed": [(5, 5), (0, 3), (1, 1), (64, 64), (65, 65), (3, 0), (0, 0), (2, 130)],
    "tiles": [(128, 128), (127, 127), (129, 129), (63, 191), (33, 32)],
    "pieces": [(7, 100), (1, 300), (130, 450), (31, 31)],
    "hidden": [(40, 25), (200, 70), (5, 1), (64, 1)],  # first queries that see no key
    "long": [(600, 600), (1, 1), (257, 700)],
}


@pytest.fixture(scope="module")
def hip():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU test ran without a visible GPU")
    return E.Backend()


def offsets(lengths):
    import torch
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def make(nq, nk, heads, kv, d, seed=0, fused=False, tail=0, spread=1.0):
    """q, k, v, g on the GPU with `tail` rows past the last sequence."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    tq, tk = sum(nq) + tail, sum(nk) + tail
    if fused and tq == tk:
        rows = r(tq, heads + 2 * kv, d)
        q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    else:
        q, k, v = r(tq, heads, d), r(tk, kv, d), r(tk, kv, d)
    q.mul_(spread)
    return q, k, v, r(tq, heads, d)


def check(hip, nq, nk, heads, kv, d, causal, seed=0, fused=False, scale=None, spread=1.0):
    print_case("packed", nq, nk, heads, kv, d, causal, seed, fused)
    q, k, v, g = make(nq, nk, heads, kv, d, seed, fused, spread=spread)
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck, scale=scale, causal=causal)
    grads = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, scale=scale,
                                          causal=causal)
    value, bound = packed(q, k, v, nq, nk, d ** -0.5 if scale is None else scale, causal, g)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        within(got, value[name], bound[name], name)


@gpu
@pytest.mark.parametrize("which", sorted(LENGTHS))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (6, 2, 32), (4, 1, 128), (3, 3, 24)])
def test_lengths(hip, which, causal, heads, kv, d):
    nq, nk = zip(*LENGTHS[which])
    check(hip, nq, nk, heads, kv, d, causal, seed=hash((which, d)) % 1000)


@gpu
@pytest.mark.parametrize("d", [1, 2, 3, 7, 8, 16, 31, 33, 40, 63, 65, 72, 80, 95, 96, 97, 100, 112,
                               127])
def test_head_dims(hip, d):
    check(hip, [70, 3, 129], [70, 40, 129], 4, 2, d, True, seed=d)


@gpu
@pytest.mark.parametrize("d", [4, 5, 6, 10, 34, 66, 98, 126])
def test_head_dims_whose_last_four_values_overlap(hip, d):
    """Every remainder by four, rows as wide as the heads and within a projection's, one row too."""
    check(hip, [70, 3, 129], [70, 40, 129], 4, 2, d, True, seed=d)
    check(hip, [33, 64], [33, 64], 2, 1, d, False, seed=d + 1, fused=True)
    check(hip, [1], [1], 1, 1, d, True, seed=d + 2)


@gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 1), (5, 5), (9, 3), (16, 2), (12, 12)])
def test_head_groups_in_a_fused_projection(hip, heads, kv):
    check(hip, [50, 1, 0, 90], [50, 1, 0, 90], heads, kv, 48, True, seed=heads, fused=True)


@gpu
@pytest.mark.parametrize("scale,spread", [(1.0, 1.0), (0.0, 1.0), (-0.3, 2.0), (0.125, 40.0)])
def test_scales_and_sharp_rows(hip, scale, spread):
    """scale 0: even weights; spread 40: nearly one key a row, scores of some hundreds."""
    check(hip, [100, 33], [100, 50], 2, 1, 64, True, seed=3, scale=scale, spread=spread)


@gpu
@pytest.mark.parametrize("count", [63, 64, 65, 200, 4097])
def test_many_short_sequences(hip, count):
    """More sequences than a wave has lanes, and than it has lanes times lanes, of 0 to 3 rows."""
    nq = [(5 * i + i // 7) % 4 for i in range(count)]
    check(hip, nq, nq, 2, 1, 16, True, seed=count)


@gpu
def test_one_offset_array_and_equal_heads(hip):
    """cu_k left out; the same values as the framework's attention of equal lengths gives."""
    import torch
    print_case("packed against short")
    b, s, h, d = 3, 48, 4, 24
    q, k, v, g = make([s] * b, [s] * b, h, h, d, seed=8)
    cu = offsets([s] * b)
    out, lse = hip.attention_packed(q, k, v, cu)
    grads = hip.attention_packed_backward(g, q, k, v, out, lse, cu)
    flat = [t.reshape(b, s, h * d).contiguous() for t in (q, k, v, g)]
    w, other = hip.attention_short(*flat[:3], h, d ** -0.5, True)
    theirs = hip.attention_short_backward(*flat[:3], w, flat[3], h, d ** -0.5, True)
    _, bound = packed(q, k, v, [s] * b, [s] * b, d ** -0.5, True, g)
    for name, x, y in zip(("out", "dq", "dk", "dv"), (out, *grads), (other, *theirs)):
        # Two results, each within the bound.
        within(x, y.reshape(x.shape).cpu().double(), 2 * bound[name], name)


@gpu
@pytest.mark.parametrize("d", [32, 64, 100])
def test_keys_that_are_not_seen_do_not_reach_a_row(hip, d):
    """NaN and infinities in the keys and values past a row's own, and in other sequences."""
    import torch
    print_case("packed unseen", d)
    nq, nk = [90, 70], [90, 130]
    q, k, v, g = make(nq, nk, 4, 2, d, seed=d)
    k[60:90], v[60:90] = math.nan, math.inf      # sequence 0: rows 60.. see them
    k[90 + 100, 0], v[90 + 100, 1] = -math.inf, math.nan  # sequence 1: rows 40..
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    dq, _, _ = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)
    kz, vz = k.clone(), v.clone()
    for t in (kz, vz):
        t[60:90] = 0
        t[90 + 100:] = 0
    value, bound = packed(q, kz, vz, nq, nk, d ** -0.5, True, g)
    for rows in (slice(0, 60), slice(90, 90 + 40)):
        for name, got in (("out", out), ("lse", lse), ("dq", dq)):
            within(got[rows], value[name][rows], bound[name][rows], f"{name} {rows}")
    assert bool(torch.isnan(out[60:90]).all()) and bool(torch.isnan(lse[60:90]).all())


@gpu
def test_values_that_are_seen_and_not_finite(hip):
    """As the formula has it: inf where a weight meets it, NaN where it has no value."""
    import torch
    print_case("packed not finite")
    nq = [20]
    q, k, v, _ = make(nq, nq, 2, 1, 64, seed=5)
    v[10, 0, 3], v[12, 0, 4], v[14, 0, 5] = math.inf, -math.inf, math.nan
    out, lse = hip.attention_packed(q, k, v, offsets(nq))
    value, bound = packed(q, k, v, nq, nq, 0.125, True)
    bound["out"] = torch.nan_to_num(bound["out"])
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
def test_rows_whose_scores_are_all_minus_infinity(hip):
    """lse = -inf, the log of nothing, and no distribution to take values by; with other keys in
    sight such a key weighs nothing."""
    import torch
    print_case("packed -inf scores")
    nq = [80, 3]
    q, k, v, _ = make(nq, nq, 2, 1, 64, seed=15)
    q = q.abs() + 0.5
    k[:5, 0, 7] = -math.inf
    out, lse = hip.attention_packed(q, k, v, offsets(nq))
    assert bool((lse[:5] == -math.inf).all()) and bool(torch.isnan(out[:5]).all())
    # Rows 5 .. 79 over keys 5 .. 79: the last query sees every key, as before.
    value, bound = packed(q[5:], k[5:], v[5:], [75, 3], [75, 3], 0.125, True)
    within(out[5:], value["out"], bound["out"], "out")
    within(lse[5:], value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e30, 2e38])
def test_values_near_the_ends_of_the_range(hip, size):
    """Values of 1e-38 keep an absolute 2^-126; larger ones their relative accuracy."""
    import torch
    print_case("packed range", size)
    nq = [70, 9]
    q, k, v, _ = make(nq, nq, 2, 2, 64, seed=6)
    v.clamp_(-1, 1).mul_(size)
    out, lse = hip.attention_packed(q, k, v, offsets(nq))
    value, bound = packed(q, k, v, nq, nq, 0.125, True)
    within(out, value["out"], bound["out"] + 2.0 ** -126, "out")


@gpu
def test_rows_past_the_last_sequence_are_left(hip):
    import torch
    print_case("packed tail")
    nq, nk, tail = [30, 65], [30, 90], 70
    q, k, v, g = make(nq, nk, 2, 1, 40, seed=7, tail=tail)
    cq, ck = offsets(nq), offsets(nk)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    hip.attention_packed(q, k, v, cq, ck, out=out, lse=lse)
    hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, grads=grads)
    for t in (out, lse, *grads):
        assert bool((t[-tail:] == 7.0).all())
    a, b = sum(nq), sum(nk)
    value, bound = packed(q[:a], k[:b], v[:b], nq, nk, 40 ** -0.5, True, g[:a])
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        within(x[:-tail], value[name], bound[name], name)


@gpu
def test_gradients_into_a_fused_projection(hip):
    """dq, dk, dv written as columns of one matrix; columns beside them stay."""
    import torch
    print_case("packed fused gradients")
    nq, h, kv, d = [40, 77], 4, 2, 33
    q, k, v, g = make(nq, nq, h, kv, d, seed=9)
    cu = offsets(nq)
    out, lse = hip.attention_packed(q, k, v, cu)
    want = hip.attention_packed_backward(g, q, k, v, out, lse, cu)
    rows = torch.full((sum(nq), h + 2 * kv + 1, d), 5.0, device="cuda")
    into = [rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:h + 2 * kv]]
    hip.attention_packed_backward(g, q, k, v, out, lse, cu, grads=into)
    for x, y in zip(into, want):
        assert torch.equal(x, y)
    assert bool((rows[:, -1] == 5.0).all())


@gpu
@pytest.mark.parametrize("want", [(True, False, False), (False, True, False), (False, False, True),
                                  (False, False, False)])
def test_parts_of_the_backward(hip, want):
    import torch
    print_case("packed parts", want)
    nq, nk = [40, 77], [50, 77]
    q, k, v, g = make(nq, nk, 4, 2, 64, seed=10)
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    every = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)
    some = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, want=want)
    for w, x, y in zip(want, some, every):
        assert (x is None) == (not w) and (x is None or torch.equal(x, y))


@gpu
def test_gradients_against_differences(hip):
    """f = sum(out g): (f(x + e) - f(x - e)) / 2 e along a direction, f from the 64-bit forward of
    the same inputs, against the kernel's gradient; e = 1e-4 leaves e^2 of the third derivative,
    far below the 1e-4 of the gradient's norm that is allowed."""
    import torch
    print_case("packed differences")
    nq, nk, d = [20, 9], [33, 9], 16
    q, k, v, g = make(nq, nk, 4, 2, d, seed=11)
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    grads = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)
    base = [t.cpu().double() for t in (q, k, v)]
    gen = torch.Generator().manual_seed(1)
    for i, got in enumerate(grads):
        step = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        f = []
        for e in (1e-4, -1e-4):
            x = [t + e * step if j == i else t for j, t in enumerate(base)]
            f.append(float((packed(*x, nq, nk, d ** -0.5, True)[0]["out"] * g.cpu()).sum()))
        slope = (f[0] - f[1]) / 2e-4
        got = got.cpu().double()
        assert abs(float((got * step).sum()) - slope) <= 1e-4 * float(got.norm() * step.norm())


@gpu
def test_same_bits_each_time_and_on_another_stream(hip):
    import torch
    print_case("packed repeat")
    nq, nk = [300, 65, 1], [300, 300, 1]
    q, k, v, g = make(nq, nk, 4, 2, 64, seed=12)
    cq, ck = offsets(nq), offsets(nk)

    def both():
        out, lse = hip.attention_packed(q, k, v, cq, ck)
        return [out, lse, *hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)]

    first = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    others = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            others.append(both())
    torch.cuda.synchronize()
    for other in others:
        for x, y in zip(first, other):
            assert torch.equal(x, y)


@gpu
def test_captured_and_replayed(hip):
    import torch
    print_case("packed graph")
    nq, nk = [100, 33], [150, 33]
    q, k, v, g = make(nq, nk, 4, 2, 64, seed=13)
    cq, ck = offsets(nq), offsets(nk)

    def both():
        out, lse = hip.attention_packed(q, k, v, cq, ck)
        return [out, lse, *hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs))
    for seed in range(3):
        fresh = make(nq, nk, 4, 2, 64, seed=20 + seed)
        for t, f in zip((q, k, v, g), fresh):
            t.copy_(f)
        want = both()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            for x, y in zip(outs, want):
                assert torch.equal(x, y)


# ------------------------------------------ few rows of many keys: split and joined
# The join adds a rounding for each of up to 32 pieces and a factor within 4 u for each, less than the
# sums over the 384 keys or more that the bounds count one by one.

def splits(hip, *args, **kw):
    """attention_packed, and whether it took a second launch."""
    before = hip.launched()
    out = hip.attention_packed(*args, **kw)
    return out, hip.launched() - before == 2


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk,heads,kv,d", [
    ([16], [2000], 2, 1, 64), ([130], [1027], 1, 1, 128), ([300], [900], 4, 2, 33),
    ([700], [700], 3, 3, 96), ([1, 0, 260, 5], [1000, 900, 390, 64], 2, 1, 32),
    ([600], [450], 2, 2, 100), ([1], [4000], 8, 1, 80), ([511, 2], [511, 513], 1, 1, 17)])
def test_split_keys(hip, nq, nk, heads, kv, d, causal):
    import torch
    print_case("packed split", nq, nk, heads, kv, d, causal)
    q, k, v, _ = make(nq, nk, heads, kv, d, seed=sum(nk) + d)
    (out, lse), split = splits(hip, q, k, v, offsets(nq), offsets(nk), causal=causal)
    assert split
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, causal)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")
    again = hip.attention_packed(q, k, v, offsets(nq), offsets(nk), causal=causal)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


# The gradients' shares are added one after the other, up to 32 for each head: the bounds' sums over
# 384 rows or more count more roundings than those.

@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk,heads,kv,d", [
    ([16], [2000], 2, 1, 64), ([1500], [40], 2, 2, 64), ([700], [700], 4, 2, 96),
    ([1027], [1027], 1, 1, 128), ([1, 0, 260, 900], [1000, 900, 390, 64], 2, 1, 33),
    ([600], [450], 2, 2, 100), ([450], [600], 3, 1, 17)])
def test_split_gradients(hip, nq, nk, heads, kv, d, causal):
    import torch
    print_case("packed split gradients", nq, nk, heads, kv, d, causal)
    q, k, v, g = make(nq, nk, heads, kv, d, seed=sum(nk) + d, tail=5)
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck, causal=causal)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, causal=causal, grads=grads)
    tq, tk = sum(nq), sum(nk)
    value, bound = packed(q[:tq], k[:tk], v[:tk], nq, nk, d ** -0.5, causal, g[:tq])
    for name, got, rows in zip(("dq", "dk", "dv"), grads, (tq, tk, tk)):
        within(got[:rows], value[name], bound[name], name)
        assert bool((got[rows:] == 7.0).all()), name
    # Each alone, on the bits of all of them.
    for n in range(3):
        alone = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, causal=causal,
                                              want=tuple(m == n for m in range(3)))
        rows = (tq, tk, tk)[n]
        assert [t is None for t in alone] == [m != n for m in range(3)]
        assert torch.equal(alone[n][:rows], grads[n][:rows])


@gpu
def test_split_gradients_not_finite_and_not_seen(hip):
    """What only later rows see does not reach a row's gradients, whichever piece holds it."""
    import torch
    print_case("packed split gradients special")
    nq, nk = [200], [900]
    q, k, v, g = make(nq, nk, 2, 1, 64, seed=51)
    cq, ck = offsets(nq), offsets(nk)
    k[800:], v[830:] = math.nan, math.inf    # rows 100.. see them
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    dq = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, want=(True, False, False))[0]
    kz, vz = k.clone(), v.clone()
    kz[800:], vz[830:] = 0, 0
    value, bound = packed(q, kz, vz, nq, nk, 0.125, True, g)
    within(dq[:100], value["dq"][:100], bound["dq"][:100], "dq")
    assert bool(torch.isnan(dq[100:]).all())
    # And a query that is not finite reaches the keys it sees, not those after them.
    q, k, v, g = make([900], [900], 2, 1, 64, seed=52)
    cu = offsets([900])
    g[700] = math.nan
    out, lse = hip.attention_packed(q, k, v, cu)
    _, dk, dv = hip.attention_packed_backward(g, q, k, v, out, lse, cu)
    assert bool(torch.isnan(dk[:701]).all()) and bool(torch.isnan(dv[:701]).all())
    gz = g.clone()
    gz[700] = 0
    value, bound = packed(q, k, v, [900], [900], 0.125, True, gz)
    within(dk[701:], value["dk"][701:], bound["dk"][701:], "dk")
    within(dv[701:], value["dv"][701:], bound["dv"][701:], "dv")


@gpu
def test_split_keys_not_finite_not_seen_and_past_the_last_sequence(hip):
    import torch
    print_case("packed split special")
    nq, nk, tail = [100, 50], [1000, 700], 9
    q, k, v, _ = make(nq, nk, 2, 1, 64, seed=31, tail=tail)
    q = q.abs() + 0.5
    k[:1000, 0, 3][::2] = -math.inf          # weighs nothing
    k[940:960], v[940:960] = math.nan, math.inf  # sequence 0: rows 40.. see them, rows 0..39 do not
    v[1000 + 20, 0, 5] = math.inf            # sequence 1: all rows see it
    cq, ck = offsets(nq), offsets(nk)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    _, split = splits(hip, q, k, v, cq, ck, out=out, lse=lse)
    assert split
    assert bool((out[150:] == 7.0).all()) and bool((lse[150:] == 7.0).all())
    assert bool(torch.isnan(out[40:100]).all()) and bool(torch.isnan(lse[40:100]).all())
    assert bool((out[100:150, :, 5] == math.inf).all())
    for i in (0, 7, 39):
        seen = [j for j in range(900 + i + 1) if j % 2]
        value, bound = packed(q[i:i + 1], k[seen], v[seen], [1], [len(seen)], 0.125, False)
        # The bound's sums run over the positions that weigh nothing too.
        within(out[i:i + 1], value["out"], 2.5 * bound["out"], "out")
        within(lse[i:i + 1], value["lse"], 2.5 * bound["lse"], "lse")
    vz = v.clone()
    vz[1000 + 20, 0, 5] = 0
    value, bound = packed(q[100:150], k[1000:1700], vz[1000:1700], [50], [700], 0.125, True)
    others = [c for c in range(64) if c != 5]
    within(out[100:150][..., others], value["out"][..., others], bound["out"][..., others], "out")
    within(lse[100:150], value["lse"], bound["lse"], "lse")


@gpu
def test_split_rows_without_keys_and_with_nothing_but_minus_infinity(hip):
    import torch
    print_case("packed split empty")
    q, k, v, _ = make([500], [400], 1, 1, 32, seed=33)
    q = q.abs() + 0.5
    k[:130, 0, 1] = -math.inf                # all that rows 100..229 see
    (out, lse), split = splits(hip, q, k, v, offsets([500]), offsets([400]))
    assert split
    assert bool((out[:100] == 0).all()) and bool((lse[:230] == -math.inf).all())
    assert bool(torch.isnan(out[100:230]).all())
    value, bound = packed(q[230:], k[130:], v[130:], [270], [270], 32 ** -0.5, True)
    # The bound's sums run over the positions that weigh nothing too.
    factor = 400 / 270 + 1
    within(out[230:], value["out"], factor * bound["out"], "out")
    within(lse[230:], value["lse"], factor * bound["lse"], "lse")


@gpu
def test_split_keys_captured_and_replayed(hip):
    import torch
    print_case("packed split graph")
    nq, nk = [40, 33], [1500, 600]
    q, k, v, g = make(nq, nk, 4, 2, 64, seed=34)
    cq, ck = offsets(nq), offsets(nk)

    def both():
        (out, lse), split = splits(hip, q, k, v, cq, ck)
        assert split
        return [out, lse, *hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs))
    for seed in range(3):
        for t, f in zip((q, k, v, g), make(nq, nk, 4, 2, 64, seed=40 + seed)):
            t.copy_(f)
        want = both()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for x, y in zip(outs, want):
                assert torch.equal(x, y)


@gpu
def test_offsets_out_of_range_stay_inside_the_tensors(hip):
    """Negative, descending and too large offsets are clamped: rows around the tensors stay."""
    import torch
    print_case("packed offsets")
    n, pad, h, d = 96, 64, 2, 32
    big = [torch.full((n + 2 * pad, h, d), 3.0, device="cuda") for _ in range(7)]
    q, k, v, g, dq, dk, dv = (t[pad:pad + n] for t in big)
    out = torch.full((n + 2 * pad, h, d), 3.0, device="cuda")
    lse = torch.full((n + 2 * pad, h), 3.0, device="cuda")
    for bad in ([0, 200], [-5, 40], [0, 50, 20, 96], [90, 10], [2 ** 31 - 1, -2 ** 31, 96]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        hip.attention_packed(q, k, v, cu, out=out[pad:pad + n], lse=lse[pad:pad + n])
        hip.attention_packed_backward(g, q, k, v, out[pad:pad + n], lse[pad:pad + n], cu,
                                      grads=[dq, dk, dv])
        torch.cuda.synchronize()
        for t in (*big, out, lse):
            assert bool((t[:pad] == 3.0).all()) and bool((t[pad + n:] == 3.0).all())


@gpu
def test_empty_tensors(hip):
    import torch
    print_case("packed empty")
    none = lambda h: torch.empty(0, h, 16, device="cuda")
    some = torch.randn(9, 2, 16, device="cuda")
    cu0 = torch.zeros(3, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    out, lse = hip.attention_packed(none(4), some, some, cu0, cu)
    assert out.shape == (0, 4, 16)
    grads = hip.attention_packed_backward(none(4), none(4), some, some, out, lse, cu0, cu)
    assert bool((grads[1] == 0).all()) and bool((grads[2] == 0).all())
    q = torch.randn(9, 4, 16, device="cuda")
    out, lse = hip.attention_packed(q, none(2), none(2), cu, cu0)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = hip.attention_packed_backward(q, q, none(2), none(2), out, lse, cu, cu0)
    assert bool((dq == 0).all()) and dk.shape == (0, 2, 16)
    hip.attention_packed(none(1), none(1), none(1), torch.zeros(1, dtype=torch.int32,
                                                               device="cuda"))


# ------------------------------------------- rows, scales and sizes of their own kind

@gpu
@pytest.mark.parametrize("d", [3, 24, 64, 67, 96, 128])
def test_rows_without_keys_beside_keys_that_are_not_finite(hip, d):
    """The first 30 queries see no key; the wave that holds them also has queries that do."""
    import torch
    print_case("packed keyless beside not finite", d)
    q, k, v, g = make([70, 5], [40, 5], 2, 1, d, seed=60 + d)
    cq, ck = offsets([70, 5]), offsets([40, 5])
    for at, value in ((0, math.nan), (0, math.inf), (17, -math.inf)):
        kx, vx = k.clone(), v.clone()
        vx[at] = value
        for keys in (k, kx):
            out, lse = hip.attention_packed(q, keys, vx, cq, ck)
            dq = hip.attention_packed_backward(g, q, keys, vx, out, lse, cq, ck,
                                               want=(True, False, False))[0]
            assert bool((out[:30] == 0).all()) and bool((lse[:30] == -math.inf).all())
            assert bool((dq[:30] == 0).all())
            kx[at] = value  # the second time the key itself too


@gpu
@pytest.mark.parametrize("nq,nk", [([70, 40], [40, 70]), ([300], [900]), ([900], [500])])
def test_scale_of_zero(hip, nq, nk):
    """Even weights over what a row sees, zeros where that is nothing, and the bits of a scale that
    is too small to matter: the same arithmetic, but for lse of one key, which is scale times its
    score: 0 or some 1e-30."""
    import torch
    print_case("packed scale 0", nq, nk)
    q, k, v, g = make(nq, nk, 4, 2, 64, seed=61)
    cq, ck = offsets(nq), offsets(nk)
    got = []
    for scale in (0.0, 1e-30):
        out, lse = hip.attention_packed(q, k, v, cq, ck, scale=scale)
        dv = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, scale=scale)[2]
        got.append((out, lse, dv))
    for n in (0, 2):
        assert bool(torch.equal(got[0][n], got[1][n])), ("out", "lse", "dv")[n]
    value, bound = packed(q, k, v, nq, nk, 0.0, True, g)
    for name, x in zip(("out", "lse", "dv"), got[0]):
        within(x, value[name], bound[name], name)


@gpu
@pytest.mark.parametrize("d", [33, 64, 128])
@pytest.mark.parametrize("nq,nk", [([90, 40], [90, 60]), ([400, 3], [700, 500])])
@pytest.mark.parametrize("which,value", [("q", math.nan), ("k", math.nan), ("v", math.nan),
                                         ("v", math.inf), ("g", math.nan), ("g", -math.inf)])
def test_gradients_of_what_is_not_finite(hip, which, value, nq, nk, d):
    """NaN and infinities in one value of one row: they are where the formula has them, the gradients
    of other heads and of rows that do not meet it are as ever."""
    import torch
    print_case("packed gradients not finite", which, value, nq, nk, d)
    data = dict(zip("qkvg", make(nq, nk, 4, 2, d, seed=65 + d)))
    data[which][50, 1, d - 2] = value
    q, k, v, g = (data[n] for n in "qkvg")
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    grads = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, True, g)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        within(got, value[name], bound[name], name)


@gpu
def test_a_step_that_is_not_finite_takes_no_longer(hip):
    """A NaN that every row sees, in a key or everywhere, and not many times a finite call's time:
    rows formed again one by one took 18 times the forward's and 55 times the backward's."""
    import torch
    print_case("packed time of NaN")
    n = [512] * 4
    q, k, v, g = make(n, n, 8, 8, 64, seed=66)
    cu = offsets(n)

    def took():
        """The least of five, in ms, of the forward and of the backward."""
        calls, best = [], [math.inf, math.inf]
        out, lse = hip.attention_packed(q, k, v, cu)
        calls.append(lambda: hip.attention_packed(q, k, v, cu))
        calls.append(lambda: hip.attention_packed_backward(g, q, k, v, out, lse, cu))
        for _ in range(5):
            for i, call in enumerate(calls):
                a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
                a.record()
                call()
                b.record()
                torch.cuda.synchronize()
                best[i] = min(best[i], a.elapsed_time(b))
        return best

    took()
    finite = took()
    k[0] = math.nan
    one = took()
    for t in (q, k, v, g):
        t.fill_(math.nan)
    every = took()
    print(finite, one, every, flush=True)
    for x in (one, every):
        assert x[0] < 8 * finite[0] and x[1] < 8 * finite[1]


# One sequence of many keys among short or empty ones: offsets that are padded to a fixed count, a
# prompt's piece beside answers that get one token each.
SKEWED = [([128] + [1] * 43, [3000] + [1] * 43, 4, 2, 64), ([300] + [0] * 50, [900] + [0] * 50, 4, 1, 32),
          ([5] * 9 + [700], [5] * 9 + [700], 2, 2, 96), ([1] * 70 + [40], [3] * 70 + [2000], 2, 1, 128)]


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk,heads,kv,d", SKEWED)
def test_one_long_sequence_among_short_ones(hip, nq, nk, heads, kv, d, causal):
    """Split with the longest known; as right with lengths that are below or far above it."""
    import torch
    print_case("packed skewed", nq, nk, heads, kv, d, causal)
    q, k, v, g = make(nq, nk, heads, kv, d, seed=sum(nk) + d)
    cq, ck = offsets(nq), offsets(nk)
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, causal, g)
    for longest in ((max(nq), max(nk)), (None, max(nk)), (1, 1), (2 ** 40, 2 ** 62), (7, None)):
        kw = dict(causal=causal, longest_q=longest[0], longest_k=longest[1])
        (out, lse), split = splits(hip, q, k, v, cq, ck, **kw)
        assert split or longest[1] != max(nk)
        grads = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck, **kw)
        # A short sequence's sums count few roundings; the join adds one and a factor within 4 u.
        for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
            within(got, value[name], bound[name] + 8 * 2.0 ** -24 * value[name].abs().nan_to_num(
                posinf=0.0), name)
        again = hip.attention_packed(q, k, v, cq, ck, **kw)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@gpu
def test_the_longest_of_one_offset_array(hip):
    """cu_k left out: its longest is the queries'."""
    import torch
    print_case("packed longest")
    n = [700] + [2] * 30
    q, k, v, _ = make(n, n, 2, 1, 64, seed=67)
    cu = offsets(n)
    (out, _), split = splits(hip, q, k, v, cu, longest_q=700)
    assert split
    assert torch.equal(out, hip.attention_packed(q, k, v, cu, cu, longest_q=700, longest_k=700)[0])


@gpu
@pytest.mark.parametrize("d", [24, 64, 100])
@pytest.mark.parametrize("power", [-100, -104, -108])
def test_small_values_keep_24_bits(hip, power, d):
    """Values from 2^-110 on are held whole in their three parts. Besides the relative bound there
    is fp32's least step, 2^-149, for each of the at most 7 roundings a key (six part products and
    the running sum), times weights and a divisor that are at most 1."""
    import torch
    print_case("packed small values", power, d)
    nq, nk = [70, 9], [100, 9]
    q, k, v, _ = make(nq, nk, 2, 1, d, seed=62)
    v = (torch.rand_like(v) + 1) * v.sign() * 2.0 ** (power - 1)
    out, _ = hip.attention_packed(q, k, v, offsets(nq), offsets(nk))
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, True)
    bound = bound["out"] + 700 * 2.0 ** -149 - 1e-37  # the last is the reference's own allowance
    assert float((value["out"].abs() > 100 * bound).double().mean()) > 0.9
    within(out, value["out"], bound, "out")


@gpu
@pytest.mark.parametrize("d", [24, 64, 100])
def test_gradients_of_small_values(hip, d):
    """g near 2^-100. dv = sum p g as the forward's sums. ds is split like a value, and loses what is
    below 2^-133: within that for each of a sum's terms, times the other factor (below 6) and the
    scale (below 1)."""
    import torch
    print_case("packed small gradients", d)
    nq, nk = [70, 9], [100, 9]
    q, k, v, g = make(nq, nk, 2, 1, d, seed=64)
    g = (torch.rand_like(g) + 1) * g.sign() * 2.0 ** -101
    cq, ck = offsets(nq), offsets(nk)
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    grads = hip.attention_packed_backward(g, q, k, v, out, lse, cq, ck)
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, True, g)
    assert float(max(t.abs().max() for t in (q, k))) < 6
    for name, got, loss in zip(("dq", "dk", "dv"), grads, (6 * 100, 6 * 140, 2.0 ** -6)):
        # Two heads add to dk and dv.
        bounds = bound[name] + loss * 2.0 ** -133 - (1 if name == "dq" else 2) * 1e-37
        assert float((value[name].abs() > 10 * bounds).double().mean()) > 0.8
        within(got, value[name], bounds, name)


@gpu
@pytest.mark.parametrize("which", sorted(LENGTHS))
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (4, 1, 128), (3, 3, 24)])
def test_lengths_of_fixed_inputs(hip, which, heads, kv, d):
    """The sets of lengths on inputs that are the same in every run."""
    nq, nk = zip(*LENGTHS[which])
    for causal in (True, False):
        check(hip, nq, nk, heads, kv, d, causal, seed=1000 * sorted(LENGTHS).index(which) + d)


# Blocks of 256 queries: without the mask from 256 of them on, with it from 512 and a mean of 2048
# queries (heads of up to 96 values).

@gpu
@pytest.mark.parametrize("d", [3, 24, 31, 64, 67, 90, 96])
def test_blocks_of_256_queries(hip, d):
    import torch
    print_case("packed 256 queries", d)
    nq, nk, heads = [700, 1, 0, 323], [200, 77, 3, 130], 64
    q, k, v, _ = make(nq, nk, heads, 4, d, seed=d)
    out, lse = hip.attention_packed(q, k, v, offsets(nq), offsets(nk), causal=False)
    value, bound = packed(q, k, v, nq, nk, d ** -0.5, False)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("d", [3, 24, 64, 90])
@pytest.mark.parametrize("n", [200, 2080])
def test_causal_blocks_of_256_queries(hip, d, n):
    """Of two heads in 64, the others the same rows in other places: as many keys as queries, or
    keys for the last of them alone."""
    import torch
    print_case("packed 256 queries, causal", d, n)
    q, k, v, _ = make([2080], [n], 64, 2, d, seed=d + n)
    q = q[:, :2].repeat(1, 32, 1).reshape(2080, 32, 2, d).transpose(1, 2).reshape(2080, 64, d)
    out, lse = hip.attention_packed(q.contiguous(), k, v, offsets([2080]), offsets([n]))
    for x in (out, lse):
        x = x.reshape(2080, 2, 32, -1)
        assert torch.equal(x, x[:, :, :1].expand_as(x))
    value, bound = packed(q[:, ::32], k, v, [2080], [n], d ** -0.5, True)
    within(out[:, ::32], value["out"], bound["out"], "out")
    within(lse[:, ::32], value["lse"], bound["lse"], "lse")


@gpu
def test_blocks_of_256_queries_not_finite_and_not_seen(hip):
    import torch
    print_case("packed 256 queries special")
    q, k, v, _ = make([2100], [2050], 64, 2, 64, seed=63)
    cq, ck = offsets([2100]), offsets([2050])
    want, want_lse = hip.attention_packed(q, k, v, cq, ck)
    k[1900], v[1900] = math.nan, math.inf  # queries 1950 .. see it
    out, lse = hip.attention_packed(q, k, v, cq, ck)
    assert bool((out[:50] == 0).all()) and bool((lse[:50] == -math.inf).all())
    assert bool(torch.isnan(out[1950:]).all()) and bool(torch.isnan(lse[1950:]).all())
    assert torch.equal(out[:1800], want[:1800]) and torch.equal(lse[:1800], want_lse[:1800])
    kz, vz = k.clone(), v.clone()
    kz[1900:], vz[1900:] = 0, 0
    value, bound = packed(q[:, ::32], kz, vz, [2100], [2050], 0.125, True)
    rows = slice(1800, 1950)
    within(out[rows, ::32], value["out"][rows], bound["out"][rows], "out")
    within(lse[rows, ::32], value["lse"][rows], bound["lse"][rows], "lse")


# ----------------------------------------------------------------- refusals

def descriptor(**changes):
    fields = dict(q=4096, k=4096, v=4096, ld_q=64, ld_k=32, ld_v=32, cu_q=4096, cu_k=4096,
                  sequences=2, total_q=10, total_k=12, heads=4, kv_heads=2, head_dim=16, scale=1.0,
                  causal=1, out=4096, ld_out=64, lse=4096)
    fields.update(changes)
    return E.AttentionPacked(**fields)


def test_workspace_and_refused_descriptors():
    """The checks that every call starts with, through the query that needs no device."""
    lib = E.load_library()
    size = lib.ehip_attention_packed_backward_workspace
    assert size(C.byref(descriptor())) >= 10 * 4 * 4
    assert size(C.byref(descriptor(sequences=0, total_q=0, total_k=0, q=None, k=None, v=None,
                                   out=None, lse=None, cu_q=None, cu_k=None))) == 0
    assert size(None) == -1
    for bad in (dict(heads=3), dict(heads=0, kv_heads=0), dict(head_dim=0), dict(head_dim=129),
                dict(ld_q=63), dict(ld_k=31), dict(ld_v=31), dict(ld_out=63), dict(q=None),
                dict(k=None), dict(v=None), dict(out=None), dict(lse=None), dict(cu_q=None),
                dict(cu_k=None), dict(sequences=-1), dict(total_q=-1), dict(total_k=-1),
                dict(total_q=2 ** 31), dict(total_k=2 ** 31), dict(sequences=2 ** 24),
                dict(total_q=2 ** 30), dict(kv_heads=-2, heads=-4), dict(ld_q=2 ** 22 + 1),
                dict(ld_k=2 ** 22 + 1), dict(ld_v=2 ** 22 + 1)):
        assert size(C.byref(descriptor(**bad))) == -1, bad
        assert b"attention_packed" in lib.ehip_last_error()
        assert lib.ehip_attention_packed_workspace(C.byref(descriptor(**bad))) == -1, bad
    forward = lib.ehip_attention_packed_workspace
    assert forward(C.byref(descriptor())) == 0  # few keys
    assert forward(C.byref(descriptor(total_k=9000))) >= 10 * 4 * (16 + 2) * 4 * 2
    assert forward(C.byref(descriptor(sequences=0, total_q=0, q=None, cu_q=None, cu_k=None))) == 0


def test_a_long_sequence_among_many_is_split():
    """With the longest known a call's workspaces hold the parts of rows that the mean leaves whole."""
    lib = E.load_library()
    sizes = (lib.ehip_attention_packed_workspace, lib.ehip_attention_packed_backward_workspace)
    for short in (0, 1, 300):
        fields = dict(sequences=44, total_q=128 + 43 * min(short, 1), total_k=16384 + 43 * short)
        long = descriptor(longest_q=128, longest_k=16384, **fields)
        # Eight pieces or more of a maximum and a sum, and of 16 values, for each row and head.
        assert sizes[0](C.byref(long)) >= 8 * long.total_q * 4 * 18 * 4
        assert sizes[1](C.byref(long)) >= 8 * long.total_q * 4 * 16 * 4
        for size in sizes:  # what fills the card without is not launched many times over
            many = descriptor(**{**fields, "sequences": 10 ** 6}, longest_q=128, longest_k=16384)
            assert 0 <= size(C.byref(many)) <= 4 * (long.total_q + 2 * long.total_k) * 4 * 17
            for bad in (dict(longest_q=-1), dict(longest_k=-1)):
                assert size(C.byref(descriptor(**fields, **bad))) == -1
                assert b"longest" in lib.ehip_last_error()


def test_no_sequences_with_a_longest():
    """Rows past the last sequence only, whatever the longest is said to be: nothing to split."""
    lib = E.load_library()
    for total_q, total_k in ((0, 0), (10, 10), (10, 5000), (5000, 10), (5000, 5000)):
        for longest in (1, 5000, 2 ** 62):
            desc = descriptor(sequences=0, total_q=total_q, total_k=total_k, longest_q=longest,
                              longest_k=longest)
            assert lib.ehip_attention_packed_workspace(C.byref(desc)) == 0
            assert lib.ehip_attention_packed_backward_workspace(C.byref(desc)) >= 0


def test_a_longest_past_everything():
    """The largest number is as good as the rows there are."""
    lib = E.load_library()
    for total in (1, 10, 9000):
        sizes = [(lib.ehip_attention_packed_workspace(C.byref(d)),
                  lib.ehip_attention_packed_backward_workspace(C.byref(d)))
                 for d in (descriptor(total_q=10, total_k=total, longest_q=q, longest_k=k)
                           for q, k in ((10, total), (2 ** 63 - 1, 2 ** 63 - 1), (11, total + 1)))]
        assert sizes[0] == sizes[1] == sizes[2] and min(sizes[0]) >= 0


def test_blocks_fit_a_launch():
    """2^32 threads: blocks of 512, so 2^23 - 1 of them."""
    size = E.load_library().ehip_attention_packed_backward_workspace
    assert size(C.byref(descriptor(sequences=2 ** 21 - 2))) >= 0
    assert size(C.byref(descriptor(sequences=2 ** 21))) == -1


def binding():
    """A Backend without a device: its argument checks only."""
    import torch
    b = E.Backend.__new__(E.Backend)
    b.torch, b.lib = torch, E.load_library()
    return b


def test_binding_refuses_layouts():
    import torch
    b = binding()
    rows = torch.zeros(6, 10, 8)
    assert b._rows(rows[:, :4], "q", (6, 4, 8)) == 80
    assert b._rows(rows[:1, 4:6], "q", (1, 2, 8)) == 16
    for bad in (rows[:, ::2], rows[:, :, ::2], rows.transpose(0, 1), rows.double(),
                rows[:, :, :1].expand(6, 10, 8), torch.zeros(1, 4, 8).expand(6, 4, 8)):
        with pytest.raises(ValueError):
            b._rows(bad, "q", tuple(bad.shape))
    with pytest.raises(ValueError):
        b._rows(rows, "q", (6, 10, 9))
    with pytest.raises(ValueError):
        b._index(torch.zeros(3), "cu", 3)
    with pytest.raises(ValueError):
        b._index(torch.zeros(6, dtype=torch.int32)[::2], "cu", 3)
    with pytest.raises(ValueError):
        b._dense(rows[:, :4, 0], "lse", (6, 4))


@gpu
def test_calls_are_refused(hip):
    """Before anything is launched, with the reason."""
    import torch
    print_case("packed refusals")
    q, k, v, g = make([4], [4], 2, 1, 16, seed=1)
    cu = offsets([4])
    out, lse = hip.attention_packed(q, k, v, cu)
    launched = hip.launched()
    for args in ((q, k, v[:3], cu), (q, k, v, cu.long()), (q[0], k, v, cu),
                 (q.cpu(), k, v, cu), (q, k, v, cu, offsets([2, 2]))):
        with pytest.raises(ValueError):
            hip.attention_packed(*args)
    with pytest.raises(RuntimeError, match="heads"):
        hip.attention_packed(torch.zeros(4, 3, 16, device="cuda"), torch.zeros(4, 2, 16,
                             device="cuda"), torch.zeros(4, 2, 16, device="cuda"), cu)
    with pytest.raises(RuntimeError, match="129"):
        hip.attention_packed(*[torch.zeros(4, 1, 129, device="cuda")] * 3, cu)
    desc = hip._packed(q, k, v, cu, None, None, True, out, lse)
    space = torch.empty(64, device="cuda")
    call = lambda at, n: hip.lib.ehip_attention_packed_backward_f32(
        C.byref(desc), g.data_ptr(), 32, out.data_ptr(), 32, None, 0, None, 0, at, n,
        hip.stream())
    assert call(None, 0) == 1 and call(space.data_ptr(), 31) == 1
    assert call(space.data_ptr() + 4, 64) == 1 and "workspace" in hip.error()
    q, k, v, _ = make([4], [900], 2, 1, 16, seed=1)
    desc = hip._packed(q, k, v, offsets([4]), offsets([900]), None, True, out, lse)
    need = hip.lib.ehip_attention_packed_workspace(C.byref(desc))
    space = torch.empty(need, device="cuda")
    call = lambda at, n: hip.lib.ehip_attention_packed_f32(C.byref(desc), at, n, hip.stream())
    assert need > 0 and call(None, 0) == 1 and call(space.data_ptr(), need - 1) == 1
    assert call(space.data_ptr() + 4, need) == 1 and "workspace" in hip.error()
    assert hip.launched() == launched
