"""Attention of one new token where the sequences of a group share their first positions, against the
formula in 64 bits with the bounds of tests/_attention64.py, and against attention_paged. Joining the
shared part with the own one adds the roundings of one more part, two for each sum, of which the
bound's n + 12 terms of a weight and m + 5 of a sum count more than there are."""
import ctypes as C
import math

import pytest

import ehip as E
from _attention64 import packed, within
from _hip import print_case

gpu = pytest.mark.gpu
KINDS = ["float32", "bfloat16", "int8"]


@pytest.fixture(scope="module")
def hip():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU test ran without a visible GPU")
    return E.Backend()


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Groups of (shared positions, [own positions of each sequence]). Whole shared pages are one for
    the group, the page in which the shared positions end is every sequence's own copy."""

    def __init__(self, hip, groups, heads, kv, d, page, kind="float32", seed=0, spread=1.0,
                 extra=1):
        import torch
        gen = torch.Generator(device="cuda").manual_seed(seed)
        lengths = [p + n for p, own in groups for n in own]
        cu = [0]
        for _, own in groups:
            cu.append(cu[-1] + len(own))
        pages, rows = 2, []
        for p, own in groups:
            whole = list(range(pages, pages + p // page))
            pages += len(whole)
            for n in own:
                mine = -(-(p + n) // page) - len(whole)
                rows.append(whole + list(range(pages, pages + mine)))
                pages += mine
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        width = max([len(r) for r in rows] + [0]) + extra
        self.table = ints([[order[i] for i in r] + [0] * (width - len(r)) for r in rows]
                          ).reshape(len(rows), width)
        kp, vp = (torch.randn(pages, page, kv, d, generator=gen, device="cuda") * spread
                  for _ in range(2))
        for (p, own), first in zip(groups, cu):
            if p % page:
                at = self.table[first:first + len(own), p // page].long()
                for pool in (kp, vp):
                    pool[at, :p % page] = pool[at[:1], :p % page]
        self.scales = None
        if kind == "int8":
            codes = [torch.empty(kp.shape, dtype=torch.int8, device="cuda") for _ in range(2)]
            self.scales = [torch.empty(pages, kv, page, device="cuda") for _ in range(2)]
            hip.cache_append(kp.view(-1, kv, d), vp.view(-1, kv, d), *codes,
                             ints([list(range(pages))]), ints([0]), ints([0, pages * page]),
                             scales=self.scales)
            kp, vp = codes
        elif kind == "bfloat16":
            kp, vp = kp.bfloat16(), vp.bfloat16()
        self.kp, self.vp, self.page = kp, vp, page
        self.q = torch.randn(len(rows), heads, d, generator=gen, device="cuda")
        self.lengths, self.cu, self.shared = lengths, cu, [p for p, _ in groups]
        self.d = d

    def held(self, lengths=None):
        """(keys, values) of all sequences one after the other, in 64 bits."""
        import torch
        out = []
        for pool, sc in zip((self.kp, self.vp), self.scales or (None, None)):
            x = pool.cpu().double()
            if sc is not None:
                x = x * sc.cpu().double().transpose(1, 2)[..., None]
            x = x.reshape(-1, *x.shape[2:])
            parts = []
            for s, n in enumerate(lengths or self.lengths):
                p = torch.arange(n)
                row = self.table[s].cpu().long()
                parts.append(x[row[p // self.page] * self.page + p % self.page])
            out.append(torch.cat(parts) if parts else x[:0])
        return out

    def run(self, hip, **how):
        # No tensor is made that was given: not in a capture.
        args = dict(scales=self.scales, **how)
        names = {"lengths": self.lengths, "group_cu": self.cu, "shared": self.shared}
        lengths, cu, shared = (args.pop(n) if n in args else ints(x) for n, x in names.items())
        q, table = args.pop("q", self.q), args.pop("table", self.table)
        return hip.attention_shared(q, self.kp, self.vp, table, lengths, cu, shared, **args)

    def expect(self, scale=None, lengths=None):
        lengths = lengths or self.lengths
        return packed(self.q, *self.held(lengths), [1] * len(lengths), lengths,
                      self.d ** -0.5 if scale is None else scale, False)


def check(hip, groups, heads, kv, d, page, kind="float32", seed=0, scale=None, longest=None,
          longest_shared=None, **how):
    print_case("shared", [(p, len(o), max(o + [0])) for p, o in groups], heads, kv, d, page, kind)
    b = Batch(hip, groups, heads, kv, d, page, kind, seed, **how)
    out, lse = b.run(hip, scale=scale, longest=longest, longest_shared=longest_shared)
    value, bound = b.expect(scale)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")
    return b, out, lse


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 64), (4, 4, 24), (8, 2, 128), (5, 1, 33),
                                        (16, 1, 128), (24, 2, 64), (6, 3, 80), (17, 1, 64),
                                        (40, 2, 128)])
def test_groups_and_heads(hip, kind, heads, kv, d):
    check(hip, [(40, [1, 2, 3]), (7, [5]), (0, [4, 4]), (200, [1, 0, 130, 17, 33]), (16, [1, 1])],
          heads, kv, d, 16, kind, seed=heads)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [2, 3, 8, 15, 16, 17, 31, 33, 64, 70, 130])
@pytest.mark.parametrize("heads", [1, 4])
def test_group_sizes(hip, kind, members, heads):
    check(hip, [(100, [1 + i % 5 for i in range(members)]), (33, [1] * 3)], heads, 1, 64, 16, kind,
          seed=members)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 3, 8, 64, 100])
def test_pages_and_shared_positions_that_end_inside(hip, kind, page):
    check(hip, [(n, [1, 4, 2 * page]) for n in (1, page, page + 1, 3 * page - 1, 127, 128, 129)],
          4, 2, 64, page, kind, seed=page)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [1, 2, 5, 8, 16, 31, 32, 40, 63, 65, 72, 96, 100, 127])
def test_head_dims(hip, kind, d):
    check(hip, [(150, [3, 37] * 10), (20, [3, 1])], 4, 2, d, 8, kind, seed=d)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [1, 2, 5, 8, 16, 31, 32, 40, 63, 65, 72, 96, 100, 127])
def test_head_dims_of_many_rows(hip, kind, d):
    check(hip, [(150, [3, 37] * 20), (97, [1] * 35)], 4, 2, d, 8, kind, seed=d)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 3, 8, 64, 100])
def test_pages_of_many_rows(hip, kind, page):
    check(hip, [(n, [1, 2 * page] * 20) for n in (1, page + 1, 3 * page - 1, 129)], 4, 2, 64, page,
          kind, seed=page)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups", [[(5000, [1] * 3)], [(3000, [2000, 1] * 12), (1, [1, 1])],
                                    [(17, [1, 1])] * 40 + [(4096, [129] * 9)],
                                    [(1025, [1] * 100)]])
def test_lengths_that_are_split(hip, kind, groups):
    check(hip, groups, 4, 2, 64, 16, kind, seed=len(groups))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale,spread", [(0.0, 1.0), (-0.2, 3.0), (0.125, 40.0)])
def test_scales_and_sharp_rows(hip, kind, scale, spread):
    check(hip, [(700, [1, 33] * 6), (9, [3, 3])], 4, 2, 64, 16, kind, seed=4, scale=scale,
          spread=spread)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_bounds_on_the_lengths(hip, kind):
    groups = [((37 * i) % 300, [(13 * i + j) % 50 for j in range(i % 7)]) for i in range(40)]
    for longest, longest_shared in ((None, None), (400, 300), (5000, 1000), (2 ** 20, 2 ** 20)):
        check(hip, groups, 4, 2, 32, 32, kind, seed=5, longest=longest,
              longest_shared=longest_shared)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_as_attention_over_the_whole_tables(hip, kind):
    """Nothing shared, and no groups: what attention_paged gives, bit for bit."""
    import torch
    groups = [(90, [1, 40, 3]), (33, [2, 2])]
    b, out, lse = check(hip, groups, 8, 2, 64, 16, kind, seed=6)
    want, want_lse = hip.attention_paged(b.q, b.kp, b.vp, b.table, ints(b.lengths),
                                         scales=b.scales)
    for how in (dict(shared=ints([0, 0])), dict(group_cu=ints([0]), shared=ints([])),
                dict(group_cu=ints([0, 0, 0])), dict(shared=ints([-1, -2 ** 31])),
                dict(shared=ints([10 ** 6, 2 ** 31 - 1])), dict(longest_shared=20)):
        o, l = b.run(hip, **how)
        assert torch.equal(o, want) and torch.equal(l, want_lse)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_are_not_shared(hip, kind):
    """In no group, alone in one, shorter than the shared positions, empty: passed whole."""
    b = Batch(hip, [(50, [3, 1, 9, 2]), (30, [4, 4, 4]), (60, [7])], 4, 2, 64, 16, kind, seed=7)
    lengths = list(b.lengths)
    lengths[1], lengths[2], lengths[5] = 0, 31, 29
    out, lse = b.run(hip, lengths=ints(lengths), group_cu=ints([0, 4, 6]), shared=ints([50, 30]))
    value, bound = b.expect(lengths=lengths)
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_bad_pages_and_lengths(hip, kind):
    """A page outside the pool among a group's shared positions, or in a sequence's own; lengths
    below zero, past `longest` or the table."""
    import torch
    b, want, want_lse = check(hip, [(40, [1, 2, 3]), (100, [5, 5, 30, 30])], 4, 2, 64, 16, kind,
                              seed=8, longest=200)
    table = b.table.clone()
    table[0, 1] = b.kp.shape[0]                      # shared by the first group
    table[4, 7], table[5, 0] = -1, 2 ** 31 - 1       # its own; shared, but of the first alone
    out, lse = b.run(hip, table=table, longest=200)
    for s in range(7):
        if s in (0, 1, 2):
            assert bool(torch.isnan(out[s]).all()) and bool(torch.isnan(lse[s]).all())
        elif s != 4:
            assert torch.equal(out[s], want[s]) and torch.equal(lse[s], want_lse[s])
    # Positions 112 on of sequence 4 are past its length.
    assert torch.equal(out[4], want[4])
    table[4, 6] = -1
    out, _ = b.run(hip, table=table, longest=200)
    assert bool(torch.isnan(out[4]).all()) and torch.equal(out[5], want[5])
    lengths = list(b.lengths)
    lengths[0], lengths[3], lengths[6] = -1, 201, 2 ** 31 - 1
    out, lse = b.run(hip, lengths=ints(lengths), longest=200)
    for s in range(7):
        if s in (0, 3, 6):
            assert bool(torch.isnan(out[s]).all()) and bool(torch.isnan(lse[s]).all())
        else:
            assert torch.equal(out[s], want[s]) and torch.equal(lse[s], want_lse[s])


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_group_offsets_that_are_none(hip, kind):
    """Out of range or descending: clamped, the others' rows are what they were, all are finite."""
    import torch
    b, want, _ = check(hip, [(40, [1, 2, 3]), (100, [5, 5, 30, 30])], 4, 2, 64, 16, kind, seed=9)
    for cu in ([0, 3, 2 ** 31 - 1], [-5, 3, 7], [-2 ** 31, 3, 7]):
        out, _ = b.run(hip, group_cu=ints(cu))
        assert torch.equal(out, want)
    for cu in ([3, 0, 7], [7, 0, 7], [100, 50, 0], [2, 2, 2]):
        out, _ = b.run(hip, group_cu=ints(cu))
        assert bool(torch.isfinite(out).all())
    many = ints([0, 7] * 500 + [0])
    out, _ = b.run(hip, group_cu=many, shared=ints([40] * 1000))
    assert bool(torch.isfinite(out).all())


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("members", [2, 40])
def test_positions_past_the_lengths_do_not_reach_a_row(hip, kind, d, members):
    import torch
    b, want, _ = check(hip, [(40, [1, 2, 3]), (130, [5, 1] * members)], 4, 2, d, 16, kind, seed=10)
    used = torch.zeros(b.kp.shape[:2], dtype=torch.bool, device="cuda")
    for s, n in enumerate(b.lengths):
        for p in range(n):
            used[b.table[s, p // 16].long(), p % 16] = True
    if kind == "int8":
        b.kp[~used], b.vp[~used] = 127, -128
        for sc in b.scales:
            sc.transpose(1, 2)[~used] = math.nan
    else:
        b.kp[~used], b.vp[~used] = math.nan, math.inf
    assert torch.equal(b.run(hip)[0], want)


@gpu
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("which,value", [("k", math.nan), ("k", math.inf), ("k", -math.inf),
                                         ("v", math.nan), ("v", math.inf)])
def test_shared_values_that_are_not_finite(hip, which, value, members, kind):
    """A key of -inf is a score of -inf where q is positive: weight 0. Else as the formula has it."""
    import torch
    print_case("shared not finite", which, value, members, kind)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, kind, seed=11)
    b.q = torch.rand_like(b.q) + 0.5
    pool = b.kp if which == "k" else b.vp
    for p in (0, 170, 299):
        pool[b.table[0, p // 16].long(), p % 16, 0, 7] = value
        if p >= 288:  # the page in which they end: every sequence's copy
            pool[b.table[:members, p // 16].long(), p % 16, 0, 7] = value
    out, lse = b.run(hip)
    want, bound = b.expect()
    if which == "k" and value != -math.inf:
        assert bool(torch.isnan(out[:members, :2]).all()) and bool(torch.isnan(lse[:members, :2]).all())
        out, lse = out[:, 2:], lse[:, 2:]
        want = {n: x[:, 2:] for n, x in want.items()}
        bound = {n: x[:, 2:] for n, x in bound.items()}
    elif which == "k":
        keep = [p for p in range(300) if p not in (0, 170, 299)]
        kx, vx = b.held()
        at = torch.cat([torch.tensor(keep + [300, 301]) + 302 * s for s in range(members)]
                       + [torch.arange(302 * members, kx.shape[0])])
        n = [299] * members + [41, 41]
        want, bound = packed(b.q, kx[at], vx[at], [1] * len(n), n, 0.125, False)
        other, other_bound = b.expect()  # the other key head has them all
        for name in want:
            want[name][:, 2:], bound[name][:, 2:] = other[name][:, 2:], other_bound[name][:, 2:]
    within(out, want["out"], bound["out"], "out")
    within(lse, want["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("members", [3, 40])
def test_scales_and_queries_that_are_not_finite(hip, members):
    import torch
    b, want, want_lse = check(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, "int8",
                              seed=12)
    b.q[1, 3, 5] = math.nan
    b.scales[1][int(b.table[0, 3]), 0, 2] = math.nan
    out, lse = b.run(hip)
    assert bool(torch.isnan(out[:members, :2]).all())
    assert bool(torch.isnan(out[1, 3]).all()) and bool(torch.isnan(lse[1, 3]))
    out[1, 3], lse[1, 3] = want[1, 3], want_lse[1, 3]
    assert torch.equal(out[:, 2:], want[:, 2:]) and torch.equal(lse[:, 2:], want_lse[:, 2:])
    assert torch.equal(out[members:], want[members:])
    # Rows that meet a NaN are formed a second time, in another order: within the same bounds.
    b.q[1, 3, 5] = 0.0
    value, bound = packed(b.q[:, :2], *[b.held()[0][:, :1]] * 2, [1] * len(b.lengths), b.lengths,
                          0.125, False)
    within(lse[:, :2], value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("members", [2, 40])
def test_shared_scores_that_are_all_minus_infinity(hip, kind, members):
    """All of the shared positions, or of the own ones, weigh nothing beside the others."""
    import torch
    print_case("shared -inf", kind, members)
    for shared in (True, False):
        b = Batch(hip, [(200, [3] * members)], 2, 1, 64, 1, kind, seed=13)
        b.q = torch.rand_like(b.q) + 0.5
        rows = b.table[:, :200] if shared else b.table[:, 200:203]
        b.kp[rows.long().reshape(-1), 0, 0, 9] = -math.inf
        out, lse = b.run(hip)
        kx, vx = b.held()
        at = torch.cat([torch.arange(200, 203) + 203 * s if shared else torch.arange(200) + 203 * s
                        for s in range(members)])
        n = [3 if shared else 200] * members
        want, bound = packed(b.q, kx[at], vx[at], [1] * members, n, 0.125, False)
        within(out, want["out"], bound["out"], "out")
        within(lse, want["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_strides_and_outputs(hip, kind):
    import torch
    b, want, want_lse = check(hip, [(100, [3] * 20), (17, [1, 1])], 4, 2, 40, 16, kind, seed=14)
    n = len(b.lengths)
    rows = torch.full((n, 9, 40), 5.0, device="cuda")
    rows[:, 4:8] = b.q
    into = torch.full((n, 6, 40), 5.0, device="cuda")
    big = torch.full((n + 1, b.table.shape[1] + 4), -9, dtype=torch.int32, device="cuda")
    big[:n, :b.table.shape[1]] = b.table
    lse = torch.empty(n, 4, device="cuda")
    b.run(hip, q=rows[:, 4:8], table=big[:n, :b.table.shape[1]], out=into[:, 1:5], lse=lse)
    assert torch.equal(into[:, 1:5], want) and torch.equal(lse, want_lse)
    assert bool((into[:, 0] == 5.0).all()) and bool((into[:, 5] == 5.0).all())


@gpu
@pytest.mark.parametrize("members", [3, 20, 80])
@pytest.mark.parametrize("kind", KINDS)
def test_pools_at_any_address(hip, kind, members):
    import torch
    b, want, _ = check(hip, [(300, [3] * members), (17, [1, 1])], 4, 2, 64, 16, kind, seed=15)
    for name in ("kp", "vp"):
        pool = getattr(b, name)
        flat = torch.zeros(pool.numel() + 3, dtype=pool.dtype, device="cuda")
        flat[3:] = pool.reshape(-1)
        setattr(b, name, flat[3:].view(pool.shape))
    out, lse = b.run(hip)
    value, bound = b.expect()
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 1)])
def test_many_groups(hip, kind, heads, kv):
    """More groups, and more sequences, than a wave has lanes, of uneven lengths."""
    groups = [((29 * i) % 70, [(11 * i + 5 * j) % 23 for j in range(1 + i % 5)])
              for i in range(150)]
    check(hip, groups, heads, kv, 32, 8, kind, seed=18)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [3, 40])
def test_values_next_to_the_largest(hip, kind, members):
    """Weighted sums before their division by the weights' are past fp32, what comes out is not."""
    print_case("shared large", kind, members)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, kind, seed=19)
    if kind == "int8":
        b.scales[1].fill_(2.0 ** 119)
        b.vp.copy_(b.vp.abs())
    else:
        b.vp.copy_((b.vp.float().abs().clamp(max=1.9) * 2.0 ** 126).to(b.vp.dtype))
    out, lse = b.run(hip)
    value, bound = b.expect()
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("power", [-70, -80, 100])
@pytest.mark.parametrize("members", [3, 40])
def test_small_and_large_scales(hip, power, members):
    """A weight times its scale runs in parts of at least 2^-133, of 2^-24 of it at the least: 2^-109
    of a position, with codes of up to 127 2^-102 in what it stands for, and as much for the sums."""
    print_case("shared scales", power, members)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, "int8", seed=20)
    b.scales[1].mul_(2.0 ** power)
    out, lse = b.run(hip)
    value, bound = b.expect()
    within(out, value["out"], bound["out"] + 302 * 2.0 ** -100, "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("power", [113, 118, 120, 122, 126])
def test_large_queries_and_small_scales(hip, power, members):
    """Queries times the whole numbers of a cache in 8 bits alone are past fp32, the scores are not."""
    print_case("shared large q", power, members)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, "int8", seed=22)
    b.scales[0].mul_(2.0 ** -power)
    b.q.mul_(2.0 ** power)
    b.kp[:, :, 0].abs_()
    b.q[::2, 0] = -b.q[::2, 0].abs()  # sums far below zero alone
    out, lse = b.run(hip)
    value, bound = b.expect()
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("power", [100, 104, 110, 118, 124])
def test_small_queries_and_large_keys(hip, power, members, kind):
    """Scores of ordinary size from queries whose parts in bf16 would lose bits."""
    print_case("shared small q", power, members, kind)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, kind, seed=23)
    b.q.mul_(2.0 ** -power)
    if kind == "int8":
        b.scales[0].mul_(2.0 ** power)
    else:
        b.kp.mul_(2.0 ** power)
    out, lse = b.run(hip)
    value, bound = b.expect()
    within(out, value["out"], bound["out"], "out")
    within(lse, value["lse"], bound["lse"], "lse")


@gpu
@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("power", [100, 110, 118, 124])
def test_small_keys_and_large_queries(hip, power, members, kind):
    """Shared fp32 keys are taken to 2^-134: a score is off by that times the sum of its |scale q|, the
    weights by twice the largest of that, relative, and lse by it. bf16 keys are exact."""
    print_case("shared small k", power, members, kind)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 64, 16, kind, seed=24)
    b.q.mul_(2.0 ** power)
    b.kp = (b.kp.float() * 2.0 ** -power).to(b.kp.dtype)
    out, lse = b.run(hip)
    value, bound = b.expect()
    off = 0.0 if kind == "bfloat16" else (
        1.01 * 2.0 ** -134 * b.q.cpu().double().abs().sum(-1) * b.d ** -0.5)
    largest = float(b.vp.float().abs().max())
    within(out, value["out"], bound["out"] + (2 * off * largest)[..., None] if kind == "float32"
           else bound["out"], "out")
    within(lse, value["lse"], bound["lse"] + off, "lse")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("which", ["k", "v"])
def test_odd_heads_that_are_not_finite(hip, kind, members, which):
    """Heads whose rows begin at any address, formed a second time: a NaN key or scale of the shared
    positions is its key head's in the group, one value's its column's."""
    import torch
    print_case("shared odd not finite", kind, members, which)
    b, want, want_lse = check(hip, [(300, [2] * members), (40, [1, 1])], 4, 2, 33, 16, kind, seed=21)
    page = int(b.table[0, 3])
    if kind == "int8":
        b.scales[which == "v"][page, 0, 2] = math.nan
    else:
        (b.kp if which == "k" else b.vp)[page, 2, 0, 7] = math.nan
    out, lse = b.run(hip)
    columns = [7] if which == "v" and kind != "int8" else list(range(33))
    assert bool(torch.isnan(out[:members, :2][..., columns]).all())
    rest = [c for c in range(33) if c not in columns]
    value, bound = b.expect()
    within(out[:members, :2][..., rest], value["out"][:members, :2][..., rest],
           bound["out"][:members, :2][..., rest], "out")
    if which == "k":
        assert bool(torch.isnan(lse[:members, :2]).all())
    else:
        within(lse[:members, :2], value["lse"][:members, :2], bound["lse"][:members, :2], "lse")
    assert torch.equal(out[:, 2:], want[:, 2:]) and torch.equal(lse[:, 2:], want_lse[:, 2:])
    assert torch.equal(out[members:], want[members:])


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("members", [3, 80])
def test_a_cache_past_32_bit_offsets(hip, kind, members):
    """The same pages at the end of pools of 2^31 values and more: the same bits."""
    import torch
    print_case("shared large cache", kind, members)
    b = Batch(hip, [(300, [2] * members), (40, [1, 1])], 8, 8, 128, 128, kind, seed=22)
    want, want_lse = b.run(hip)
    pages, count = 16400, b.kp.shape[0]
    at = pages - 1 - torch.arange(count, device="cuda")
    for name in ("kp", "vp"):
        pool = getattr(b, name)
        big = torch.zeros(pages, *pool.shape[1:], dtype=pool.dtype, device="cuda")
        assert big.numel() > 2 ** 31
        big[at] = pool
        setattr(b, name, big)
    if b.scales is not None:
        scales = [torch.zeros(pages, *x.shape[1:], device="cuda") for x in b.scales]
        for big, x in zip(scales, b.scales):
            big[at] = x
        b.scales = scales
    b.table = (pages - 1 - b.table).to(torch.int32)
    out, lse = b.run(hip)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    del b, big
    torch.cuda.empty_cache()


@gpu
def test_no_sequences(hip):
    import torch
    print_case("shared no sequences")
    kp = torch.zeros(2, 4, 1, 8, device="cuda")
    out, lse = hip.attention_shared(torch.empty(0, 2, 8, device="cuda"), kp, kp,
                                    torch.empty(0, 3, dtype=torch.int32, device="cuda"), ints([]),
                                    ints([0, 0]), ints([5]))
    assert out.shape == (0, 2, 8) and lse.shape == (0, 2)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_same_bits_each_time_on_other_streams_and_in_a_graph(hip, kind):
    import torch
    b, want, want_lse = check(hip, [(1000, [30] * 20), (40, [1, 1]), (300, [5, 0, 5])], 8, 2, 64,
                              16, kind, seed=16, longest=1100, longest_shared=1024)
    n, cu, shared = ints(b.lengths), ints(b.cu), ints(b.shared)

    def step():
        return b.run(hip, lengths=n, group_cu=cu, shared=shared, longest=1100, longest_shared=1024)

    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(step())
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
        b.q.copy_(torch.randn_like(b.q))
        n.copy_(ints([x - i if x > 30 else x for x in b.lengths]))
        shared.copy_(ints([1000 - 100 * i, 40 - 30 * i, 290]))
        cu.copy_(ints([0, 20 - 7 * i, 22, 25]) if i != 2 else ints([0, 20, 22, 22]))
        o, l = step()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert torch.equal(outs[0], o) and torch.equal(outs[1], l)


@gpu
def test_answers_to_prompts_step_by_step(hip):
    """Prompts are written once, their answers grow by a token a step: each step's attention is that
    of packed attention over all that was written."""
    import torch
    print_case("shared steps")
    gen = torch.Generator(device="cuda").manual_seed(17)
    prompts, members, page, kv, d = [37, 100], [3, 4], 16, 2, 64
    normal = lambda *n: torch.randn(*n, generator=gen, device="cuda")
    weight, freqs = 1 + 0.2 * normal(d), hip.rotary_frequencies(d)
    pages, rows, starts = 0, [], []
    for p, m in zip(prompts, members):
        whole = list(range(pages, pages + p // page))
        pages += len(whole)
        for _ in range(m):
            rows.append(whole + [pages, pages + 1])
            pages += 2
            starts.append(p)
    width = max(len(r) for r in rows)
    table = ints([r + [0] * (width - len(r)) for r in rows])
    kp, vp = (torch.zeros(pages, page, kv, d, device="cuda") for _ in range(2))
    n = len(rows)
    keys, values = [], []
    # Each prompt's rows, written for every answer (whole pages by all, the same values).
    for g, p in enumerate(prompts):
        k, v = normal(p, kv, d), normal(p, kv, d)
        at = torch.arange(p, dtype=torch.int32, device="cuda")
        _, k = hip.norm_rotate(k, k, at, freqs, weight, weight)
        for s in range(sum(members[:g]), sum(members[:g + 1])):
            hip.cache_append(k, v, kp, vp, table[s:s + 1], ints([0]), ints([0, p]))
            keys.append(k)
            values.append(v)
    group_cu, shared = ints([0, 3, 7]), ints(prompts)
    for step in range(20):
        at = ints([x + step for x in starts])
        fused = normal(n, 4 + 2 * kv, d)
        q, k = hip.norm_rotate(fused[:, :4], fused[:, 4:6], at, freqs, weight, weight)
        hip.cache_append(k, fused[:, 6:], kp, vp, table, at)
        keys = [torch.cat([a, k[s:s + 1]]) for s, a in enumerate(keys)]
        values = [torch.cat([a, fused[s:s + 1, 6:]]) for s, a in enumerate(values)]
        lengths = [x + step + 1 for x in starts]
        out, lse = hip.attention_shared(q, kp, vp, table, ints(lengths), group_cu, shared)
        if step % 6 == 0 or step == 19:
            value, bound = packed(q, torch.cat(keys), torch.cat(values), [1] * n, lengths, 0.125,
                                  False)
            within(out, value["out"], bound["out"], "out")
            within(lse, value["lse"], bound["lse"], "lse")


# ----------------------------------------------------------------- refusals

def cache(**changes):
    d = dict(k_pages=64, v_pages=64, type=0, pages=4, page_size=16, kv_heads=2, head_dim=64,
             table=64, ld_table=4, table_width=4, sequences=3, k_scales=None, v_scales=None)
    d.update(changes)
    return E.Cache(*[d[n] for n, _ in E.Cache._fields_])


REFUSED = [(dict(type=3), 4, 64, 1, 64), (dict(type=2), 4, 64, 1, 64), (dict(head_dim=129), 4, 64, 1, 64),
           ({}, 3, 64, 1, 64), ({}, 0, 64, 1, 64), ({}, 4, -1, 1, 64), ({}, 4, 2 ** 31, 1, 64),
           ({}, 4, 64, -1, 64), ({}, 4, 64, 2 ** 24, 64), ({}, 4, 64, 1, -1),
           ({}, 4, 64, 1, 2 ** 30 + 1), (dict(sequences=2 ** 20), 4, 64, 1, 2 ** 30)]


@pytest.mark.parametrize("changes,heads,longest,groups,longest_shared", REFUSED)
def test_refused_queries(changes, heads, longest, groups, longest_shared):
    """The query answers without a device."""
    lib = E.load_library()
    assert lib.ehip_attention_shared_workspace(C.byref(cache(**changes)), heads, longest, groups,
                                               longest_shared) == -1
    assert b"attention_shared" in lib.ehip_last_error()


def test_workspace_query():
    lib = E.load_library()
    ask = lambda g=2, n=64, **c: lib.ehip_attention_shared_workspace(C.byref(cache(**c)), 4, 64, g, n)
    assert ask() > 0 and ask(sequences=0) == 0 and ask(g=0) > 0 and ask(n=0) > 0


@gpu
def test_refused_calls(hip):
    import torch
    print_case("shared refused")
    lib = hip.lib

    def call(changes={}, q=64, ld_q=1 << 20, heads=4, lengths=64, longest=64, cu=64, shared=64,
             groups=2, most=64, out=64, ld_out=1 << 20, w=64, n=1 << 40):
        return lib.ehip_attention_shared_f32(C.byref(cache(**changes)), q, ld_q, heads, lengths,
                                             longest, cu, shared, groups, most, 1.0, out, ld_out,
                                             None, w, n, None)

    for changes, heads, longest, groups, most in REFUSED:
        assert call(changes, heads=heads, longest=longest, groups=groups, most=most) == 1
    for bad in (dict(q=None), dict(lengths=None), dict(cu=None), dict(shared=None), dict(out=None),
                dict(ld_q=255), dict(ld_out=255), dict(w=None), dict(w=72), dict(n=100)):
        assert call(**bad) == 1, bad
    b = Batch(hip, [(20, [1, 1])], 4, 2, 64, 16)
    for how in (dict(group_cu=ints([[0, 2]])), dict(group_cu=ints([])), dict(shared=ints([20, 20])),
                dict(shared=torch.tensor([20], device="cuda")), dict(q=b.q[0]),
                dict(lengths=ints([21])), dict(group_cu=ints([0, 2]).cpu())):
        with pytest.raises(ValueError):
            b.run(hip, **how)
