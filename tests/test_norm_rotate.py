"""Norms of query and key heads with the rotation by position, and their gradients, against 64 bits.

u = 2^-24. A head's sum of D squares is a chain of eight, then six additions: with the mean, eps,
root and division r is within 12 u of itself, y = x r w within 14 u |y|. The sine and cosine of the
reduced angle, rounded once to fp32, are within 4 u: 0.79 for that rounding, at most 2.5 for the
series' own, 2^-28 for what it leaves out.
  out:  20 u (|y_a| + |y_b|), two roundings included; 14 u |y| where nothing turns
  turned gradient t:  e = 6 u (|g_a| + |g_b|)
  m = mean(w t x r):  mean of |w x r| (e + 30 u |t|)
  dx = r (w t - x r m):  r (|w| e + 20 u (|w t| + |x r m|) + |x r| times m's)
  dw:   sum of |x r| (e + 14 u |t|), and u for each of the n terms of the magnitudes' sum
"""
import ctypes as C
import math

import pytest

import ehip as E
from _hip import print_case

gpu = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def hip():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU test ran without a visible GPU")
    return E.Backend()


def turned(x, cos, sin, rotary, interleaved, magnitudes=False):
    """The pairs of x (tokens, heads, D) turned; with `magnitudes` the sums |a| + |b| at both."""
    import torch
    i = torch.arange(rotary // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
    y = x.clone()
    xa, xb = x[..., a], x[..., b]
    if magnitudes:
        y[..., a] = y[..., b] = xa.abs() + xb.abs()
    else:
        c, s = cos[:, None], sin[:, None]
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def formula(x, w, angle, rotary, interleaved, eps, g=None):
    """(values, bounds) of one of q and k: out, and with g of dx and dw. 64 bits, on the CPU."""
    import torch
    cos, sin = torch.cos(angle), torch.sin(angle)
    d = x.shape[-1]
    r = torch.ones_like(x[..., :1]) if w is None else 1 / torch.sqrt((x * x).mean(-1, keepdim=True)
                                                                      + eps)
    y = x * r * w if w is not None else x
    value = {"out": turned(y, cos, sin, rotary, interleaved)}
    bound = {"out": 20 * U * turned(y.abs(), cos, sin, rotary, interleaved, True)}
    if g is not None:
        t = turned(g, cos, -sin, rotary, interleaved)
        e = 6 * U * turned(g.abs(), cos, sin, rotary, interleaved, True)
        if w is None:
            value["dx"], bound["dx"] = t, e
        else:
            xr = x * r
            m = (w * t * xr).mean(-1, keepdim=True)
            em = ((w * xr).abs() * (e + 30 * U * t.abs())).mean(-1, keepdim=True)
            value["dx"] = r * (w * t - xr * m)
            bound["dx"] = r * (w.abs() * e + 20 * U * ((w * t).abs() + (xr * m).abs())
                               + xr.abs() * em)
            value["dw"] = (t * xr).sum((0, 1))
            n = x.shape[0] * x.shape[1]
            bound["dw"] = (xr.abs() * (e + 14 * U * t.abs())).sum((0, 1)) + (n + 8) * U * (
                t * xr).abs().sum((0, 1))
    return value, {k: 1.01 * b + 1e-37 for k, b in bound.items()}


def within(got, value, bound, what):
    import torch
    got = got.detach().cpu().double()
    assert got.shape == value.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    off = torch.nan_to_num((got - value).abs() - bound, nan=0.0)
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over"


def make(tokens, h, kv, d, rotary, seed=0, fused=False, norm=(True, True), far=False):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *n: torch.randn(*n, generator=gen, device="cuda")
    if fused:
        rows = normal(tokens, h + 2 * kv, d)
        q, k = rows[:, :h], rows[:, h:h + kv]
    else:
        q, k = normal(tokens, h, d), normal(tokens, kv, d)
    top = 2 ** 31 - 1 if far else 5000
    at = torch.randint(-top if far else 0, top, (tokens,), generator=gen, device="cuda")
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    freqs = 10000.0 ** (-2 * i / max(1, rotary))
    w = [1 + 0.3 * normal(d) if n else None for n in norm]
    return (q, k, at.to(torch.int32), freqs, *w), (normal(tokens, h, d), normal(tokens, kv, d))


def check(hip, tokens, h, kv, d, rotary, interleaved=False, eps=1e-6, back=True, **how):
    import torch
    print_case("norm_rotate", tokens, h, kv, d, rotary, interleaved, how)
    what, grads = make(tokens, h, kv, d, rotary, **how)
    q, k, at, freqs, *w = what
    outs = hip.norm_rotate(*what, eps=eps, interleaved=interleaved)
    got = hip.norm_rotate_backward(*grads, *what, eps=eps, interleaved=interleaved) if back else None
    angle = at.cpu().double()[:, None] * freqs.cpu()[None, :]
    for i, name in enumerate("qk"):
        value, bound = formula(what[i].cpu().double(),
                               None if w[i] is None else w[i].cpu().double(), angle, rotary,
                               interleaved, eps, grads[i].cpu().double())
        within(outs[i], value["out"], bound["out"], name)
        if back:
            within(got[i], value["dx"], bound["dx"], "d" + name)
            if w[i] is None:
                assert got[2 + i] is None
            else:
                within(got[2 + i], value["dw"], bound["dw"], "d" + name + "_weight")
    return what, grads, outs, got


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [1, 2, 3, 4, 6, 7, 8, 15, 16, 24, 33, 63, 64, 77, 80, 96, 127, 128,
                               160, 201, 256])
def test_head_sizes(hip, d, interleaved):
    check(hip, 7, 5, 2, d, d // 2 * 2, interleaved, seed=d)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(8, 2), (64, 0), (64, 2), (64, 6), (64, 32), (65, 64),
                                      (96, 48), (100, 10), (128, 126), (128, 64), (256, 2),
                                      (256, 128), (250, 246)])
def test_parts_of_a_head(hip, d, rotary, interleaved):
    check(hip, 6, 3, 3, d, rotary, interleaved, seed=d + rotary)


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 3, 63, 64, 257, 1000, 4099])
@pytest.mark.parametrize("h,kv", [(1, 1), (4, 1), (6, 3), (16, 16)])
def test_tokens_and_heads(hip, tokens, h, kv):
    check(hip, tokens, h, kv, 24, 24, seed=tokens)


@gpu
def test_many_tokens(hip):
    """More than the backward's blocks have at a time."""
    check(hip, 20011, 3, 1, 64, 64, seed=1)


@gpu
@pytest.mark.parametrize("tokens,h,kv,d", [(20011, 3, 1, 64), (4099, 16, 16, 24), (30000, 1, 1, 128),
                                           (8192, 16, 4, 64), (65536, 2, 1, 16)])
def test_weights_gradients_of_many_tokens(hip, tokens, h, kv, d):
    """No share is lost on the way. The sums are no chain of all terms: a lane adds those of its wave's
    turns, one in 4096 of the tokens with at most all heads each, the lanes of a wave join in 6 steps,
    its waves in 4, up to 1024 blocks in 16 and 64. So many times u of the magnitudes' sum, beside
    the terms' own errors, is what they may be off by. Without the terms of any eight tokens in a
    row, a part of what a block has, the result would not pass."""
    import torch
    print_case("norm_rotate dw", tokens, h, kv, d)
    what, grads = make(tokens, h, kv, d, d, seed=15)
    got = hip.norm_rotate_backward(*grads, *what)
    angle = what[2].cpu().double()[:, None] * what[3].cpu()[None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    for i, name in enumerate("qk"):
        x, g, w = what[i].cpu().double(), grads[i].cpu().double(), what[4 + i]
        xr = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        t = turned(g, cos, -sin, d, False)
        e = 6 * U * turned(g.abs(), cos, sin, d, False, True)
        terms, value = t * xr, (t * xr).sum((0, 1))
        depth = -(-tokens // 4096) * x.shape[1] + 6 + 4 + 16 + 64
        bound = 1.01 * ((xr.abs() * (e + 14 * U * t.abs())).sum((0, 1))
                        + depth * U * terms.abs().sum((0, 1)))
        within(got[2 + i], value, bound, f"d{name}_weight")
        for at in range(0, tokens - 8, tokens // 7):
            with pytest.raises(AssertionError):
                within(value - terms[at:at + 8].sum((0, 1)), value, bound, "")


@gpu
@pytest.mark.parametrize("norm", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("fused", [False, True])
def test_norms_and_fused_rows(hip, norm, fused):
    check(hip, 33, 8, 2, 40, 32, norm=norm, fused=fused, seed=2)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(hip, interleaved):
    """Angles of up to 2^31: the sine of fp32's product would have no digit."""
    check(hip, 50, 2, 1, 64, 64, interleaved, far=True, seed=3)


@gpu
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-2, 100.0])
def test_eps(hip, eps):
    check(hip, 9, 3, 1, 32, 32, eps=eps, seed=4)


@gpu
def test_heads_of_zeros_and_what_is_not_finite(hip):
    """A head of zeros gives zeros; a NaN or an infinity stays in its head."""
    import torch
    print_case("norm_rotate not finite")
    (q, k, at, freqs, wq, wk), (gq, gk) = make(5, 4, 2, 32, 16, seed=5)
    want = hip.norm_rotate(q, k, at, freqs, wq, wk)
    q[1, 2] = 0.0
    q[2, 0, 3], q[3, 1, 31], k[4, 1, 0] = math.nan, math.inf, -math.inf
    outs = hip.norm_rotate(q, k, at, freqs, wq, wk)
    assert bool((outs[0][1, 2] == 0).all())
    assert bool(torch.isnan(outs[0][2, 0]).all())
    assert bool(torch.isnan(outs[0][3, 1, 31])) and bool((outs[0][3, 1, 16:31] == 0).all())
    assert bool(torch.isnan(outs[1][4, 1, 0]))
    for got, old, bad in ((outs[0], want[0], [(1, 2), (2, 0), (3, 1)]), (outs[1], want[1], [(4, 1)])):
        same = torch.ones(got.shape[:2], dtype=torch.bool, device="cuda")
        for t, h in bad:
            same[t, h] = False
        assert torch.equal(got[same], old[same])
    # Without a norm what is not rotated is what came in, whatever stands beside it.
    outs = hip.norm_rotate(q, k, at, freqs)
    for x, y in zip(outs, (q, k)):
        assert torch.equal(torch.nan_to_num(x[..., 16:], nan=7.0),
                           torch.nan_to_num(y[..., 16:], nan=7.0))
    grads = hip.norm_rotate_backward(gq, gk, q, k, at, freqs, wq, wk)
    assert bool(torch.isnan(grads[0][2, 0]).all()) and bool(torch.isfinite(grads[0][0]).all())


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(hip, interleaved):
    """Central differences of the formula in 64 bits, steps of 1e-6: their own error is below
    1e-8 (h^2 times a third derivative of some 10^2, and 1e-16 / h)."""
    import torch
    print_case("norm_rotate differences", interleaved)
    what, grads = make(3, 2, 1, 10, 8, seed=6)
    got = hip.norm_rotate_backward(*grads, *what, interleaved=interleaved)
    q, k, at, freqs, wq, wk = [t.cpu().double() for t in what]
    angle = at[:, None] * freqs[None, :]

    def loss(x, w, g):
        return float((formula(x, w, angle, 8, interleaved, 1e-6)[0]["out"] * g.cpu().double()).sum())

    for x, w, g, dx, dw in ((q, wq, grads[0], got[0], got[2]), (k, wk, grads[1], got[1], got[3])):
        for place, target in ((x, dx), (w, dw)):
            flat, d = place.view(-1), target.cpu().double().reshape(-1)
            for i in range(0, flat.numel(), 3):
                keep = float(flat[i])
                flat[i] = keep + 1e-6
                up = loss(x, w, g)
                flat[i] = keep - 1e-6
                down = loss(x, w, g)
                flat[i] = keep
                assert abs((up - down) / 2e-6 - float(d[i])) < 2e-5 * max(1.0, abs(float(d[i])))


@gpu
def test_in_place_and_strides(hip):
    """Written over q and k, into columns of wider rows, and the gradients over theirs."""
    import torch
    print_case("norm_rotate in place")
    what, grads, outs, got = check(hip, 21, 4, 2, 48, 32, fused=True, seed=7)
    q, k, at, freqs, wq, wk = what
    into = torch.full((21, 9, 48), 5.0, device="cuda")
    hip.norm_rotate(*what, out=(into[:, 1:5], into[:, 6:8]))
    assert torch.equal(into[:, 1:5], outs[0]) and torch.equal(into[:, 6:8], outs[1])
    assert bool((into[:, [0, 5, 8]] == 5.0).all())
    rows = torch.cat([q, k, torch.full((21, 2, 48), 3.0, device="cuda")], 1)
    q2, k2 = rows[:, :4], rows[:, 4:6]
    assert hip.norm_rotate(q2, k2, at, freqs, wq, wk, out=(q2, k2))[0] is q2
    assert torch.equal(q2, outs[0]) and torch.equal(k2, outs[1])
    assert bool((rows[:, 6:] == 3.0).all())
    gq, gk = grads[0].clone(), grads[1].clone()
    hip.norm_rotate_backward(gq, gk, *what, grads=(gq, gk))
    assert torch.equal(gq, got[0]) and torch.equal(gk, got[1])
    qx, kx = q.clone(), k.clone()
    hip.norm_rotate_backward(*grads, qx, kx, at, freqs, wq, wk, grads=(qx, kx))
    assert torch.equal(qx, got[0]) and torch.equal(kx, got[1])


@gpu
def test_parts_that_are_not_asked_for(hip):
    import torch
    print_case("norm_rotate parts")
    what, grads, outs, got = check(hip, 12, 4, 2, 32, 32, seed=8)
    q, k, at, freqs, wq, wk = what
    alone, none = hip.norm_rotate(q, None, at, freqs, wq)
    assert none is None and torch.equal(alone, outs[0])
    part = hip.norm_rotate_backward(grads[0], None, q, None, at, freqs, wq)
    assert torch.equal(part[0], got[0])
    assert part[1] is None and part[3] is None
    # How tokens are spread over waves goes by the heads of both, so a weight's gradient may be added
    # up in another order: n numbers in any order are off by (n - 1) U of the sum of their sizes,
    # which the formula's bound counts as (n + 8) U.
    angle = at.cpu().double()[:, None] * freqs.cpu()[None, :]
    value, bound = formula(q.cpu().double(), wq.cpu().double(), angle, 32, False, 1e-6,
                           grads[0].cpu().double())
    within(part[2], value["dw"], bound["dw"], "dq_weight")
    for skip in range(4):
        want = [i != skip for i in range(4)]
        part = hip.norm_rotate_backward(*grads, *what, want=want)
        assert part[skip] is None
        assert all(torch.equal(part[i], got[i]) for i in range(4) if i != skip)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 63, 65, 1000])
@pytest.mark.parametrize("h,kv,d", [(1, 0, 8), (1, 1, 24), (2, 1, 64), (1, 2, 32), (3, 2, 16),
                                    (1, 1, 128), (5, 3, 20), (1, 0, 256)])
def test_tokens_that_share_a_wave(hip, h, kv, d, tokens, interleaved):
    if kv > 0:
        check(hip, tokens, h, kv, d, d // 2 * 2, interleaved, seed=tokens)
        return
    what, grads = make(tokens, h, 1, d, d // 2 * 2, seed=tokens)
    q, _, at, freqs, wq, _ = what
    out, _ = hip.norm_rotate(q, None, at, freqs, wq, interleaved=interleaved)
    got = hip.norm_rotate_backward(grads[0], None, q, None, at, freqs, wq, interleaved=interleaved)
    angle = at.cpu().double()[:, None] * freqs.cpu()[None, :]
    value, bound = formula(q.cpu().double(), wq.cpu().double(), angle, d // 2 * 2, interleaved,
                           1e-6, grads[0].cpu().double())
    within(out, value["out"], bound["out"], "out")
    within(got[0], value["dx"], bound["dx"], "dx")
    within(got[2], value["dw"], bound["dw"], "dw")


@gpu
def test_no_tokens(hip):
    import torch
    print_case("norm_rotate no tokens")
    what, grads = make(0, 4, 2, 32, 32, seed=9)
    outs = hip.norm_rotate(*what)
    got = hip.norm_rotate_backward(*grads, *what)
    assert outs[0].shape == (0, 4, 32) and got[1].shape == (0, 2, 32)
    assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())


@gpu
def test_rows_past_two_to_the_31(hip):
    """Offsets past 32 bits: the last rows of a matrix with wide rows."""
    import torch
    print_case("norm_rotate far rows")
    ld, tokens = 1 << 22, 520
    rows = torch.empty(tokens * ld, device="cuda").view(tokens, ld // 32, 32)
    gen = torch.Generator(device="cuda").manual_seed(10)
    q, k = rows[:, :2], rows[:, 2:3]
    q.copy_(torch.randn(tokens, 2, 32, generator=gen, device="cuda"))
    k.copy_(torch.randn(tokens, 1, 32, generator=gen, device="cuda"))
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    freqs = hip.rotary_frequencies(32)
    w = torch.ones(32, device="cuda")
    want = hip.norm_rotate(q.contiguous(), k.contiguous(), at, freqs, w, w)
    got = hip.norm_rotate(q, k, at, freqs, w, w, out=(q, k))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_same_bits_each_time_on_other_streams_and_in_a_graph(hip):
    import torch
    what, grads, outs, got = check(hip, 300, 8, 2, 64, 64, seed=11)
    torch.cuda.synchronize()
    both = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            both.append((hip.norm_rotate(*what), hip.norm_rotate_backward(*grads, *what)))
    torch.cuda.synchronize()
    for o, g in both:
        assert all(torch.equal(a, b) for a, b in zip((*o, *g), (*outs, *got)))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = (*hip.norm_rotate(*what), *hip.norm_rotate_backward(*grads, *what))
        graphs.append((graph, res))
    for step in range(3):
        what[0].copy_(torch.randn(300, 8, 64, device="cuda"))
        what[2].add_(step)
        want = (*hip.norm_rotate(*what), *hip.norm_rotate_backward(*grads, *what))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def descriptor(**changes):
    """Pointers that are never followed: every call is refused."""
    d = dict(q=64, k=64, ld_q=128, ld_k=64, tokens=4, heads=4, kv_heads=2, head_dim=32, rotary=32,
             positions=64, freqs=64, q_weight=64, k_weight=64, eps=1e-6, interleaved=0)
    d.update(changes)
    return E.NormRotate(*[d[n] for n, _ in E.NormRotate._fields_])


REFUSED = [dict(tokens=-1), dict(heads=-1), dict(kv_heads=-1), dict(heads=0, kv_heads=0),
           dict(head_dim=0), dict(head_dim=257, rotary=0, ld_q=2000, ld_k=2000), dict(rotary=3),
           dict(rotary=34), dict(rotary=-2), dict(eps=-1.0), dict(eps=math.nan), dict(ld_q=127),
           dict(ld_k=63), dict(tokens=2 ** 31), dict(heads=2 ** 24, ld_q=2 ** 30)]


@pytest.mark.parametrize("changes", REFUSED)
def test_refused_descriptors(changes):
    """The query answers without a device."""
    lib = E.load_library()
    assert lib.ehip_norm_rotate_backward_workspace(C.byref(descriptor(**changes))) == -1
    assert b"norm_rotate_backward" in lib.ehip_last_error()
    assert lib.ehip_norm_rotate_backward_workspace(None) == -1


def test_workspace_query():
    lib = E.load_library()
    ask = lambda **c: lib.ehip_norm_rotate_backward_workspace(C.byref(descriptor(**c)))
    assert ask() > 0 and ask(tokens=0) == 0 and ask(q_weight=None, k_weight=None) == 0
    assert ask(tokens=2 ** 31 - 1) <= 1024 * 2 * 256 * 4


@gpu
def test_refused_calls(hip):
    import torch
    print_case("norm_rotate refused")
    lib = hip.lib
    for changes in REFUSED + [dict(q=None), dict(k=None), dict(positions=None), dict(freqs=None)]:
        d = descriptor(**changes)
        assert lib.ehip_norm_rotate_f32(C.byref(d), 64, 2 ** 31, 64, 2 ** 31, None) == 1, changes
        assert lib.ehip_norm_rotate_backward_f32(C.byref(d), 64, 2 ** 31, 64, 2 ** 31, 64, 2 ** 31,
                                                 64, 2 ** 31, None, None, None, 0, None) == 1, changes
    d = descriptor()
    forward = lambda *a: lib.ehip_norm_rotate_f32(C.byref(d), *a, None)
    assert forward(None, 128, 64, 64) == 1 and forward(64, 128, None, 64) == 1
    assert forward(64, 127, 64, 64) == 1 and forward(64, 128, 64, 63) == 1
    back = lambda gq=64, lgq=128, gk=64, lgk=64, ldq=128, ldk=64, w=64, n=1 << 20: (
        lib.ehip_norm_rotate_backward_f32(C.byref(d), gq, lgq, gk, lgk, 64, ldq, 64, ldk, 64, 64, w,
                                          n, None))
    assert back(gq=None) == 1 and back(gk=None) == 1 and back(lgq=127) == 1 and back(lgk=63) == 1
    assert back(ldq=127) == 1 and back(ldk=63) == 1
    assert back(w=None) == 1 and back(w=72) == 1 and back(n=16) == 1
    d = descriptor(q_weight=None)
    assert back() == 1
    what, grads = make(4, 4, 2, 32, 32)
    q, k, at, freqs, wq, wk = what
    for bad in ((q[0], k), (q, k[:3]), (q, k[..., :16]), (q.double(), k), (q.transpose(0, 1), k)):
        with pytest.raises(ValueError):
            hip.norm_rotate(*bad, at, freqs, wq, wk)
    for bad in ((at.long(), freqs), (at[:3], freqs), (at, freqs.float()), (None, freqs),
                (at, freqs[::2])):
        with pytest.raises(ValueError):
            hip.norm_rotate(q, k, *bad, wq, wk)
    with pytest.raises(ValueError):
        hip.norm_rotate(q, k, at, freqs, wq[:16], wk)
    with pytest.raises(ValueError):
        hip.norm_rotate(q, None, at, freqs, wq, wk)
    with pytest.raises(ValueError):
        hip.norm_rotate(q, k.cpu(), at, freqs, wq, wk)
    with pytest.raises(RuntimeError):
        hip.norm_rotate(q, k, at, hip.rotary_frequencies(34), wq, wk)
