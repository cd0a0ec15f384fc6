"""Log probabilities of given tokens with entropy, top alternatives and gradients, against 64 bits.

u = 2^-24. A row of n logits: the sum of n exponentials, each within 4 u of its value (the device exp
is within 2 ulp, its argument x - m is rounded once, |x - m| exp(x - m) <= 0.37 of one) is off by
(n + 8) u of itself whatever the order, so log of it by that; lse rounds at |lse| u and |m| u on top.
  lse:     e = (n + 10) u + 2 u |lse|
  logprob: e + u |x_t - lse|
  entropy: each term p (lse - x) relative (n + 16) u, plus u |x - m| p: (n + 20) u (1 + |H| + sum p |x - m|)
  dx:      p off by (|x| + |lse|) u + e + 4 u, times (|g| + |g_H| (|x - lse| + |H|)), plus p |g_H| times
           what x - lse and H are off by, plus four roundings
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


def exact(x, t, g=None, ge=None):
    """64-bit results and bounds of finite rows (-inf allowed beside finite logits)."""
    import torch
    x, t = x.detach().cpu().double(), t.cpu().long()
    n = x.shape[1]
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    p = logp.exp()
    zero = torch.zeros_like(p)
    h = -torch.where(p > 0, p * logp, zero).sum(1)
    m = x.amax(1)
    e = (n + 10) * U + 2 * U * lse.abs()
    one = torch.arange(x.shape[0])
    lp = logp[one, t]
    value = {"lse": lse, "logprob": lp, "entropy": h}
    spread = torch.where(p > 0, p * (m[:, None] - x), zero).sum(1)
    eh = (n + 20) * U * (1 + h.abs() + spread)
    bound = {"lse": e, "logprob": e + U * torch.nan_to_num(lp.abs(), posinf=0.0),
             "entropy": eh}
    if g is not None:
        g, ge = g.cpu().double()[:, None], ge.cpu().double()[:, None]
        z = torch.where(p > 0, logp, zero)
        dx = -p * (g + ge * (z + h[:, None]))
        dx[one, t] += g[:, 0]
        xa = torch.where(p > 0, x.abs(), zero)
        rel = U * (xa + lse.abs()[:, None] + z.abs()) + e[:, None] + 8 * U
        value["dx"] = dx
        bound["dx"] = (p * (rel * (g.abs() + ge.abs() * (z.abs() + h.abs()[:, None]))
                            + ge.abs() * (eh[:, None] + e[:, None]
                                          + 3 * U * (xa + lse.abs()[:, None] + h.abs()[:, None])))
                       + 4 * U * dx.abs() + 2 * U * p * g.abs() + 1e-37)
    return value, {k: 1.01 * b for k, b in bound.items()}


def near(got, value, bound, what):
    import torch
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(value)), what
    fine = torch.isfinite(value)
    rest = ~fine & ~torch.isnan(value)
    assert torch.equal(got[rest], value[rest]), what
    off = ((got - value).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over"


def best(x, top):
    """Indices of the largest logits, equal ones by index, NaN first, -0 as 0."""
    import torch
    y = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x).cpu().double()
    y = y + torch.isnan(x).cpu() * 1.0
    key = torch.where(torch.isnan(x).cpu(), torch.ones_like(y), torch.zeros_like(y))
    out = []
    for row, nan in zip(y.tolist(), key.tolist()):
        order = sorted(range(len(row)), key=lambda j: (-nan[j], -row[j], j))
        out.append(order[:top])
    return torch.tensor(out, dtype=torch.int32).reshape(x.shape[0], top)


def check(hip, x, t, top=0, g=None, ge=None):
    import torch
    print_case("logprobs", tuple(x.shape), top, x.stride(0))
    logprob, entropy, lse, best_lp, index = hip.token_logprobs(x, t, top=top)
    value, bound = exact(x, t, g, ge)
    for name, got in (("logprob", logprob), ("entropy", entropy), ("lse", lse)):
        near(got, value[name], bound[name], name)
    if top:
        want = best(x, top)
        assert torch.equal(index.cpu(), want)
        lp = x.cpu().double().gather(1, want.long()) - value["lse"][:, None]
        near(best_lp, lp, bound["lse"][:, None] + 1.01 * U * torch.nan_to_num(lp.abs(), posinf=0.),
             "top")
    if g is not None:
        near(hip.token_logprobs_backward(x, t, lse, entropy, g, ge), value["dx"], bound["dx"],
             "dlogits")


def make(rows, vocab, seed=0, spread=2.0, pad=0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab + pad, generator=gen, device="cuda")[:, :vocab] * spread
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))[:, :vocab]
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").to(torch.int32)
    g = torch.randn(rows, generator=gen, device="cuda")
    return x, t, g, torch.randn(rows, generator=gen, device="cuda")


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 121, 255, 256, 257, 1000, 1023, 1024, 1025,
                                   4096, 8191, 10007, 32000, 50257, 70001])
def test_vocabularies(hip, vocab):
    x, t, g, ge = make(5, vocab, seed=vocab)
    check(hip, x, t, min(vocab, 20), g, ge)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 7, 64, 300, 1500])
def test_rows(hip, rows):
    x, t, g, ge = make(rows, 1231, seed=rows)
    check(hip, x, t, 3, g, ge)


@gpu
@pytest.mark.parametrize("pad", [1, 3, 4, 13])
@pytest.mark.parametrize("vocab", [97, 5000, 40001])
def test_strides_and_alignment(hip, vocab, pad):
    x, t, g, ge = make(4, vocab, seed=pad, pad=pad)
    assert x.stride(0) == vocab + pad
    check(hip, x, t, 9, g, ge)


@gpu
@pytest.mark.parametrize("vocab", [200, 3000, 32000, 130001])
@pytest.mark.parametrize("top", [1, 2, 20, 64, 100, 128])
def test_tops(hip, vocab, top):
    x, t, _, _ = make(3, vocab, seed=top)
    check(hip, x, t, top)


@gpu
@pytest.mark.parametrize("vocab", [128, 1500, 32000, 100003])
def test_ties_go_to_the_lowest_index(hip, vocab):
    """Whole-number logits, one value only, the top at the row's end, ascending and descending
    rows, zeros of both signs."""
    import torch
    x, t, _, _ = make(7, vocab, seed=1)
    x[0].round_()
    x[1] = 0.5
    x[2].copy_(torch.arange(vocab, device="cuda") / 64)
    x[3].copy_(torch.arange(vocab, device="cuda").flip(0) / 64)
    x[4].clamp_(max=0).mul_(0.0)  # 0 and -0
    x[5] = -1.0
    x[5, -40:] = 3.0
    x[6] = (torch.arange(vocab, device="cuda") % 7).float()
    for top in (5, 128):
        check(hip, x, t, top)


@gpu
@pytest.mark.parametrize("top", [3, 50])
def test_tops_of_rows_in_one_block(hip, top):
    """Segments that come after the list is full: better ones at the end, none, a NaN or +inf in the
    second or the last, thousands of equal ones, little but -inf."""
    import torch
    print_case("logprobs one block", top)
    x, t, _, _ = make(520, 20001, seed=top)
    x[0].copy_(torch.arange(20001, device="cuda") / 64)
    x[1].copy_(torch.arange(20001, device="cuda").flip(0) / 64)
    x[2, 9000], x[2, 20000] = math.nan, 50.0
    x[3, 20000], x[3, 8191] = math.nan, math.inf
    x[4, 8192:] = 4.0
    x[5] = -math.inf
    x[5, 17000:17002] = 1.0
    x[6] = -math.inf
    x[6, ::977] = torch.randn(21, device="cuda")
    x[7, :8192] = -3.0e38
    index = hip.token_logprobs(x, t, top=top)[4]
    assert torch.equal(index[:12].cpu(), best(x[:12], top))
    assert torch.equal(index[500:520].cpu(), best(x[500:], top))


@gpu
@pytest.mark.parametrize("vocab", [130, 2000, 33001])
def test_masked_and_extreme_logits(hip, vocab):
    """-inf beside others, the lowest float as a mask, one token left, logits of 1e4 and 1e30."""
    import torch
    x, t, g, ge = make(6, vocab, seed=2)
    x[0, ::2] = -math.inf
    x[1, 1:] = -math.inf
    t[1] = 0
    x[2, 5:] = torch.finfo(torch.float32).min
    x[3] *= 1e4
    x[4, vocab - 1] = 90.0
    x[5] -= 300.0
    check(hip, x, t, 20, g, ge)
    x[3] = x[3].sign() * 1e30
    logprob, entropy, lse, top, index = hip.token_logprobs(x, t, top=2)
    assert float(lse[3]) == pytest.approx(1e30, rel=1e-6)
    assert bool(torch.isfinite(entropy).all())


@gpu
@pytest.mark.parametrize("vocab", [130, 33001, 90000])
def test_rows_without_a_distribution(hip, vocab):
    """All -inf; +inf; NaN; and targets outside the vocabulary, each without touching the rows
    beside it."""
    import torch
    print_case("logprobs none", vocab)
    x, t, g, ge = make(7, vocab, seed=3)
    want = hip.token_logprobs(x, t, top=4)
    dx0 = hip.token_logprobs_backward(x, t, want[2], want[1], g, ge)
    y = x.clone()
    y[1] = -math.inf
    y[2, vocab // 2] = math.inf
    y[3, 7] = math.nan
    t[4], t[5] = -1, vocab
    logprob, entropy, lse, top, index = hip.token_logprobs(y, t, top=4)
    dx = hip.token_logprobs_backward(y, t, lse, entropy, g, ge)
    assert float(lse[1]) == -math.inf and float(entropy[1]) == 0 and float(logprob[1]) == -math.inf
    assert bool((top[1] == -math.inf).all()) and index[1].tolist() == [0, 1, 2, 3]
    assert bool((dx[1] == 0).all())
    for r in (2, 3):
        assert all(bool(torch.isnan(z[r]).all()) for z in (logprob, entropy, lse, top, dx))
        assert torch.equal(index[r].cpu(), best(y[r:r + 1], 4)[0])
    for r in (4, 5):
        assert bool(torch.isnan(logprob[r])) and bool(torch.isnan(dx[r]).all())
        for a, b in zip((entropy, lse, top, index), want[1:]):
            assert torch.equal(a[r], b[r])
    for r in (0, 6):
        for a, b in zip((logprob, entropy, lse, top, index, dx), (*want, dx0)):
            assert torch.equal(a[r], b[r])


@gpu
def test_parts_that_are_not_asked_for(hip):
    import torch
    print_case("logprobs parts")
    x, t, g, ge = make(9, 5000, seed=4)
    full = hip.token_logprobs(x, t, top=3)
    a = hip.token_logprobs(x, top=3, want_entropy=False)
    assert a[0] is None and a[1] is None
    assert all(torch.equal(p, q) for p, q in zip(a[2:], full[2:]))
    b = hip.token_logprobs(x, t)
    assert b[3] is None and b[4] is None
    assert all(torch.equal(p, q) for p, q in zip(b[:3], full[:3]))
    plain = hip.token_logprobs_backward(x, t, full[2], None, g)
    zero = hip.token_logprobs_backward(x, t, full[2], full[1], g, torch.zeros_like(g))
    assert torch.equal(plain, zero)


@gpu
def test_as_the_cross_entropy(hip):
    """The mean loss of the framework's cross-entropy, and its gradient for one row each."""
    import torch
    print_case("logprobs against cross entropy")
    x, t, _, _ = make(64, 1000, seed=5)
    loss, probs = hip.cross_entropy(x, t)
    logprob, entropy, lse, _, _ = hip.token_logprobs(x, t)
    value, bound = exact(x, t)
    # A mean of 64, each within its bound, and the other's own of the same size.
    assert abs(float(loss) + float(logprob.double().mean())) <= 2 * float(bound["logprob"].max())
    g = torch.full((64,), -1.0 / 64, device="cuda")
    dx = hip.token_logprobs_backward(x, t, lse, None, g)
    theirs = hip.cross_entropy_backward(probs, t, torch.ones(1, device="cuda"))
    _, b = exact(x, t, g, torch.zeros_like(g))
    near(dx, theirs.cpu().double(), 2 * b["dx"], "dx")


@gpu
def test_gradient_in_place_and_in_wider_rows(hip):
    import torch
    print_case("logprobs in place")
    x, t, g, ge = make(6, 3001, seed=6, pad=7)
    _, entropy, lse, _, _ = hip.token_logprobs(x, t)
    want = hip.token_logprobs_backward(x, t, lse, entropy, g, ge)
    wide = torch.full((6, 3010), 5.0, device="cuda")
    hip.token_logprobs_backward(x, t, lse, entropy, g, ge, dlogits=wide[:, 4:3005])
    assert torch.equal(wide[:, 4:3005], want)
    assert bool((wide[:, :4] == 5.0).all()) and bool((wide[:, 3005:] == 5.0).all())
    hip.token_logprobs_backward(x, t, lse, entropy, g, ge, dlogits=x)
    assert torch.equal(x, want)


@gpu
def test_gradients_against_differences(hip):
    """The slope of sum(g logprob + ge entropy) along a direction, by central differences in 64
    bits."""
    import torch
    print_case("logprobs differences")
    x, t, g, ge = make(5, 300, seed=7)
    _, entropy, lse, _, _ = hip.token_logprobs(x, t)
    dx = hip.token_logprobs_backward(x, t, lse, entropy, g, ge).cpu().double()
    step = torch.randn(x.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    f = []
    for e in (1e-4, -1e-4):
        v, _ = exact(x.cpu().double() + e * step, t)
        f.append(float((g.cpu() * v["logprob"] + ge.cpu() * v["entropy"]).sum()))
    slope = (f[0] - f[1]) / 2e-4
    assert abs(float((dx * step).sum()) - slope) <= 1e-4 * float(dx.norm() * step.norm())


@gpu
@pytest.mark.parametrize("rows,vocab", [(3, 100000), (200, 1000)])
def test_same_bits_on_other_streams_and_in_a_graph(hip, rows, vocab):
    import torch
    print_case("logprobs repeat", rows, vocab)
    x, t, g, ge = make(rows, vocab, seed=8)

    def both():
        r = hip.token_logprobs(x, t, top=5)
        return [*r, hip.token_logprobs_backward(x, t, r[2], r[1], g, ge)]

    want = both()
    torch.cuda.synchronize()
    got = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for one in got for a, b in zip(one, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        graphs.append((graph, outs))
    for seed in range(3):
        x.copy_(make(rows, vocab, seed=30 + seed)[0])
        want = both()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
@pytest.mark.parametrize("vocab,top", [(32771, 0), (32771, 9), (40960, 5)])
def test_more_logits_than_the_caches_hold(hip, vocab, top):
    """2^26 logits and more are read past the caches: the bits of the same rows in two calls, which
    are not, and some rows against 64 bits."""
    import torch
    rows = -(-2 ** 26 // vocab)
    rows += rows % 2
    x, t, _, _ = make(rows, vocab, seed=vocab + top)
    got = hip.token_logprobs(x, t, top=top)
    half = rows // 2
    assert half >= 512  # whole rows a block, as in one call
    parts = [hip.token_logprobs(x[at:at + half], t[at:at + half], top=top) for at in (0, half)]
    for a, b, c in zip(got, *parts):
        assert (a is None) == (b is None)
        assert a is None or torch.equal(a, torch.cat([b, c]))
    some = torch.arange(0, rows, rows // 6, device="cuda")
    value, bound = exact(x[some], t[some])
    for name, y in zip(("logprob", "entropy", "lse"), got):
        near(y[some], value[name], bound[name], name)
    if top:
        assert torch.equal(got[4][some].cpu(), best(x[some], top))


def test_refused_sizes():
    """The checks that every call starts with, through the query that needs no device."""
    lib = E.load_library()
    size = lib.ehip_token_logprobs_workspace
    assert size(4, 1000, 10) >= 0 and size(0, 1, 1) >= 0
    for bad in ((-1, 10, 0), (4, 0, 0), (4, 10, -1), (4, 10, 11), (4, 1000, 129), (4, 2 ** 31, 0),
                (2 ** 24, 10, 0)):
        assert size(*bad) == -1, bad
        assert b"token_logprobs" in lib.ehip_last_error()


@gpu
def test_calls_are_refused(hip):
    import torch
    print_case("logprobs refusals")
    x, t, g, ge = make(4, 100)
    _, entropy, lse, _, _ = hip.token_logprobs(x, t)
    launched = hip.launched()
    for args in ((x, t.long()), (x, t[:3]), (x.half(), t), (x[0], t), (x.T, t), (x, t.cpu()),
                 (x[:, ::2], t)):
        with pytest.raises(ValueError):
            hip.token_logprobs(*args)
    for top in (101, -1):
        with pytest.raises(RuntimeError):
            hip.token_logprobs(x, t, top=top)
    for args in ((x, t, lse[:3], entropy, g), (x, t, lse, entropy, g[:3]),
                 (x, t, lse, entropy[:3], g, ge), (x, t, lse, entropy, g, ge[:2]),
                 (x, t, lse.double(), entropy, g)):
        with pytest.raises(ValueError):
            hip.token_logprobs_backward(*args)
    with pytest.raises(RuntimeError):
        hip.token_logprobs_backward(x, t, lse, None, g, ge)
    assert hip.launched() == launched
    empty = hip.token_logprobs(x[:0], t[:0], top=2)
    assert empty[0].shape == (0,) and empty[3].shape == (0, 2)
