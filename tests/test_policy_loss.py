"""The clipped policy loss and its gradients against the formula in 64 bits.

u = 2^-24. d = p - o is exact in 64 bits and rounded once; the device exp is within 2 ulp, so a ratio
is within er = (5 + |d|) u of itself. x = f - p likewise; exp(x) - x - 1 is a series of positive
weight below |x| = 1, within 12 u of itself, and past it the difference of numbers within
(5 + |x|) u of exp(x): ek = 12 u kl, or (6 + |x|) u (exp(x) + |x| + 1). exp(x) - 1 the same.
  term:   e = ratio |A| (er + 2 u) + beta ek + 4 u (ratio |A| + beta kl + c |H|)
  loss:   sum of w e, and one rounding; the sums and weights are in 64 bits
  slope:  ratio |A| (er + 2 u) + beta er' + 4 u of the magnitudes; times w: three roundings and w's two
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


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def formula(lp, old, adv, cu, clip_low=0.2, clip_high=0.2, ref=None, kl_weight=0.0, entropy=None,
            entropy_weight=0.0, mask=None, by_sequence=False, mean_by_sequence=None, grad=1.0):
    """(values, bounds), 64 bits, on the CPU."""
    import torch
    lp, old, adv = (t.cpu().double() for t in (lp, old, adv))
    n = lp.numel()
    offsets = cu.tolist()
    which = torch.full((n,), -1)
    for s in range(len(offsets) - 1):
        which[offsets[s]:offsets[s + 1]] = s
    counts = which >= 0
    if mask is not None:
        counts = counts & (mask.cpu() != 0)
    if by_sequence and len(offsets) == 1:
        adv = torch.zeros(1, dtype=torch.float64)  # of no sequence: not used
    a = adv[which.clamp_min(0)] if by_sequence else adv
    if by_sequence if mean_by_sequence is None else mean_by_sequence:
        size = torch.zeros(max(1, len(offsets) - 1), dtype=torch.float64).index_add_(
            0, which[counts], torch.ones(int(counts.sum()), dtype=torch.float64))
        w = 1 / (size[which.clamp_min(0)] * max(1, int((size > 0).sum())))
    else:
        w = torch.full((n,), 1.0 / max(1, int(counts.sum())), dtype=torch.float64)
    w = torch.where(counts, w, torch.zeros_like(w))
    zero = torch.zeros_like(lp)
    keep = lambda t: torch.where(counts, t, zero)
    d = keep(lp - old)
    ratio = d.exp()
    a = keep(a)
    clipped = torch.where(a < 0, ratio < 1 - clip_low, ratio > 1 + clip_high) & counts
    limit = torch.where(a < 0, torch.full_like(a, 1 - clip_low), torch.full_like(a, 1 + clip_high))
    used = torch.where(clipped, limit, ratio)
    term, slope = -used * a, torch.where(clipped, zero, -ratio * a)
    er = (5 + d.abs()) * U
    e = used * a.abs() * (er + 6 * U)
    es = slope.abs() * (er + 6 * U)
    kl = zero
    ek = zero
    if ref is not None:
        x = keep(ref.cpu().double() - lp)
        rise = torch.expm1(x)
        kl = torch.where(x.abs() < 0.01, x * x / 2 * (1 + x / 3 * (1 + x / 4 * (1 + x / 5))), rise - x)
        ek = torch.where(x.abs() < 1, 12 * U * kl, (6 + x.abs()) * U * (x.exp() + x.abs() + 1))
        er2 = torch.where(x.abs() < 1, 12 * U * rise.abs(), (6 + x.abs()) * U * (x.exp() + 1))
        term, slope = term + kl_weight * kl, slope - kl_weight * rise
        e = e + abs(kl_weight) * (ek + 4 * U * kl)
        es = es + abs(kl_weight) * (er2 + 4 * U * rise.abs())
    if entropy is not None:
        h = keep(entropy.cpu().double())
        term = term - entropy_weight * h
        e = e + 4 * U * abs(entropy_weight) * h.abs()
    total = max(1.0, float(counts.sum()))
    value = {"loss": (w * term).sum().reshape(1),
             "stats": torch.stack([keep(kl).sum(), clipped.double().sum(), keep(ratio).sum()]) / total,
             "g_logprob": grad * w * slope}
    bound = {"loss": (w * e).sum().reshape(1), "stats": torch.stack(
        [keep(ek).sum(), zero.sum(), keep(ratio * er).sum()]) / total,
        "g_logprob": abs(grad) * w * es + 6 * U * value["g_logprob"].abs()}
    if entropy is not None:
        value["g_entropy"] = -grad * w * entropy_weight
        bound["g_entropy"] = 6 * U * value["g_entropy"].abs()
    return value, {k: 1.01 * (bound[k] + U * value[k].abs()) + 1e-37 for k in value}


def within(got, value, bound, what):
    import torch
    got = got.detach().cpu().double()
    assert got.shape == value.shape, what
    assert bool(torch.isfinite(got).all()), what
    off = (got - value).abs() - bound
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over"


def make(lengths, by_sequence=False, ref=True, entropy=True, masked=0.3, seed=0, spread=0.3,
         behind=0, before=0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = before + sum(lengths) + behind
    normal = lambda m: torch.randn(m, generator=gen, device="cuda")
    cu = [before]
    for x in lengths:
        cu.append(cu[-1] + x)
    lp = -normal(n).abs() * 2
    return (lp, lp + spread * normal(n), normal(len(lengths) if by_sequence else n), ints(cu)), dict(
        ref=lp + spread * normal(n) if ref else None, kl_weight=0.1 if ref else 0.0,
        entropy=normal(n).abs() if entropy else None, entropy_weight=0.02 if entropy else 0.0,
        mask=(torch.rand(n, generator=gen, device="cuda") >= masked) if masked else None,
        by_sequence=by_sequence)


def check(hip, what, how, grad=0.75):
    import torch
    print_case("policy", what[3].numel() - 1, what[0].numel(), how["by_sequence"])
    g = torch.full((1,), grad, device="cuda")
    loss, stats, weights = hip.policy_loss(*what, **how)
    g_logprob, g_entropy = hip.policy_loss_backward(g, *what, weights, **how)
    value, bound = formula(*what, **how, grad=grad)
    for name, got in (("loss", loss), ("stats", stats), ("g_logprob", g_logprob),
                      ("g_entropy", g_entropy)):
        if name in value:
            within(got, value[name], bound[name], name)
        else:
            assert got is None
    return loss, stats, weights, g_logprob, g_entropy


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("lengths", [[1], [2, 0, 3], [511], [512], [513], [1024, 1025], [63, 64, 65],
                                     [0, 0, 7, 0], [5000], [1] * 700, [100] * 70, [3000, 1, 1, 2500],
                                     [8192], [8193, 9000], [255, 256, 257], [9] * 256, [9] * 257])
def test_lengths(hip, lengths, by_sequence):
    for masked in (0.0, 0.4):
        check(hip, *make(lengths, by_sequence, masked=masked, seed=len(lengths)))


@gpu
@pytest.mark.parametrize("lengths", [[500], [30] * 40, [4000] * 3])
def test_a_loss_of_terms_that_cancel(hip, lengths):
    """Neighbours have the advantages a and -a and nearly the same ratio. A term is a product in 64
    bits with a series that is 2^-37 off: 2^-36 of it with what is rounded, and the result 2^-24."""
    import torch
    what, how = make(lengths, ref=False, entropy=False, masked=0.0, seed=21, spread=0.05)
    lp, old, a, cu = what
    a = a.view(-1, 2)[:, :1].repeat(1, 2) * torch.tensor([1.0, -1.0], device="cuda")
    a = a.reshape(-1)
    d = (lp - old).view(-1, 2)
    old = (lp.view(-1, 2) - d[:, :1] - torch.tensor([0.0, 1e-4], device="cuda")).reshape(-1)
    print_case("policy cancel", lengths)
    loss, _, _ = hip.policy_loss(lp, old, a.contiguous(), cu, 0.9, 9.0, **how)
    term = (-(lp.double() - old.double()).exp() * a.double()).cpu()
    want, size = float(term.mean()), float(term.abs().mean())
    assert abs(want) < 1e-3 * size
    assert abs(float(loss) - want) <= 2.0 ** -36 * size + 2.0 ** -24 * abs(want)


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 63, 64, 65])
def test_about_as_many_as_one_block_takes(hip, by_sequence, count):
    check(hip, *make([1 + i % 9 for i in range(count)], by_sequence, seed=count))
    check(hip, *make([520] * (count // 2), by_sequence, seed=count, entropy=False, before=3))


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
def test_many_sequences(hip, by_sequence):
    """More than one joining block has, of which one block has more than its threads again."""
    lengths = [(37 * i) % 23 for i in range(3000)]
    lengths[1500] = 20000
    check(hip, *make(lengths, by_sequence, seed=1))
    check(hip, *make([2] * 20000, by_sequence, seed=2, entropy=False))


@gpu
@pytest.mark.parametrize("ref", [False, True])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("by_sequence", [False, True])
def test_terms(hip, ref, entropy, by_sequence):
    check(hip, *make([40, 7, 600], by_sequence, ref=ref, entropy=entropy, seed=3))


@gpu
@pytest.mark.parametrize("advantages,means", [(False, True), (True, False)])
def test_advantages_and_means_apart(hip, advantages, means):
    what, how = make([40, 0, 7, 600], advantages, seed=4)
    check(hip, what, dict(how, mean_by_sequence=means))


@gpu
@pytest.mark.parametrize("spread", [1e-4, 1e-2, 1.0, 5.0])
@pytest.mark.parametrize("low,high", [(0.2, 0.2), (0.0, 0.0), (1.0, 3.0), (2.0, 1e30)])
def test_ratios_and_limits(hip, low, high, spread):
    what, how = make([300, 40], seed=5, spread=spread)
    check(hip, what, dict(how, clip_low=low, clip_high=high))


@gpu
def test_ratios_next_to_their_limits(hip):
    """Which side is exact: the neighbours in fp32 of a difference at the limit."""
    import torch
    print_case("policy limits")
    limits = [math.log1p(-0.2), math.log1p(0.28)]
    d = []
    for x in limits:
        near = torch.tensor([x], dtype=torch.float32)
        for step in (-math.inf, math.inf):
            at = near.clone()
            for _ in range(5):
                d.append(float(at))
                at = torch.nextafter(at, torch.tensor([step]))
    lp = torch.tensor(d * 2, dtype=torch.float32)
    n = lp.numel()
    adv = torch.cat([torch.ones(n // 2), -torch.ones(n // 2)]).cuda()
    what = (lp.cuda(), torch.zeros(n, device="cuda"), adv, ints([0, n]))
    how = dict(clip_low=0.2, clip_high=0.28, by_sequence=False)
    check(hip, what, how, grad=1.0)


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
def test_sequences_without_a_token_that_counts(hip, by_sequence):
    import torch
    what, how = make([40, 30, 0, 50], by_sequence, seed=6, masked=0.0)
    mask = torch.ones(120, dtype=torch.uint8, device="cuda")
    mask[40:70] = 0
    mask[80] = 255
    check(hip, what, dict(how, mask=mask))
    mask.zero_()
    out = check(hip, what, dict(how, mask=mask))
    assert all(bool((x == 0).all()) for x in out[:2]) and bool((out[3] == 0).all())


@gpu
def test_masked_tokens_are_not_looked_at(hip):
    import torch
    what, how = make([40, 700, 3], seed=7)
    want = check(hip, what, how)
    off = ~how["mask"]
    for t, bad in ((what[0], math.nan), (what[1], math.inf), (what[2], -math.inf),
                   (how["ref"], math.nan), (how["entropy"], math.inf)):
        t[off] = bad
    got = check(hip, what, how)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
def test_tokens_of_no_sequence(hip, by_sequence):
    """Before the first and behind the last: they do not count, and get gradients of 0."""
    import torch
    what, how = make([40, 700], by_sequence, seed=8, behind=1500, before=600, masked=0.0)
    what[0][:600], what[1][1340:] = math.nan, math.inf
    out = check(hip, what, how)
    assert bool((out[3][:600] == 0).all()) and bool((out[3][1340:] == 0).all())
    assert bool((out[4][1340:] == 0).all())


@gpu
def test_no_tokens_and_no_sequences(hip):
    import torch
    for lengths, behind in (([], 0), ([0, 0], 0), ([], 1000)):
        out = check(hip, *make(lengths, seed=9, behind=behind))
        assert float(out[0]) == 0 and bool((out[3] == 0).all())


@gpu
def test_what_is_not_finite(hip):
    """An advantage of 0 has no part in the loss however large the ratio; a token that cannot come
    any more has ratio 0; a NaN shows."""
    import torch
    print_case("policy not finite")
    lp = torch.tensor([-1.0, -math.inf, -2.0, 0.0], device="cuda")
    old = torch.tensor([-1.0, -1.0, -math.inf, -200.0], device="cuda")
    adv = torch.tensor([2.0, 3.0, 0.0, 1.0], device="cuda")
    cu = ints([0, 4])
    loss, stats, weights = hip.policy_loss(lp, old, adv, cu)
    assert abs(float(loss) + (2 + 0 + 0 + 1.2) / 4) < 1e-6 and float(stats[1]) == 0.5
    g, _ = hip.policy_loss_backward(torch.ones(1, device="cuda"), lp, old, adv, cu, weights)
    assert g.tolist() == [-0.5, 0.0, 0.0, 0.0]
    ref = torch.tensor([-1.0, -1.0, -math.inf, 0.0], device="cuda")
    loss, stats, _ = hip.policy_loss(lp, old, adv, cu, ref=ref, kl_weight=0.1)
    assert float(loss) == math.inf and float(stats[0]) == math.inf
    loss, stats, _ = hip.policy_loss(lp, old, adv, cu, ref=ref)
    assert abs(float(loss) + 0.8) < 1e-6 and float(stats[0]) == math.inf
    adv[0] = math.nan
    assert math.isnan(float(hip.policy_loss(lp, old, adv, cu)[0]))


@gpu
@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("lengths", [[400] * 8, [3000] * 40])
@pytest.mark.parametrize("far", [79.0, 81.0, 88.0, 90.0, 95.0])
def test_terms_past_fp32_with_weights_that_bring_them_back(hip, far, lengths, by_sequence):
    """exp(95) is 2^137; with a token's share of the mean it is in range again, in the loss, the means
    and the gradients. Of a policy's token that the sampler or the reference held for certain, and the
    other way round: ratios below fp32's normal numbers, times advantages of 10^30."""
    import torch
    print_case("policy far", far, len(lengths), by_sequence)
    what, how = make(lengths, seed=13, masked=0.2)
    how["mean_by_sequence"] = by_sequence
    lp, old, adv, cu = what
    n = lp.numel()
    for i in (5, n // 2, n - 7):
        old[i], adv[i] = lp[i] - far, -1e-3
    for i in (9, n // 3):
        how["ref"][i] = lp[i] + far
    for i in (17, n - 3):
        old[i], adv[i] = lp[i] + far, 1e30
    how["mask"][[5, 9, 17, n // 3, n // 2, n - 7, n - 3]] = True
    check(hip, what, how)
    how.update(ref=None, kl_weight=0.0)
    check(hip, what, how)


@gpu
def test_gradient_against_differences(hip):
    """Central differences of the formula in 64 bits, no token next to a limit."""
    import torch
    print_case("policy differences")
    what, how = make([5, 9, 4], True, seed=10)
    _, _, weights = hip.policy_loss(*what, **how)
    got, _ = hip.policy_loss_backward(torch.ones(1, device="cuda"), *what, weights, **how)
    lp = what[0].cpu().double()
    for i in range(18):
        up, down = lp.clone(), lp.clone()
        up[i] += 1e-6
        down[i] -= 1e-6
        a, b = (formula(x, *what[1:], **how)[0]["loss"] for x in (up, down))
        assert abs(float(a - b) / 2e-6 - float(got[i])) < 1e-7


@gpu
def test_with_the_token_scores(hip):
    """A training step's path: scores of the logits, the loss, its gradients, the logits' gradient,
    against 64 bits through torch's own graph, and against the sum of the operators' bounds: some
    300 u of the largest gradient (a row of 50 logits, scores within 64 u)."""
    import torch
    print_case("policy with scores")
    gen = torch.Generator(device="cuda").manual_seed(11)
    lengths, vocab = [7, 0, 12, 30], 50
    n = sum(lengths) + 3
    logits = torch.randn(n, vocab, generator=gen, device="cuda") * 2
    targets = torch.randint(0, vocab, (n,), generator=gen, device="cuda").to(torch.int32)
    cu = ints([0, 7, 7, 19, 49])
    lp, entropy, lse, _, _ = hip.token_logprobs(logits, targets)
    old = lp + 0.3 * torch.randn(n, generator=gen, device="cuda")
    ref = lp + 0.3 * torch.randn(n, generator=gen, device="cuda")
    adv = torch.randn(4, generator=gen, device="cuda")
    mask = torch.rand(n, generator=gen, device="cuda") < 0.8
    how = dict(ref=ref, kl_weight=0.1, entropy=entropy, entropy_weight=0.02, mask=mask,
               by_sequence=True)
    loss, _, weights = hip.policy_loss(lp, old, adv, cu, **how)
    g, ge = hip.policy_loss_backward(torch.ones(1, device="cuda"), lp, old, adv, cu, weights, **how)
    dlogits = hip.token_logprobs_backward(logits, targets, lse, entropy, g, ge)
    x = logits.cpu().double().requires_grad_()
    logp = torch.log_softmax(x, 1)
    p = logp.gather(1, targets.cpu().long()[:, None])[:, 0]
    h = -(logp.exp() * logp).sum(1)
    which = torch.repeat_interleave(torch.arange(4), torch.tensor(lengths + [])) if n else None
    m = mask.cpu()[:49]
    size = torch.zeros(4, dtype=torch.float64).index_add_(0, which[m], torch.ones(
        int(m.sum()), dtype=torch.float64))
    w = m / (size[which].clamp_min(1) * (size > 0).sum())
    a = adv.cpu().double()[which]
    ratio = (p[:49] - old.cpu().double()[:49]).exp()
    limited = torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    d = ref.cpu().double()[:49] - p[:49]
    want = (w * (-limited + float(torch.tensor(0.1)) * (d.exp() - d - 1)
                 - float(torch.tensor(0.02)) * h[:49])).sum()
    want.backward()
    assert abs(float(loss) - float(want)) < 300 * U * (1 + abs(float(want)))
    off = (dlogits.cpu().double() - x.grad).abs().max()
    assert float(off) < 300 * U * float(x.grad.abs().max())
    assert bool((dlogits[49:] == 0).all())


@gpu
def test_same_bits_each_time_on_other_streams_and_in_a_graph(hip):
    import torch
    what, how = make([700, 3, 0, 1500], True, seed=12)
    want = check(hip, what, how)
    g = torch.full((1,), 0.75, device="cuda")

    def step():
        loss, stats, weights = hip.policy_loss(*what, **how)
        return (loss, stats, weights, *hip.policy_loss_backward(g, *what, weights, **how))

    torch.cuda.synchronize()
    both = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            both.append(step())
    torch.cuda.synchronize()
    for got in both:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        what[0].add_(0.05 * torch.randn_like(what[0]))
        what[3].copy_(ints([0, 600 + i, 603, 700, 2203]))
        how["mask"].copy_(torch.rand(2203, device="cuda") < 0.5)
        eager = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def descriptor(**changes):
    d = dict(logprob=64, old_logprob=64, advantage=64, ref_logprob=64, entropy=64, mask=64, cu=64,
             sequences=3, tokens=10, advantage_by_sequence=0, mean_by_sequence=0, clip_low=0.2,
             clip_high=0.2, kl_weight=0.1, entropy_weight=0.1)
    d.update(changes)
    return E.Policy(*[d[n] for n, _ in E.Policy._fields_])


REFUSED = [dict(sequences=-1), dict(tokens=-1), dict(sequences=2 ** 24), dict(tokens=2 ** 31 - 1),
           dict(clip_low=-0.1), dict(clip_high=-0.1), dict(clip_low=math.nan),
           dict(clip_high=math.nan), dict(kl_weight=math.inf), dict(entropy_weight=math.nan),
           dict(ref_logprob=None), dict(entropy=None)]


@pytest.mark.parametrize("changes", REFUSED)
def test_refused_descriptors(changes):
    """The query answers without a device."""
    lib = E.load_library()
    assert lib.ehip_policy_loss_workspace(C.byref(descriptor(**changes))) == -1
    assert b"policy_loss" in lib.ehip_last_error()
    assert lib.ehip_policy_loss_workspace(None) == -1


def test_workspace_query():
    lib = E.load_library()
    ask = lambda **c: lib.ehip_policy_loss_workspace(C.byref(descriptor(**c)))
    assert ask() > 0 and ask(tokens=0, ref_logprob=None) > 0
    assert ask(kl_weight=0.0, ref_logprob=None, entropy_weight=0.0, entropy=None) == ask()


@gpu
def test_refused_calls(hip):
    import torch
    print_case("policy refused")
    lib = hip.lib
    for changes in REFUSED + [dict(logprob=None), dict(old_logprob=None), dict(advantage=None),
                              dict(cu=None)]:
        d = descriptor(**changes)
        assert lib.ehip_policy_loss_f32(C.byref(d), 64, 64, 64, 64, 1 << 30, None) == 1, changes
        assert lib.ehip_policy_loss_backward_f32(C.byref(d), 64, 64, 64, 64, None) == 1, changes
    d = descriptor()
    call = lambda loss=64, weights=64, w=64, n=1 << 30: lib.ehip_policy_loss_f32(
        C.byref(d), loss, 64, weights, w, n, None)
    assert call(loss=None) == 1 and call(weights=None) == 1 and call(w=None) == 1
    assert call(w=72) == 1 and call(n=16) == 1
    assert lib.ehip_policy_loss_backward_f32(C.byref(d), None, 64, 64, 64, None) == 1
    assert lib.ehip_policy_loss_backward_f32(C.byref(d), 64, None, 64, 64, None) == 1
    (lp, old, adv, cu), how = make([4, 5], seed=13)
    for bad in ((lp[:8], old, adv, cu), (lp, old.double(), adv, cu), (lp, old, adv[:4], cu),
                (lp, old, adv, cu.long()), (lp[None], old, adv, cu), (lp, old, adv, cu[:0]),
                (lp.cpu(), old, adv, cu)):
        with pytest.raises(ValueError):
            hip.policy_loss(*bad, **how)
    with pytest.raises(ValueError):
        hip.policy_loss(lp, old, adv, cu, mask=torch.ones(9, device="cuda"))
    with pytest.raises(ValueError):
        hip.policy_loss(lp, old, adv, cu, by_sequence=True)
    with pytest.raises(RuntimeError):
        hip.policy_loss(lp, old, adv, cu, kl_weight=0.1)
    _, _, weights = hip.policy_loss(lp, old, adv, cu)
    with pytest.raises(ValueError):
        hip.policy_loss_backward(torch.ones(1, device="cuda"), lp, old, adv, cu, weights[:2])
