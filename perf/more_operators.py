"""The operators of sampling answers in groups and training on them, as calls of `ehip.Backend`.

Several answers are sampled to each prompt and the model is trained on them. Around attention over
packed sequences, the paged cache and the token scores that takes: norms of query and key heads with
the rotation by position (forward and backward), a cache in 8 bits that is quantised as it is
written, read by attention and read back as rows, attention of one new token for sequences that
share their first positions, and the clipped policy loss with its gradients.

  own                   run the framework's kernels; else the operators in elementary torch
  listed()              the cases, each a dict of plain values with a name
  draw(rng)             one more case of the same ranges
  prepare(case, seed)   what the caller holds before the call, on the GPU
  run(state)            one pass; returns its outputs
  work(case)            bytes and operations a pass cannot do without
  exact(case, seed)     the same outputs in 64 bits
"""
import math
import os
import random
import sys

import torch

own = False

_handles = {}


def backend():
    """The framework's binding; imported from the repository's root, the working folder."""
    if "hip" not in _handles:
        package = os.path.join(os.getcwd(), "cpp-ai-engine_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import ehip
        _handles["hip"] = ehip.Backend()
    return _handles["hip"]


# ----------------------------------------------------------------------- the cases

# Norms of the query and key heads and their rotation by position, with gradients where `train`
# says so. `rotary`: values of a head that are rotated; `far`: positions up to a million, as in long
# documents, else each token's place in a sequence of up to 8192; `fused`: q and k are columns of
# one projection's rows.
ROTATE = [
    # The token that each answer of a batch has just been given: latency.
    {"name": "rotate_step", "kind": "rotate", "tokens": 64, "heads": 32, "kv_heads": 8,
     "head_dim": 128, "rotary": 128, "interleaved": False, "norm": True, "far": False,
     "fused": True, "train": False},
    # A long document, read: a part of each head is rotated, neighbours are the pairs.
    {"name": "rotate_long", "kind": "rotate", "tokens": 30011, "heads": 12, "kv_heads": 4,
     "head_dim": 96, "rotary": 48, "interleaved": True, "norm": True, "far": True,
     "fused": False, "train": False},
    # One layer of the scaled Transformer's training step (16 x 512 tokens, 16 heads of 64).
    {"name": "rotate_train", "kind": "rotate", "tokens": 8192, "heads": 16, "kv_heads": 16,
     "head_dim": 64, "rotary": 64, "interleaved": False, "norm": True, "far": False,
     "fused": True, "train": True},
]
# A piece of each prompt is written into the pages, and all that is held is read back as the rows
# that the piece attends to.
PIECE = [
    # A few words follow in four conversations: latency.
    {"name": "piece_short", "kind": "piece", "sequences": 4, "longest": 16, "spread": 1,
     "held": 64, "kv_heads": 4, "head_dim": 64, "page": 16, "cache": "int8"},
    # A server's batch of prompts that arrive in pieces.
    {"name": "piece_prompt", "kind": "piece", "sequences": 16, "longest": 2048, "spread": 2,
     "held": 6000, "kv_heads": 8, "head_dim": 128, "page": 16, "cache": "int8"},
]
# One new token per sequence over a cache in 8 bits.
DECODE = [
    # One answer being written by the scaled Transformer: latency.
    {"name": "decode8_one", "kind": "decode", "sequences": 1, "longest": 500, "spread": 3,
     "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "cache": "int8"},
    # A server's batch: many answers of all lengths, grouped heads.
    {"name": "decode8_batch", "kind": "decode", "sequences": 64, "longest": 8192, "spread": 4,
     "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "cache": "int8"},
]
# The same where the sequences of a group share their first positions, the prompt's. `most`: answers
# to one prompt, `prompt`: the longest prompt, `longest`: the longest answer so far.
SHARED = [
    # Sixteen answers to one short question by the scaled Transformer: latency.
    {"name": "shared_one", "kind": "shared", "groups": 1, "most": 16, "prompt": 400, "longest": 100,
     "spread": 5, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "cache": "fp32"},
    # A training batch's sampling: eight prompts, up to sixteen answers each.
    {"name": "shared_batch", "kind": "shared", "groups": 8, "most": 16, "prompt": 6000,
     "longest": 1024, "spread": 6, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32,
     "cache": "bf16"},
    # Many questions about one long document.
    {"name": "shared_long", "kind": "shared", "groups": 1, "most": 64, "prompt": 30000,
     "longest": 300, "spread": 7, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
     "cache": "int8"},
]
# The clipped policy loss of sampled answers and its gradients. `by_answer`: an advantage for each
# answer, and the mean of the answers' means; else one for each token, and the mean over tokens.
POLICY = [
    # A few short answers: latency.
    {"name": "policy_step", "kind": "policy", "sequences": 32, "longest": 64, "spread": 8,
     "by_answer": True, "reference": True, "entropy": False, "mask": True},
    # A large batch.
    {"name": "policy_train", "kind": "policy", "sequences": 2048, "longest": 4096, "spread": 9,
     "by_answer": False, "reference": True, "entropy": True, "mask": True},
]

EPS = 1e-6
CLIP_LOW, CLIP_HIGH, KL, ENTROPY = 0.2, 0.28, 0.05, 0.01


def listed():
    return ROTATE + PIECE + DECODE + SHARED + POLICY


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "piece", "decode", "shared", "shared", "policy"])
    dims = [24, 32, 40, 64, 64, 80, 96, 128, 128, rng.randint(8, 128)]
    pages = [1, 8, 16, 16, 32, 64, 100]
    while True:
        c = {"kind": kind}
        if kind == "rotate":
            kv, d = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice(dims + [160, 256])
            c.update(tokens=_log(rng, 1, 65536), kv_heads=kv,
                     heads=kv * rng.choice([1, 1, 2, 3, 4, 8]), head_dim=d,
                     rotary=2 * (d // 2 if rng.random() < 0.6 else rng.randint(1, d // 2)),
                     interleaved=rng.random() < 0.4, norm=rng.random() < 0.8,
                     far=rng.random() < 0.4, fused=rng.random() < 0.6,
                     train=rng.random() < 0.5)
            if c["tokens"] * (c["heads"] + kv) * d > 1 << (25 if c["train"] else 27):
                continue
        elif kind == "piece":
            c.update(sequences=_log(rng, 1, 64), longest=_log(rng, 1, 4096),
                     spread=rng.randint(0, 999), held=_log(rng, 1, 8192),
                     kv_heads=rng.choice([1, 2, 4, 8, 16]), head_dim=rng.choice(dims),
                     page=rng.choice(pages),
                     cache=rng.choice(["int8", "int8", "bf16", "fp32"]))
            new, held = lengths(c)
            if (sum(new) + sum(held)) * c["kv_heads"] * c["head_dim"] > 1 << 26:
                continue
        elif kind == "decode":
            kv = rng.choice([1, 2, 4, 8, 16])
            c.update(sequences=_log(rng, 1, 128), longest=_log(rng, 16, 65536),
                     spread=rng.randint(0, 999), kv_heads=kv,
                     heads=kv * rng.choice([1, 1, 2, 4, 5, 8]), head_dim=rng.choice(dims),
                     page=rng.choice(pages), cache="int8")
            if c["sequences"] * c["longest"] * kv * c["head_dim"] > 64 * 8192 * 8 * 128:
                continue
        elif kind == "shared":
            kv = rng.choice([1, 2, 4, 8, 16])
            c.update(groups=_log(rng, 1, 16), most=_log(rng, 1, 64), prompt=_log(rng, 16, 32768),
                     longest=_log(rng, 1, 2048), spread=rng.randint(0, 999), kv_heads=kv,
                     heads=kv * rng.choice([1, 1, 2, 4, 5, 8]), head_dim=rng.choice(dims),
                     page=rng.choice(pages), cache=rng.choice(["int8", "bf16", "fp32"]))
            # The plain form holds every sequence's keys and values.
            prompt, own_ = lengths(c)
            n = sum(len(x) for x in own_)
            longest = max(a + max(b) for a, b in zip(prompt, own_))
            if n * longest * kv * c["head_dim"] > 64 * 30300 * 8 * 128:
                continue
        else:
            c.update(sequences=_log(rng, 1, 4096), longest=_log(rng, 16, 16384),
                     spread=rng.randint(0, 999), by_answer=rng.random() < 0.5,
                     reference=rng.random() < 0.7, entropy=rng.random() < 0.5,
                     mask=rng.random() < 0.6)
            if c["sequences"] * c["longest"] > 2048 * 4096:
                continue
        return c


def lengths(case):
    """Of a piece: (new tokens, positions held before) of each sequence. Of a decoding step:
    positions. Shared: (prompts, answers to each). Policy: tokens. `spread` 0: all of the longest
    length."""
    rng = random.Random(case["spread"])
    even, longest = case["spread"] == 0, case["longest"]
    low = max(1, longest // 64)
    if case["kind"] == "shared":
        prompts = [case["prompt"] if even or i == 0 else _log(rng, max(1, case["prompt"] // 16),
                                                              case["prompt"])
                   for i in range(case["groups"])]
        answers = [case["most"] if even or i == 0 else rng.randint(1, case["most"])
                   for i in range(case["groups"])]
        return prompts, [[longest if even else _log(rng, low, longest) for _ in range(n)]
                         for n in answers]
    n = [longest if even or i == 0 else _log(rng, low, longest) for i in range(case["sequences"])]
    if case["kind"] == "piece":
        return n, [case["held"] if even else rng.randint(0, case["held"]) for _ in n]
    return n


def _offsets(values):
    out = [0]
    for x in values:
        out.append(out[-1] + x)
    return out


# ---------------------------------------------------------------------- the inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _table(gen, held, page):
    """A page table for sequences of `held` positions, its pages in any order, and their
    number, some unused ones included."""
    each = [-(-x // page) for x in held]
    pages = sum(each) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(held), max(1, max(each)), dtype=torch.int32, device="cuda")
    used = torch.arange(table.shape[1], device="cuda")[None, :] < _ints(each)[:, None]
    table[used] = order[:sum(each)]
    return table, pages


def _quantise(x):
    """(codes, scales) of rows of values: the nearest whole numbers of 127ths of the largest
    magnitude, ties to even; the quotients in 64 bits, as they may lie next to a half."""
    scale = x.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = torch.round(x.double() / safe.double()[..., None]).clamp_(-127, 127)
    return codes.to(torch.int8), scale


def _pools(gen, case, pages, kind):
    """Pools of keys and values (and scales) of a cache: empty, or as earlier tokens left them."""
    page, kv, d = case["page"], case["kv_heads"], case["head_dim"]
    state = {}
    for name in ("k", "v"):
        if kind == "empty":
            x = torch.zeros(pages, page, kv, d, device="cuda")
        else:
            x = _normal(gen, pages, page, kv, d)
        if case["cache"] == "int8":
            codes, scale = _quantise(x)
            state[name + "_pages"] = codes
            state[name + "_scales"] = scale.transpose(1, 2).contiguous()
        else:
            state[name + "_pages"] = x.to(torch.bfloat16) if case["cache"] == "bf16" else x
    state["scales"] = ((state["k_scales"], state["v_scales"]) if case["cache"] == "int8"
                       else None)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"case": case, "kind": kind}
    if kind == "rotate":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        if case["fused"]:  # q, k and v of one projection
            rows = _normal(gen, t, h + 2 * kv, d).mul_(2.0)
            q, k = rows[:, :h], rows[:, h:h + kv]
        else:
            q, k = _normal(gen, t, h, d).mul_(2.0), _normal(gen, t, kv, d).mul_(2.0)
        at = torch.arange(t, device="cuda")
        at = at * 33 % 1000003 if case["far"] else at % 8192
        rotary = case["rotary"]
        i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
        state.update(q=q, k=k, positions=at.to(torch.int32),
                     freqs=torch.pow(torch.full_like(i, 10000.0), -2.0 * i / rotary),
                     q_weight=1.0 + 0.2 * _normal(gen, d) if case["norm"] else None,
                     k_weight=1.0 + 0.2 * _normal(gen, d) if case["norm"] else None)
        if case["train"]:
            state.update(g_q=_normal(gen, t, h, d), g_k=_normal(gen, t, kv, d))
    elif kind == "piece":
        new, held = lengths(case)
        kv, d = case["kv_heads"], case["head_dim"]
        upto = [a + b for a, b in zip(new, held)]
        table, pages = _table(gen, upto, case["page"])
        rows = _normal(gen, sum(new), 2 * kv, d)  # one projection's keys and values
        state.update(_pools(gen, case, pages, "held"), k=rows[:, :kv], v=rows[:, kv:],
                     table=table, starts=_ints(held), cu=_ints(_offsets(new)),
                     zeros=_ints([0] * len(new)), cu_all=_ints(_offsets(upto)), tokens=sum(upto))
    elif kind == "decode":
        held = lengths(case)
        table, pages = _table(gen, held, case["page"])
        state.update(_pools(gen, case, pages, "held"), table=table, lengths=_ints(held),
                     q=_normal(gen, len(held), case["heads"], case["head_dim"]).mul_(1.5),
                     longest=case["longest"], scale=1.0 / math.sqrt(case["head_dim"]))
    elif kind == "shared":
        prompts, answers = lengths(case)
        page = case["page"]
        # A group's whole pages of the prompt first, then each answer's own: the page in which the
        # prompt ends is every answer's own copy.
        own_ = [[n + p % page for n in group] for p, group in zip(prompts, answers)]
        whole = [p // page for p in prompts]
        flat, pages = _table(gen, [w * page for w in whole] + [n for g in own_ for n in g], page)
        width = max(w + max(-(-n // page) for n in g) for w, g in zip(whole, own_))
        n = sum(len(g) for g in answers)
        table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        state.update(_pools(gen, case, pages, "held"))
        s = 0
        for g, (w, group) in enumerate(zip(whole, own_)):
            first = s
            for m in group:
                last = -(-m // page)
                table[s, :w] = flat[g, :w]
                table[s, w:w + last] = flat[len(whole) + s, :last]
                s += 1
            part = prompts[g] % page
            if part:
                at = table[first:s, w].long()
                for name in ("k_pages", "v_pages"):
                    state[name][at, :part] = state[name][at[:1], :part]
                if state["scales"] is not None:
                    for scales in state["scales"]:
                        scales[at, :, :part] = scales[at[:1], :, :part]
        held = [p + m for p, g in zip(prompts, answers) for m in g]
        state.update(table=table, lengths=_ints(held),
                     group_cu=_ints(_offsets([len(g) for g in answers])), shared=_ints(prompts),
                     q=_normal(gen, n, case["heads"], case["head_dim"]).mul_(1.5),
                     longest=max(held), longest_shared=max(prompts),
                     scale=1.0 / math.sqrt(case["head_dim"]))
    else:
        n = lengths(case)
        t, s = sum(n), len(n)
        cu = _ints(_offsets(n))
        logprob = -_normal(gen, t).abs_().mul_(1.5)
        # Most ratios are near one, some are clipped.
        old = torch.clamp_max(logprob + 0.15 * _normal(gen, t), 0.0)
        state.update(logprob=logprob, old=old, cu=cu,
                     advantage=_normal(gen, s if case["by_answer"] else t),
                     ref=(torch.clamp_max(logprob + 0.1 * _normal(gen, t), 0.0)
                          if case["reference"] else None),
                     entropy=_normal(gen, t).abs_() if case["entropy"] else None, mask=None,
                     grad=torch.full((1,), 0.75, device="cuda"))
        if case["mask"]:  # the prompt's tokens are not trained on; one answer has no others
            at = torch.arange(t, device="cuda")
            which = torch.searchsorted(cu.long(), at, right=True) - 1
            part = torch.rand(s, generator=gen, device="cuda") * 0.5
            part[s // 2] = 1.0 if s > 1 else 0.25
            size = (cu[1:] - cu[:-1])[which]
            state["mask"] = (at - cu[which]).float() >= part[which] * size.float()
    return state


# -------------------------------------------------------------- the plain operators

def _turned(x, cos, sin, rotary, interleaved):
    """The first `rotary` values of every head, turned by the tokens' angles."""
    head, rest = x[..., :rotary], x[..., rotary:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :rotary // 2], head[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_rotate(state):
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["freqs"][None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    rotary, pairs = case["rotary"], case["interleaved"]
    result = {}
    for name in ("q", "k"):
        x, w = state[name], state[name + "_weight"]
        y = x
        if w is not None:
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            y = x * r * w
        result[name] = _turned(y, cos, sin, rotary, pairs)
        if case["train"]:
            u = _turned(state["g_" + name], cos, -sin, rotary, pairs)
            if w is None:
                result["d" + name] = u
                continue
            mean = (w * u * x).mean(-1, keepdim=True)
            result["d" + name] = r * (w * u - x * r * r * mean)
            result["d" + name + "_weight"] = (u * x * r).sum((0, 1))
    return result


def _values(state, name):
    """What a cache's pages hold, in fp32."""
    x = state[name + "_pages"].float()
    return x if state["scales"] is None else x * state[name + "_scales"].transpose(1, 2)[..., None]


def _plain_piece(state):
    page = state["case"]["page"]
    table, cu = state["table"].long(), state["cu"].long()
    t = torch.arange(state["k"].shape[0], device=cu.device)
    s = torch.searchsorted(cu, t, right=True) - 1
    at = state["starts"].long()[s] + t - cu[s]
    where = table[s, at // page]
    for name in ("k", "v"):
        pages = state[name + "_pages"]
        if state["scales"] is None:
            pages[where, at % page] = state[name].to(pages.dtype)
        else:
            codes, scale = _quantise(state[name])
            pages[where, at % page] = codes
            state[name + "_scales"][where, :, at % page] = scale
    cu = state["cu_all"].long()
    t = torch.arange(state["tokens"], device=cu.device)
    s = torch.searchsorted(cu, t, right=True) - 1
    where, at = table[s, (t - cu[s]) // page], (t - cu[s]) % page
    result = {}
    for name in ("k", "v"):
        x = state[name + "_pages"][where, at].float()
        if state["scales"] is not None:
            x = x * state[name + "_scales"][where, :, at][..., None]
        result[name] = x
    return result


def _plain_attention(state):
    """Attention of one token per sequence over the positions that its table names."""
    kv, d = state["k_pages"].shape[2:]
    s, h = state["q"].shape[:2]
    table = state["table"].long()
    q = state["q"].reshape(s, kv, h // kv, d)
    k = _values(state, "k")[table].reshape(s, -1, kv, d).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(q, k) * state["scale"]
    seen = torch.arange(k.shape[3], device=q.device)[None, :] < state["lengths"][:, None]
    del k
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    v = _values(state, "v")[table].reshape(s, -1, kv, d).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(e / total, v)
    return {"out": out.reshape(s, h, d), "lse": (torch.log(total) + top).reshape(s, h)}


def _plain_policy(state):
    """In 64 bits: a ratio may lie next to its clip, and the sums are long."""
    case = state["case"]
    lp, cu = state["logprob"].double(), state["cu"].long()
    t = torch.arange(lp.shape[0], device=lp.device)
    s = torch.searchsorted(cu, t, right=True) - 1
    counted = torch.ones_like(lp) if state["mask"] is None else state["mask"].double()
    a = state["advantage"].double()
    if case["by_answer"]:
        a = a[s]
        n = torch.zeros(cu.shape[0] - 1, dtype=lp.dtype, device=lp.device)
        n = n.index_add_(0, s, counted)
        each = torch.where(n > 0, 1.0 / n, torch.zeros_like(n)) / (n > 0).sum()
        w = each[s] * counted
    else:
        w = counted / counted.sum()
    ratio = torch.exp(lp - state["old"].double())
    clipped = torch.where(a < 0, ratio < 1.0 - CLIP_LOW, ratio > 1.0 + CLIP_HIGH)
    bound = torch.where(a < 0, torch.full_like(a, 1.0 - CLIP_LOW), torch.full_like(a, 1.0 + CLIP_HIGH))
    loss = -torch.where(clipped, bound, ratio) * a
    g = -torch.where(clipped, torch.zeros_like(a), ratio * a)
    kl = torch.zeros_like(lp)
    if state["ref"] is not None:
        x = state["ref"].double() - lp
        kl = torch.exp(x) - x - 1.0
        loss = loss + KL * kl
        g = g + KL * (1.0 - torch.exp(x))
    if state["entropy"] is not None:
        loss = loss - ENTROPY * state["entropy"].double()
    up = state["grad"].double()
    total = counted.sum()
    result = {"loss": (w * loss).sum().reshape(1).float(),
              "stats": torch.stack([(counted * kl).sum() / total,
                                    (counted * clipped).sum() / total,
                                    (counted * ratio).sum() / total]).float(),
              "g_logprob": (up * w * g).float()}
    if state["entropy"] is not None:
        result["g_entropy"] = (-ENTROPY * up * w).float()
    return result


# --------------------------------------------------------------------- one pass

def run(state):
    kind, case = state["kind"], state["case"]
    if not own:
        return {"rotate": _plain_rotate, "piece": _plain_piece, "decode": _plain_attention,
                "shared": _plain_attention, "policy": _plain_policy}[kind](state)
    hip = backend()
    if kind == "rotate":
        how = dict(eps=EPS, interleaved=case["interleaved"])
        what = (state["q"], state["k"], state["positions"], state["freqs"], state["q_weight"],
                state["k_weight"])
        q, k = hip.norm_rotate(*what, **how)
        result = {"q": q, "k": k}
        if case["train"]:
            dq, dk, dq_weight, dk_weight = hip.norm_rotate_backward(state["g_q"], state["g_k"],
                                                                    *what, **how)
            result.update(dq=dq, dk=dk)
            if case["norm"]:
                result.update(dq_weight=dq_weight, dk_weight=dk_weight)
        return result
    if kind == "piece":
        cache = (state["k_pages"], state["v_pages"], state["table"])
        hip.cache_append(state["k"], state["v"], *cache, state["starts"], state["cu"],
                         scales=state["scales"])
        k, v = hip.cache_read(*cache, state["zeros"], state["cu_all"], state["tokens"],
                              scales=state["scales"])
        return {"k": k, "v": v}
    if kind == "decode":
        out, lse = hip.attention_paged(state["q"], state["k_pages"], state["v_pages"],
                                       state["table"], state["lengths"],
                                       longest=state["longest"], scales=state["scales"])
        return {"out": out, "lse": lse}
    if kind == "shared":
        out, lse = hip.attention_shared(state["q"], state["k_pages"], state["v_pages"],
                                        state["table"], state["lengths"], state["group_cu"],
                                        state["shared"], longest=state["longest"],
                                        longest_shared=state["longest_shared"],
                                        scales=state["scales"])
        return {"out": out, "lse": lse}
    what = (state["logprob"], state["old"], state["advantage"], state["cu"])
    how = dict(clip_low=CLIP_LOW, clip_high=CLIP_HIGH, ref=state["ref"],
               kl_weight=KL if state["ref"] is not None else 0.0, entropy=state["entropy"],
               entropy_weight=ENTROPY if state["entropy"] is not None else 0.0,
               mask=state["mask"], by_sequence=case["by_answer"])
    loss, stats, weights = hip.policy_loss(*what, **how)
    g_logprob, g_entropy = hip.policy_loss_backward(state["grad"], *what, weights, **how)
    result = {"loss": loss, "stats": stats, "g_logprob": g_logprob}
    if state["entropy"] is not None:
        result["g_entropy"] = g_entropy
    return result


# ------------------------------------------------------------------------- the work

def work(case):
    kind = case["kind"]
    if kind == "rotate":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        # Forward: read, written; backward: values and gradients read, gradients written.
        return {"bytes": (20 if case["train"] else 8) * n, "flops": (24 if case["train"] else 8) * n}
    kv, d = case.get("kv_heads", 0), case.get("head_dim", 0)
    # A position's bytes in one of the pools.
    row = {"int8": kv * d + 4 * kv, "bf16": 2 * kv * d, "fp32": 4 * kv * d}.get(case.get("cache"))
    if kind == "piece":
        new, held = lengths(case)
        # New rows read and written into the pages, all rows read from there and written.
        n, m = sum(new), sum(new) + sum(held)
        return {"bytes": 2 * (n + m) * (4 * kv * d + row), "flops": 4 * n * kv * d}
    if kind == "decode":
        held = lengths(case)
        return {"bytes": 2 * sum(held) * row + 8 * len(held) * case["heads"] * d,
                "flops": 4 * sum(held) * case["heads"] * d}
    if kind == "shared":
        prompts, answers = lengths(case)
        once = sum(prompts) + sum(sum(g) for g in answers)
        pairs = sum(p * len(g) + sum(g) for p, g in zip(prompts, answers))
        n = sum(len(g) for g in answers)
        return {"bytes": 2 * once * row + 8 * n * case["heads"] * d,
                "flops": 4 * pairs * case["heads"] * d}
    t = sum(lengths(case))
    # Log probabilities and gradients, and what there is of the others.
    each = (4 + 4 + 4 + 4 * case["reference"] + 8 * case["entropy"] + case["mask"]
            + 4 * (not case["by_answer"]))
    return {"bytes": each * t, "flops": 60 * t}


# ------------------------------------------------------------------------ in 64 bits

def _exact_rotate(case, state):
    half, d = case["rotary"] // 2, case["head_dim"]
    i = torch.arange(half, device="cuda")
    a = 2 * i if case["interleaved"] else i
    b = 2 * i + 1 if case["interleaved"] else i + half
    angle = torch.outer(state["positions"].double(), state["freqs"])
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    result = {}
    for name in ("q", "k"):
        x = state[name].double()
        w = state[name + "_weight"]
        y = x
        if w is not None:
            w = w.double()
            r = torch.rsqrt(x.square().sum(-1, keepdim=True) / d + EPS)
            y = x * r * w
        z = torch.complex(y[..., a], y[..., b]) * turn
        y = y.clone()
        y[..., a], y[..., b] = z.real, z.imag
        result[name] = y
        if case["train"]:
            g = state["g_" + name].double()
            z = torch.complex(g[..., a], g[..., b]) * turn.conj()
            u = g.clone()
            u[..., a], u[..., b] = z.real, z.imag
            if w is None:
                result["d" + name] = u
            else:
                hat = x * r
                dot = (u * w * hat).sum(-1, keepdim=True) / d
                result["d" + name] = (u * w - hat * dot) * r
                result["d" + name + "_weight"] = torch.einsum("thd,thd->d", u, hat)
    return result


def _pages64(state, name):
    x = state[name + "_pages"].double()
    if state["scales"] is not None:
        x *= state[name + "_scales"].double().permute(0, 2, 1).unsqueeze(3)
    return x


def _exact_piece(case, state):
    page, table = case["page"], state["table"].tolist()
    new, held = lengths(case)
    result = {}
    for name in ("k", "v"):
        pool = _pages64(state, name)
        pool = pool.view(-1, *pool.shape[2:])
        parts, at = [], 0
        for s, (n, start) in enumerate(zip(new, held)):
            p = torch.arange(start, device="cuda")
            parts.append(pool[_ints(table[s]).long()[p // page] * page + p % page])
            x = state[name][at:at + n].double()
            at += n
            if case["cache"] == "int8":
                top = x.abs().amax(2, keepdim=True)
                scale = (top / 127).float().double()  # the scale is kept in 32 bits
                x = torch.round(x / scale.clamp_min(1e-300)).clamp(-127, 127) * scale
            elif case["cache"] == "bf16":
                x = x.to(torch.float32).to(torch.bfloat16).double()  # from 32 bits: exact, once
            parts.append(x)
        result[name] = torch.cat(parts)
    return result


def _exact_attention(case, state):
    page, held = case["page"], state["lengths"].tolist()
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    table = state["table"].cpu()
    out = torch.zeros(len(held), h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(held), h, dtype=torch.float64, device="cuda")
    pools = [_pages64(state, name) for name in ("k", "v")]
    for s, n in enumerate(held):
        which = table[s, :-(-n // page)].long().cuda()
        k, v = (pool[which].reshape(-1, kv, d)[:n] for pool in pools)
        for c in range(kv):
            at = slice(c * (h // kv), (c + 1) * (h // kv))
            x = state["q"][s, at].double() @ k[:, c].T / math.sqrt(d)
            lse[s, at] = torch.logsumexp(x, 1)
            out[s, at] = torch.softmax(x, 1) @ v[:, c]
    return {"out": out, "lse": lse}


def _exact_policy(case, state):
    n = lengths(case)
    cpu = {name: state[name].cpu().double() for name in ("logprob", "old", "advantage", "ref",
                                                         "entropy", "grad")
           if state[name] is not None}
    mask = torch.ones(sum(n), dtype=torch.bool) if state["mask"] is None else state["mask"].cpu()
    sizes = [int(m.sum()) for m in mask.split(n)]
    answers, total = sum(1 for m in sizes if m), sum(sizes)
    loss, stats = 0.0, [0.0, 0.0, 0.0]
    g_logprob = torch.zeros(sum(n), dtype=torch.float64)
    g_entropy = torch.zeros(sum(n), dtype=torch.float64)
    at = 0
    for s, (m, size) in enumerate(zip(n, sizes)):
        rows = torch.arange(at, at + m)[mask[at:at + m]]
        at += m
        if size == 0:
            continue
        w = 1.0 / (answers * size) if case["by_answer"] else 1.0 / total
        lp = cpu["logprob"][rows]
        a = cpu["advantage"][s] if case["by_answer"] else cpu["advantage"][rows]
        d = lp - cpu["old"][rows]
        ratio = d.exp()
        limited = torch.minimum(ratio * a, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a)
        free = limited == ratio * a
        term, g = -limited, -(a * ratio) * free
        if "ref" in cpu:
            x = cpu["ref"][rows] - lp
            kl = torch.expm1(x) - x
            term = term + KL * kl
            g = g - KL * torch.expm1(x)
            stats[0] += float(kl.sum())
        if "entropy" in cpu:
            term = term - ENTROPY * cpu["entropy"][rows]
            g_entropy[rows] = -ENTROPY * w * cpu["grad"]
        loss += w * float(term.sum())
        stats[1] += float((~free).sum())
        stats[2] += float(ratio.sum())
        g_logprob[rows] = g * w * cpu["grad"]
    result = {"loss": torch.tensor([loss], dtype=torch.float64),
              "stats": torch.tensor(stats, dtype=torch.float64) / total, "g_logprob": g_logprob}
    if "entropy" in cpu:
        result["g_entropy"] = g_entropy
    return {name: x.cuda() for name, x in result.items()}


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotate": _exact_rotate, "piece": _exact_piece, "decode": _exact_attention,
            "shared": _exact_attention, "policy": _exact_policy}[case["kind"]](case, state)
