"""The operators of packed and cached attention and of token scores, as calls of `ehip.Backend`.

A Transformer that was trained with this framework is trained further and asked for tokens
through four operators: attention over packed sequences of different lengths (forward and
backward, grouped heads), the write of new keys and values into a paged cache, attention of
one new token per sequence over that cache, and the log probabilities of given tokens with
entropy and top alternatives (forward and backward).

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

# Attention over packed sequences, forward: a prompt is read, or a batch is scored. `longest` is
# the longest sequence, `spread` seeds the others' lengths, `prefix` the most keys that a
# sequence holds from before (a prompt that arrives in pieces), `fused` says that q, k and v
# are columns of one projection's rows.
PROMPT = [
    # The character model's heads (4 of 24) over a few lines of text: latency.
    {"name": "prompt_short", "kind": "prompt", "sequences": 8, "longest": 64, "spread": 1,
     "prefix": 0, "heads": 4, "kv_heads": 4, "head_dim": 24, "causal": True, "fused": True,
     "empty": False},
    # Requests of very different lengths, each after a part that is already cached; one has no
    # new tokens at all.
    {"name": "prompt_ragged", "kind": "prompt", "sequences": 24, "longest": 1537, "spread": 2,
     "prefix": 700, "heads": 16, "kv_heads": 4, "head_dim": 64, "causal": True, "fused": False,
     "empty": True},
    # One long document.
    {"name": "prompt_long", "kind": "prompt", "sequences": 1, "longest": 16384, "spread": 3,
     "prefix": 0, "heads": 8, "kv_heads": 2, "head_dim": 128, "causal": True, "fused": True,
     "empty": False},
]
# The same with its gradients: one layer of a training step.
TRAIN = [
    # The scaled Transformer's attention (16 x 512 tokens, 16 heads of 64).
    {"name": "train_lm", "kind": "train", "sequences": 16, "longest": 512, "spread": 0,
     "prefix": 0, "heads": 16, "kv_heads": 16, "head_dim": 64, "causal": True, "fused": False,
     "empty": False},
    # Documents of odd lengths packed into one batch, grouped heads of 96.
    {"name": "train_packed", "kind": "train", "sequences": 11, "longest": 2011, "spread": 4,
     "prefix": 0, "heads": 12, "kv_heads": 4, "head_dim": 96, "causal": True, "fused": True,
     "empty": True},
]
# One new token per sequence over the pages of a cache.
DECODE = [
    # One answer being written by the scaled Transformer: latency.
    {"name": "decode_one", "kind": "decode", "sequences": 1, "longest": 500, "spread": 5,
     "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "bf16": False},
    # A server's batch: many answers of all lengths, grouped heads, a cache in 16 bits.
    {"name": "decode_batch", "kind": "decode", "sequences": 64, "longest": 4096, "spread": 6,
     "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "bf16": True},
    # Two very long documents: the length has to be split to fill the card.
    {"name": "decode_long", "kind": "decode", "sequences": 2, "longest": 131072, "spread": 0,
     "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "bf16": False},
]
# New keys and values into the pages.
APPEND = [
    # The token that each answer of a batch has just been given.
    {"name": "append_step", "kind": "append", "sequences": 64, "longest": 1, "spread": 0,
     "held": 4000, "kv_heads": 8, "head_dim": 128, "page": 32, "bf16": True},
    # Whole prompts, read from a fused projection.
    {"name": "append_prompt", "kind": "append", "sequences": 16, "longest": 2048, "spread": 7,
     "held": 300, "kv_heads": 8, "head_dim": 128, "page": 16, "bf16": False},
]
# Log probabilities of given tokens; `ties`: logits as a head in 16 bits leaves them.
SCORE = [
    # The last position of a batch of answers, with the alternatives shown to the user.
    {"name": "score_step", "kind": "score", "rows": 8, "vocab": 32000, "top": 8, "ties": True,
     "train": False},
    # A training step on the scores: log probability, entropy and their gradients.
    {"name": "score_train", "kind": "score", "rows": 8192, "vocab": 32000, "top": 0,
     "ties": False, "train": True},
]


def listed():
    return PROMPT + TRAIN + DECODE + APPEND + SCORE


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "append",
                       "score", "score"])
    dims = [24, 32, 40, 64, 64, 80, 96, 128, 128, rng.randint(8, 128)]
    while True:
        c = {"kind": kind}
        if kind in ("prompt", "train"):
            kv = rng.choice([1, 2, 3, 4, 8, 16])
            c.update(sequences=_log(rng, 1, 64), longest=_log(rng, 16, 16384),
                     spread=rng.randint(0, 999),
                     prefix=_log(rng, 1, 4096) if rng.random() < 0.4 else 0,
                     kv_heads=kv, heads=kv * rng.choice([1, 1, 2, 3, 4, 8]),
                     head_dim=rng.choice(dims), causal=rng.random() < 0.8,
                     fused=rng.random() < 0.5, empty=rng.random() < 0.3)
            nq, nk = lengths(c)
            # The plain form holds sequences x heads x longest x longest scores.
            scores = len(nq) * c["heads"] * max(nq) * max(nk)
            limit = (1 << 31) // (1 if kind == "prompt" else 3)
            if scores > limit or scores * c["head_dim"] > (128 << 31) // 3 or sum(nq) > 65536:
                continue
        elif kind == "decode":
            kv = rng.choice([1, 2, 4, 8, 16])
            c.update(sequences=_log(rng, 1, 128), longest=_log(rng, 16, 131072),
                     spread=rng.randint(0, 999), kv_heads=kv,
                     heads=kv * rng.choice([1, 1, 2, 4, 5, 8]), head_dim=rng.choice(dims),
                     page=rng.choice([1, 8, 16, 16, 32, 64, 100]), bf16=rng.random() < 0.5)
            if c["sequences"] * c["longest"] * kv * c["head_dim"] > 2 * 131072 * 8 * 128:
                continue
        elif kind == "append":
            c.update(sequences=_log(rng, 1, 128), longest=_log(rng, 1, 4096),
                     spread=rng.randint(0, 999), held=_log(rng, 1, 4096),
                     kv_heads=rng.choice([1, 2, 4, 8, 16]), head_dim=rng.choice(dims),
                     page=rng.choice([1, 8, 16, 16, 32, 64, 100]), bf16=rng.random() < 0.5)
            if c["sequences"] * (c["longest"] + c["held"]) * c["kv_heads"] * c["head_dim"] > 1 << 27:
                continue
        else:
            c.update(rows=_log(rng, 1, 8192), vocab=_log(rng, 100, 160000),
                     train=rng.random() < 0.4, ties=rng.random() < 0.5)
            c["top"] = 0 if c["train"] else min(c["vocab"], rng.choice([0, 1, 5, 8, 20, 50]))
            if c["rows"] * c["vocab"] > 8192 * 32000 // (16 if c["top"] else 1):
                continue
        return c


def lengths(case):
    """(new tokens, keys) of each sequence. `spread` 0: all of the longest length."""
    rng = random.Random(case["spread"])
    n, longest = case["sequences"], case["longest"]
    low = max(1, longest // 64)
    new = [longest if case["spread"] == 0 or i == 0 else _log(rng, low, longest)
           for i in range(n)]
    if case.get("empty") and n > 2:
        new[1], new[2] = 0, 1
    if case["kind"] == "append":
        return new, [rng.randint(0, case["held"]) if case["spread"] else case["held"]
                     for _ in range(n)]
    prefix = case.get("prefix", 0)
    return new, [a + (rng.randint(0, prefix) if prefix else 0) for a in new]


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
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    used = at < _ints(each)[:, None]
    table[used] = order[:sum(each)]
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = {"case": case, "kind": kind}
    if kind in ("prompt", "train"):
        nq, nk = lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        tq, tk = sum(nq), sum(nk)
        if case["fused"] and tq == tk:
            rows = _normal(gen, tq, h + 2 * kv, d)
            q, k, v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
        else:
            q, k, v = _normal(gen, tq, h, d), _normal(gen, tk, kv, d), _normal(gen, tk, kv, d)
        q.mul_(1.5)  # scores with a spread of 1.5, as trained heads have them
        state.update(q=q, k=k, v=v, cu_q=_ints(_offsets(nq)), cu_k=_ints(_offsets(nk)),
                     nq=nq, nk=nk, scale=1.0 / math.sqrt(d))
        if kind == "train":
            state["g"] = _normal(gen, tq, h, d)
    elif kind == "decode":
        held, _ = lengths(case)
        kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
        table, pages = _table(gen, held, page)
        dtype = torch.bfloat16 if case["bf16"] else torch.float32
        state.update(q=_normal(gen, case["sequences"], case["heads"], d).mul_(1.5),
                     k_pages=_normal(gen, pages, page, kv, d).to(dtype),
                     v_pages=_normal(gen, pages, page, kv, d).to(dtype), table=table,
                     lengths=_ints(held), longest=case["longest"], scale=1.0 / math.sqrt(d))
    elif kind == "append":
        new, held = lengths(case)
        kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
        table, pages = _table(gen, [a + b for a, b in zip(new, held)], page)
        dtype = torch.bfloat16 if case["bf16"] else torch.float32
        rows = _normal(gen, sum(new), 2 * kv, d)  # one projection's keys and values
        state.update(k=rows[:, :kv], v=rows[:, kv:], table=table, starts=_ints(held),
                     cu=_ints(_offsets(new)),
                     k_pages=torch.zeros(pages, page, kv, d, dtype=dtype, device="cuda"),
                     v_pages=torch.zeros(pages, page, kv, d, dtype=dtype, device="cuda"))
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = _normal(gen, rows, vocab).mul_(2.5)
        if case["ties"]:
            logits = logits.bfloat16().float()
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        # Half of the targets are what the model itself would answer.
        best = logits.argmax(1)
        even = torch.arange(rows, device="cuda") % 2 == 0
        state.update(logits=logits, targets=torch.where(even, best, targets).to(torch.int32),
                     top=case["top"])
        if case["train"]:
            state.update(g_logprob=_normal(gen, rows), g_entropy=_normal(gen, rows).mul_(0.01))
    return state


# -------------------------------------------------------------- the plain operators

def _padded(x, cu, n):
    """(sequences, longest, ...) from packed rows, and which of its rows are real."""
    at = torch.arange(max(1, max(n)), device=x.device)[None, :]
    real = at < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(real, cu[:-1, None] + at, torch.zeros_like(at)).long()
    return torch.where(real[:, :, None, None], x[rows], torch.zeros((), device=x.device)), real


def _by_head(x, groups):
    """(sequences, n, groups * each, d) -> (sequences * groups, each * n, d)."""
    s, n, h, d = x.shape
    x = x.reshape(s, n, groups, h // groups, d).permute(0, 2, 3, 1, 4)
    return x.reshape(s * groups, (h // groups) * n, d).contiguous()


def _from_head(x, s, groups, n):
    """The inverse of _by_head."""
    d = x.shape[-1]
    x = x.reshape(s, groups, x.shape[1] // n, n, d).permute(0, 3, 1, 2, 4)
    return x.reshape(s, n, -1, d)


def _softmax_parts(scores):
    """(weights, lse) of rows some of which have no score above -inf: those get zeros."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(-1)
    return e / torch.where(total == 0, torch.ones_like(total), total), lse


def _plain_packed(state):
    case = state["case"]
    kv = case["kv_heads"]
    group = case["heads"] // kv
    (q, real_q), (k, real_k), (v, _) = (_padded(state[x], state["cu_" + y], state["n" + y])
                                        for x, y in (("q", "q"), ("k", "k"), ("v", "k")))
    s, nq, nk = q.shape[0], q.shape[1], k.shape[1]
    qh, kh, vh = _by_head(q, kv), _by_head(k, kv), _by_head(v, kv)
    scores = torch.matmul(qh, kh.transpose(1, 2).contiguous()) * state["scale"]
    seen = real_k[:, None, :].expand(s, nq, nk)
    if case["causal"]:
        shift = (state["cu_k"][1:] - state["cu_k"][:-1]) - (state["cu_q"][1:] - state["cu_q"][:-1])
        i = torch.arange(nq, device=q.device)[None, :, None]
        j = torch.arange(nk, device=q.device)[None, None, :]
        seen = seen & (j <= i + shift[:, None, None])
    seen = seen[:, None, None].expand(s, kv, group, nq, nk).reshape(s * kv, group * nq, nk)
    weights, lse = _softmax_parts(scores.masked_fill(~seen, -math.inf))
    del scores
    out = _from_head(torch.matmul(weights, vh), s, kv, nq)[real_q]
    lse = _from_head(lse[..., None], s, kv, nq)[real_q].squeeze(-1)
    if state["kind"] == "prompt":
        return {"out": out, "lse": lse}
    g, _ = _padded(state["g"], state["cu_q"], state["nq"])
    o, _ = _padded(out, state["cu_q"], state["nq"])
    gh, oh = _by_head(g, kv), _by_head(o, kv)
    delta = (gh * oh).sum(-1, keepdim=True)
    dv = torch.matmul(weights.transpose(1, 2).contiguous(), gh)
    ds = weights * (torch.matmul(gh, vh.transpose(1, 2).contiguous()) - delta) * state["scale"]
    dq = torch.matmul(ds, kh)
    dk = torch.matmul(ds.transpose(1, 2).contiguous(), qh)
    return {"out": out, "lse": lse, "dq": _from_head(dq, s, kv, nq)[real_q],
            "dk": _from_head(dk, s, kv, nk)[real_k], "dv": _from_head(dv, s, kv, nk)[real_k]}


def _plain_decode(state):
    kv, d = state["k_pages"].shape[2:]
    s, h = state["q"].shape[:2]
    table = state["table"].long()
    k = state["k_pages"][table].float().reshape(s, -1, kv, d).permute(0, 2, 1, 3)
    v = state["v_pages"][table].float().reshape(s, -1, kv, d).permute(0, 2, 1, 3)
    q = state["q"].reshape(s, kv, h // kv, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * state["scale"]
    j = torch.arange(k.shape[2], device=q.device)
    seen = j[None, :] < state["lengths"][:, None]
    weights, lse = _softmax_parts(scores.masked_fill(~seen[:, None, None, :], -math.inf))
    out = torch.matmul(weights, v.contiguous())
    return {"out": out.reshape(s, h, d), "lse": lse.reshape(s, h)}


def _plain_append(state):
    k_pages, v_pages = state["k_pages"], state["v_pages"]
    page, cu = k_pages.shape[1], state["cu"].long()
    t = torch.arange(state["k"].shape[0], device=cu.device)
    s = torch.searchsorted(cu, t, right=True) - 1
    at = state["starts"].long()[s] + t - cu[s]
    where = state["table"].long()[s, at // page]
    k_pages[where, at % page] = state["k"].to(k_pages.dtype)
    v_pages[where, at % page] = state["v"].to(v_pages.dtype)
    return {"k_pages": k_pages, "v_pages": v_pages}


def _plain_score(state):
    x, t = state["logits"], state["targets"].long()[:, None]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.log(total) - (e * (x - top)).sum(1, keepdim=True) / total
    out = {"logprob": (x.gather(1, t) - lse).squeeze(1), "entropy": entropy.squeeze(1),
           "lse": lse.squeeze(1)}
    if state["top"]:
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        out["top"] = best[:, :state["top"]] - lse
        out["top_index"] = index[:, :state["top"]].to(torch.int32)
    if "g_logprob" in state:
        logp = x - lse
        dx = torch.exp(logp) * (-state["g_logprob"][:, None]
                                - state["g_entropy"][:, None] * (logp + entropy))
        out["dlogits"] = dx.scatter_add_(1, t, state["g_logprob"][:, None])
    return out


# --------------------------------------------------------------------- one pass

def run(state):
    if not own:
        return {"prompt": _plain_packed, "train": _plain_packed, "decode": _plain_decode,
                "append": _plain_append, "score": _plain_score}[state["kind"]](state)
    hip, kind = backend(), state["kind"]
    if kind in ("prompt", "train"):
        q, k, v, causal = state["q"], state["k"], state["v"], state["case"]["causal"]
        out, lse = hip.attention_packed(q, k, v, state["cu_q"], state["cu_k"], causal=causal)
        if kind == "prompt":
            return {"out": out, "lse": lse}
        dq, dk, dv = hip.attention_packed_backward(state["g"], q, k, v, out, lse, state["cu_q"],
                                                   state["cu_k"], causal=causal)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if kind == "decode":
        out, lse = hip.attention_paged(state["q"], state["k_pages"], state["v_pages"],
                                       state["table"], state["lengths"],
                                       longest=state["longest"])
        return {"out": out, "lse": lse}
    if kind == "append":
        hip.cache_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                         state["table"], state["starts"], state["cu"])
        return {"k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    logprob, entropy, lse, top, index = hip.token_logprobs(state["logits"], state["targets"],
                                                           top=state["top"])
    result = {"logprob": logprob, "entropy": entropy, "lse": lse}
    if state["top"]:
        result.update(top=top, top_index=index)
    if "g_logprob" in state:
        result["dlogits"] = hip.token_logprobs_backward(
            state["logits"], state["targets"], lse, entropy, state["g_logprob"],
            state["g_entropy"])
    return result


# ------------------------------------------------------------------------- the work

def work(case):
    kind = case["kind"]
    if kind in ("prompt", "train"):
        nq, nk = lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(nq, nk))
        q, k = 4 * sum(nq) * h * d, 4 * sum(nk) * kv * d
        if kind == "prompt":
            return {"bytes": 2 * q + 2 * k + 4 * sum(nq) * h, "flops": 4 * d * h * pairs}
        # Forward: q, k, v read, out written; backward: q, k, v, out, g read, dq, dk, dv written.
        return {"bytes": 5 * q + 6 * k + 8 * sum(nq) * h, "flops": 14 * d * h * pairs}
    if kind == "decode":
        held, _ = lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        each = 2 if case["bf16"] else 4
        return {"bytes": 2 * sum(held) * kv * d * each + 8 * len(held) * h * d,
                "flops": 4 * sum(held) * h * d}
    if kind == "append":
        new, _ = lengths(case)
        each = 4 + (2 if case["bf16"] else 4)
        return {"bytes": 2 * sum(new) * case["kv_heads"] * case["head_dim"] * each, "flops": 0}
    n = case["rows"] * case["vocab"]
    # Forward reads the logits; the backward reads them again and writes as many.
    return {"bytes": (12 if case["train"] else 4) * n, "flops": (10 if case["train"] else 5) * n}


# ------------------------------------------------------------------------ in 64 bits

def _exact_packed(case, state):
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    cq, ck = _offsets(state["nq"]), _offsets(state["nk"])
    q, k, v = (state[x].double() for x in "qkv")
    scale = 1.0 / math.sqrt(d)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=q.dtype, device=q.device)
    grads = {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    for s in range(len(state["nq"])):
        rows, keys = slice(cq[s], cq[s + 1]), slice(ck[s], ck[s + 1])
        n, m = state["nq"][s], state["nk"][s]
        if n == 0:
            continue
        hidden = None
        if case["causal"]:
            hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
        for head in range(h):
            c = head // (h // kv)
            a, b, w = q[rows, head], k[keys, c], v[keys, c]
            x = (a @ b.T).mul_(scale)
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(x, 1)
            p = x.sub_(z[:, None]).exp_()
            lse[rows, head] = z
            out[rows, head] = p @ w
            if case["kind"] == "train":
                g = state["g"][rows, head].double()
                grads["dv"][keys, c] += p.T @ g
                mean = (p @ w * g).sum(1, keepdim=True)
                y = p.mul_((g @ w.T).sub_(mean)).mul_(scale)
                grads["dq"][rows, head] = y @ b
                grads["dk"][keys, c] += y.T @ a
    result = {"out": out, "lse": lse}
    if case["kind"] == "train":
        result.update(grads)
    return result


def _exact_decode(case, state):
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    page, held = case["page"], lengths(case)[0]
    table = state["table"].cpu()
    out = torch.zeros(len(held), h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(held), h, dtype=torch.float64, device="cuda")
    for s, n in enumerate(held):
        which = table[s, :-(-n // page)].long().cuda()
        k = state["k_pages"].index_select(0, which).reshape(-1, kv, d)[:n].double()
        v = state["v_pages"].index_select(0, which).reshape(-1, kv, d)[:n].double()
        for c in range(kv):
            at = slice(c * (h // kv), (c + 1) * (h // kv))
            x = state["q"][s, at].double() @ k[:, c].T / math.sqrt(d)
            lse[s, at] = torch.logsumexp(x, 1)
            out[s, at] = torch.softmax(x, 1) @ v[:, c]
    return {"out": out, "lse": lse}


def _exact_append(case, state):
    page = case["page"]
    table, new, held = state["table"].tolist(), *lengths(case)
    pools = {"k": state["k_pages"].double(), "v": state["v_pages"].double()}
    at = 0
    for s, (n, start) in enumerate(zip(new, held)):
        t = torch.arange(start, start + n, device="cuda")
        where = _ints(table[s]).long()[t // page] * page + t % page
        for name in ("k", "v"):
            flat = pools[name].view(-1, *pools[name].shape[2:])
            flat[where] = state[name][at:at + n].double()
        at += n
    return {"k_pages": pools["k"], "v_pages": pools["v"]}


def _exact_score(case, state):
    parts = {}
    step = max(1, (1 << 27) // case["vocab"])
    for at in range(0, case["rows"], step):
        part = slice(at, at + step)
        x = state["logits"][part].double()
        t = state["targets"][part].long()
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        p = logp.exp()
        h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
        one = torch.arange(x.shape[0], device=x.device)
        got = {"logprob": logp[one, t], "entropy": h, "lse": lse}
        if case["top"]:
            order = torch.argsort(-x, dim=1, stable=True)[:, :case["top"]]
            got["top"], got["top_index"] = logp.gather(1, order), order.to(torch.int32)
        if case["train"]:
            g, e = state["g_logprob"][part].double(), state["g_entropy"][part].double()
            dx = -p * g[:, None] - e[:, None] * p * (logp + h[:, None])
            dx[one, t] += g
            got["dlogits"] = dx
        for name, value in got.items():
            parts.setdefault(name, []).append(value)
    return {name: torch.cat(value) for name, value in parts.items()}


def exact(case, seed):
    state = prepare(case, seed)
    return {"prompt": _exact_packed, "train": _exact_packed, "decode": _exact_decode,
            "append": _exact_append, "score": _exact_score}[case["kind"]](case, state)
