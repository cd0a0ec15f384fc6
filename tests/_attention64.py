"""Attention over the pairs that lengths and a causal mask leave, in 64 bits on the CPU, with the
gradients, and how far a result in 32 bits may be from it.

u = 2^-24 is half a unit in the last place of fp32. A sum of n terms in any order is off by at
most (n - 1) u of the sum of the terms' magnitudes to first order; the bounds below take n + 4
for the terms' own roundings (a product on three bf16 parts of each factor drops at most 2^-25 of
it, two roundings' worth), and add the second order by taking everything times 1.01.
  score:   ds = scale (D + 4) u |q|.|k| + u |s|            (the scaling rounds once)
  weight:  exp's argument s - lse is rounded and each of s, lse too, the device exp and a logarithm
           are within 2 ulp: relative error  rho = 2 max_j ds + u (|s| + |lse| + |s - lse|) + (n + 12) u
  out:     rho sum p |v| + (n + 4) u sum p |v|, then one rounding
and so on through the products of the backward; every bound is an elementwise product of
magnitudes, so a term that is dropped or misplaced stands out where terms are few.
"""
import math

import torch

U = 2.0 ** -24


def _sequence(q, k, v, g, scale, causal):
    """One sequence and head: dict of (value, bound) of out, lse, dq, dk, dv."""
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    seen = torch.ones(n, m, dtype=torch.bool)
    if causal:
        seen = seen.tril(m - n)
    none = ~seen.any(1)
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=q.dtype)
    lse = torch.where(none, torch.full_like(lse, -math.inf), lse)
    p = torch.where(seen, torch.exp(s - torch.where(none, torch.zeros_like(lse), lse)[:, None]),
                    torch.zeros_like(s))
    vz = v
    out = torch.where(none[:, None], torch.zeros(n, d, dtype=q.dtype), _masked(p, seen, vz))
    a = torch.where(seen, q.abs() @ k.abs().T, torch.zeros_like(s)) * abs(scale)
    sf = torch.where(seen, s, torch.zeros_like(s))
    lf = torch.where(none, torch.zeros_like(lse), lse)
    ds_err = (d + 4) * U * a + U * sf.abs()
    top = ds_err.amax(1) if m else torch.zeros(n, dtype=q.dtype)
    rho = (2 * top[:, None] + U * (sf.abs() + lf.abs()[:, None] + (sf - lf[:, None]).abs())
           + (m + 12) * U)
    rho = rho.amax(1, keepdim=True) if m else torch.zeros(n, 1, dtype=q.dtype)
    res = {"out": (out, 1.01 * (rho + (m + 5) * U) * _masked(p, seen, v.abs()) + 1e-37),
           "lse": (lse, 1.01 * (top + (m + 4) * U + 2 * U * lf.abs() + 4 * U))}
    if g is None:
        return res
    delta = (g * out).sum(1, keepdim=True)
    dp = torch.where(seen, g @ v.T, torch.zeros_like(s))
    x = torch.where(seen, p * (dp - delta), torch.zeros_like(s))
    dp_err = torch.where(seen, (d + 4) * U * (g.abs() @ v.abs().T), torch.zeros_like(s))
    delta_err = ((d + 4) * U * (g * out).abs().sum(1, keepdim=True)
                 + (g.abs() * res["out"][1]).sum(1, keepdim=True))
    x_err = p * (rho * (dp - delta).abs() + dp_err + delta_err + 3 * U * (dp.abs() + delta.abs()))
    scale_ = abs(scale)
    res["dq"] = (_masked(x, seen, k) * scale,
                 1.01 * scale_ * (_masked(x_err, seen, k.abs())
                                  + (m + 5) * U * _masked(x.abs(), seen, k.abs())) + 1e-37)
    t = seen.T
    res["dk"] = (_masked(x.T, t, q) * scale,
                 1.01 * scale_ * (_masked(x_err.T, t, q.abs())
                                  + (n + 5) * U * _masked(x.abs().T, t, q.abs())) + 1e-37)
    res["dv"] = (_masked(p.T, t, g),
                 1.01 * (_masked((p * rho).T, t, g.abs())
                         + (n + 5) * U * _masked(p.T, t, g.abs())) + 1e-37)
    return res


def _masked(w, seen, x):
    """w @ x over the pairs seen only: 0 times a NaN that is not seen is not part of the sum."""
    if bool(torch.isfinite(x).all()):
        return torch.where(seen, w, torch.zeros_like(w)) @ x
    out = torch.zeros(w.shape[0], x.shape[1], dtype=x.dtype)
    for i in range(w.shape[0]):
        out[i] = (w[i, seen[i], None] * x[seen[i]]).sum(0)
    return out


def packed(q, k, v, nq, nk, scale, causal, g=None):
    """(values, bounds) of out, lse and with g of dq, dk, dv: dicts of float64 tensors shaped as
    the packed inputs (tokens, heads, head_dim); lse (tokens, heads)."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    g = None if g is None else g.detach().cpu().double()
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    value = {"out": torch.zeros_like(q), "lse": torch.zeros(q.shape[:2], dtype=q.dtype)}
    if g is not None:
        value.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    bound = {n: torch.zeros_like(t) for n, t in value.items()}
    a = b = 0
    for n, m in zip(nq, nk):
        rows, keys = slice(a, a + n), slice(b, b + m)
        for h in range(heads):
            c = h // group
            r = _sequence(q[rows, h], k[keys, c], v[keys, c], None if g is None else g[rows, h],
                          scale, causal)
            for name, (x, e) in r.items():
                at = (keys, c) if name in ("dk", "dv") else (rows, h)
                value[name][at] += x
                # Every head of a group adds its own sum, and one rounding of the whole.
                bound[name][at] += e + U * group * x.abs()
        a, b = a + n, b + m
    return value, bound


def within(got, value, bound, what):
    got = got.detach().cpu().double()
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    same = ~fine & ~torch.isnan(value)
    assert torch.equal(got[same], value[same]), f"{what}: infinities differ"
    off = (got - value).abs()[fine] - bound[fine]
    if off.numel():
        at = int(off.argmax())
        assert float(off[at]) <= 0, (
            f"{what}: {float(got[fine][at])!r} is {float((got - value).abs()[fine][at]):.3e} from "
            f"{float(value[fine][at])!r}, bound {float(bound[fine][at]):.3e}")
