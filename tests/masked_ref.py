"""Masked attention in binary64, with elementwise bounds on what a kernel of given roundings may be off by.

``u`` is half a step of binary32 (2^-24) and ``w`` half a step of the storage type of P, dS and the results
(2^-8 for bf16, 2^-24 for binary32).  Every bound is first order in these, doubled for the rest.
"""

from __future__ import annotations

import math

import torch

U = 2.0**-24


def visible(S, window=0, doc=None, prefix=None):
    """[B, S, S] (B 1 without doc and prefix)."""
    i, j = torch.arange(S)[:, None], torch.arange(S)[None, :]
    see = (j <= i) & ((i - j < window) if window else torch.ones(S, S, dtype=torch.bool))
    see = see[None]
    if prefix is not None:
        see = see | (j[None] < prefix[:, None, None])
    if doc is not None:
        see = see & (doc[:, :, None] == doc[:, None, :]) & (doc[:, :, None] >= 0)
    return see


def reference(q, k, v, do, see, cap=0.0, slopes=None, storage=torch.bfloat16):
    """{"o", "dq", "dk", "dv"}: (value, bound), from q [B, H, S, D], k and v [B, Hkv, S, D] in any type."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    B, H, S, D = q.shape
    Hkv, group = k.shape[1], H // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    w = torch.finfo(storage).eps / 2
    sigma = 1 / math.sqrt(D)
    s = sigma * q @ kk.mT
    s_err = sigma * (q.abs() @ kk.abs().mT) * U * (D + 4)  # a dot of D terms, the scale
    t, slope_of_cap, g_err = s, torch.ones_like(s), torch.zeros_like(s)
    if cap:
        x = torch.tanh(s / cap)
        t, slope_of_cap = cap * x, 1 - x * x
        s_err = s_err + 16 * U * cap  # the tanh's absolute error
        g_err = 2 * (16 * U + s_err / cap)
    if slopes is not None:
        at = torch.arange(S, dtype=torch.float64)
        bias = slopes.double()[:, None, None] * (at[:, None] - at[None, :]).abs()
        t = t - bias
        s_err = s_err + 4 * U * bias
    t = t.masked_fill(~see[:, None], -math.inf)
    top = t.amax(-1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(t - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    lse = torch.where(total > 0, top + total.clamp_min(1e-300).log(), 0.0)
    # relative error of a weight: its score's, the roundings of the exponent's argument, exp2 itself, the sum of S
    big = torch.where(see[:, None], t.abs(), 0.0) + lse.abs() + top.abs().clamp_max(1e30) * (total > 0)
    p_err = p * (s_err + 8 * U * big + (S + 16) * U)
    p_err = p_err + p * p_err.sum(-1, keepdim=True)  # through the sum
    o = p @ vv
    o_err = 2 * ((p_err + w * p) @ vv.abs() + S * U * (p @ vv.abs())) + w * o.abs()
    dp = do @ vv.mT
    delta = (do * o).sum(-1, keepdim=True)
    d_err = (do.abs() * (o_err + D * U * o.abs())).sum(-1, keepdim=True)
    dp_err = (do.abs() @ vv.abs().mT) * U * (D + 4)
    ds = p * (dp - delta) * slope_of_cap
    ds_err = p * (dp_err + d_err) * slope_of_cap + (dp - delta).abs() * (p_err * slope_of_cap + p * g_err) + w * ds.abs()
    ds_err = ds_err + 8 * U * ds.abs()

    def heads(x):
        return x.reshape(B, Hkv, group, S, D).sum(2)

    n = S * group
    dq, dq_err = sigma * ds @ kk, sigma * (ds_err + S * U * ds.abs()) @ kk.abs()
    dk, dk_err = heads(sigma * ds.mT @ q), heads(sigma * (ds_err + n * U * ds.abs()).mT @ q.abs())
    dv, dv_err = heads(p.mT @ do), heads((p_err + (w + n * U) * p).mT @ do.abs())
    tiny = 1e-30
    return {"o": (o, o_err + tiny), **{name: (x, 2 * e + w * x.abs() + tiny)
                                       for name, x, e in (("dq", dq, dq_err), ("dk", dk, dk_err), ("dv", dv, dv_err))}}


def check(name, got, value, bound):
    got = got.detach().double().cpu()
    assert got.shape == value.shape
    assert torch.isfinite(got).all(), f"{name}: {int((~torch.isfinite(got)).sum())} values are not finite"
    off = (got - value).abs() / bound
    assert off.max() <= 1, f"{name}: {float(off.max()):.3g} times the bound, at {torch.nonzero(off > 1)[:4].tolist()}"
