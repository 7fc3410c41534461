"""Performance cases of attention with document, prefix and distance masks, rotary positions and layer norm.

The users are training jobs that pack documents of unequal length into one sequence: positions restart in every
document, attention stays inside it, scores may be capped or biased by distance, and rows may end in padding.  Each
case is one operator forward and backward, or forward alone where a program evaluates.  ``listed()`` holds the sizes
that stand for the OPEN-1B family (16 x 128 heads, 4 KV heads, d 2048, sequences of 2048 to 8192) and the small, odd
and binary32 ones beside them; ``draw`` spreads over the same ranges.

``run`` computes the operators from elementary torch operations in binary32 while ``own`` is False, and through the
framework's entry points where it is True.  ``exact`` evaluates the definitions in binary64.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def _attn(name=None, *, B, H, Hkv, S, D, dtype="bf16", window=0, softcap=0.0, alibi=False, doc=0, pad=False, prefix=0,
          heads_last=False, grad=True):
    case = dict(kind="attn", B=B, H=H, Hkv=Hkv, S=S, D=D, dtype=dtype, window=window, softcap=softcap, alibi=alibi,
                doc=doc, pad=pad, prefix=prefix, heads_last=heads_last, grad=grad)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a unit-test-sized binary32 model with distance bias: launches and latency count
        _attn("attn_f32_short", B=2, H=4, Hkv=2, S=197, D=64, dtype="f32", alibi=True, doc=60),
        # one short sequence of grouped heads at evaluation
        _attn("attn_short_eval", B=1, H=16, Hkv=4, S=333, D=128, softcap=50.0, grad=False),
        # OPEN-1B training on packed documents, q, k and v as the projections leave them
        _attn("attn_packed_docs", B=4, H=16, Hkv=4, S=4096, D=128, doc=900, heads_last=True),
        # a multi-head micro-batch with capped scores, one document to a row
        _attn("attn_capped_mha", B=4, H=16, Hkv=16, S=2048, D=128, softcap=50.0),
        # evaluation of one long sequence with distance bias
        _attn("attn_alibi_long", B=1, H=16, Hkv=16, S=8192, D=128, alibi=True, grad=False),
        # prompts with a bidirectional prefix, right-padded to the longest of the batch
        _attn("attn_prefix_padded", B=8, H=12, Hkv=4, S=1501, D=64, pad=True, prefix=256, window=512),
        # the queries of one short sequence, rotated
        dict(name="rotary_short", kind="rotary", B=1, T=61, H=16, D=128, R=128, layout="half", dtype="bf16",
             positions=True, view=False, grad=True),
        # the queries of a packed micro-batch, positions restarting in each document, tables scaled to a longer context
        dict(name="rotary_packed", kind="rotary", B=4, T=4096, H=16, D=128, R=128, layout="interleaved", dtype="bf16",
             positions=True, view=False, grad=True),
        # a quarter of each head rotated, heads cut from a joint projection
        dict(name="rotary_partial", kind="rotary", B=2, T=2047, H=12, D=128, R=32, layout="half", dtype="f32",
             positions=False, view=True, grad=True),
        # the norm of one short sequence
        dict(name="layer_norm_short", kind="layer_norm", rows=37, D=2048, dtype="bf16", bias=True, grad=True),
        # the residual stream's norm over a micro-batch
        dict(name="layer_norm_stream", kind="layer_norm", rows=16384, D=2048, dtype="bf16", bias=True, grad=True),
        # an odd width in binary32, no bias
        dict(name="layer_norm_odd", kind="layer_norm", rows=4099, D=5005, dtype="f32", bias=False, grad=True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rotary", "layer_norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "attn":
        Hkv, group = rng.choice([(1, 1), (2, 1), (4, 1), (16, 1), (1, 4), (2, 3), (4, 4), (2, 8), (3, 2)])
        S, B = int(_log(rng, 1, 8192)), rng.choice([1, 1, 2, 3, 4, 8])
        while B * Hkv * group * S * S > (16 if dtype == "f32" else 64) * 2048 * 2048:
            S = S * 2 // 3
        S = max(S, 1)
        return _attn(B=B, H=Hkv * group, Hkv=Hkv, S=S, D=rng.choice([64, 128]), dtype=dtype,
                     window=rng.choice([0, 0, 0, 17, 256, 512]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                     alibi=rng.random() < 0.3, doc=rng.choice([0, 0, 1]) and max(1, int(_log(rng, 4, 2048))),
                     pad=rng.random() < 0.3, prefix=rng.choice([0, 0, 0, 1]) and max(1, S // rng.choice([2, 5, 9])),
                     heads_last=rng.random() < 0.5, grad=rng.random() < 0.7)
    if kind == "rotary":
        D = rng.choice([64, 80, 96, 128, 128, 256])
        B, T = rng.choice([1, 1, 2, 4]), int(_log(rng, 1, 8192))
        R = rng.choice([D, D, D // 2, D // 4])
        return dict(kind=kind, B=B, T=T, H=rng.choice([1, 3, 4, 12, 16]), D=D, R=R,
                    layout=rng.choice(["half", "interleaved"]), dtype=dtype, positions=rng.random() < 0.6,
                    view=rng.random() < 0.4, grad=rng.random() < 0.7)
    D = int(_log(rng, 16, 16384))
    if rng.random() < 0.6:
        D = max(64, D // 64 * 64)
    return dict(kind=kind, rows=int(_log(rng, 1, max(2, min(131072, (1 << 25) // D)))), D=D, dtype=dtype,
                bias=rng.random() < 0.6, grad=rng.random() < 0.8)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _structure(case, seed):
    """Document numbers [B, S] (-1 where a row is padded) and prefix lengths [B], or None where the case has none.

    A row's documents have a multiset of lengths that the case fixes; the seed orders them.
    """
    B, S = case["B"], case["S"]
    rng = random.Random(seed)
    doc = None
    if case["doc"] or case["pad"]:
        doc = np.zeros((B, S), dtype=np.int32)
        for b in range(B):
            fixed = random.Random(1000 * S + b)
            used = S - (fixed.randrange(0, max(1, S // 2)) if case["pad"] and b else 0)
            lengths = []
            while sum(lengths) < used:
                n = max(1, int(fixed.expovariate(1.0 / case["doc"]))) if case["doc"] else used
                lengths.append(min(n, used - sum(lengths)))
            rng.shuffle(lengths)
            ends = np.cumsum(lengths)
            doc[b, :used] = np.searchsorted(ends, np.arange(used), side="right")
            doc[b, used:] = -1
    prefix = None
    if case["prefix"]:
        prefix = np.array([max(0, case["prefix"] - 11 * b) for b in range(B)], dtype=np.int32)
    return doc, prefix


def _slopes(H):
    """The usual geometric slopes of a linear distance bias."""
    return 2.0 ** (-8.0 * (np.arange(H) + 1) / H)


def _rotary_tables(case):
    """cos, sin [T, R/2] of positions on a context stretched four times, frequencies split as YaRN splits them."""
    R, theta, factor, original = case["R"], 500000.0, 4.0, 2048.0
    freq = theta ** (-np.arange(0, R, 2) / R)
    turns = original * freq / (2 * math.pi)
    keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    freq = freq / factor * (1 - keep) + freq * keep
    angle = np.arange(case["T"])[:, None] * freq[None]
    scale = 0.1 * math.log(factor) + 1.0
    return ((scale * np.cos(angle)).astype(np.float32), (scale * np.sin(angle)).astype(np.float32))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, kind, grad = DTYPES[case["dtype"]], case["kind"], case["grad"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dt)

    s = dict(case=case)
    if kind == "attn":
        B, H, Hkv, S, D = (case[n] for n in ("B", "H", "Hkv", "S", "D"))

        def heads(n):
            return normal(B, S, n, D).transpose(1, 2) if case["heads_last"] else normal(B, n, S, D)

        doc, prefix = _structure(case, seed)
        s.update(q=heads(H), k=heads(Hkv), v=heads(Hkv), dy=heads(H),
                 doc=None if doc is None else torch.from_numpy(doc).cuda(),
                 prefix=None if prefix is None else torch.from_numpy(prefix).cuda(),
                 slopes=torch.from_numpy(_slopes(H).astype(np.float32)).cuda() if case["alibi"] else None)
        leaves = ("q", "k", "v")
    elif kind == "rotary":
        B, T, H, D = (case[n] for n in ("B", "T", "H", "D"))
        cos, sin = _rotary_tables(case)
        x = normal(B, T, 3 * H, D)[:, :, H:2 * H] if case["view"] else normal(B, T, H, D)
        positions = None
        if case["positions"]:
            rng = random.Random(seed)
            positions = np.zeros((B, T), dtype=np.int32)
            for b in range(B):
                at = 0
                while at < T:
                    n = min(T - at, max(1, int(rng.expovariate(1.0 / 700))))
                    positions[b, at:at + n] = np.arange(n)
                    at += n
            positions = torch.from_numpy(positions).cuda()
        s.update(x=x, dy=normal(B, H, T, D), cos=torch.from_numpy(cos).cuda(), sin=torch.from_numpy(sin).cuda(),
                 positions=positions)
        leaves = ("x",)
    else:
        rows, D = case["rows"], case["D"]
        # a residual stream: rows of unequal scale, a few wide channels, a mean that is not zero
        x = torch.randn(rows, D, device="cuda", generator=gen) * (1 + 3 * torch.rand(rows, 1, device="cuda", generator=gen))
        x = x * (1 + 4 * (torch.rand(D, device="cuda", generator=gen) < 0.01)) + 0.3
        s.update(x=x.to(dt), w=1 + normal(D, scale=0.1), b=normal(D, scale=0.1) if case["bias"] else None,
                 dy=normal(rows, D))
        leaves = ("x", "w", "b") if case["bias"] else ("x", "w")
    if grad:
        for n in leaves:
            s[n].requires_grad_()
    s["leaves"] = leaves
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def _visible(case, doc, prefix):
    """The pairs (query, key) that take part, [B or 1, 1, S, S]."""
    at = torch.arange(case["S"], device="cuda")
    far = at[:, None] - at[None, :]
    see = (far >= 0) & (far < case["window"]) if case["window"] else far >= 0
    see = see[None]
    if prefix is not None:
        see = see | (at[None, None, :] < prefix[:, None, None])
    if doc is not None:
        see = see & (doc[:, :, None] == doc[:, None, :]) & (doc >= 0)[:, :, None]
    return see[:, None]


def _plain_attention(s):
    case = s["case"]
    group = case["H"] // case["Hkv"]
    q = s["q"].float()
    k, v = (s[n].float().repeat_interleave(group, dim=1) for n in ("k", "v"))
    t = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(case["D"]))
    if case["softcap"]:
        t = case["softcap"] * torch.tanh(t / case["softcap"])
    if s["slopes"] is not None:
        at = torch.arange(case["S"], device="cuda", dtype=torch.float32)
        t = t - s["slopes"][:, None, None] * (at[:, None] - at[None, :]).abs()
    t = t.masked_fill(~_visible(case, s["doc"], s["prefix"]), -math.inf)
    top = t.detach().amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(t - top)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.to(s["q"].dtype)


def _plain_rotary(s):
    case = s["case"]
    x, R = s["x"].float().transpose(1, 2), case["R"]
    cos, sin = s["cos"][None, None], s["sin"][None, None]
    if s["positions"] is not None:
        at = s["positions"].long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    if case["layout"] == "half":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., R:]], -1).to(s["x"].dtype)


def _plain_layer_norm(s):
    x = s["x"].float()
    x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].float()
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(s["x"].dtype)


def _own_forward(s):
    from __graft_entry__ import load_package

    load_package()
    from open_transformers_amd.nn.functional import layer_norm, rotary_heads
    from open_transformers_amd.nn.masked_attention import masked_flash_attention

    case = s["case"]
    if case["kind"] == "attn":
        return masked_flash_attention(s["q"], s["k"], s["v"], window=case["window"], softcap=case["softcap"],
                                      slopes=s["slopes"], doc_ids=s["doc"], prefix=s["prefix"])
    if case["kind"] == "rotary":
        return rotary_heads(s["x"], s["cos"], s["sin"], positions=s["positions"], layout=case["layout"])
    return layer_norm(s["x"], s["w"], s["b"], EPS)


def run(state):
    s, kind = state, state["case"]["kind"]
    with torch.set_grad_enabled(s["case"]["grad"]):
        if own:
            y = _own_forward(s)
        else:
            y = {"attn": _plain_attention, "rotary": _plain_rotary, "layer_norm": _plain_layer_norm}[kind](s)
    out = dict(y=y)
    if s["case"]["grad"]:
        grads = torch.autograd.grad(y, [s[n] for n in s["leaves"]], s["dy"])
        out.update({"d" + n: g for n, g in zip(s["leaves"], grads)})
    return out


# ---- definitions in binary64 --------------------------------------------------------------------------------------

def _exact_attention(case, s):
    """One head at a time, the softmax's gradient written out."""
    B, H, Hkv, S, D = (case[n] for n in ("B", "H", "Hkv", "S", "D"))
    group, cap, scale = H // Hkv, case["softcap"], 1 / math.sqrt(D)
    at = torch.arange(S, device="cuda", dtype=torch.float64)
    slopes = s["slopes"].double() if s["slopes"] is not None else None
    y = torch.zeros((B, H, S, D), device="cuda", dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(y), *(torch.zeros((B, Hkv, S, D), device="cuda", dtype=torch.float64) for _ in "kv")
    for b in range(B):
        see = _visible(case, None if s["doc"] is None else s["doc"][b:b + 1],
                       None if s["prefix"] is None else s["prefix"][b:b + 1])[0, 0]
        for h in range(H):
            q, k, v = s["q"][b, h].double(), s["k"][b, h // group].double(), s["v"][b, h // group].double()
            t = scale * (q @ k.t())
            slope_of_cap = 1.0
            if cap:
                t = torch.tanh(t / cap)
                slope_of_cap = 1 - t * t
                t = cap * t
            if slopes is not None:
                t = t - slopes[h] * (at[:, None] - at[None, :]).abs()
            t[~see] = -math.inf
            top = t.max(-1, keepdim=True).values
            top[top == -math.inf] = 0
            p = torch.exp(t - top)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            y[b, h] = p @ v
            if case["grad"]:
                g = s["dy"][b, h].double()
                dv[b, h // group] += p.t() @ g
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * slope_of_cap * scale
                dq[b, h] = ds @ k
                dk[b, h // group] += ds.t() @ q
    return dict(y=y, dq=dq, dk=dk, dv=dv) if case["grad"] else dict(y=y)


def _exact_rotary(case, s):
    """Every pair as a complex number turned by cos + i sin; the gradient turns by the conjugate."""
    R = case["R"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    turn = turn[None, :, None] if s["positions"] is None else turn[s["positions"].long()][:, :, None]

    def rotate(x, by):
        x = x.double().clone()
        first, second = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = dict(y=rotate(s["x"].detach(), turn).transpose(1, 2))
    if case["grad"]:
        out["dx"] = rotate(s["dy"].transpose(1, 2), turn.conj())
    return out


def _exact_layer_norm(case, s):
    x, w, D = s["x"].detach().double(), s["w"].detach().double(), case["D"]
    centred = x - x.sum(-1, keepdim=True) / D
    rstd = 1 / torch.sqrt((centred ** 2).sum(-1, keepdim=True) / D + EPS)
    unit = centred * rstd
    out = dict(y=unit * w + (s["b"].detach().double() if case["bias"] else 0.0))
    if case["grad"]:
        g = s["dy"].double()
        gw = g * w
        out["dx"] = rstd * (gw - gw.sum(-1, keepdim=True) / D - unit * ((gw * unit).sum(-1, keepdim=True) / D))
        out["dw"] = (g * unit).sum(0)
        if case["bias"]:
            out["db"] = g.sum(0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attention, "rotary": _exact_rotary, "layer_norm": _exact_layer_norm}[case["kind"]](case, s)


# ---- work ---------------------------------------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of the batch, for one head."""
    doc, prefix = _structure(case, 0)
    S, total = case["S"], 0
    at = np.arange(S)
    for b in range(case["B"]):
        ids = np.zeros(S, dtype=np.int64) if doc is None else doc[b]
        first = np.searchsorted(np.where(ids < 0, S, ids), np.where(ids < 0, S, ids), side="left")
        last = np.searchsorted(np.where(ids < 0, S, ids), np.where(ids < 0, S, ids), side="right")
        lo = np.maximum(first, at - case["window"] + 1) if case["window"] else first
        n = at + 1 - lo
        if prefix is not None:  # keys of the prefix that the causal band does not hold already
            end = np.minimum(prefix[b], last)
            n = n + np.maximum(0, np.minimum(end, lo) - first) + np.maximum(0, end - np.maximum(at + 1, first))
        total += int(n[ids >= 0].sum())
    return total


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "attn":
        B, H, Hkv, S, D = (case[n] for n in ("B", "H", "Hkv", "S", "D"))
        q, kv = B * H * S * D * size, B * Hkv * S * D * size
        # forward: q k v in, o out; backward: q k v o do in, dq dk dv out
        moved = (2 * q + 2 * kv) + ((4 * q + 4 * kv) if case["grad"] else 0)
        return dict(bytes=moved, flops=_pairs(case) * H * D * (14 if case["grad"] else 4))
    if case["kind"] == "rotary":
        n, once = case["B"] * case["T"] * case["H"] * case["D"], case["T"] * case["R"] * 4
        passes = 2 if case["grad"] else 1
        return dict(bytes=passes * (2 * n * size + once), flops=passes * 3 * n * case["R"] // case["D"])
    n, params = case["rows"] * case["D"], case["D"] * size
    # forward: x in, y out; backward: x dy in, dx out
    return dict(bytes=(5 if case["grad"] else 2) * n * size + (5 if case["grad"] else 2) * params,
                flops=(20 if case["grad"] else 8) * n)
