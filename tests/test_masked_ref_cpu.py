"""The binary64 reference of the masked attention's GPU tests, against torch's autograd and against differences."""

from __future__ import annotations

import math

import pytest
import torch

from masked_ref import reference, visible


def _plain(q, k, v, see, cap, slopes):
    S, group = q.shape[2], q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    t = q @ k.mT / math.sqrt(q.shape[3])
    if cap:
        t = cap * torch.tanh(t / cap)
    if slopes is not None:
        at = torch.arange(S, dtype=torch.float64)
        t = t - slopes[:, None, None] * (at[:, None] - at[None]).abs()
    p = torch.where(see[:, None], torch.exp(t), 0.0)
    return (p / p.sum(-1, keepdim=True).clamp_min(1e-300)) @ v


@pytest.mark.parametrize("cap,alibi,window,docs", [(0.0, False, 0, False), (5.0, False, 3, True), (2.0, True, 0, True)])
def test_reference_gradients(cap, alibi, window, docs):
    gen = torch.Generator().manual_seed(3)
    B, H, Hkv, S, D = 2, 4, 2, 9, 8
    q, k, v, do = (torch.randn(B, n, S, D, generator=gen, dtype=torch.float64) for n in (H, Hkv, Hkv, H))
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0], dtype=torch.float64) if alibi else None
    doc = torch.tensor([[0] * 4 + [1] * 5, [-1] * 2 + [3] * 6 + [-1]]) if docs else None
    prefix = torch.tensor([2, 5])
    see = visible(S, window, doc, prefix)
    r = reference(q, k, v, do, see, cap, slopes)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = _plain(*leaves, see, cap, slopes)
    grads = torch.autograd.grad(o, leaves, do)
    for name, want in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)):
        torch.testing.assert_close(r[name][0], want, rtol=1e-9, atol=1e-9)
    # and against differences
    step, d = 1e-6, torch.randn(q.shape, generator=gen, dtype=torch.float64)
    diff = ((_plain(q + step * d, k, v, see, cap, slopes) - _plain(q - step * d, k, v, see, cap, slopes)) * do).sum()
    torch.testing.assert_close((r["dq"][0] * d).sum(), diff / (2 * step), rtol=1e-6, atol=1e-6)


def test_visible():
    see = visible(6, 2, torch.tensor([[0, 0, 1, 1, -1, 1]]), torch.tensor([4]))[0]
    want = ["110000", "110000", "001100", "001100", "000000", "001101"]
    assert ["".join(str(int(x)) for x in row) for row in see] == want
