"""Masked attention on the GPU against binary64, at the sizes, masks and layouts where it can go wrong."""

from __future__ import annotations

import pytest
import torch

from masked_ref import check, reference, visible
from open_transformers_amd.nn import functional as F
from open_transformers_amd.nn.masked_attention import document_positions, masked_flash_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def docs_of(kind, B, S, gen):
    if kind is None:
        return None
    d = torch.zeros(B, S, dtype=torch.int32)
    for b in range(B):
        if kind == "packed":
            cuts = torch.sort(torch.randint(0, S + 1, (max(1, S // 40),), generator=gen)).values
            d[b] = torch.bucketize(torch.arange(S), cuts, right=True).int()
        elif kind == "right":
            d[b, max(1, S - 1 - 23 * b):] = -1
        elif kind == "left":
            d[b, :min(S - 1, 17 * b + 5)] = -1
        elif kind == "none":  # a row that is all padding
            d[b] = -1 if b == 0 else 7
        elif kind == "scattered":  # documents interleaved, in no order
            d[b] = torch.randint(-1, 4, (S,), generator=gen).int() * 1000003
            d[b][d[b] < 0] = -2**31
        elif kind == "single":
            d[b] = torch.arange(S).int()
    return d


def make(B, H, Hkv, S, D, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed + 1000 * S + B)
    return [(torch.randn(B, n, S, D, generator=gen) * scale).to(dtype) for n in (H, Hkv, Hkv, H)], gen


def run(q, k, v, do, **kw):
    kw = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o = masked_flash_attention(*leaves, **kw)
    return [o.detach(), *torch.autograd.grad(o, leaves, do.to(DEV))]


def compare(got, r):
    for (name, (value, bound)), x in zip(r.items(), got):
        check(name, x, value, bound)


CASES = [
    # dtype, B, H, Hkv, S, D, window, cap, alibi, docs, prefix
    (BF, 1, 1, 1, 1, 64, 0, 0.0, False, None, False),
    (F32, 2, 2, 1, 1, 128, 0, 30.0, True, None, False),
    (BF, 2, 2, 1, 2, 128, 0, 0.0, False, "none", False),
    (BF, 1, 2, 2, 31, 64, 0, 0.0, True, None, False),
    (F32, 1, 2, 2, 32, 64, 5, 0.0, False, None, False),
    (BF, 1, 3, 1, 33, 128, 0, 20.0, False, "packed", False),
    (F32, 2, 3, 3, 63, 128, 0, 0.0, False, "left", False),
    (BF, 1, 4, 2, 64, 64, 1, 0.0, False, None, False),
    (BF, 2, 4, 4, 65, 128, 0, 0.0, False, "right", True),
    (F32, 1, 4, 2, 127, 64, 40, 0.0, True, "scattered", False),
    (BF, 2, 2, 1, 128, 128, 0, 0.0, False, None, False),
    (BF, 2, 4, 1, 129, 128, 0, 50.0, True, "scattered", True),
    (F32, 2, 4, 1, 129, 128, 0, 50.0, True, "scattered", True),
    (BF, 2, 4, 2, 200, 64, 17, 0.0, False, None, True),
    (F32, 2, 4, 2, 200, 64, 17, 0.0, False, None, True),
    (BF, 3, 2, 2, 257, 128, 0, 0.0, False, "packed", False),
    (BF, 2, 2, 2, 257, 64, 0, 0.0, False, "none", False),
    (F32, 1, 2, 2, 191, 128, 0, 0.0, False, "single", False),
    (BF, 1, 2, 1, 515, 128, 64, 5.0, True, "packed", True),
    (BF, 2, 2, 1, 640, 64, 0, 0.0, True, "right", True),
    (F32, 1, 2, 1, 320, 128, 0, 0.0, False, None, False),
]


@pytest.mark.parametrize("dtype,B,H,Hkv,S,D,window,cap,alibi,docs,prefix", CASES)
def test_against_binary64(dtype, B, H, Hkv, S, D, window, cap, alibi, docs, prefix):
    (q, k, v, do), gen = make(B, H, Hkv, S, D, dtype)
    doc = docs_of(docs, B, S, gen)
    slopes = 2.0 ** -(torch.arange(H, dtype=F32) + 1) if alibi else None
    pre = torch.tensor([(S * (b + 1)) // (B + 2) for b in range(B)], dtype=torch.int32) if prefix else None
    got = run(q, k, v, do, window=window, softcap=cap, slopes=slopes, doc_ids=doc, prefix=pre)
    see = visible(S, window, doc, pre)
    compare(got, reference(q, k, v, do, see, cap, slopes, dtype))
    empty = ~see.any(-1)[:, None].expand(B, H, S)
    assert (got[0].cpu()[empty] == 0).all() and (got[1].cpu()[empty] == 0).all()


@pytest.mark.parametrize("heads", [1, 8])
@pytest.mark.parametrize("dtype,B,H,Hkv,S,D,window,cap,alibi,docs,prefix", [c for c in CASES if c[4] > 64])
def test_full_grids_against_binary64(dtype, B, H, Hkv, S, D, window, cap, alibi, docs, prefix, heads):
    """The same rows many times over, so that blocks of 128 rows fill the device: a workgroup's waves share their tiles
    (in CASES, from S = 129, they do not), and with many key/value heads dK/dV walks a group's heads in one.  One repetition
    against binary64, the others against it bit for bit."""
    H, Hkv = H * heads, Hkv * heads
    n = -(-780 // (B * Hkv * -(-S // 128))) if heads > 1 else -(-260 // (B * H * -(-S // 128)))
    (q, k, v, do), gen = make(B, H, Hkv, S, D, dtype)
    doc = docs_of(docs, B, S, gen)
    slopes = 2.0 ** -(torch.arange(H, dtype=F32) / heads + 1) if alibi else None
    pre = torch.tensor([(S * (b + 1)) // (B + 2) for b in range(B)], dtype=torch.int32) if prefix else None
    over = [t if t is None else torch.cat([t] * n) for t in (q, k, v, do, doc, pre)]
    got = run(*over[:4], window=window, softcap=cap, slopes=slopes, doc_ids=over[4], prefix=over[5])
    for x in got:
        for i in range(1, n):
            assert torch.equal(x[i * B:(i + 1) * B], x[:B])
    compare([x[:B] for x in got], reference(q, k, v, do, visible(S, window, doc, pre), cap, slopes, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_scores(dtype):
    """Maxima that move by far more than the threshold of the running rescale, in both directions."""
    (q, k, v, do), _ = make(1, 2, 2, 300, 64, dtype, scale=6.0)
    do = do / 6
    compare(run(q, k, v, do), reference(q, k, v, do, visible(300), storage=dtype))


def test_heads_of_a_group_together_and_apart():
    """Enough workgroups that dK/dV walks a group's heads in one, and too few; both add up to the same gradients."""
    (q, k, v, do), _ = make(64, 16, 8, 70, 64, BF)
    got = run(q, k, v, do)
    few = run(q[:4], k[:4], v[:4], do[:4])
    for a, b in zip(got[:2], few[:2]):
        assert torch.equal(a[:4], b)
    compare([t[:4] for t in got], reference(q[:4], k[:4], v[:4], do[:4], visible(70)))
    compare(few, reference(q[:4], k[:4], v[:4], do[:4], visible(70)))


def test_window_of_the_length_and_beyond_is_none():
    (q, k, v, do), _ = make(1, 2, 1, 150, 64, BF)
    plain = run(q, k, v, do)
    for window in (150, 151, 2**31 - 1):
        for a, b in zip(plain, run(q, k, v, do, window=window)):
            assert torch.equal(a, b)


def test_prefix_beyond_the_row_and_negative():
    (q, k, v, do), _ = make(3, 2, 1, 150, 64, BF)
    pre = torch.tensor([2**31 - 1, -2**31, 150], dtype=torch.int32)
    got = run(q, k, v, do, prefix=pre)
    compare(got, reference(q, k, v, do, visible(150, prefix=pre.clamp(0, 150))))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_seen_does_not_reach(dtype, bad):
    """Non-finite values in padding, in another document and in later tokens change nothing that does not see them."""
    B, H, Hkv, S, D = 2, 4, 2, 210, 64
    (q, k, v, do), gen = make(B, H, Hkv, S, D, dtype)
    doc = torch.zeros(B, S, dtype=torch.int32)
    doc[:, 90:] = 1
    doc[:, 180:] = -1
    clean = [t.clone() for t in (q, k, v, do)]
    for t in (q, k, v, do):
        t[:, :, 180:] = bad  # padding
        t[1, :, 100:110] = bad  # tokens of the second document: it sees them, the first does not
    r = reference(*clean, visible(S, doc=doc), storage=dtype)
    o, dq, dk, dv = (t.cpu() for t in run(q, k, v, do, doc_ids=doc))
    for name, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        value, bound = r[name]
        check(name, t[0, :, :180], value[0, :, :180], bound[0, :, :180])
        check(name, t[1, :, :90], value[1, :, :90], bound[1, :, :90])
        assert (t[:, :, 180:] == 0).all()
    # queries before the bad keys of their own document do not see them; queries after do
    check("o", o[1, :, 90:100], r["o"][0][1, :, 90:100], r["o"][1][1, :, 90:100])
    check("dq", dq[1, :, 90:100], r["dq"][0][1, :, 90:100], r["dq"][1][1, :, 90:100])
    assert torch.isnan(o[1, :, 110:180]).any(-1).all()
    # keys after every bad query are seen by good ones only, whose own weights are not numbers
    assert not torch.isfinite(dk[1, :, 90:100]).all() and not torch.isfinite(dv[1, :, 90:100]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_bad_gradients_stay_with_their_keys(dtype):
    """A query whose gradient is not a number spoils its own dq and the dk, dv of the keys that it sees."""
    (q, k, v, do), _ = make(1, 2, 1, 170, 128, dtype)
    r = reference(q, k, v, do, visible(170, window=20), storage=dtype)
    do = do.clone()
    do[:, :, 100] = float("nan")
    o, dq, dk, dv = (t.cpu() for t in run(q, k, v, do, window=20))
    check("o", o, *r["o"])
    for name, t, first, last in (("dq", dq, 100, 101), ("dk", dk, 81, 101), ("dv", dv, 81, 101)):
        assert torch.isnan(t[:, :, first:last]).any(-1).all()
        for part in (slice(0, first), slice(last, 170)):
            check(name, t[:, :, part], r[name][0][:, :, part], r[name][1][:, :, part])


def test_seen_infinities_come_through():
    (q, k, v, do), _ = make(1, 1, 1, 70, 64, BF)
    v[0, 0, 3, 5] = float("inf")
    o = run(q, k, v, do)[0].cpu()
    assert torch.isfinite(o[0, 0, :3]).all() and (o[0, 0, 3:, 5] == float("inf")).all()
    assert torch.isfinite(o[0, 0, :, :5]).all()


LAYOUTS = {
    "heads_last": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
    "joint": lambda t: torch.cat([t, t, t], 3)[..., t.shape[3]:2 * t.shape[3]],
    "columns_first": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
    "unaligned": lambda t: torch.cat([t.new_zeros(3), t.reshape(-1)])[3:].view(t.shape),
    "batch_last": lambda t: t.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3),
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts(layout, dtype):
    (q, k, v, do), gen = make(2, 4, 2, 75, 64, dtype)
    doc = docs_of("packed", 2, 75, gen)
    plain = run(q, k, v, do, doc_ids=doc)
    lay = LAYOUTS[layout]
    leaves = [lay(t.to(DEV)).requires_grad_() for t in (q, k, v)]
    o = masked_flash_attention(*leaves, doc_ids=doc.to(DEV))
    got = [o, *torch.autograd.grad(o, leaves, lay(do.to(DEV)))]
    for a, b in zip(plain, got):
        assert torch.equal(a, b)
    if layout == "heads_last":
        assert o.transpose(1, 2).is_contiguous()


def test_broadcast_heads_and_gradients():
    """One key head shared by expansion: its gradient is the sum; a gradient that is itself an expansion."""
    (q, k, v, _), _ = make(2, 4, 1, 75, 64, F32)
    do = torch.ones(2, 4, 75, 64)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o = masked_flash_attention(leaves[0], leaves[1].expand(2, 4, 75, 64), leaves[2].expand(2, 4, 75, 64))
    o.sum().backward()
    compare([o, *(t.grad for t in leaves)], reference(q, k, v, do, visible(75), storage=F32))


def test_repeats_bit_for_bit_and_on_a_side_stream():
    (q, k, v, do), gen = make(2, 8, 2, 333, 128, BF)
    doc = docs_of("packed", 2, 333, gen)
    first = run(q, k, v, do, doc_ids=doc, softcap=30.0)
    for a, b in zip(first, run(q, k, v, do, doc_ids=doc, softcap=30.0)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(q, k, v, do, doc_ids=doc, softcap=30.0)
    side.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    """Two captured passes, replayed in turn with eager passes between, on inputs that change."""
    (q, k, v, do), gen = make(2, 4, 2, 200, 64, BF)
    doc = docs_of("packed", 2, 200, gen).to(DEV)
    ins = [t.to(DEV) for t in (q, k, v)]
    do = do.to(DEV)

    def step(window):
        leaves = [t.detach().requires_grad_() for t in ins]
        o = masked_flash_attention(*leaves, window=window, doc_ids=doc)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for window in (0, 50):
            step(window)
    torch.cuda.current_stream().wait_stream(side)
    for window in (0, 50):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(window)
        graphs.append((g, out, window))
    for n in range(3):
        gen.manual_seed(n)
        for t in ins:
            t.copy_(torch.randn(t.shape, generator=gen))
        for g, out, window in graphs:
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, step(window)):
                assert torch.equal(a, b)


def test_more_work_items_than_the_grid_holds():
    B, H = 524300, 2  # rows of one token: the result is v
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, do = (torch.randn(B, H, 1, 64, device=DEV, generator=gen, dtype=BF) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = masked_flash_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    assert torch.equal(o, v) and torch.equal(dv, do)
    assert float(dq.abs().max()) <= 0.1 and float(dk.abs().max()) <= 0.1  # dO.v - dO.o: zero but for roundings


def test_offsets_beyond_32_bits():
    """Batch rows that lie 2^31 elements apart."""
    (q, k, v, do), _ = make(2, 2, 1, 130, 64, BF)
    base = torch.zeros((1 << 31) + (1 << 20), dtype=BF, device=DEV)
    far = []
    for n, t in enumerate((q, k, v)):
        view = base[n << 17:].as_strided(t.shape, ((1 << 31), t.shape[2] * 64, 64, 1))
        view.copy_(t)
        far.append(view)
    leaves = [t.detach().requires_grad_() for t in far]
    o = masked_flash_attention(*leaves)
    got = [o.detach(), *torch.autograd.grad(o, leaves, do.to(DEV))]
    for a, b in zip(run(q, k, v, do), got):
        assert torch.equal(a, b)


def test_long_row():
    """16384 tokens, documents of all lengths, window; sampled queries against binary64."""
    S = 16384
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(1, n, S, 64, device=DEV, generator=gen, dtype=BF) for n in (2, 1, 1))
    cuts = torch.sort(torch.randint(0, S, (9,), device=DEV, generator=gen)).values
    doc = torch.bucketize(torch.arange(S, device=DEV), cuts, right=True).int()[None]
    o = masked_flash_attention(q, k, v, window=5000, doc_ids=doc).double()
    for i in torch.randint(0, S, (50,), device=DEV, generator=gen).tolist() + [0, S - 1]:
        see = (doc[0] == doc[0, i]) & (torch.arange(S, device=DEV) <= i) & (torch.arange(S, device=DEV) > i - 5000)
        p = torch.softmax((q[0, :, i].double() @ k[0, 0, see].double().T) / 8, -1)
        want, bound = p @ v[0, 0, see].double(), p @ v[0, 0, see].double().abs()
        # roundings of the weights and of the result, 2^-8 each; scores and sums are far below
        assert ((o[0, :, i] - want).abs() <= 2.0**-8 * (1.02 * bound + want.abs())).all()


def test_document_positions():
    doc = torch.tensor([[0, 0, 0, 4, 4, 4, 4, -1], [-1, 2, 2, 3, 3, 3, 2, 2]], dtype=torch.int32)
    want = [[0, 1, 2, 0, 1, 2, 3, 0], [0, 0, 1, 0, 1, 2, 0, 1]]
    assert document_positions(doc.to(DEV)).tolist() == want


def test_a_trace_replays_the_operator():
    (q, k, v, _), gen = make(1, 2, 1, 40, 64, BF)
    args = [t.to(DEV) for t in (q, k, v)] + [docs_of("packed", 1, 40, gen).to(DEV)]

    def f(q, k, v, doc):
        return masked_flash_attention(q, k, v, doc_ids=doc)

    traced = torch.jit.trace(f, args, check_trace=False)
    others = [torch.randn_like(t) for t in args[:3]] + [torch.zeros_like(args[3])]
    assert torch.equal(traced(*others), f(*others))


def test_refusals_on_the_gpu():
    x = torch.zeros(1, 2, 8, 64, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="head_dim"):
        masked_flash_attention(x[..., :32], x[..., :32], x[..., :32])
    with pytest.raises(ValueError, match="multiple of n_kv_heads"):
        masked_flash_attention(x.expand(1, 2, 8, 64).repeat(1, 2, 1, 1)[:, :3], x, x)
    with pytest.raises(ValueError, match="do not fit"):
        masked_flash_attention(x, x[:, :, :4], x[:, :, :4])
    with pytest.raises(ValueError, match="dtypes differ"):
        masked_flash_attention(x, x.float(), x)
    with pytest.raises(ValueError, match="not supported"):
        masked_flash_attention(x.half(), x.half(), x.half())
    with pytest.raises(ValueError, match="empty"):
        masked_flash_attention(x[:, :, :0], x[:, :, :0], x[:, :, :0])
    for window in (-1, 1.5, True, 2**31):
        with pytest.raises(ValueError, match="window"):
            masked_flash_attention(x, x, x, window=window)
    for cap in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            masked_flash_attention(x, x, x, softcap=cap)
    with pytest.raises(ValueError, match="slopes must be"):
        masked_flash_attention(x, x, x, slopes=torch.zeros(3, device=DEV))
    with pytest.raises(ValueError, match="no gradient"):
        masked_flash_attention(x, x, x, slopes=torch.zeros(2, device=DEV, requires_grad=True))
    with pytest.raises(ValueError, match="doc_ids must be"):
        masked_flash_attention(x, x, x, doc_ids=torch.zeros(1, 8, device=DEV, dtype=torch.int64))
    with pytest.raises(ValueError, match="prefix must be"):
        masked_flash_attention(x, x, x, prefix=torch.zeros(2, device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="is on cpu"):
        masked_flash_attention(x, x, x, doc_ids=torch.zeros(1, 8, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm"):
        masked_flash_attention(x.cpu(), x, x)


def test_packed_layer_run():
    """Rotary positions that restart, attention inside documents and layer norm in a row, as a packed batch uses them:
    each document gets what it gets alone."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    H, Hkv, D, lengths = 4, 2, 64, (37, 100, 64)
    S = sum(lengths)
    x = torch.randn(1, S, (H + 2 * Hkv) * D, device=DEV, generator=gen, dtype=F32)
    w, b = (torch.randn(H * D, device=DEV, generator=gen) for _ in "wb")
    doc = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(lengths, device=DEV)).int()[None]
    from open_transformers_amd.rope import scaled_rope_tables

    cos, sin = (torch.from_numpy(t).to(DEV) for t in scaled_rope_tables(S, 32, 1e4, 2.0))

    def block(x, doc):
        T = x.shape[1]
        q, k, v = x.view(1, T, H + 2 * Hkv, D).split([H, Hkv, Hkv], 2)
        at = document_positions(doc)
        q, k = (F.rotary_heads(t, cos, sin, positions=at) for t in (q, k))
        o = masked_flash_attention(q, k, v.transpose(1, 2), doc_ids=doc)
        return F.layer_norm(F.merge_heads(o), w, b)

    leaf = x.clone().requires_grad_()
    y = block(leaf, doc)
    dy = torch.randn(y.shape, device=DEV, generator=gen)
    y.backward(dy)
    at = 0
    for n in lengths:
        alone = x[:, at:at + n].clone().requires_grad_()
        ya = block(alone, torch.zeros(1, n, dtype=torch.int32, device=DEV))
        ya.backward(dy[:, at:at + n])
        # the same sums in another order of tiles: a few hundred roundings of binary32 on values of order 1 to 10
        torch.testing.assert_close(y[:, at:at + n], ya, rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(leaf.grad[:, at:at + n], alone.grad, rtol=1e-4, atol=1e-4)
        at += n


@pytest.mark.parametrize("S,n", [(512, 1), (512, 40)])
@pytest.mark.parametrize("L", [2, 3, 512])
def test_gradients_of_rows_that_see_few_keys(L, S, n):
    """D_i is formed from O before its rounding.  An error uniform within half a step of bf16, 2^-8 of the low end of a
    binade, is 2^-8 sqrt(0.54 / 3) = 0.00166 of the value in the mean square.  dQ and dK bear that once for the result and
    once for dS.  O bears the rounding of P, 0.0011 where two keys share a row, and D_i hands on 1.7 times O's error (the
    factor of two keys, where it is largest): sqrt(2 * 0.00166^2 + 0.0019^2) = 0.0030 in all.  O rounded before D_i is
    formed would add another 0.0029."""
    (q, k, v, do), _ = make(1, 4, 4, S, 128, BF)
    doc = (torch.arange(S) // L).int()[None]
    got = run(*[torch.cat([t] * n) for t in (q, k, v, do)], doc_ids=torch.cat([doc] * n))
    for (name, (value, _)), x in list(zip(reference(q, k, v, do, visible(S, 0, doc)).items(), got))[1:3]:
        off = (x[:1].double().cpu() - value).norm() / value.norm()
        assert off < 0.0030, (name, float(off))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cap,alibi", [(0.0, False), (30.0, False), (0.0, True)])
@pytest.mark.parametrize("S,n,window", [(1, 1, 0), (1, 300, 0), (40, 2, 1), (200, 1, 1), (200, 80, 1)])
def test_rows_that_see_one_key(S, n, window, cap, alibi, dtype):
    """Their weight is 1 whatever the score, so o is v, and dq and dk are 0, to the bit."""
    (q, k, v, do), _ = make(1, 4, 2, S, 128, dtype, scale=2.0)
    slopes = torch.full((4,), 0.5) if alibi else None
    o, dq, dk, _ = run(*[torch.cat([t] * n) for t in (q, k, v, do)], window=window, softcap=cap, slopes=slopes)
    assert torch.equal(o[:1].cpu(), v.repeat_interleave(2, 1))
    assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("S", [70, 300])
def test_recomputed_and_unpacked_activations(S):
    """Under checkpointing and through saved-tensor hooks, the same bytes; without a gradient, the same output."""
    from torch.utils.checkpoint import checkpoint

    (q, k, v, do), gen = make(2, 4, 2, S, 64, BF)
    kw = dict(doc_ids=docs_of("packed", 2, S, gen).to(DEV), slopes=torch.full((4,), 0.1, device=DEV), softcap=20.0)
    want = run(q, k, v, do, **kw)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    with torch.no_grad():
        assert torch.equal(masked_flash_attention(*leaves, **kw), want[0])
    o = checkpoint(lambda *t: masked_flash_attention(*t, **kw), *leaves, use_reentrant=False)
    for a, b in zip((o, *torch.autograd.grad(o, leaves, do.to(DEV))), want):
        assert torch.equal(a, b)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        o = masked_flash_attention(*leaves, **kw)
    for a, b in zip(torch.autograd.grad(o, leaves, do.to(DEV)), want[1:]):
        assert torch.equal(a, b)
