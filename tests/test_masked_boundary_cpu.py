"""What masked attention, rotary heads, layer norm and the scaled tables refuse before anything reaches the GPU, and the
tables against the formulas in binary64.  No test here launches a kernel."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from open_transformers_amd import _lib, rope
from open_transformers_amd.nn import functional as F
from open_transformers_amd.nn.masked_attention import document_positions, masked_flash_attention

P = 0x10000  # an aligned address that nothing reads
BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32


def strides(n, S=100, D=64, **change):
    s = (ctypes.c_long * (3 * n))(*([4 * S * D, S * D, D] * n))
    for i, v in change.items():
        s[int(i[1:])] = v
    return s


def fwd(q=P, k=P, v=P, o=P, low=P, lse=P, slopes=None, doc=None, prefix=None, table=None, st=None, B=1, H=4, Hkv=2, S=100,
        D=64, window=0, cap=0.0, dtype=BF16):
    st = strides(4) if st is None else st
    return _lib.load().otx_mask_attn_fwd(q, k, v, o, low, lse, slopes, doc, prefix, table, ctypes.addressof(st) if st else None,
                                         B, H, Hkv, S, D, window, cap, dtype, None)


def bwd(lse=P, dq=P, low=P, st=None, ws=P, nbytes=1 << 40, doc=None, table=None, **sizes):
    st = strides(8) if st is None else st
    a = dict(B=1, H=4, Hkv=2, S=100, D=64, window=0, cap=0.0, dtype=BF16) | sizes
    return _lib.load().otx_mask_attn_bwd(P, P, P, P, low, lse, P, dq, P, P, None, doc, None, table, ctypes.addressof(st),
                                         *a.values(), ws, nbytes, None)


def refused(rc, message):
    assert rc == _lib.OTX_EINVAL
    assert message in _lib.load().otx_last_error().decode()


@pytest.mark.parametrize("message,change", [
    ("positive", dict(S=0)), ("positive", dict(B=-1)), ("multiple of Hkv", dict(H=3)), ("head_dim", dict(D=96)),
    ("2^24", dict(S=(1 << 24) + 1)), ("too large", dict(B=1 << 20, H=1 << 12)), ("dtype", dict(dtype=7)),
    ("window", dict(window=-1)), ("softcap", dict(cap=-1.0)), ("softcap", dict(cap=float("nan"))),
    ("softcap", dict(cap=float("inf"))), ("softcap", dict(cap=1e-30)), ("softcap", dict(cap=1e5)),
    ("block table", dict(doc=P)), ("block table", dict(doc=P, table=P + 4)), ("null pointer", dict(lse=None)),
    ("null pointer argument: q", dict(q=None)), ("q must be 16-byte", dict(q=P + 8)), ("o must be 16-byte", dict(o=P + 2)),
    ("o_low", dict(low=P + 8)), ("k: stride", dict(st=strides(4, i3=-8))), ("v: stride", dict(st=strides(4, i8=68))),
    ("row stride", dict(st=strides(4, i2=1 << 22)))])
def test_attention_forward_refusals(message, change):
    refused(fwd(**change), message)


@pytest.mark.parametrize("message,change", [
    ("null pointer", dict(lse=None)), ("null pointer argument: dq", dict(dq=None)), ("256-byte", dict(ws=P + 16)),
    ("too small", dict(nbytes=100)), ("null pointer", dict(ws=None)), ("dv: stride", dict(st=strides(8, i23=4))),
    ("dout: stride", dict(st=strides(8, i12=12))), ("multiple of Hkv", dict(Hkv=3)), ("o_low", dict(low=P + 1)),
    ("block table", dict(doc=P))])
def test_attention_backward_refusals(message, change):
    refused(bwd(**change), message)


def test_attention_sizes():
    lib = _lib.load()
    assert lib.otx_mask_attn_table_bytes(2, 65) == 2 * 2 * 16 and lib.otx_mask_attn_table_bytes(0, 5) == 0
    rows = lambda B, H, S: -(-B * H * S * 4 // 256) * 256
    need = lib.otx_mask_attn_bwd_workspace_bytes
    assert need(1, 4, 4, 100, 64, 0) == rows(1, 4, 100)
    assert need(1, 4, 2, 100, 64, 0) == rows(1, 4, 100) + 4 * 100 * 64 * 8  # partial sums of two heads a group
    assert need(64, 16, 8, 100, 64, 0) == rows(64, 16, 100) < need(64, 16, 8, 100, 64, 1)
    assert need(1, 4, 3, 100, 64, 0) == 0 and need(1, 4, 2, 100, 80, 0) == 0
    refused(bwd(nbytes=need(1, 4, 2, 100, 64, 0) - 1), "too small")


def test_rotary_refusals():
    def call(x=P, cos=P, sin=P, y=2 * P, st=None, B=2, T=5, H=3, D=64, R=32, tables=5, layout=1, dtype=BF16, positions=None):
        st = strides(2) if st is None else st
        return _lib.load().otx_rotary(x, cos, sin, positions, y, ctypes.addressof(st), B, T, H, D, R, tables, layout, 0,
                                      dtype, None)

    for message, change in (
            ("positive", dict(T=0)), ("rotated columns", dict(R=0)), ("rotated columns", dict(R=31)),
            ("rotated columns", dict(R=66)), ("tables", dict(tables=4)), ("tables", dict(tables=0, positions=P)),
            ("layout", dict(layout=2)), ("dtype", dict(dtype=9)), ("null", dict(cos=None)), ("alias", dict(y=P)),
            ("too large", dict(B=1 << 20, T=1 << 10, tables=1 << 10)), ("too large", dict(H=65536)),
            ("negative stride", dict(st=strides(2, i4=-1)))):
        refused(call(**change), message)


def test_layer_norm_refusals():
    lib = _lib.load()

    def forward(x=P, w=P, y=P, mean=P, rows=3, D=5, eps=1e-5, dtype=F32):
        return lib.otx_layer_norm_fwd(x, w, None, y, mean, P, rows, D, eps, dtype, None)

    def backward(rows=3, D=5, dtype=F32, wdtype=F32, ws=P, nbytes=1 << 30, dw=P):
        return lib.otx_layer_norm_bwd(P, P, P, P, P, P, dw, None, rows, D, dtype, wdtype, ws, nbytes, None)

    for message, change in (("positive", dict(rows=0)), ("positive", dict(D=0)), ("too large", dict(D=(1 << 24) + 1)),
                            ("dtype", dict(dtype=5)), ("eps", dict(eps=-1.0)), ("eps", dict(eps=float("nan"))),
                            ("null", dict(w=None)), ("null", dict(mean=None))):
        refused(forward(**change), message)
    for message, change in (("positive", dict(rows=-1)), ("dtype", dict(wdtype=3)), ("null", dict(dw=None)),
                            ("null", dict(ws=None)), ("16-byte", dict(ws=P + 4)), ("too small", dict(nbytes=8))):
        refused(backward(**change), message)
    assert lib.otx_layer_norm_bwd_workspace_bytes(3, 5) == 1 * 5 * 2 * 4  # 32 rows of 8 threads in a workgroup
    assert lib.otx_layer_norm_bwd_workspace_bytes(0, 5) == 0


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(1, 4, 2, 64)
    c = torch.zeros(4, 32)
    for call in (lambda: masked_flash_attention(x, x, x), lambda: F.rotary_heads(x, c, c),
                 lambda: F.layer_norm(x, torch.ones(64))):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()
    with pytest.raises(TypeError):
        masked_flash_attention(None, x, x)


def test_document_positions():
    ids = torch.tensor([[4, 4, 4, 2, 2, 4, -1, -1], [7, 8, 9, 9, 9, 9, 9, 9]], dtype=torch.int32)
    assert document_positions(ids).tolist() == [[0, 1, 2, 0, 1, 0, 0, 1], [0, 0, 0, 1, 2, 3, 4, 5]]
    assert document_positions(ids[:, :1]).tolist() == [[0], [0]]
    assert document_positions(ids[:, :0]).shape == (2, 0)
    with pytest.raises(ValueError, match="must be"):
        document_positions(ids[0])


@pytest.mark.parametrize("R,theta,factor,original", [(64, 1e4, 1.0, 128), (128, 1e4, 4.0, 2048), (32, 5e5, 8.0, 4096),
                                                     (2, 1e4, 2.0, 16), (96, 100.0, 16.0, 64)])
def test_scaled_tables(R, theta, factor, original):
    """Entry by entry from the formulas, in Python's binary64; a rounding to binary32 and a last place of cos at the
    greatest angle, 300 (2^-45), are what may differ."""
    bound = 2.0**-24 * 1.4 + 2.0**-44
    for method in ("linear", "yarn"):
        cos, sin = rope.scaled_rope_tables(301, R, theta, factor, method, original_len=original)
        assert cos.dtype == sin.dtype == np.float32 and cos.shape == sin.shape == (301, R // 2)
        scale = 1.0 if method == "linear" else 0.1 * math.log(factor) + 1.0
        if method == "yarn":
            at = [R * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R - 1)
        for i in range(R // 2):
            f = theta ** (-2 * i / R)
            if method == "linear":
                f /= factor
            else:
                ramp = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
                f = f * (1 - ramp) + f / factor * ramp
            for p in (0, 1, 7, 300):
                assert abs(float(cos[p, i]) - scale * math.cos(p * f)) <= bound * scale
                assert abs(float(sin[p, i]) - scale * math.sin(p * f)) <= bound * scale
    cos, _ = rope.scaled_rope_tables(3, R, theta, factor, "yarn", original_len=original, attention_factor=0.5)
    assert (cos[0] == 0.5).all()


def test_scaled_tables_refusals():
    for kw, match in ((dict(seq_len=0), "positions"), (dict(rotary_dim=3), "rotated columns"), (dict(factor=0.5), "factor"),
                      (dict(factor=float("nan")), "factor"), (dict(method="ntk"), "method"), (dict(theta=1.0), "theta"),
                      (dict(method="yarn"), "original_len"), (dict(attention_factor=0.0), "attention_factor"),
                      (dict(method="yarn", original_len=64, beta_fast=1.0, beta_slow=2.0), "beta_fast")):
        a = dict(seq_len=4, rotary_dim=8, theta=1e4) | kw
        with pytest.raises(ValueError, match=match):
            rope.scaled_rope_tables(**a)
