"""Attention with document, prefix and distance masks, for packed and padded batches.

``causal_flash_attention`` (nn/flash_attention.py) computes one causal sequence per row under the bitwise
contract.  ``masked_flash_attention`` serves batches that it does not take: documents packed into one row
(attention stays inside each), rows that end in padding, a prefix that every query sees, windows and
lengths that are no multiple of 32, scores capped by a tanh or biased by distance.  Its products run on
the matrix units of the storage type (bf16: with P and dS rounded to bf16, sums in binary32), so it is
several times faster and not under that contract; its results repeat bit for bit all the same.
"""

from __future__ import annotations

import torch

from . import _nodes

__all__ = ["masked_flash_attention", "document_positions"]

_DTYPES = (torch.bfloat16, torch.float32)
_CAPS = (2.0**-20, 2.0**13)  # a cap's scores err by about 2^-22 of it: 2^-9, half a step of bf16, at the greatest


def _check_mask(name: str, t: torch.Tensor | None, shape: tuple[int, ...], dtype: torch.dtype,
                device: torch.device) -> torch.Tensor | None:
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor or None")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, q on {device}")
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    if t.requires_grad:
        raise ValueError(f"{name} is a constant of this operator and gets no gradient: detach it")
    return t.contiguous()


def masked_flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, softcap: float = 0.0,
                           slopes: torch.Tensor | None = None, doc_ids: torch.Tensor | None = None,
                           prefix: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped-query attention of q [B, H, S, D] over k, v [B, Hkv, S, D]; D 64 or 128, any S, bf16 or float32.

    Query i sees key j when both are of one document and j lies in the causal band or in the prefix:

        doc_ids[b, i] == doc_ids[b, j] >= 0  and  ((j <= i and (window == 0 or i - j < window)) or j < prefix[b])

    ``doc_ids`` int32 [B, S] (None: one document per row; negative: padding), ``prefix`` int32 [B] (None: 0),
    ``window`` in keys, the query's own included (0: all).  Scores are q.k / sqrt(D), capped to
    softcap * tanh(score / softcap) where ``softcap`` (2^-20 .. 2^13) is not 0, less slopes[h] * |i - j| where ``slopes``
    (float32 [H], constants) are given.  A query that sees nothing, as one of padding, gets zeros, and its
    gradients are zero; what lies in rows that a query does not see, NaN included, does not reach it.

    q, k and v may be views whose last dimension is contiguous and whose rows start at 16-byte boundaries, as the
    transposed output of a projection; others are copied.  The result has q's order of dimensions in memory.
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.device.type != "cuda" or t.is_meta:
            raise RuntimeError(f"{name} is on {t.device}: this operator is the ROCm (HIP) backend and only accepts GPU tensors")
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-D [B, H, S, D], got shape {tuple(t.shape)}")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"q, k, v dtypes differ: {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dtype not in _DTYPES:
        raise ValueError(f"dtype {q.dtype} not supported (bfloat16 or float32)")
    if not (q.device == k.device == v.device):
        raise ValueError("q, k, v must be on the same device")
    B, H, S, D = q.shape
    Hkv = k.shape[1]
    if tuple(v.shape) != tuple(k.shape) or tuple(k.shape) != (B, Hkv, S, D):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if min(B, H, Hkv, S) == 0:
        raise ValueError(f"empty attention: q {tuple(q.shape)}, k {tuple(k.shape)}")
    if H % Hkv != 0:
        raise ValueError(f"n_heads ({H}) must be a multiple of n_kv_heads ({Hkv})")
    if D not in (64, 128):
        raise ValueError(f"head_dim {D} not supported (64 or 128)")
    if not isinstance(window, int) or isinstance(window, bool) or not 0 <= window < 1 << 31:
        raise ValueError(f"window must be 0 (all keys) or a positive number of keys, got {window!r}")
    softcap = float(softcap)
    if softcap != 0.0 and not _CAPS[0] <= softcap <= _CAPS[1]:
        raise ValueError(f"softcap must be 0 (none) or in [{_CAPS[0]}, {_CAPS[1]}], got {softcap}")
    slopes = _check_mask("slopes", slopes, (H,), torch.float32, q.device)
    doc_ids = _check_mask("doc_ids", doc_ids, (B, S), torch.int32, q.device)
    prefix = _check_mask("prefix", prefix, (B,), torch.int32, q.device)
    return _nodes.call("masked_attention", q, k, v, slopes, doc_ids, prefix, window, softcap)


def document_positions(doc_ids: torch.Tensor) -> torch.Tensor:
    """The position of every token within its document, int32 [B, S]: a run of equal ``doc_ids`` counts from 0."""
    if doc_ids.dim() != 2:
        raise ValueError(f"doc_ids must be [B, S], got {tuple(doc_ids.shape)}")
    at = torch.arange(doc_ids.shape[1], device=doc_ids.device, dtype=torch.int32).expand(doc_ids.shape)
    first = torch.ones_like(doc_ids, dtype=torch.bool)
    first[:, 1:] = doc_ids[:, 1:] != doc_ids[:, :-1]
    return at - torch.where(first, at, 0).cummax(1).values.to(torch.int32)
