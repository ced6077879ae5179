"""Eviction from a KV cache by accumulated attention weight.

``accumulate_attention_weights`` adds up the attention probability that each
cached key received from given queries: a decode step's, a prompt's last
queries (the rows that the vertical_and_slash estimator looks at), or all of
them.  ``evict_cache`` keeps the first and last rows of every head's cache and,
of the rest, those with the greatest weight, and packs them.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _native
from ._cache import check_output, check_query, check_same, lengths_arg, overlap, rows_arg

__all__ = ["accumulate_attention_weights", "evict_cache", "EvictedCache"]


class EvictedCache(NamedTuple):
    """k, v ``[B,H,keep,D]``, weights ``[B,H,keep]``, index (int32, the row each
    came from, -1 past the length) and the new lengths (int32 ``[B]``)."""

    k: torch.Tensor
    v: torch.Tensor
    weights: torch.Tensor
    index: torch.Tensor
    lengths: torch.Tensor


def _check_weights(name: str, w, shape: tuple, device: torch.device) -> None:
    if isinstance(w, torch.Tensor) and w.shape == shape and w.dtype is torch.float32 \
            and w.get_device() == device.index and w.is_contiguous():
        return
    if not isinstance(w, torch.Tensor) or w.shape != shape:
        got = tuple(w.shape) if isinstance(w, torch.Tensor) else type(w).__name__
        raise ValueError(f"{name} must be {shape}, got {got}")
    if w.dtype is not torch.float32:
        raise TypeError(f"{name} must be float32, got {w.dtype}")
    if w.device != device:
        raise ValueError(f"{name} is on {w.device}, expected {device}")
    if shape[-1] > 1 and w.stride(-1) != 1:
        raise ValueError(f"{name} needs unit stride along the keys")


def accumulate_attention_weights(q: torch.Tensor, k: torch.Tensor,
                                 weights: torch.Tensor | None = None,
                                 lengths: torch.Tensor | None = None, *,
                                 lse: torch.Tensor | None = None, scale: float | None = None,
                                 causal: bool = True,
                                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``weights + sum over heads and rows of softmax(scale q k^T)``, float32 ``[B,Hkv,C]``.

    ``q`` ``[B,Hq,S_q,D]`` are the last ``S_q`` tokens of the caches ``k``
    ``[B,Hkv,C,D]`` with ``lengths[b]`` valid rows (None: C); the heads of a
    group add up in their key/value head.  ``causal`` as in
    ``shared_prefix_attention``.  ``lse`` ``[B,Hq,S_q]`` is the rows'
    log-sum-exp where it is known -- from ``shared_prefix_attention`` with
    ``return_lse``, so that the weights are those of that attention, prefix
    included -- otherwise it is computed from the keys.  The result is written
    to ``out``: by default to ``weights`` itself, or to a new tensor without
    it.  Entries past a length are those of ``weights``, or 0."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be [B,Hq,S_q,D]")
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be [B,Hkv,C,D]")
    B, Hq, S_q, D = q.shape
    Hkv, C = k.shape[1], k.shape[2]
    code = check_query(q, Hkv)
    check_same("k", k, q, (B, Hkv, C, D))
    dev = q.device
    clen = None if lengths is None else lengths_arg("lengths", lengths, B, C, dev)
    if weights is not None:
        _check_weights("weights", weights, (B, Hkv, C), dev)
    if out is None:
        out = weights if weights is not None else \
            torch.empty((B, Hkv, C), dtype=torch.float32, device=dev)
    else:
        _check_weights("out", out, (B, Hkv, C), dev)
        if weights is not None and weights is not out and overlap(out, weights) and (
                out.data_ptr() != weights.data_ptr() or out.stride() != weights.stride()):
            raise ValueError("out overlaps weights without being the same view")
    check_output("out", out)
    if overlap(out, q) or overlap(out, k):
        raise ValueError("out overlaps q or k")
    if lse is not None:
        if not isinstance(lse, torch.Tensor) or lse.shape != (B, Hq, S_q):
            raise ValueError(f"lse must be {(B, Hq, S_q)}")
        if lse.dtype is not torch.float32 or lse.device != dev:
            raise TypeError(f"lse must be float32 on {dev}")
        lse = lse.contiguous()
        if overlap(out, lse):
            raise ValueError("out overlaps lse")
    if B == 0 or C == 0:
        return out
    if Hq == 0 or S_q == 0:
        if weights is None:
            return out.zero_()
        return out if out.data_ptr() == weights.data_ptr() else out.copy_(weights)
    dk = max(32, (D + 7) & ~7)
    hold: list = []
    args = _native.ATTN_WEIGHTS_ARGS.pack(
        *rows_arg(q, dk - D, hold), *rows_arg(k, dk - D, hold), 0 if lse is None else lse.data_ptr(),
        0 if clen is None else clen.data_ptr(),
        *((weights.data_ptr(), *weights.stride()[:2]) if weights is not None else (0, 0, 0)),
        out.data_ptr(), *out.stride()[:2], B, Hq, Hkv, S_q, C, dk, code, 1 if causal else 0,
        1.0 / math.sqrt(D) if scale is None else scale)
    _native.call_packed("mi_attn_weights", args, dev)
    return out


def evict_cache(k: torch.Tensor, v: torch.Tensor, weights: torch.Tensor, keep: int,
                lengths: torch.Tensor | None = None, *, sink: int = 0, recent: int = 0,
                out: tuple | None = None) -> EvictedCache:
    """Packs the rows worth keeping of the caches ``k`` / ``v`` ``[B,H,C,D]``.

    Of every head's ``n = lengths[b]`` valid rows (None: C) it keeps
    ``min(n, keep)``: the first ``sink``, the last ``recent``, then those with
    the greatest ``weights`` ``[B,H,C]`` (float32; ties go to the lower index,
    NaN ranks below everything).  They keep their order.  Rows past the new
    length are 0 and their index is -1.  ``out=(k, v, weights)`` are optional
    destinations of ``keep`` rows, which must not overlap the inputs."""
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be [B,H,C,D]")
    _native.require_cuda(k)
    _native.dtype_code(k)
    B, H, C, D = k.shape
    dev = k.device
    check_same("v", v, k, (B, H, C, D))
    if not 1 <= D <= 1024:
        raise NotImplementedError(f"head_dim={D}: evict_cache takes 1 to 1024")
    _check_weights("weights", weights, (B, H, C), dev)
    keep, sink, recent = int(keep), int(sink), int(recent)
    if keep < 1 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError(f"need keep >= 1 and sink + recent <= keep; got keep={keep}, "
                         f"sink={sink}, recent={recent}")
    clen = None if lengths is None else lengths_arg("lengths", lengths, B, C, dev)
    shape = (B, H, keep, D)
    if out is None:
        ko, vo = k.new_empty(shape), k.new_empty(shape)
        wo = weights.new_empty(shape[:3])
    else:
        ko, vo, wo = out
        check_same("out[0]", ko, k, shape)
        check_same("out[1]", vo, k, shape)
        _check_weights("out[2]", wo, shape[:3], dev)
        outs = (ko, vo, wo)
        for i, x in enumerate(outs):
            if i < 2 and D > 1 and x.stride(-1) != 1:
                raise ValueError(f"out[{i}] needs unit stride along the head dim")
            check_output(f"out[{i}]", x)
            if any(overlap(x, y) for y in (k, v, weights)) or any(
                    overlap(x, y) for y in outs[:i]):
                raise ValueError(f"out[{i}] overlaps an input or another output")
    index = torch.empty(shape[:3], dtype=torch.int32, device=dev)
    new_len = torch.empty((B,), dtype=torch.int32, device=dev)
    res = EvictedCache(ko, vo, wo, index, new_len)
    if B == 0 or H == 0:
        if B:  # no heads: the lengths alone
            n = clen.clamp(0, C) if clen is not None else torch.full_like(new_len, C)
            new_len.copy_(n.clamp_max(keep))
        return res
    if D > 1:
        k = k if k.stride(-1) == 1 else k.contiguous()
        v = v if v.stride(-1) == 1 else v.contiguous()
    args = _native.EVICT_ARGS.pack(
        k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], weights.data_ptr(),
        *weights.stride()[:2], ko.data_ptr(), *ko.stride()[:3], vo.data_ptr(), *vo.stride()[:3],
        wo.data_ptr(), *wo.stride()[:2], index.data_ptr(), new_len.data_ptr(),
        0 if clen is None else clen.data_ptr(), B, H, C, D, keep, sink, recent)
    _native.call_packed("mi_evict_cache", args, dev)
    return res
