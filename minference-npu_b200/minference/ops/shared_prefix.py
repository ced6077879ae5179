"""Attention of new tokens over a shared prefix and per-sequence caches.

After the prefill of one long prompt, a batch of sequences continues from it:
each new token attends to the prompt's keys, which every sequence shares, and
to its own sequence's cache.  ``shared_prefix_attention`` reads the shared keys
once for the whole batch, splits both caches along their length, and joins the
parts by their log-sum-exp.  Without a prefix it is the decode attention of a
batch of caches with their own lengths and grouped key/value heads, where
``dense_attention`` takes one length and repeated heads.
"""

from __future__ import annotations

import math

import torch

from .. import _native
from ._cache import check_output, check_query, check_same, lengths_arg, overlap, rows_arg
from ._common import output as _common_out

__all__ = ["shared_prefix_attention"]

_NONE = (0, 0, 0, 0)


def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor | None,
                            v_prefix: torch.Tensor | None, k: torch.Tensor | None,
                            v: torch.Tensor | None, lengths: torch.Tensor | None = None, *,
                            prefix_lengths: torch.Tensor | None = None,
                            scale: float | None = None, causal: bool = True,
                            return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of the new tokens ``q`` ``[B,Hq,S_q,D]``.

    ``k_prefix`` / ``v_prefix`` ``[G,Hkv,P,D]`` (or ``[Hkv,P,D]``: one prefix)
    hold G prefixes, each shared by ``B/G`` consecutive sequences; ``k`` / ``v``
    ``[B,Hkv,C,D]`` are the sequences' own caches, in which the new tokens are
    the last of the ``lengths[b]`` valid rows.  Either pair may be None.
    ``Hq`` is a multiple of ``Hkv``: consecutive query heads share a key/value
    head.  A token sees the first ``prefix_lengths[g]`` prefix keys and, if
    ``causal``, the own keys up to itself (bottom-right aligned), otherwise
    every valid own key.  Lengths are integer device tensors (None: whole),
    clamped to the capacity; rows past them are never used, whatever they hold.
    Values within a length must be finite (one that a token does not see is
    still multiplied by 0).  A token that sees nothing gives 0; one whose query
    holds a NaN gives NaN, in the log-sum-exp too.

    ``scale`` defaults to ``1/sqrt(D)``.  Returns the output, of q's dtype, or
    with ``return_lse`` the pair (output, lse float32 ``[B,Hq,S_q]``: natural
    log of the sum of exponentials, -inf where nothing is seen).  ``out`` is an
    optional caller-owned view, which must not overlap the inputs."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be [B,Hq,S_q,D]")
    B, Hq, S_q, D = q.shape
    if (k_prefix is None) != (v_prefix is None) or (k is None) != (v is None):
        raise ValueError("keys and values come in pairs")
    if k is None and k_prefix is None:
        raise ValueError("neither a prefix nor a cache to attend to")
    if k_prefix is not None and k_prefix.dim() == 3 and v_prefix.dim() == 3:
        k_prefix, v_prefix = k_prefix[None], v_prefix[None]
    kv = k if k is not None else k_prefix
    if kv.dim() != 4:
        raise ValueError("keys must be [B,Hkv,C,D] and prefix keys [G,Hkv,P,D] or [Hkv,P,D]")
    Hkv = kv.shape[1]
    code = check_query(q, Hkv)
    G, P, C = 1, 0, 0
    plen = clen = None
    if k_prefix is not None:
        if k_prefix.dim() != 4:
            raise ValueError("prefix keys must be [G,Hkv,P,D] or [Hkv,P,D]")
        G, P = k_prefix.shape[0], k_prefix.shape[2]
        shape = (G, Hkv, P, D)
        check_same("k_prefix", k_prefix, q, shape)
        check_same("v_prefix", v_prefix, q, shape)
        if G < 1 or B % G:
            raise ValueError(f"{B} sequences over {G} prefixes")
        if prefix_lengths is not None:
            plen = lengths_arg("prefix_lengths", prefix_lengths, G, P, q.device)
    elif prefix_lengths is not None:
        raise ValueError("prefix_lengths without a prefix")
    if k is not None:
        C = k.shape[2]
        shape = (B, Hkv, C, D)
        check_same("k", k, q, shape)
        check_same("v", v, q, shape)
        if lengths is not None:
            clen = lengths_arg("lengths", lengths, B, C, q.device)
    elif lengths is not None:
        raise ValueError("lengths without own caches")

    dk = max(32, (D + 7) & ~7)
    if out is None:
        res = q.new_empty((B, Hq, S_q, dk))
    else:
        check_same("out", out, q, (B, Hq, S_q, D))
        check_output("out", out)
        for name, x in (("q", q), ("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k", k),
                        ("v", v)):
            if x is not None and overlap(out, x):
                raise ValueError(f"out overlaps {name}")
        if dk == D:
            res = _common_out(out, (B, Hq, S_q, D), q)
        else:
            res = q.new_empty((B, Hq, S_q, dk))
    lse = torch.empty((B, Hq, S_q), dtype=torch.float32, device=q.device) if return_lse else None
    hold: list = []
    pad = dk - D
    args = _native.SHARED_PREFIX_ARGS.pack(
        *rows_arg(q, pad, hold),
        *(rows_arg(k_prefix, pad, hold) if P else _NONE),
        *(rows_arg(v_prefix, pad, hold) if P else _NONE),
        *(rows_arg(k, pad, hold) if C else _NONE), *(rows_arg(v, pad, hold) if C else _NONE),
        res.data_ptr(), *res.stride()[:3], 0 if lse is None else lse.data_ptr(),
        plen.data_ptr() if plen is not None and P else 0,
        clen.data_ptr() if clen is not None and C else 0, B, Hq, Hkv, S_q, G, P, C, dk, code,
        1 if causal else 0, 1.0 / math.sqrt(D) if scale is None else scale)
    _native.call_packed("mi_shared_prefix_fwd", args, q.device)
    if dk != D:
        res = res[..., :D] if out is None else out.copy_(res[..., :D])
    return (res, lse) if return_lse else res
