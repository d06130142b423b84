"""Sliding-window attention with sinks, and its single-token form over a ring cache.

Query ``i`` of a sequence attends to key ``j`` when both lie inside ``window`` of each other (``i - window < j <= i``
for ``causal``, ``|i - j| < window`` otherwise) or ``j`` is one of the first ``sinks`` tokens (static fields, forcings:
whatever every step has to see).  Query heads may share key heads.  Cost and memory grow with ``sequence x window``:
no score matrix is stored, and key tiles out of sight are never read.

Kernels: ``csrc/window_attention_sm100.cu`` (bf16, tcgen05), ``csrc/window_attention.cu`` (fp32 and the shapes that
the tensor cores do not take) and ``csrc/window_step.cu`` (one token over the cache).  Softmax statistics and sums
are fp32; the gradients use no atomics, so a pass gives the same bits every time.  Second and forward-mode derivatives
are refused on the GPU.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from tornado_gcm_b200.ops import _ext


def window_mask(sequence: int, window: int, sinks: int = 0, causal: bool = True,
                lengths: Optional[torch.Tensor] = None, device=None) -> torch.Tensor:
    """``(…, sequence, sequence)`` truth values: query (row) sees key (column)."""
    i = torch.arange(sequence, device=device)[:, None]
    j = torch.arange(sequence, device=device)[None, :]
    see = ((i - j).abs() < window) | (j < sinks)
    if causal:
        see = see & (j <= i)
    if lengths is not None:
        see = see & (j < lengths.to(j.device)[:, None, None])
    return see


def _torch_form(q, k, v, window, sinks, causal, lengths, scale):
    """Dense masked attention in elementary torch operations (CPU tensors)."""
    see = window_mask(q.shape[1], window, sinks, causal, lengths, q.device)
    see = see[:, None] if see.ndim == 3 else see
    n = q.shape[2] // k.shape[2]
    c = torch.float64 if q.dtype == torch.float64 else torch.float32
    qh, kh, vh = (t.transpose(1, 2).to(c) for t in (q, k.repeat_interleave(n, 2), v.repeat_interleave(n, 2)))
    if lengths is not None:  # what lies behind the end may hold anything
        behind = (torch.arange(q.shape[1], device=q.device) >= lengths.to(q.device)[:, None])[:, None, :, None]
        kh, vh = kh.masked_fill(behind, 0.0), vh.masked_fill(behind, 0.0)
    s = (qh @ kh.transpose(-1, -2) * scale).masked_fill(~see, -math.inf)
    dead = (s == -math.inf).all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
    return (p @ vh).transpose(1, 2).to(q.dtype)


def _scale(q: torch.Tensor, scale: Optional[float], name: str) -> float:
    if scale is None:
        return q.shape[-1] ** -0.5
    scale = float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{name}: the scale must be positive and finite, got {scale}")
    return scale


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int, sinks: int = 0,
                     causal: bool = True, lengths: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """``(B, S, H, D)`` attention of ``q (B, S, H, D)`` over ``k, v (B, S, Hk, D)``; ``Hk`` divides ``H``.

    bf16 or fp32, ``D`` up to 128, any strides with a contiguous last axis.  ``lengths``: int32 ``(B,)``, the number
    of valid keys of every sequence (keys and values behind may hold anything, NaN included; the queries there are
    computed like any other, and what they hold reaches the gradients of the keys they see).  A query that sees no
    key, or scores of minus infinity alone, gives zeros and no gradient, one that sees a score of NaN or plus infinity
    gives NaN.  A valid key's value, or in the backward pass any operand, that is not finite may also reach what lies
    in one block of 128 tokens with those that see it: the tensor cores multiply whole tiles, masked weights being
    zeros.  ``scale`` (positive) defaults to ``D ** -0.5``.
    """
    if window < 1:
        raise ValueError(f"window_attention: the window must hold at least the token itself, got {window}")
    if sinks < 0:
        raise ValueError(f"window_attention: sinks must not be negative, got {sinks}")
    scale = _scale(q, scale, "window_attention")
    if not q.is_cuda:
        if q.ndim != 4 or k.shape != v.shape or q.shape[2] % k.shape[2]:
            raise ValueError("window_attention: q (B, S, H, D) and k, v (B, S, Hk, D) with Hk dividing H expected")
        return _torch_form(q, k, v, window, sinks, causal, lengths, scale)
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    return _ext.op("window_attention")(
        q, k, v, int(window), int(sinks), bool(causal), lengths, scale, _ext.error_flag(q.device))


def window_slot(token: torch.Tensor, slots: int, sinks: int) -> torch.Tensor:
    """The cache slot of a token number: itself at first, then round and round behind the sinks."""
    return torch.where(token < slots, token, sinks + (token - sinks) % (slots - sinks))


def window_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, lengths: torch.Tensor, *, sinks: int = 0,
                          scale: Optional[float] = None) -> torch.Tensor:
    """One new token of every sequence: puts ``k, v (B, Hk, D)`` in the caches and returns the attention of
    ``q (B, H, D)`` over what they then hold.

    ``k_cache, v_cache``: ``(B, sinks + window, Hk, D)``, changed in place.  ``lengths``: int32 ``(B,)``, the tokens
    that each sequence had before this one (the caller adds one afterwards; calling again with the same lengths
    writes the same slots).  A negative length marks a sequence that takes no part: zeros, its cache untouched.
    The result equals the last row of :func:`window_attention` with ``causal`` over the whole history.  It has no
    gradient: with gradients enabled and an input that requires one the call is refused.
    """
    scale = _scale(q, scale, "window_attention_step")
    if q.is_cuda:
        return _ext.op("window_attention_step")(q, k, v, k_cache, v_cache, lengths, int(sinks), scale)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, k_cache, v_cache)):
        raise RuntimeError("window_attention_step: no gradient; call it under torch.no_grad()")
    for t in (k_cache, v_cache):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise RuntimeError("window_attention_step: cache elements share a single memory location")
    cap = k_cache.shape[1]
    if not 0 <= sinks < cap:
        raise ValueError("window_attention_step: sinks must lie between 0 and the cache's slots")
    at = lengths.long()
    on = (at >= 0).nonzero().flatten()
    slot = window_slot(at[on], cap, sinks)
    k_cache[on, slot], v_cache[on, slot] = k[on], v[on]
    see = torch.arange(cap)[None, None, None] <= at[:, None, None, None]
    n = q.shape[1] // k.shape[1]
    c = torch.float64 if q.dtype == torch.float64 else torch.float32
    kh, vh = (t.repeat_interleave(n, 2).transpose(1, 2).to(c) for t in (k_cache, v_cache))
    s = (q.to(c)[:, :, None] @ kh.transpose(-1, -2) * scale).masked_fill(~see, -math.inf)
    dead = (s == -math.inf).all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
    vh = vh.masked_fill(~see.transpose(-1, -2), 0.0)
    return (p @ vh)[:, :, 0].to(q.dtype)


def fill_window_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                      sinks: int = 0, lengths: Optional[torch.Tensor] = None) -> None:
    """Puts a whole history ``k, v (B, S, Hk, D)`` in the caches, as that many steps would have left them.

    ``lengths (B,)``: valid tokens of every sequence (what lies behind is not stored); a negative one leaves the
    sequence's cache as it is.  The caches hold values alone: no gradient reaches the history through them.
    """
    k, v = k.detach(), v.detach()
    S, cap = k.shape[1], k_cache.shape[1]
    if not 0 <= sinks < cap:
        raise ValueError("fill_window_cache: sinks must lie between 0 and the cache's slots")
    if lengths is None:
        keep = torch.arange(S, device=k.device)
        if S > cap:
            keep = torch.cat([keep[:sinks], keep[S - (cap - sinks):]])
        slot = window_slot(keep, cap, sinks)
        k_cache[:, slot], v_cache[:, slot] = k[:, keep].to(k_cache.dtype), v[:, keep].to(v_cache.dtype)
        return
    if lengths.shape != (k.shape[0],):
        raise ValueError(f"fill_window_cache: one length for each of {k.shape[0]} sequences expected, got {tuple(lengths.shape)}")
    if S == 0:
        return
    # The token that each slot holds behind `lengths` steps: itself among the sinks, behind them the latest one of
    # its residue; negative, or beyond the length, where the slot has not been written yet.
    last = lengths.to(k.device).long().clamp(max=S)[:, None] - 1
    slot = torch.arange(cap, device=k.device)
    held = last - (last - slot) % (cap - sinks)
    token = torch.where(slot < sinks, slot, torch.where(held >= sinks, held, -1))
    on = ((token >= 0) & (token <= last))[:, :, None, None]
    at = token.clamp(min=0, max=S - 1)[:, :, None, None].expand(-1, -1, *k.shape[2:])
    for cache, t in ((k_cache, k), (v_cache, v)):
        cache.copy_(torch.where(on, t.gather(1, at).to(cache.dtype), cache))
