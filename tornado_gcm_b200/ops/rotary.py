"""Head norms and rotary positions of queries and keys in one pass (``csrc/rotary.cu``).

:func:`qk_norm_rotary` normalises every query and key head (layer norm or root-mean-square norm over the head's
values, with optional scale and shift shared by the heads) and turns the first ``rotary_dim`` values by the angle
of the token's position.  :func:`rotary_table` makes the cosines and sines once, in fp64, for whole-numbered or
real positions (time steps, longitudes, level indices), with the two usual stretchings for sequences longer than
those trained on.  Forward and backward are one kernel each for queries and keys together; the statistics and the
parameter gradients are held in fp32, and the parameter gradients are added in a fixed order.  Second and forward-mode
derivatives are refused on the GPU.
"""

from __future__ import annotations

from typing import Optional

import torch

from tornado_gcm_b200.ops import _ext

NORM_CODES = {"none": 0, "rms": 1, "layer": 2}


def rotary_table(positions, rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None,
                 factor: float = 1.0, device=None) -> torch.Tensor:
    """``(P, rotary_dim / 2, 2)`` fp32 cosines and sines of ``positions · base^(-2i / rotary_dim)``.

    ``positions``: a count (positions 0 … P-1) or a 1-D tensor of real positions.  ``scaling="linear"`` divides the
    positions by ``factor``; ``scaling="base"`` raises the base by ``factor^(rotary_dim / (rotary_dim - 2))``, which
    leaves the fastest pair alone and slows the slowest one by ``factor``.  Computed in fp64: an fp32 angle of a
    position near 1e5 would be wrong by a hundredth of a radian.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_table: rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in (None, "linear", "base"):
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    if not factor > 0.0:
        raise ValueError(f"rotary_table: factor must be positive, got {factor}")
    if isinstance(positions, int):
        positions = torch.arange(positions, dtype=torch.float64)
    pos = torch.as_tensor(positions, dtype=torch.float64)
    if pos.ndim != 1:
        raise ValueError("rotary_table: positions must be a count or a 1-D tensor")
    if scaling == "linear":
        pos = pos / factor
    elif scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=pos.device) / rotary_dim)
    ang = pos[:, None] * freq
    return torch.stack([ang.cos(), ang.sin()], -1).float().to(device or pos.device)


def _torch_form(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps):
    """The same in elementary torch operations (CPU tensors)."""
    out = []
    cs = None
    if table is not None and table.shape[1]:
        if positions is None and q.shape[1] > table.shape[0]:
            raise ValueError(f"qk_norm_rotary: the table has {table.shape[0]} positions, the sequence {q.shape[1]}")
        if positions is not None and bool((positions < 0).any()):
            raise IndexError("qk_norm_rotary: a position is negative")
        cs = table[: q.shape[1]] if positions is None else table[positions.long()]
        cs = cs.unsqueeze(-3)  # (…, S, 1, R/2, 2)
    for x, w, b in ((q, qw, qb), (k, kw, kb)):
        y = x.float() if x.dtype != torch.float64 else x
        if norm == "layer":
            y = y - y.mean(-1, keepdim=True)
        if norm != "none":
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w
        if b is not None:
            y = y + b
        if cs is not None:
            r = 2 * cs.shape[-2]
            cos, sin = cs[..., 0].to(y.dtype), cs[..., 1].to(y.dtype)
            if interleaved:
                u, v = y[..., 0:r:2], y[..., 1:r:2]
                turned = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
            else:
                u, v = y[..., : r // 2], y[..., r // 2: r]
                turned = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
            y = torch.cat([turned, y[..., r:]], -1)
        out.append(y.to(x.dtype))
    return tuple(out)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor] = None,
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, *,
                   norm: str = "layer", interleaved: bool = False, positions: Optional[torch.Tensor] = None,
                   eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """Normalised and rotated ``q (B, S, H, D)`` and ``k (B, S, Hk, D)`` (bf16 or fp32, any strides with a
    contiguous last axis: slices of a packed projection need no copy).

    ``table``: :func:`rotary_table`; its width sets how much of the head turns, ``None`` turns nothing.  On the GPU it
    has no gradient, and one that requires it is refused.
    ``positions``: rows of the table, int32 or int64, ``(B, S)`` or ``(S,)``; ``None`` means 0 … S-1.  A position
    outside the table is reported through the device error flag (:func:`tornado_gcm_b200.ops._ext.check_error_flag`)
    and takes the nearest row; on the CPU it raises ``IndexError``.  ``norm``: ``"layer"``, ``"rms"`` or ``"none"``; weights and shifts are fp32 vectors
    of ``D`` values.  ``interleaved``: pairs are neighbours (2i, 2i+1) instead of (i, i + rotary_dim/2).
    """
    if norm not in NORM_CODES:
        raise ValueError(f"qk_norm_rotary: norm must be one of {sorted(NORM_CODES)}, got {norm!r}")
    if norm == "none" and any(t is not None for t in (q_weight, k_weight, q_bias, k_bias)):
        raise ValueError("qk_norm_rotary: norm='none' takes no weights or shifts")
    if not q.is_cuda:
        return _torch_form(q, k, table, positions, q_weight, k_weight, q_bias, k_bias, norm, interleaved, eps)
    if q.stride(-1) != 1:
        q = q.contiguous()
    if k.stride(-1) != 1:
        k = k.contiguous()
    return _ext.op("qk_norm_rotary")(
        q, k, table, positions, q_weight, k_weight, q_bias, k_bias, NORM_CODES[norm], bool(interleaved), float(eps),
        _ext.error_flag(q.device))
