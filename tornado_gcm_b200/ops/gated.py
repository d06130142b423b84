"""Gated linear layer ``act(x Wgᵀ + bg) * (x Wuᵀ + bu)`` in BF16 on the tensor cores (``csrc/gated.cu``).

Both projections, the activation and the product are one kernel: the two accumulators of a hidden value sit side
by side in tensor memory and only the product is written.  The backward pass recomputes the projections (nothing
of the hidden size is kept for it), gets both pre-activation gradients in that kernel's epilogue and needs one
product for ``dx`` and one for both weight gradients.  A few tokens (a forecast step) take a kernel that streams
the weights once.

Like the column MLPs (:mod:`tornado_gcm_b200.ops.linear`) the layer computes in the BF16 zone: fp32 inputs and
master weights are rounded to BF16 on entry, and the gradients reach them through that cast.
"""

from __future__ import annotations

from typing import Optional

import torch

from tornado_gcm_b200.ops import _ext
from tornado_gcm_b200.ops.linear import ACT_CODES


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                 b_up: Optional[torch.Tensor] = None, *, activation: str = "silu") -> torch.Tensor:
    """``(…, F)`` from ``x (…, K)`` and the weights ``(F, K)``; ``activation`` one of ``ops.linear.ACT_CODES``.

    On the GPU the result is BF16 and so is the arithmetic's input, and only first derivatives in reverse mode are
    there (others are refused); on the CPU it has ``x``'s type.
    """
    act = ACT_CODES.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation must be one of {sorted(ACT_CODES)}, got {activation!r}")
    if x.is_cuda:
        return _ext.op("gated_linear")(x, w_gate, w_up, b_gate, b_up, act, _ext.error_flag(x.device))
    if w_gate.ndim != 2 or w_gate.shape != w_up.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"gated_linear: weights (hidden, features) that match x expected, got x {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    if (b_gate is None) != (b_up is None):
        raise ValueError("gated_linear: both biases or none")
    from tornado_gcm_b200.neural.standard_layers import apply_activation

    lin = torch.nn.functional.linear
    return apply_activation(activation, lin(x, w_gate, b_gate)) * lin(x, w_up, b_up)
