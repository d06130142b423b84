"""Global gradient norm and clipping over a list of tensors (``csrc/gradnorm.cu``).

``norm = sqrt(Σ g²)`` over every gradient, ``g ← g · min(1, max_norm / (norm + 1e-6))`` — the rule of
``torch.nn.utils.clip_grad_norm_`` — in one read for the norm and one read and write for the result, whatever
the number of tensors.  The squares of 16 bytes of values are added in fp32 (in fp64 where they leave its range) and
from there on in fp64, in a fixed order, so the norm neither overflows nor depends on the run.  The calls have no
gradient; the tensors they write may not overlap each other or gradients still to be read.  Nothing synchronises with the host: the norm stays a 0-d device tensor, and a call can be
captured in a CUDA graph.

With ``out`` the clipped gradients go to other buffers of the same shapes: bf16 gradients can be widened to the
fp32 buffers of an optimizer, or gathered in one flat buffer, in the same pass.
"""

from __future__ import annotations

from typing import Iterable, Optional, Sequence

import torch

from tornado_gcm_b200.ops import _ext


def _plain_norm(grads) -> torch.Tensor:
    return torch.stack([g.detach().double().square().sum() for g in grads]).sum().sqrt().float()


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all ``grads`` (fp32, bf16 or fp64; one device) as a 0-d fp32 tensor."""
    grads = [g for g in grads if g is not None]
    if not grads:
        return torch.zeros(())
    if not grads[0].is_cuda:
        return _plain_norm(grads)
    return _ext.op("grad_norm")(grads)


def clip_grad_norm(grads: Iterable[torch.Tensor], max_norm: float,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Clips ``grads`` to a global norm of ``max_norm``, in place or into ``out``; returns the norm before.

    ``out`` has one dense tensor for each gradient, of its shape; bf16 gradients may have fp32 outputs and
    the other way round.  A norm that is infinite or NaN scales as the formula says (to zero or NaN).
    """
    if not float(max_norm) >= 0.0:
        raise ValueError(f"clip_grad_norm: max_norm must not be negative, got {max_norm}")
    if out is None:
        grads = out_list = [g for g in grads if g is not None]
    else:
        grads, out_list = list(grads), list(out)
        if len(out_list) != len(grads):
            raise ValueError(f"clip_grad_norm: {len(out_list)} outputs for {len(grads)} gradients")
        if any(g is None for g in grads):
            raise ValueError("clip_grad_norm: with `out` every gradient must be there")
    if not grads:
        return torch.zeros(())
    if grads[0].is_cuda:
        return _ext.op("clip_grad_norm")(grads, [] if out is None else out_list, float(max_norm))
    with torch.no_grad():
        for g, o in zip(grads, out_list):
            if g.shape != o.shape:
                raise ValueError("clip_grad_norm: an output has another shape than its gradient")
        norm = _plain_norm(grads)
        coef = torch.clamp(float(max_norm) / (norm + 1e-6), max=1.0)
        for g, o in zip(grads, out_list):
            o.copy_(g * coef.to(g.dtype) if g.dtype == torch.float64 else g.float() * coef)
        return norm
