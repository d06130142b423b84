"""A transformer that steps column states through time, next to the hybrid model.

Every sequence is one column (or region): ``statics`` tokens of time-independent fields first (orography, land mask,
latitude: the attention's sinks, in sight of every step), then one token for each 6-hour state.  The model predicts
the increment to the next state.  Training sees whole histories at once; a forecast keeps a ring cache of the window
and costs the same for every step, however long it runs.

    python -m tornado_gcm_b200.models.sequence --steps 50 --length 512 --forecast 40

trains on synthetic damped waves and compares the cached forecast with the whole-history form.
"""

from __future__ import annotations

import argparse
import math
import time
from typing import Optional

import torch
import torch.nn as nn

from tornado_gcm_b200.neural.sequence_layers import SequenceTransformer, WindowCache, without_padding
from tornado_gcm_b200.ops import _ext
from tornado_gcm_b200.ops.gradnorm import clip_grad_norm


class SequenceEmulator(nn.Module):
    def __init__(self, features: int, static_features: int, *, statics: int = 4, d_model: int = 384, num_heads: int = 6,
                 kv_heads: Optional[int] = None, num_layers: int = 4, d_ff: int = 1024, window: int = 120,
                 activation: str = "silu", norm: str = "rms", max_positions: int = 16384):
        super().__init__()
        self.features, self.statics, self.window = features, statics, window
        self.embed = nn.Linear(features, d_model)
        self.embed_static = nn.Linear(static_features, statics * d_model) if statics else None
        self.body = SequenceTransformer(d_model, num_heads, num_layers, d_ff, window, kv_heads=kv_heads, sinks=statics,
                                        activation=activation, norm=norm, max_positions=max_positions)
        self.head = nn.Linear(d_model, features)
        nn.init.zeros_(self.head.weight)
        nn.init.zeros_(self.head.bias)

    def _tokens(self, states: torch.Tensor, static: Optional[torch.Tensor]) -> torch.Tensor:
        x = self.embed(states)
        if self.embed_static is None:
            return x
        return torch.cat([self.embed_static(static).unflatten(-1, (self.statics, -1)), x], 1)

    def forward(self, states: torch.Tensor, static: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, cache: Optional[WindowCache] = None) -> torch.Tensor:
        """``states (B, T, features)`` and ``static (B, static_features)`` to the next state of every step.
        ``lengths`` int32 ``(B,)``: valid states of each sequence (negative: it takes no part), what lies behind is taken
        for zeros; ``cache`` takes the valid history in."""
        if lengths is not None:
            states = without_padding(states, lengths)
            lengths = torch.where(lengths < 0, lengths, lengths + self.statics)
        h = self.body(self._tokens(states, static), lengths, cache=cache)
        return states + self.head(h[:, self.statics:])

    def loss(self, states: torch.Tensor, static: Optional[torch.Tensor] = None,
             lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Mean squared error of the predicted next states, over the valid ones."""
        if lengths is not None:
            states = without_padding(states, lengths)
        err = (self(states[:, :-1], static, None if lengths is None else (lengths - 1).clamp(min=0))
               - states[:, 1:]).square().mean(-1)
        if lengths is None:
            return err.mean()
        on = torch.arange(err.shape[1], device=err.device) < (lengths - 1)[:, None]
        return (err * on).sum() / on.sum().clamp(min=1)

    @torch.no_grad()
    def forecast(self, states: torch.Tensor, static: Optional[torch.Tensor] = None, *, steps: int) -> torch.Tensor:
        """``(B, steps, features)``: the states that follow ``states (B, T, features)``, one cached step at a time.
        The tables of rotations grow to the forecast's length; what a kernel reported on the way is raised at the end."""
        if steps < 1:
            raise ValueError(f"forecast: at least one step expected, got {steps}")
        self.body.reserve(self.statics + states.shape[1] + steps - 1)
        cache = self.body.new_cache(states.shape[0], states.device)
        state = self(states, static, cache=cache)[:, -1]
        out = [state]
        for _ in range(steps - 1):
            state = state + self.head(self.body.step(self.embed(state), cache))
            out.append(state)
        _ext.check_error_flag(states.device)
        return torch.stack(out, 1)


def train_step(model: SequenceEmulator, optimizer: torch.optim.Optimizer, states: torch.Tensor,
               static: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
               max_grad_norm: float = 1.0, check_errors: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """One optimizer step; the loss and the gradients' norm before clipping, both 0-d device tensors.

    ``check_errors``: read the device error flag afterwards (one host synchronisation) and raise if a kernel's bounded
    wait ran out or a table's index was out of range since it was last read."""
    optimizer.zero_grad(set_to_none=True)
    loss = model.loss(states, static, lengths)
    loss.backward()
    norm = clip_grad_norm([p.grad for p in model.parameters()], max_grad_norm)
    optimizer.step()
    if check_errors:
        _ext.check_error_flag(states.device)
    return loss.detach(), norm


def synthetic_columns(batch: int, length: int, features: int, static_features: int, *, seed: int = 0,
                      device="cpu") -> tuple[torch.Tensor, torch.Tensor]:
    """Sums of damped waves whose frequencies depend on the column's static fields: ``(B, T, F)`` and ``(B, S)``."""
    g = torch.Generator().manual_seed(seed)
    static = torch.rand(batch, static_features, generator=g)
    t = torch.arange(length)[None, :, None]
    freq = 2 * math.pi / (8 + 40 * static[:, None, :1] + 4 * torch.arange(features)[None, None, :] / features)
    phase = 2 * math.pi * torch.rand(batch, 1, features, generator=g)
    states = torch.sin(freq * t + phase) * torch.exp(-t / (20.0 * length))
    return states.to(device), static.to(device)


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=512)
    ap.add_argument("--features", type=int, default=37)
    ap.add_argument("--window", type=int, default=120)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--width", type=int, default=384)
    ap.add_argument("--forecast", type=int, default=40)
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = SequenceEmulator(a.features, 3, d_model=a.width, num_heads=a.width // 64, num_layers=a.layers,
                             d_ff=8 * a.width // 3 // 8 * 8, window=a.window).to(a.device)
    opt = torch.optim.AdamW(model.parameters(), lr=a.lr, betas=(0.9, 0.95))
    states, static = synthetic_columns(a.batch, a.length + 1, a.features, 3, device=a.device)
    losses = []
    start = time.perf_counter()
    for i in range(a.steps):
        shown = i % 10 == 0 or i == a.steps - 1
        loss, norm = train_step(model, opt, states, static, check_errors=shown)
        if shown:
            losses.append(float(loss))
            print(f"step {i}: loss {losses[-1]:.3e}, gradient norm {float(norm):.3e}, "
                  f"{(time.perf_counter() - start) / (i + 1) * 1e3:.1f} ms a step")
    history = states[:, : a.length // 2]
    ahead = model.forecast(history, static, steps=a.forecast)
    with torch.no_grad():  # the same states through the whole-history form
        whole = model(torch.cat([history, ahead[:, :-1]], 1), static)[:, history.shape[1] - 1:]
    gap = float((ahead - whole).norm() / whole.norm())
    print(f"forecast of {a.forecast} steps: rms error {float((ahead - states[:, a.length // 2:][:, :a.forecast]).square().mean().sqrt()):.3e}, "
          f"cached against whole-history form {gap:.2e}")
    return {"losses": losses, "gap": gap}


if __name__ == "__main__":
    main()
