"""Transformer layers for long sequences: time steps of a column or region, or the tokens of a grid.

The column transformer (:mod:`tornado_gcm_b200.neural.transformer_layers`) attends over the levels of one column,
a few dozen tokens without a mask.  Sequences of 6-hour steps or of grid points are thousands of tokens long; these
layers see a sliding window of them and the first ``sinks`` tokens (static fields, forcings), know positions by
rotation, may share key heads between query heads, and use a gated feed-forward block.  On the GPU everything between
the projections runs in this framework's kernels, in the BF16 zone with fp32 master weights:
``ops.rotary.qk_norm_rotary``, ``ops.window_attention`` and ``ops.gated.gated_linear``; the plain projections are
library products.  ``step`` runs the same block for one new token over a ring cache, for forecasts: no gradient goes
through it, nor through a cache.
"""

from __future__ import annotations

import dataclasses
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from tornado_gcm_b200.ops.gated import gated_linear
from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table
from tornado_gcm_b200.ops.window_attention import fill_window_cache, window_attention, window_attention_step


def _linear(x: torch.Tensor, lin: nn.Linear) -> torch.Tensor:
    """The layer in ``x``'s type (master weights are cast, gradients reach them through the cast)."""
    return F.linear(x, lin.weight.to(x.dtype), None if lin.bias is None else lin.bias.to(x.dtype))


def without_padding(x: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
    """``x (B, S, features)`` with zeros behind each sequence's end, whatever was there: a product with a weight of zero
    would carry NaN from it into gradients."""
    behind = torch.arange(x.shape[1], device=x.device) >= lengths.to(x.device)[:, None]
    return x.masked_fill(behind[..., None], 0.0)


def _zone(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.bfloat16) if x.is_cuda else x


@dataclasses.dataclass
class WindowCache:
    """Keys and values of the tokens in sight, one pair of ``(B, sinks + window, heads, head_dim)`` for each block,
    the number of tokens that every sequence has seen (int32 ``(B,)``; negative: it takes no part), the position of
    its next token (``(B,)``) where that is another number than its count, and the host's bound on positions: the next
    token of every sequence stands at ``reach`` or before it."""

    k: list
    v: list
    lengths: torch.Tensor
    positions: Optional[torch.Tensor] = None
    reach: int = 0


class WindowSelfAttention(nn.Module):
    """Causal or two-sided self-attention in a sliding window, with normalised and rotated queries and keys."""

    def __init__(self, d_model: int, num_heads: int, window: int, *, kv_heads: Optional[int] = None, sinks: int = 0,
                 causal: bool = True, norm: str = "rms", rotary_dim: Optional[int] = None, interleaved: bool = False,
                 max_positions: int = 16384, rotary_scaling: Optional[str] = None, rotary_factor: float = 1.0,
                 use_bias: bool = False):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if d_model % num_heads or num_heads % kv_heads:
            raise ValueError(f"{num_heads} heads must divide {d_model} features and be a multiple of {kv_heads} key heads")
        self.num_heads, self.kv_heads, self.head_dim = num_heads, kv_heads, d_model // num_heads
        self.window, self.sinks, self.causal, self.norm, self.interleaved = window, sinks, causal, norm, interleaved
        self.qkv = nn.Linear(d_model, (num_heads + 2 * kv_heads) * self.head_dim, bias=use_bias)
        self.out = nn.Linear(d_model, d_model, bias=use_bias)
        for lin in (self.qkv, self.out):
            nn.init.xavier_normal_(lin.weight)
        if norm != "none":
            self.q_weight, self.k_weight = (nn.Parameter(torch.ones(self.head_dim)) for _ in range(2))
        else:
            self.q_weight = self.k_weight = None
        if norm == "layer":
            self.q_bias, self.k_bias = (nn.Parameter(torch.zeros(self.head_dim)) for _ in range(2))
        else:
            self.q_bias = self.k_bias = None
        rotary_dim = self.head_dim // 2 * 2 if rotary_dim is None else rotary_dim
        self.rotary = dict(rotary_dim=rotary_dim, scaling=rotary_scaling, factor=rotary_factor)
        self.register_buffer("table", rotary_table(max_positions, **self.rotary) if rotary_dim else None, persistent=False)
        self._outgrown = []

    def reserve(self, positions: int) -> None:
        """Makes the table of rotations hold at least ``positions`` positions.  A CUDA graph captured before keeps the
        table that it was captured with."""
        if self.table is not None and positions > self.table.shape[0]:
            self._outgrown.append(self.table)  # captured graphs read it still
            self.table = rotary_table(max(positions, 2 * self.table.shape[0]), **self.rotary, device=self.table.device)

    def _heads(self, x: torch.Tensor, positions: Optional[torch.Tensor]):
        """``x (B, S, d_model)`` to rotated q and k and plain v, all ``(B, S, heads, head_dim)`` without copies of v."""
        H, Hk, D = self.num_heads, self.kv_heads, self.head_dim
        q, k, v = (t.unflatten(-1, (-1, D)) for t in _linear(x, self.qkv).split([H * D, Hk * D, Hk * D], -1))
        q, k = qk_norm_rotary(q, k, self.table, self.q_weight, self.k_weight, self.q_bias, self.k_bias, norm=self.norm,
                              interleaved=self.interleaved, positions=positions)
        return q, k, v

    def forward(self, x: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, cache: Optional[tuple] = None) -> torch.Tensor:
        """``x (B, S, d_model)``; ``lengths`` int32 ``(B,)``: valid tokens; ``cache``: a pair that takes the keys and
        values of this whole history's valid tokens."""
        q, k, v = self._heads(x, positions)
        if cache is not None:
            fill_window_cache(k, v, *cache, sinks=self.sinks, lengths=lengths)
        o = window_attention(q, k, v, window=self.window, sinks=self.sinks, causal=self.causal, lengths=lengths)
        return _linear(o.flatten(-2), self.out)

    @torch.no_grad()
    def step(self, x: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
             positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token ``x (B, d_model)`` behind ``lengths`` earlier ones, at ``positions (B,)`` or, without, at
        ``lengths``."""
        if not self.causal:
            raise ValueError("a two-sided window has no one-token form")
        positions = None if self.table is None else (lengths.clamp(min=0) if positions is None else positions)[:, None]
        q, k, v = (t[:, 0] for t in self._heads(x[:, None], positions))
        return _linear(window_attention_step(q, k, v, k_cache, v_cache, lengths, sinks=self.sinks).flatten(-2), self.out)

    def new_cache(self, batch: int, device, dtype) -> tuple:
        shape = (batch, self.sinks + self.window, self.kv_heads, self.head_dim)
        return torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape, device=device, dtype=dtype)


class GatedFeedForward(nn.Module):
    """``down(act(gate(x)) * up(x))``."""

    def __init__(self, d_model: int, d_ff: int, activation: str = "silu", use_bias: bool = False):
        super().__init__()
        self.activation = activation
        self.gate = nn.Linear(d_model, d_ff, bias=use_bias)
        self.up = nn.Linear(d_model, d_ff, bias=use_bias)
        self.down = nn.Linear(d_ff, d_model, bias=use_bias)
        for lin in (self.gate, self.up, self.down):
            nn.init.xavier_normal_(lin.weight)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, activation=self.activation)
        return _linear(h, self.down)


class SequenceBlock(nn.Module):
    """Pre-norm block: window attention, then the gated feed-forward; the residual stream is fp32."""

    def __init__(self, d_model: int, num_heads: int, d_ff: int, window: int, *, activation: str = "silu", **attention):
        super().__init__()
        self.ln1, self.ln2 = nn.LayerNorm(d_model), nn.LayerNorm(d_model)
        self.attn = WindowSelfAttention(d_model, num_heads, window, **attention)
        self.ffn = GatedFeedForward(d_model, d_ff, activation)

    def forward(self, x: torch.Tensor, lengths=None, positions=None, cache=None) -> torch.Tensor:
        x = x + self.attn(_zone(self.ln1(x)), lengths, positions, cache)
        return x + self.ffn(_zone(self.ln2(x)))

    @torch.no_grad()
    def step(self, x: torch.Tensor, k_cache, v_cache, lengths, positions=None) -> torch.Tensor:
        x = x + self.attn.step(_zone(self.ln1(x)), k_cache, v_cache, lengths, positions)
        return x + self.ffn(_zone(self.ln2(x)))


class SequenceTransformer(nn.Module):
    """A stack of :class:`SequenceBlock` with a final norm; ``(B, S, d_model)`` fp32 in and out."""

    def __init__(self, d_model: int, num_heads: int, num_layers: int, d_ff: int, window: int, **block):
        super().__init__()
        self.layers = nn.ModuleList(SequenceBlock(d_model, num_heads, d_ff, window, **block) for _ in range(num_layers))
        self.final_ln = nn.LayerNorm(d_model)

    def forward(self, x: torch.Tensor, lengths=None, positions=None, cache: Optional[WindowCache] = None) -> torch.Tensor:
        """``lengths`` int32 ``(B,)``: valid tokens of each sequence; what lies behind may hold anything and is taken
        for zeros.  ``cache`` takes the history in; with ``lengths`` each sequence's valid tokens only, so that its
        steps go on behind them (a negative length: the sequence takes no part).  ``positions``, ``(S,)`` or
        ``(B, S)``: those of the tokens; steps go on behind the last valid one (a sequence without tokens: at the
        first)."""
        if lengths is not None:
            x = without_padding(x, lengths)
        for i, layer in enumerate(self.layers):
            x = layer(x, lengths, positions, None if cache is None else (cache.k[i], cache.v[i]))
        if cache is not None:
            if lengths is None:
                cache.lengths.fill_(x.shape[1])
            else:
                cache.lengths.copy_(lengths.clamp(max=x.shape[1]))
            cache.positions, cache.reach = None, x.shape[1]
            if positions is not None and x.shape[1]:
                cache.reach = int(positions.max()) + 1
                at = positions.expand(x.shape[:2])
                last = at.gather(1, (cache.lengths.long() - 1).clamp(min=0)[:, None])[:, 0]
                cache.positions = last + (cache.lengths > 0)
        return self.final_ln(x)

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: WindowCache, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token ``(B, d_model)`` of every sequence; the cache takes it in.  ``positions (B,)``: where these tokens
        stand, if not right behind the last ones; later steps go on behind them.

        A token behind the table of rotations (``max_positions``; see :meth:`reserve`) is refused where the host can
        tell: positions given to a step, or steps replayed from a CUDA graph, are only seen by the kernel, which
        reports them through the device error flag (:func:`tornado_gcm_b200.ops._ext.check_error_flag`).
        """
        if positions is not None:
            cache.positions = positions.clone()
        elif (rows := self.positions()) is not None and cache.reach >= rows:
            raise IndexError(f"a token at position {cache.reach} of a table of {rows}: reserve() more positions first")
        for i, layer in enumerate(self.layers):
            x = layer.step(x, cache.k[i], cache.v[i], cache.lengths, cache.positions)
        if cache.positions is not None:
            cache.positions += cache.lengths >= 0
        cache.lengths += cache.lengths >= 0
        cache.reach += 1
        return self.final_ln(x)

    def positions(self) -> Optional[int]:
        """Positions that the tables of rotations hold; ``None`` without rotation."""
        tables = [layer.attn.table for layer in self.layers if layer.attn.table is not None]
        return min(t.shape[0] for t in tables) if tables else None

    def reserve(self, positions: int) -> None:
        """Makes every block's table of rotations hold at least ``positions`` positions."""
        for layer in self.layers:
            layer.attn.reserve(positions)

    def new_cache(self, batch: int, device=None) -> WindowCache:
        """An empty cache for ``batch`` sequences."""
        p = self.final_ln.weight
        device = p.device if device is None else torch.device(device)
        dtype = torch.bfloat16 if device.type == "cuda" else p.dtype
        pairs = [layer.attn.new_cache(batch, device, dtype) for layer in self.layers]
        return WindowCache([k for k, _ in pairs], [v for _, v in pairs],
                           torch.zeros(batch, dtype=torch.int32, device=device))
