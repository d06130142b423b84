"""The sequence operators' CPU forms and the model built on them (no GPU)."""

import math

import pytest
import torch

from tornado_gcm_b200.models import sequence
from tornado_gcm_b200.neural.sequence_layers import SequenceTransformer, WindowSelfAttention
from tornado_gcm_b200.ops import accounting
from tornado_gcm_b200.ops.gated import gated_linear
from tornado_gcm_b200.ops.gradnorm import clip_grad_norm, grad_norm
from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table
from tornado_gcm_b200.ops.window_attention import (fill_window_cache, window_attention, window_attention_step,
                                                   window_mask)


def _randn(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=dtype)


def test_rotary_table_scalings_and_refusals():
    t = rotary_table(8, 6)
    assert t.shape == (8, 3, 2) and t.dtype == torch.float32
    ang = torch.arange(8.0, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.tensor([0.0, 2.0, 4.0]).double() / 6)
    assert torch.allclose(t.double(), torch.stack([ang.cos(), ang.sin()], -1), atol=1e-7)
    assert torch.equal(rotary_table(torch.arange(8) * 4, 6, scaling="linear", factor=4.0), t)
    b = rotary_table(8, 6, scaling="base", factor=3.0)  # the fastest pair stays, the slowest is three times slower
    assert torch.allclose(b[:, 0], t[:, 0]) and torch.allclose(
        torch.atan2(b[1:, -1, 1], b[1:, -1, 0]) * 3, torch.atan2(t[1:, -1, 1], t[1:, -1, 0]), rtol=1e-5)
    for bad in (dict(rotary_dim=5), dict(rotary_dim=0), dict(rotary_dim=4, scaling="cubic"), dict(rotary_dim=4, factor=0.0)):
        with pytest.raises(ValueError):
            rotary_table(8, **bad)


def test_qk_norm_rotary_preserves_lengths_and_relative_positions():
    q, k = _randn(2, 7, 3, 8, seed=1), _randn(2, 7, 1, 8, seed=2)
    t = rotary_table(100, 8).double()
    for inter in (False, True):
        a = qk_norm_rotary(q, k, t, norm="none", interleaved=inter)
        assert torch.allclose(a[0].norm(dim=-1), q.norm(dim=-1), atol=1e-6)
        b = qk_norm_rotary(q, k, t, norm="none", interleaved=inter, positions=torch.arange(7) + 60)
        dots = lambda y: torch.einsum("bihd,bjkd->bhij", y[0], y[1].expand(2, 7, 1, 8))  # noqa: E731
        assert torch.allclose(dots(a), dots(b), atol=1e-5)
    y = qk_norm_rotary(q, k, None, torch.full((8,), 2.0), None, torch.ones(8), None, norm="layer")[0]
    assert torch.allclose(y, torch.nn.functional.layer_norm(q, (8,), torch.full((8,), 2.0).double(), torch.ones(8).double()))


@pytest.mark.parametrize("causal", [True, False])
def test_window_attention_is_masked_attention(causal):
    q, k, v = _randn(2, 12, 4, 6, seed=1), _randn(2, 12, 2, 6, seed=2), _randn(2, 12, 2, 6, seed=3)
    L = torch.tensor([12, 5], dtype=torch.int32)
    o = window_attention(q, k, v, window=3, sinks=2, causal=causal, lengths=L)
    for b in range(2):
        for h in range(4):
            for i in range(12):
                see = [j for j in range(int(L[b])) if (abs(i - j) < 3 or j < 2) and (j <= i or not causal)]
                want = torch.zeros(6, dtype=torch.float64)
                if see:
                    p = torch.softmax(torch.stack([q[b, i, h] @ k[b, j, h // 2] for j in see]) / math.sqrt(6), 0)
                    want = sum(w * v[b, j, h // 2] for w, j in zip(p, see))
                assert torch.allclose(o[b, i, h], want, atol=1e-12)
    assert window_mask(12, 3, 2, causal, L).shape == (2, 12, 12)


def test_window_step_and_fill_on_the_cpu():
    window, sinks, steps = 4, 2, 15
    q, k, v = _randn(2, steps, 2, 6, seed=1, dtype=torch.float32), _randn(2, steps, 1, 6, seed=2, dtype=torch.float32), _randn(2, steps, 1, 6, seed=3, dtype=torch.float32)
    want = window_attention(q, k, v, window=window, sinks=sinks)
    kc, vc = torch.zeros(2, 6, 1, 6), torch.zeros(2, 6, 1, 6)
    for t in range(steps):
        n = torch.full((2,), t, dtype=torch.int32)
        o = window_attention_step(q[:, t], k[:, t], v[:, t], kc, vc, n, sinks=sinks)
        assert torch.allclose(o, want[:, t], atol=1e-6)
        kf, vf = torch.zeros_like(kc), torch.zeros_like(vc)
        fill_window_cache(k[:, : t + 1], v[:, : t + 1], kf, vf, sinks=sinks)
        assert torch.equal(kf, kc) and torch.equal(vf, vc)
    before = kc.clone()
    o = window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, torch.tensor([-1, steps], dtype=torch.int32), sinks=sinks)
    assert (o[0] == 0).all() and torch.equal(kc[0], before[0]) and not torch.equal(kc[1], before[1])
    with pytest.raises(ValueError):
        window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, torch.zeros(2, dtype=torch.int32), sinks=6)


def test_cpu_refusals():
    x, w = _randn(4, 6), _randn(8, 6, seed=1)
    for call in (lambda: gated_linear(x, w, w[:4]), lambda: gated_linear(x[:, :4], w, w),
                 lambda: gated_linear(x, w, w, w[:, 0]), lambda: gated_linear(x, w, w, activation="softplus"),
                 lambda: clip_grad_norm([x], -1.0), lambda: clip_grad_norm([x], 1.0, out=[w]),
                 lambda: clip_grad_norm([x, None], 1.0, out=[x, x]),
                 lambda: window_attention(x[None, None], x[None, None], x[None, None], window=0),
                 lambda: WindowSelfAttention(32, 3, 4), lambda: WindowSelfAttention(32, 4, 4, kv_heads=3)):
        with pytest.raises(ValueError):
            call()
    two_sided = WindowSelfAttention(32, 4, 4, causal=False)
    with pytest.raises(ValueError):
        two_sided.step(torch.zeros(1, 32), *two_sided.new_cache(1, "cpu", torch.float32), torch.zeros(1, dtype=torch.int32))


def test_clip_grad_norm_on_the_cpu_follows_torch():
    ts = [_randn(5, 3, seed=i, dtype=torch.float32).requires_grad_() for i in range(3)]
    for t in ts:
        t.grad = _randn(5, 3, seed=9, dtype=torch.float32)
    mine = [t.grad.clone() for t in ts]
    out = [torch.zeros(5, 3) for _ in ts]
    n = torch.nn.utils.clip_grad_norm_(ts, 0.3)
    assert torch.allclose(grad_norm(mine), n)
    assert torch.allclose(clip_grad_norm(mine, 0.3, out=out), n)
    assert all(torch.allclose(o, t.grad, rtol=1e-5) for o, t in zip(out, ts))
    assert torch.allclose(clip_grad_norm(mine, 0.3), n)
    assert all(torch.allclose(o, t.grad, rtol=1e-5) for o, t in zip(mine, ts))
    assert clip_grad_norm([None, None], 1.0) == 0


@pytest.mark.parametrize("norm,kv_heads", [("rms", 1), ("layer", 2), ("none", 2)])
def test_transformer_step_equals_whole_history(norm, kv_heads):
    torch.manual_seed(0)
    m = SequenceTransformer(32, 2, 2, 48, 5, kv_heads=kv_heads, sinks=2, norm=norm, max_positions=64)
    x = _randn(3, 20, 32, dtype=torch.float32)
    whole = m(x)
    cache = m.new_cache(3)
    got = torch.stack([m.step(x[:, t], cache) for t in range(20)], 1)
    assert torch.allclose(got, whole, atol=1e-5)
    half = m.new_cache(3)
    m(x[:, :12], cache=half)
    got = torch.stack([m.step(x[:, t], half) for t in range(12, 20)], 1)
    assert torch.allclose(got, whole[:, 12:], atol=1e-5) and (half.lengths == 20).all()


def test_padded_states_do_not_reach_the_loss():
    torch.manual_seed(0)
    m = sequence.SequenceEmulator(5, 3, statics=2, d_model=32, num_heads=2, num_layers=1, d_ff=40, window=6, max_positions=64)
    torch.nn.init.normal_(m.head.weight, std=0.1)
    states, static = sequence.synthetic_columns(2, 16, 5, 3)
    L = torch.tensor([16, 9], dtype=torch.int32)
    a = m.loss(states, static, L)
    a.backward()
    grads = [p.grad.clone() for p in m.parameters()]
    junk = states.clone()
    junk[1, 9:] = 7.0
    for p in m.parameters():
        p.grad = None
    b = m.loss(junk, static, L)
    b.backward()
    assert torch.allclose(a, b) and all(torch.allclose(x, p.grad, atol=1e-6) for x, p in zip(grads, m.parameters()))


def test_example_trains_and_forecasts():
    r = sequence.main(["--device", "cpu", "--steps", "21", "--batch", "2", "--length", "32", "--features", "4",
                       "--window", "8", "--layers", "1", "--width", "64", "--forecast", "12", "--lr", "3e-3"])
    assert r["losses"][-1] < 0.5 * r["losses"][0] and r["gap"] < 1e-5


def test_accounting_counts_the_backward_pass_of_native_nodes():
    x, w = torch.empty(10, 16), torch.empty(24, 16)
    assert accounting._flops("gated_linear", (x, w, w, None, None, 4)) == (4 * 10 * 24 * 16, "bf16")
    assert accounting._flops("gated_linear", (x.requires_grad_(), w, w, None, None, 4)) == (12 * 10 * 24 * 16, "bf16")
    q = torch.empty(1, 100, 2, 8, dtype=torch.bfloat16)
    assert accounting._flops("window_attention", (q, q, q, 10, 2, True, None, 1.0)) == (4 * 100 * 2 * 8 * 12, "bf16")
