"""The sequence operators on the GPU where they are easily wrong: narrow windows and sharp scores, scores of minus
infinity, values that are not finite where they should not matter, derivatives that the operators do not have,
shared memory, capture in a graph, other streams and broadcast gradients.

Tolerances are those of ``test_sequence_ops.py``; where a third rounding to bf16 comes in the 2-norm of the error is
held to sqrt(3) * 1.7e-3 = 3e-3.
"""

import math

import pytest
import torch

from tests.test_sequence_ops import DEV, TOL, _attn64, _close, _gated_inputs, _qk64, _randn, _see
from tornado_gcm_b200.ops import _ext

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs CUDA")]

BF = torch.bfloat16


# ── precision ──────────────────────────────────────────────────────────────
@pytest.mark.parametrize("D", [64, 128, 30])
@pytest.mark.parametrize("S,window,sinks,causal,sharp", [
    (300, 2, 0, True, 1), (300, 2, 1, False, 1), (300, 3, 0, True, 1), (300, 3, 1, True, 4), (1000, 2, 0, False, 1),
    (1000, 3, 0, True, 4), (300, 200, 0, True, 4), (700, 64, 4, False, 4)])
def test_window_attention_gradients_of_few_or_sharp_weights(D, S, window, sinks, causal, sharp):
    """Two or three keys to a row, or weights close to one and zero: dP - delta cancels, whatever the sequence's length.
    Three roundings to bf16: of the weights in the forward product, of dS, and of the result."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    q, k, v = (_randn(2, S, h, D, seed=i, dtype=BF, scale=s).requires_grad_()
               for i, (h, s) in enumerate(((4, sharp), (2, 1), (2, 1))))
    do = _randn(2, S, 4, D, seed=5, dtype=BF)
    grads = torch.autograd.grad(window_attention(q, k, v, window=window, sinks=sinks, causal=causal), [q, k, v], do)
    r = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o64 = _attn64(*r, _see(S, window, sinks, causal, None, 2), D ** -0.5)
    for n, a, b in zip(("dq", "dk", "dv"), grads, torch.autograd.grad(o64, r, do.double())):
        _close(a, b, 3e-3, n)
    _ext.check_error_flag(DEV)


# ── what is not finite ─────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 30), (torch.float32, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_whose_every_score_is_minus_infinity_give_zeros(dtype, D, causal):
    from tornado_gcm_b200.ops.window_attention import window_attention, window_attention_step

    B, S = 1, 600
    q, k, v = (_randn(B, S, 1, D, seed=i, dtype=dtype) for i in range(3))
    k[..., 3] = 1.0
    cfg = dict(window=300, causal=causal)
    rows = torch.tensor([0, 5, 100, 130, 400, 599], device=DEV)
    q[:, rows] = 0.0
    want = window_attention(q, k, v, **cfg)
    q[:, rows, :, 3] = -math.inf
    got = window_attention(q, k, v, **cfg)
    assert (got[:, rows] == 0).all()
    others = torch.ones(S, dtype=torch.bool, device=DEV).index_fill_(0, rows, False)
    assert torch.equal(got[:, others], want[:, others])
    lengths = torch.full((B,), S - 1, dtype=torch.int32, device=DEV)
    o = window_attention_step(q[:, 5], k[:, 7], v[:, 7], k.clone(), v.clone(), lengths)
    assert (o == 0).all()


@pytest.mark.parametrize("T", [4, 300])
def test_gated_relu_keeps_nan(T):
    from tornado_gcm_b200.ops.gated import gated_linear

    ts = [t.requires_grad_() for t in _gated_inputs(T, 64, 96, True)]
    with torch.no_grad():
        ts[3][7] = math.nan
    h = gated_linear(*ts, activation="relu")
    bad = torch.zeros(96, dtype=torch.bool, device=DEV)
    bad[7] = True
    assert torch.equal(h.isnan(), bad.expand(T, 96))
    dwu = torch.autograd.grad(h, ts[2], torch.ones_like(h))[0]  # du = dh * act
    assert torch.equal(dwu.isnan(), bad[:, None].expand(96, 64))


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("H,Hk,D,R,S", [(5, 1, 64, 64, 30), (3, 2, 32, 16, 9), (1, 1, 16, 16, 70), (5, 3, 40, 20, 9)])
def test_qk_norm_rotary_without_epsilon(H, Hk, D, R, S, norm, dtype):
    """eps = 0 is sound where no head is constant; head counts that leave lanes of the last load idle."""
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    q, k = (_randn(2, S, h, D, seed=h, dtype=dtype).requires_grad_() for h in (H, Hk))
    w = [(1 + _randn(D, seed=s, scale=0.2)).requires_grad_() for s in (3, 4)]
    b = [_randn(D, seed=s).requires_grad_() for s in (5, 6)] if norm == "layer" else [None, None]
    table = rotary_table(S, R, device=DEV)
    y = qk_norm_rotary(q, k, table, *w, *b, norm=norm, eps=0.0)
    leaves = [t for t in (q, k, *w, *b) if t is not None]
    up = [_randn(*t.shape, seed=9, dtype=dtype) for t in y]
    grads = torch.autograd.grad(y, leaves, up)
    r = {id(t): t.detach().double().requires_grad_() for t in leaves}
    pos = torch.arange(S, device=DEV)
    y64 = [_qk64(r[id(x)], r[id(w[i])], r.get(id(b[i])), table, pos, norm, False, 0.0) for i, x in enumerate((q, k))]
    for a, c in zip(y, y64):
        _close(a, c, TOL[dtype])
    for i, (a, c) in enumerate(zip(grads, torch.autograd.grad(y64, list(r.values()), [u.double() for u in up]))):
        _close(a, c, TOL[a.dtype], f"gradient {i}")


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("D,R,inter", [(64, 32, False), (64, 32, True), (64, 30, True), (40, 20, False), (64, 0, False)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_values_outside_the_rotation_pass_as_they_are(D, R, inter, bad, dtype):
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    q = _randn(1, 5, 3, D, seed=1, dtype=dtype)
    q[0, 2, 1, R + 3] = bad
    q.requires_grad_()
    table = rotary_table(5, R, device=DEV) if R else None
    up = _randn(1, 5, 3, D, seed=2, dtype=dtype)
    up[0, 2, 1, R + 3] = bad
    y, _ = qk_norm_rotary(q, q.detach(), table, norm="none", interleaved=inter)
    (g,) = torch.autograd.grad(y, q, up)
    for a, src in ((y, q), (g, up)):
        odd = ~torch.isfinite(a)
        assert int(odd.sum()) == 1 and bool(odd[0, 2, 1, R + 3])
        assert torch.equal(a[..., R:].nan_to_num(9.0, 8.0), src.detach()[..., R:].nan_to_num(9.0, 8.0))


def test_padding_of_the_model_may_hold_anything():
    from tornado_gcm_b200.models import sequence

    torch.manual_seed(0)
    m = sequence.SequenceEmulator(9, 3, statics=2, d_model=128, num_heads=2, num_layers=2, d_ff=80, window=30,
                                  max_positions=256).to(DEV)
    torch.nn.init.normal_(m.head.weight, std=0.1)
    states, static = sequence.synthetic_columns(3, 150, 9, 3, device=DEV)
    L = torch.tensor([150, 70, 0], dtype=torch.int32, device=DEV)
    res = []
    for junk in (0.0, math.nan):
        s = states.clone()
        s[1, 70:], s[2] = junk, junk
        m.zero_grad()
        loss = m.loss(s, static, L)
        loss.backward()
        res.append([loss.detach()] + [p.grad.clone() for p in m.parameters()])
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(*res))


# ── derivatives ────────────────────────────────────────────────────────────
def _three():
    """The operators that have a backward pass: a call, its differentiable inputs."""
    from tornado_gcm_b200.ops.gated import gated_linear
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table
    from tornado_gcm_b200.ops.window_attention import window_attention

    table = rotary_table(40, 64, device=DEV)
    return {
        "gated": (lambda *t: (gated_linear(*t),), list(_gated_inputs(40, 64, 96, True))),
        "qk": (lambda q, k, w: qk_norm_rotary(q, k, table, w, norm="rms"),
               [_randn(2, 40, 4, 64, seed=1, dtype=BF), _randn(2, 40, 2, 64, seed=2, dtype=BF), 1 + _randn(64, seed=3, scale=0.1)]),
        "attn": (lambda q, k, v: (window_attention(q, k, v, window=9, sinks=1),),
                 [_randn(2, 40, h, 64, seed=h + i, dtype=BF) for i, h in enumerate((4, 2, 2))]),
        "attn fp32": (lambda q, k, v: (window_attention(q, k, v, window=9, sinks=1),),
                      [_randn(2, 40, h, 32, seed=h + i) for i, h in enumerate((4, 2, 2))]),
    }


NAMES = ["gated", "qk", "attn", "attn fp32"]


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name):
    call, ts = _three()[name]
    ts = [t.requires_grad_() for t in ts]
    ys = call(*ts)
    plain = torch.autograd.grad(ys, ts, [torch.ones_like(y) for y in ys], retain_graph=True)
    first = torch.autograd.grad(ys, ts, [torch.ones_like(y) for y in ys], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, first))  # the first derivative is there all the same
    for f in first:
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(f.float().square().sum(), ts, allow_unused=True, retain_graph=True)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
    import torch.autograd.forward_ad as fwAD

    call, ts = _three()[name]
    for i in range(len(ts)):
        with fwAD.dual_level(), torch.set_grad_enabled(grad):
            duals = [fwAD.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ts)]
            with pytest.raises(NotImplementedError, match="no forward-mode"):
                call(*duals)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_window_step_has_no_gradient_and_says_so(dtype):
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    base = [_randn(2, h, 32, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2))] + [
        torch.zeros(2, 6, 2, 32, dtype=dtype, device=DEV) for _ in range(2)]
    want = window_attention_step(*base, n)
    for i in range(5):
        ts = [t.clone().requires_grad_() if j == i else t.clone() for j, t in enumerate(base)]
        with pytest.raises(RuntimeError, match="no gradient"):
            window_attention_step(*ts, n)
        with torch.no_grad():
            assert torch.equal(window_attention_step(*ts, n), want)


def test_a_table_that_requires_a_gradient_is_refused():
    """The kernels have none for the table; on the CPU it can be learned."""
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    q = _randn(1, 6, 2, 32, seed=1)
    want = qk_norm_rotary(q, q, rotary_table(6, 32, device=DEV), norm="rms")
    table = rotary_table(6, 32, device=DEV).requires_grad_()
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="no gradient for the table"):
            qk_norm_rotary(x, x, table, norm="rms")
        with torch.no_grad():
            got = qk_norm_rotary(x, x, table, norm="rms")
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_writes_are_seen_by_autograd():
    """A value that a graph has saved and an operator then overwrites is an error, not a wrong gradient."""
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm
    from tornado_gcm_b200.ops.window_attention import window_attention, window_attention_step

    w = torch.ones((), device=DEV, requires_grad=True)
    q = _randn(2, 1, 32, seed=1)
    kc, vc = torch.zeros(2, 6, 1, 32, device=DEV), torch.zeros(2, 6, 1, 32, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    for cache in (kc, vc):
        y = (cache * w).sum()
        window_attention_step(q, q, q, kc, vc, n)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
    g, o = _randn(100, seed=2), torch.empty(100, device=DEV)
    y = (g * w).sum()
    clip_grad_norm([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    y = (o * w).sum()
    before = g._version
    clip_grad_norm([g], 0.1, out=[o])
    assert g._version == before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    a = _randn(2, 9, 1, 32, seed=3).requires_grad_()
    lengths = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    y = window_attention(a, a, a, window=3, lengths=lengths).sum()
    lengths -= 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_caches_whose_sequences_share_memory_are_refused():
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    q = _randn(3, 1, 32, seed=1)
    own, shared = torch.zeros(3, 6, 1, 32, device=DEV), torch.zeros(1, 6, 1, 32, device=DEV).expand(3, 6, 1, 32)
    n = torch.zeros(3, dtype=torch.int32, device=DEV)
    for kc, vc in ((shared, own), (own, shared)):
        with pytest.raises(RuntimeError, match="single memory location"):
            window_attention_step(q, q, q, kc, vc, n)


# ── the model's caches ─────────────────────────────────────────────────────
def _body():
    from tornado_gcm_b200.neural.sequence_layers import SequenceTransformer

    torch.manual_seed(0)
    return SequenceTransformer(128, 2, 2, 96, 40, kv_heads=1, sinks=3, max_positions=256).to(DEV)


def test_steps_behind_a_ragged_history():
    m = _body()
    x = _randn(4, 106, 128, seed=1)
    L = [100, 57, 2, 0]
    padded = x[:, :100].clone()
    for b, n in enumerate(L):
        padded[b, n:] = math.nan
    with torch.no_grad():
        cache = m.new_cache(4)
        m(padded, torch.tensor(L, dtype=torch.int32, device=DEV), cache=cache)
        got = torch.stack([m.step(x[:, 100 + t], cache) for t in range(6)], 1)
        for b, n in enumerate(L):
            whole = m(torch.cat([x[b:b + 1, :n], x[b:b + 1, 100:]], 1))[:, n:]
            _close(got[b:b + 1], whole, 1e-2)
    assert cache.lengths.tolist() == [n + 6 for n in L]
    _ext.check_error_flag(DEV)


def test_steps_behind_a_history_at_given_positions():
    m = _body()
    x = _randn(2, 30, 128, seed=1)
    pos = torch.stack([torch.arange(30) + 20, torch.arange(30) + 101]).to(DEV)
    with torch.no_grad():
        whole = m(x, None, pos)
        cache = m.new_cache(2)
        m(x[:, :24], None, pos[:, :24], cache=cache)
        got = torch.stack([m.step(x[:, 24 + t], cache) for t in range(6)], 1)
    _close(got, whole[:, 24:], 1e-2)


def test_forecast_past_the_table_of_positions():
    from tornado_gcm_b200.models import sequence

    res = []
    for rows in (20, 256):
        torch.manual_seed(0)
        m = sequence.SequenceEmulator(9, 3, statics=2, d_model=128, num_heads=2, num_layers=1, d_ff=80, window=12,
                                      max_positions=rows).to(DEV)
        torch.nn.init.normal_(m.head.weight, std=0.1)
        states, static = sequence.synthetic_columns(2, 16, 9, 3, device=DEV)
        res.append(m.forecast(states, static, steps=40))
    assert torch.equal(*res)
    _ext.check_error_flag(DEV)


# ── graphs, streams, broadcast gradients ───────────────────────────────────
def _pass(call, ts):
    ys = call(*ts)
    ups = [torch.linspace(-1, 1, y.numel(), device=DEV).to(y.dtype).view_as(y) for y in ys]
    grads = torch.autograd.grad(ys, ts, ups)
    return [y.detach() for y in ys] + list(grads)  # a graph kept alive would tie the capture to this stream


@pytest.mark.parametrize("name", NAMES)
def test_training_pass_in_a_graph_and_on_another_stream(name):
    call, ts = _three()[name]
    ts = [t.requires_grad_() for t in ts]
    want = _pass(call, ts)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _pass(call, ts)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = _pass(call, ts)
    with torch.no_grad():
        for t in ts:
            t.mul_(0.75)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(_pass(call, ts), captured))
    _ext.check_error_flag(DEV)


def test_wide_gated_pass_in_a_graph():
    """Sizes that split dW over the tokens, so every kernel of the pass is captured, with its place in the order."""
    from tornado_gcm_b200.ops.gated import gated_linear

    ts = [t.requires_grad_() for t in _gated_inputs(4096, 128, 264, True)]
    call = lambda *t: (gated_linear(*t, activation="gelu_tanh"),)  # noqa: E731
    _pass(call, ts)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = _pass(call, ts) + _pass(call, ts)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    want = _pass(call, ts)
    assert all(torch.equal(a, b) for a, b in zip(want + want, captured))
    _ext.check_error_flag(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_steps_in_a_graph_and_on_another_stream(dtype):
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    q, k, v = (_randn(3, h, 64, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    fresh = lambda: [torch.zeros(3, 12, 2, 64, dtype=dtype, device=DEV) for _ in range(2)]  # noqa: E731
    n = torch.tensor([0, 5, 30], dtype=torch.int32, device=DEV)

    def steps(kc, vc, n):
        outs = []
        for _ in range(4):
            outs.append(window_attention_step(q, k, v, kc, vc, n, sinks=2))
            n += 1
        return outs

    a, b, c = fresh(), fresh(), fresh()
    want = steps(*a, n.clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = steps(*b, n.clone())
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want + a, got + b))
    m = n.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = steps(*c, m)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want + a, captured + c)) and torch.equal(m, n + 4)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("axis", [0, 1])
def test_gradients_that_are_broadcast(name, axis):
    """A mean over tokens or sequences hands back a gradient with a stride of zero."""
    call, ts = _three()[name]
    ts = [t.requires_grad_() for t in ts]
    ys = call(*ts)
    ups = [_randn(*y.shape, seed=7, dtype=y.dtype).select(axis, 0).unsqueeze(axis) for y in ys]
    got = torch.autograd.grad(ys, ts, [u.expand_as(y) for u, y in zip(ups, ys)], retain_graph=True)
    want = torch.autograd.grad(ys, ts, [u.expand_as(y).contiguous() for u, y in zip(ups, ys)])
    for i, (a, b) in enumerate(zip(got, want)):
        _close(a, b, TOL[a.dtype], f"gradient {i}")
