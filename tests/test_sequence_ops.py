"""The sequence operators on the GPU against their definitions in fp64: gated linear layer, head norms with rotation,
window attention and its one-token step, gradient clipping.

Tolerances follow from the formats.  An fp32 result is a sum of n products accumulated in fp32: the relative error
of the whole output stays below 2e-5 at the sizes used.  A bf16 result is rounded once (half a unit in the 8th bit,
2^-9 at most, 1.7e-3 in the root mean square); where an operand of a second product is rounded to bf16 on the way
(softmax weights, their gradients, the gradients of the two projections) another 1.7e-3 comes in, so the 2-norm of
the error is held to 4e-3 of the result's, 1.6 times the 2.4e-3 that the two roundings give.
"""

import math

import pytest
import torch

from tornado_gcm_b200.ops import _ext

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs CUDA")]

DEV = "cuda"
TOL = {torch.float32: 2e-5, torch.bfloat16: 4e-3}


def _randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(DEV)


def _close(a, b, tol, what=""):
    a, b = a.detach().double(), b.detach().double()
    assert a.shape == b.shape, (what, a.shape, b.shape)
    assert torch.isfinite(a).all(), what
    err, ref = float((a - b).norm()), float(b.norm())
    assert err <= tol * ref + 1e-30, (what, err / (ref + 1e-30))


# ── gated linear layer ─────────────────────────────────────────────────────
def _act64(name, z):
    F = torch.nn.functional
    return {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu, "tanh": torch.tanh,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[name](z)


def _gated_inputs(T, K, Fh, bias, seed=0):
    bf = torch.bfloat16
    x, wg, wu = (_randn(*s, seed=seed + i, dtype=bf, scale=c)
                 for i, (s, c) in enumerate([((T, K), 1.0), ((Fh, K), K ** -0.5), ((Fh, K), K ** -0.5)]))
    b = [_randn(Fh, seed=seed + 5 + i, dtype=bf, scale=0.3) if bias else None for i in range(2)]
    return x, wg, wu, b[0], b[1]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu", "relu", "tanh", "none"])
@pytest.mark.parametrize("T,K,F,bias", [(300, 136, 264, True), (5, 72, 40, True)])
def test_gated_linear_activations(T, K, F, bias, act):
    from tornado_gcm_b200.ops.gated import gated_linear

    _check_gated(gated_linear, T, K, F, bias, act)


@pytest.mark.parametrize("T,K,F,bias", [
    (1, 8, 8, False), (1, 1024, 512, True), (2, 64, 100, True), (3, 200, 33, False), (8, 384, 1000, True),
    (9, 64, 128, False), (17, 64, 129, True), (128, 64, 128, False), (129, 72, 136, True), (255, 384, 384, False),
    (257, 40, 264, True), (513, 264, 520, True), (1000, 520, 257, True), (2049, 384, 1000, True),
    (300, 37, 65, True), (1, 37, 5, True), (4096, 128, 256, False), (70, 1024, 640, False)])
def test_gated_linear_shapes(T, K, F, bias):
    from tornado_gcm_b200.ops.gated import gated_linear

    _check_gated(gated_linear, T, K, F, bias, "silu")


def _check_gated(gated_linear, T, K, F, bias, act):
    ts = _gated_inputs(T, K, F, bias)
    leaves = [t.requires_grad_() for t in ts if t is not None]
    dh = _randn(T, F, seed=9, dtype=torch.bfloat16)
    with torch.no_grad():
        h0 = gated_linear(*ts, activation=act)
    h = gated_linear(*ts, activation=act)
    grads = torch.autograd.grad(h, leaves, dh)
    assert torch.equal(h0, h)
    ref = [t.detach().double().requires_grad_() if t is not None else None for t in ts]
    lin = torch.nn.functional.linear
    h64 = _act64(act, lin(ref[0], ref[1], ref[3])) * lin(ref[0], ref[2], ref[4])
    g64 = torch.autograd.grad(h64, [t for t in ref if t is not None], dh.double())
    _close(h, h64, TOL[torch.bfloat16], "h")
    for i, (a, b) in enumerate(zip(grads, g64)):
        assert a.dtype == torch.bfloat16
        _close(a, b, TOL[torch.bfloat16], f"gradient {i}")
    _ext.check_error_flag(DEV)


def test_gated_linear_strided_and_batched_inputs():
    from tornado_gcm_b200.ops.gated import gated_linear

    x, wg, wu, bg, bu = _gated_inputs(192, 64, 96, True)
    wide = _randn(192, 200, seed=3, dtype=torch.bfloat16)
    for v in (wide[:, 8:72], wide[:, 3:67], x.t().contiguous().t(), x[:1].expand(192, 64)):
        _close(gated_linear(v, wg, wu, bg, bu), gated_linear(v.contiguous(), wg, wu, bg, bu), 1e-7)
    both = torch.cat([wg, wu])  # halves of one packed weight
    _close(gated_linear(x, both[:96], both[96:], bg, bu), gated_linear(x, wg, wu, bg, bu), 1e-7)
    y = gated_linear(x.reshape(4, 48, 64), wg, wu, bg, bu)
    assert y.shape == (4, 48, 96) and torch.equal(y.reshape(192, 96), gated_linear(x, wg, wu, bg, bu))
    assert gated_linear(x[:0], wg, wu, bg, bu).shape == (0, 96)
    # gradients of a broadcast input and a strided upstream gradient
    row = x[:1].detach().clone().requires_grad_()
    h = gated_linear(row.expand(192, 64), wg, wu, bg, bu)
    up = _randn(96, 192, seed=4, dtype=torch.bfloat16).t()
    (g,) = torch.autograd.grad(h, row, up)
    r64 = row.detach().double().requires_grad_()
    lin = torch.nn.functional.linear
    h64 = torch.nn.functional.silu(lin(r64.expand(192, 64), wg.double(), bg.double())) * lin(
        r64.expand(192, 64), wu.double(), bu.double())
    (g64,) = torch.autograd.grad(h64, r64, up.double())
    _close(g, g64, 2e-2)  # the 192 rows' gradients are bf16 and add up outside the operator


def test_gated_linear_gradient_against_differences():
    """Directional derivative of sum(h * dh) along random directions of every input, by central differences in fp64."""
    from tornado_gcm_b200.ops.gated import gated_linear

    ts = [t.requires_grad_() for t in _gated_inputs(64, 48, 80, True, seed=20)]
    dh = _randn(64, 80, seed=30, dtype=torch.bfloat16)
    grads = torch.autograd.grad(gated_linear(*ts, activation="gelu_tanh"), ts, dh)

    def f(v):
        lin = torch.nn.functional.linear
        return float((_act64("gelu_tanh", lin(v[0], v[1], v[3])) * lin(v[0], v[2], v[4]) * dh.double()).sum())

    base = [t.detach().double() for t in ts]
    for i in range(5):
        d = grads[i].double().sign()  # along the gradient's signs: no cancellation
        e = 1e-5
        hi, lo = ([b + s * e * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
        num, ana = (f(hi) - f(lo)) / (2 * e), float((grads[i].double() * d).sum())
        assert abs(num - ana) <= 4e-3 * abs(num), (i, num, ana)


def test_gated_linear_fp32_master_weights():
    from tornado_gcm_b200.ops.gated import gated_linear

    w = [_randn(40, 24, seed=i, scale=0.2).requires_grad_() for i in range(2)]
    x = _randn(30, 24, seed=7).requires_grad_()
    h = gated_linear(x, *w)
    assert h.dtype == torch.bfloat16
    g = torch.autograd.grad(h, [x, *w], torch.ones_like(h))
    assert all(t.dtype == torch.float32 for t in g)


def test_gated_linear_refusals():
    from tornado_gcm_b200.ops.gated import gated_linear

    x, wg, wu, bg, bu = _gated_inputs(4, 16, 24, True)
    with pytest.raises(ValueError):
        gated_linear(x, wg, wu, activation="step")
    with pytest.raises(ValueError):
        gated_linear(x, wg, wu[:8])
    with pytest.raises(ValueError):
        gated_linear(x[:, :8], wg, wu)
    with pytest.raises(ValueError):
        gated_linear(x, wg, wu, bg)
    with pytest.raises(RuntimeError, match="biases"):
        gated_linear(x, wg, wu, bg[:3], bu)
    with pytest.raises(RuntimeError, match="one device"):
        gated_linear(x, wg.cpu(), wu)


# ── head norms and rotation ────────────────────────────────────────────────
def _qk64(x, w, b, table, positions, norm, inter, eps):
    y = x
    if norm == "layer":
        y = y - y.mean(-1, keepdim=True)
    if norm != "none":
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    if table is None:
        return y
    cs = table.double()[positions.long()]
    cs = (cs[None] if cs.ndim == 3 else cs)[:, :, None]
    n = cs.shape[-2]
    i = torch.arange(n, device=y.device)
    a, c = (2 * i, 2 * i + 1) if inter else (i, i + n)
    out = y.clone()
    out[..., a] = y[..., a] * cs[..., 0] - y[..., c] * cs[..., 1]
    out[..., c] = y[..., c] * cs[..., 0] + y[..., a] * cs[..., 1]
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,Hk,D,R,norm,inter", [
    (2, 37, 6, 2, 64, 64, "layer", False), (2, 37, 6, 2, 64, 32, "rms", True), (1, 1, 1, 1, 16, 16, "layer", False),
    (3, 5, 3, 3, 40, 20, "layer", True), (3, 5, 3, 3, 40, 20, "rms", False), (1, 130, 5, 1, 128, 128, "rms", False),
    (2, 9, 4, 4, 80, 40, "none", False), (2, 9, 4, 1, 24, 10, "layer", False), (1, 7, 2, 2, 256, 256, "layer", False),
    (2, 3, 2, 1, 13, 6, "layer", False), (2, 3, 2, 1, 7, 2, "rms", True), (2, 300, 8, 8, 32, 0, "layer", False),
    (1, 4, 16, 4, 96, 96, "rms", True), (5, 1, 16, 4, 64, 64, "layer", False), (1, 2, 1, 1, 1, 0, "rms", False)])
def test_qk_norm_rotary(B, S, H, Hk, D, R, norm, inter, dtype):
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    rows = _randn(B, S, (H + 2 * Hk) * D, seed=1, dtype=dtype, scale=2.0) + 0.5
    q = rows[..., :H * D].unflatten(-1, (H, D)).detach().requires_grad_()  # views of a packed projection
    k = rows[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)).detach().requires_grad_()
    par = [None] * 4
    if norm != "none":
        par[0], par[1] = ((1 + _randn(D, seed=s, scale=0.2)).requires_grad_() for s in (3, 4))
    if norm == "layer":
        par[2], par[3] = _randn(D, seed=5).requires_grad_(), _randn(D, seed=6).requires_grad_()
    table = rotary_table(S + 10, R, device=DEV) if R else None
    pos = torch.stack([torch.arange(S) + 3 * b % 10 for b in range(B)]).to(DEV)
    yq, yk = qk_norm_rotary(q, k, table, *par, norm=norm, interleaved=inter, positions=pos)
    gq, gk = _randn(B, S, H, D, seed=7, dtype=dtype), _randn(B, S, Hk, D, seed=8, dtype=dtype)
    leaves = [q, k] + [t for t in par if t is not None]
    grads = torch.autograd.grad([yq, yk], leaves, [gq, gk])
    with torch.no_grad():
        y2 = qk_norm_rotary(q, k, table, *par, norm=norm, interleaved=inter, positions=pos)
    assert torch.equal(y2[0], yq) and torch.equal(y2[1], yk)
    r = {id(t): t.detach().double().requires_grad_() for t in leaves}
    get = lambda t: None if t is None else r[id(t)]  # noqa: E731
    e = [_qk64(r[id(x)], get(w), get(b), table, pos, norm, inter, 1e-5) for x, w, b in ((q, par[0], par[2]), (k, par[1], par[3]))]
    g64 = torch.autograd.grad(e, [r[id(t)] for t in leaves], [gq.double(), gk.double()])
    for a, b, n in zip((yq, yk), e, "qk"):
        _close(a, b, TOL[dtype], n)
    for i, (a, b) in enumerate(zip(grads, g64)):
        if D == 1 and i < 2:
            continue  # one value normalised by itself: the gradient is eps's alone, a difference of equal numbers
        assert a.dtype == leaves[i].dtype
        _close(a, b, TOL[a.dtype], f"gradient {i}")
    _ext.check_error_flag(DEV)


def test_qk_norm_rotary_positions_and_types():
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    q, k = _randn(2, 6, 2, 32, seed=1), _randn(2, 6, 1, 32, seed=2)
    t = rotary_table(64, 32, device=DEV)
    a = qk_norm_rotary(q, k, t)
    for pos in (torch.arange(6, device=DEV), torch.arange(6, device=DEV, dtype=torch.int32),
                torch.arange(6, device=DEV).expand(2, 6), torch.arange(0, 12, device=DEV)[::2] // 2):
        b = qk_norm_rotary(q, k, t, positions=pos)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a position outside the table is reported and clamped
    qk_norm_rotary(q, k, t, positions=torch.full((6,), 64, device=DEV))
    with pytest.raises(RuntimeError, match="out of bounds"):
        _ext.check_error_flag(DEV)
    # shifting every position leaves the products of rotated heads alone
    u = qk_norm_rotary(q, k, t, positions=torch.arange(6, device=DEV) + 50)
    dots = lambda y: torch.einsum("bihd,bjkd->bhij", y[0].double(), y[1].double().expand(2, 6, 1, 32))  # noqa: E731
    _close(dots(u), dots(a), 1e-5)


def test_qk_norm_rotary_refusals():
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table

    q, k = _randn(2, 6, 2, 32, seed=1), _randn(2, 6, 1, 32, seed=2)
    t = rotary_table(6, 32, device=DEV)
    with pytest.raises(ValueError):
        qk_norm_rotary(q, k, t, norm="batch")
    with pytest.raises(ValueError):
        qk_norm_rotary(q, k, t, torch.ones(32, device=DEV), norm="none")
    for bad in (dict(k=k.bfloat16()), dict(k=k[:1]), dict(k=k[..., :16]), dict(table=t[:5]), dict(table=t.double()),
                dict(table=rotary_table(6, 64, device=DEV)), dict(positions=torch.zeros(5, device=DEV, dtype=torch.int32)),
                dict(positions=torch.zeros(6, device=DEV)), dict(q_weight=torch.ones(16, device=DEV))):
        a = dict(dict(q=q, k=k, table=t), **bad)
        with pytest.raises(RuntimeError, match="qk_norm_rotary"):
            qk_norm_rotary(**a)


# ── window attention ───────────────────────────────────────────────────────
def _see(S, window, sinks, causal, lengths, B):
    i, j = torch.arange(S, device=DEV)[:, None], torch.arange(S, device=DEV)
    see = ((i - j).abs() < window) | (j < sinks)
    if causal:
        see = see & (j <= i)
    L = torch.full((B,), S, device=DEV) if lengths is None else lengths.long()
    return see[None] & (j < L[:, None, None])


def _attn64(q, k, v, see, scale):
    n = q.shape[2] // k.shape[2]
    qh, kh, vh = (t.transpose(1, 2) for t in (q, k.repeat_interleave(n, 2), v.repeat_interleave(n, 2)))
    s = (qh @ kh.transpose(-1, -2) * scale).masked_fill(~see[:, None], -math.inf)
    dead = ~see.any(-1)[:, None, :, None]
    p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
    return (p @ vh).transpose(1, 2)


ATTN = [  # B, S, H, Hk, D, window, sinks, causal, lengths
    (1, 1, 1, 1, 64, 1, 0, True, None), (2, 7, 2, 1, 64, 3, 0, True, None), (1, 128, 2, 2, 64, 128, 0, True, None),
    (1, 129, 2, 2, 64, 64, 1, True, None), (2, 300, 4, 2, 64, 100, 4, True, None),
    (1, 300, 4, 1, 128, 50, 3, False, None), (2, 513, 2, 2, 64, 200, 17, False, (513, 130)),
    (3, 260, 2, 1, 64, 40, 2, True, (0, 1, 260)), (2, 400, 2, 2, 32, 33, 0, False, (399, 40)),
    (1, 700, 6, 2, 64, 130, 140, True, None), (1, 700, 3, 1, 128, 1, 0, False, None),
    (2, 257, 2, 2, 16, 300, 0, True, None), (1, 384, 2, 2, 80, 128, 129, False, (200,)),
    (2, 65, 2, 1, 13, 20, 3, True, (65, 30)), (1, 1100, 4, 4, 64, 256, 5, True, None),
    (1, 900, 2, 1, 96, 77, 0, True, (850,)), (1, 520, 8, 1, 64, 90, 300, True, None), (2, 200, 2, 2, 24, 64, 64, True, (7, 150)),
    # sinks ahead of the queries that see them, beyond their window
    (1, 600, 2, 1, 64, 20, 300, False, None), (2, 230, 2, 2, 128, 100, 200, False, (230, 180)), (1, 200, 1, 1, 64, 1, 200, False, None),
    (1, 640, 2, 2, 128, 500, 1, True, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,Hk,D,window,sinks,causal,lengths", ATTN)
def test_window_attention(B, S, H, Hk, D, window, sinks, causal, lengths, dtype):
    from tornado_gcm_b200.ops.window_attention import window_attention

    q, k, v = (_randn(B, S, h, D, seed=i, dtype=dtype).requires_grad_() for i, h in enumerate((H, Hk, Hk)))
    do = _randn(B, S, H, D, seed=5, dtype=dtype)
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    cfg = dict(window=window, sinks=sinks, causal=causal, lengths=L)
    o = window_attention(q, k, v, **cfg)
    grads = torch.autograd.grad(o, [q, k, v], do)
    again = torch.autograd.grad(window_attention(q, k, v, **cfg), [q, k, v], do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))  # the same bits every time
    r = [t.detach().double().requires_grad_() for t in (q, k, v)]
    see = _see(S, window, sinks, causal, L, B)
    o64 = _attn64(*r, see, D ** -0.5)
    g64 = torch.autograd.grad(o64, r, do.double())
    _close(o, o64, TOL[dtype], "o")
    assert (o.transpose(1, 2)[~see.any(-1)[:, None].expand(B, H, S)] == 0).all()  # rows that see nothing
    for n, a, b in zip(("dq", "dk", "dv"), grads, g64):
        # a softmax over one key has no gradient: what is left of ds is the rounding of equal numbers
        if float(b.norm()) < 1e-6 * float(do.double().norm()):
            assert float(a.double().norm()) <= 1e-2 * float(do.double().norm()), n
            continue
        _close(a, b, TOL[dtype], n)
    _ext.check_error_flag(DEV)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 32)])
def test_window_attention_keys_behind_the_end_may_hold_anything(dtype, D):
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, S, H = 3, 300, 2
    L = torch.tensor([300, 140, 0], dtype=torch.int32, device=DEV)
    q, k, v = (_randn(B, S, H, D, seed=i, dtype=dtype) for i in range(3))
    do = _randn(B, S, H, D, seed=5, dtype=dtype)
    out = []
    for junk in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kk, vv = k.clone(), v.clone()
        for b in range(B):
            kk[b, int(L[b]):], vv[b, int(L[b]):] = junk, junk
        a = [t.requires_grad_() for t in (q.clone(), kk, vv)]
        o = window_attention(*a, window=70, sinks=3, lengths=L)
        out.append([o, *torch.autograd.grad(o, a, do)])
    for other in out[1:]:
        for a, b in zip(out[0], other):
            assert torch.isfinite(b).all() and torch.equal(a, b)
    assert (out[0][0][2] == 0).all() and (out[0][2][2] == 0).all()
    assert (out[0][3][1, 140:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_attention_large_scores_and_strides(dtype):
    """Scores of several hundred in both directions, and operands that are slices of one packed projection."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, S, H, Hk, D = 2, 260, 4, 2, 64
    rows = _randn(B, S, (H + 2 * Hk) * D, seed=1, dtype=dtype, scale=6.0)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in rows.split([H * D, Hk * D, Hk * D], -1))
    o = window_attention(q, k, v, window=90, sinks=2)
    assert torch.equal(o, window_attention(q.contiguous(), k.contiguous(), v.contiguous(), window=90, sinks=2))
    o64 = _attn64(q.double(), k.double(), v.double(), _see(S, 90, 2, True, None, B), D ** -0.5)
    # fp32: a score near 300 carries an error of 300 * 2^-23 or so into its exponential
    _close(o, o64, {torch.float32: 2e-4, torch.bfloat16: 4e-3}[dtype])
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(o, window_attention(heads_first, k, v, window=90, sinks=2))
    shifted = torch.empty(B * S * H * D + 1, dtype=dtype, device=DEV)[1:].view(B, S, H, D).copy_(q)  # off 16 bytes
    _close(window_attention(shifted, k, v, window=90, sinks=2), o, TOL[dtype])


def test_window_attention_on_another_stream_and_in_a_graph():
    from tornado_gcm_b200.ops.window_attention import window_attention

    q, k, v = (_randn(1, 400, 2, 64, seed=i, dtype=torch.bfloat16) for i in range(3))
    want = window_attention(q, k, v, window=99, sinks=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = window_attention(q, k, v, window=99, sinks=1)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = window_attention(q, k, v, window=99, sinks=1)
    k.add_(1.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, window_attention(q, k, v, window=99, sinks=1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 72, 128, 30])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_window_attention_passes_on_what_is_not_finite(dtype, D, causal, bad):
    """One key holds NaN, or an infinity in one component: the queries that get a NaN or plus infinity for a score
    give NaN, all others what they would give anyway.  The key stands at another place of its tile in every batch."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, S, H, W = 64, 200, 1, 90
    q, k, v = (_randn(B, S, H, D, seed=i, dtype=dtype) for i in range(3))
    b = torch.arange(B, device=DEV)
    k[b, 64 + b, 0, 3] = 0.0
    sound = window_attention(q, k, v, window=W, causal=causal)
    k[b, 64 + b, 0, 3] = bad
    got = window_attention(q, k, v, window=W, causal=causal)
    i, j = torch.arange(S, device=DEV)[None], (64 + b)[:, None]
    see = ((i - j) < W) & (i >= j) if causal else (i - j).abs() < W
    hit = see if bad != bad else see & (q[:, :, 0, 3] > 0)
    assert torch.equal(got.isnan().all(-1)[..., 0], hit)
    assert torch.equal(got.isnan().any(-1)[..., 0], hit)
    apart = ~see[..., None, None].expand_as(got)
    assert torch.equal(got[apart], sound[apart])
    qg, kg, vg = (t.clone().requires_grad_() for t in (q, k, v))
    dq, _, dv = torch.autograd.grad(window_attention(qg, kg, vg, window=W, causal=causal), [qg, kg, vg],
                                    torch.ones_like(q))
    assert dq[hit].isnan().all()
    seen = torch.stack([torch.zeros(S, dtype=torch.bool, device=DEV)] * B)
    for n in range(S):  # keys that a query with NaN for a result sees
        far = ((i - n) < W) & (i >= n) if causal else (i - n).abs() < W
        seen[:, n] = (hit & far).any(-1)
    assert dv[seen].isnan().all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 30),
                                     (torch.float32, 32)])
@pytest.mark.parametrize("S,window,sinks,causal,length", [
    (300, 1, 0, True, None), (300, 1, 0, False, None), (300, 7, 0, True, 1), (300, 400, 1, False, 1),
    (700, 3, 1, True, 1), (1, 5, 2, True, None), (40, 1, 0, False, None)])
def test_window_attention_one_key_has_no_score_gradient(dtype, D, S, window, sinks, causal, length):
    """Where every query sees one key or none its weight is 1 whatever the score: dq and dk are zeros, dv sums dO."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, H, Hk = 2, 4, 2
    q, k, v, g = (_randn(B, S, h, D, seed=i, dtype=dtype).requires_grad_() for i, h in enumerate((H, Hk, Hk, H)))
    n = None if length is None else torch.full((B,), length, dtype=torch.int32, device=DEV)
    o = window_attention(q, k, v, window=window, sinks=sinks, causal=causal, lengths=n)
    dq, dk, dv = torch.autograd.grad(o, [q, k, v], g)
    assert not dq.any() and not dk.any()
    i, j = torch.arange(S, device=DEV)[:, None], torch.arange(S, device=DEV)[None]
    see = (j < (S if length is None else length)) & (((i - j).abs() < window) | (j < sinks))
    if causal:
        see &= i >= j
    assert (see.sum(1) <= 1).all()
    want = torch.einsum("ij,bihd->bjhd", see.double(), g.detach().double().view(B, S, Hk, H // Hk, D).sum(3))
    # weights of 1 within an ulp or two of fp32; one rounding of the result
    _close(dv, want, 4e-3 if dtype == torch.bfloat16 else 2e-6, "dv")


@pytest.mark.parametrize("scale", [0.0, -0.125, float("inf"), float("nan"), 1e-60])
def test_window_attention_scale_refusals(scale):
    from tornado_gcm_b200.ops.window_attention import window_attention, window_attention_step

    q = torch.zeros(1, 4, 1, 64, device=DEV)
    with pytest.raises((RuntimeError, ValueError), match="scale must be positive and finite"):
        window_attention(q, q, q, window=2, scale=scale)
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises((RuntimeError, ValueError), match="scale must be positive and finite"):
        window_attention_step(q[:, 0], q[:, 0], q[:, 0], q.clone(), q.clone(), n, scale=scale)


def test_window_attention_refusals():
    from tornado_gcm_b200.ops.window_attention import window_attention

    q, k, v = (_randn(2, 9, h, 16, seed=i) for i, h in enumerate((4, 2, 2)))
    for bad in (dict(window=0), dict(window=2, sinks=-1)):
        with pytest.raises(ValueError):
            window_attention(q, k, v, **bad)
    L = torch.tensor([9, 9], device=DEV, dtype=torch.int32)
    for a in ((q[:, :, :3], k, v), (q, k, v[:, :5]), (q, k.bfloat16(), v), (q[..., :8], k, v), (q[0], k, v),
              (q.half(), k.half(), v.half())):
        with pytest.raises(RuntimeError, match="window_attention"):
            window_attention(*a, window=3)
    for bad in (L.long(), L[:1], L.cpu()):
        with pytest.raises(RuntimeError, match="lengths"):
            window_attention(q, k, v, window=3, lengths=bad)
    with pytest.raises(RuntimeError, match="head_dim"):
        window_attention(*(torch.zeros(1, 4, 1, 136, device=DEV) for _ in range(3)), window=3)


# ── one token over the cache ───────────────────────────────────────────────
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hk,D,window,sinks,steps", [(4, 2, 64, 6, 2, 20), (1, 1, 16, 1, 0, 4), (6, 2, 40, 5, 1, 17),
                                                       (8, 1, 128, 9, 0, 25), (2, 2, 13, 4, 3, 12), (10, 2, 64, 7, 1, 9)])
def test_window_step_equals_the_sequence_form(H, Hk, D, window, sinks, steps, dtype):
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    B = 3
    q, k, v = (_randn(B, steps, h, D, seed=i, dtype=dtype) for i, h in enumerate((H, Hk, Hk)))
    want = _attn64(q.double(), k.double(), v.double(), _see(steps, window, sinks, True, None, B), D ** -0.5)
    kc = torch.full((B, window + sinks, Hk, D), float("nan"), dtype=dtype, device=DEV)  # empty slots are never read
    vc = kc.clone()
    n = torch.zeros(B, dtype=torch.int32, device=DEV)
    for t in range(steps):
        for _ in range(2):  # a repeated call with the same lengths writes the same slots
            o = window_attention_step(q[:, t], k[:, t], v[:, t], kc, vc, n, sinks=sinks)
        _close(o, want[:, t], TOL[dtype], f"step {t}")
        n += 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hk,D,cap,sinks", [(1, 16, 4, 64, 516, 4), (5, 4, 4, 64, 1000, 0), (2, 8, 2, 128, 4099, 3),
                                                (7, 3, 1, 24, 77, 7), (40, 4, 2, 32, 300, 1)])
def test_window_step_long_caches(B, H, Hk, D, cap, sinks, dtype):
    from tornado_gcm_b200.ops.window_attention import fill_window_cache, window_attention, window_attention_step

    lengths = [-1 if b % 4 == 3 else (b + 1) * 2 * cap // B - 1 for b in range(B)]
    q, k, v = (_randn(B, h, D, seed=i, dtype=dtype) for i, h in enumerate((H, Hk, Hk)))
    kc, vc = (_randn(B, cap, Hk, D, seed=5 + i, dtype=dtype) for i in range(2))
    before = kc.clone()
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    for b, t in enumerate(lengths):
        if t < 0:
            continue
        slot = t if t < cap else sinks + (t - sinks) % (cap - sinks)
        kk, vv = kc[b].double(), vc[b].double()
        kk[slot], vv[slot] = k[b].double(), v[b].double()
        seen = min(t + 1, cap)
        kk, vv = (x[:seen].repeat_interleave(H // Hk, 1) for x in (kk, vv))
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[b].double(), kk) * D ** -0.5, -1)
        want[b] = torch.einsum("hn,nhd->hd", p, vv)
        before[b, slot] = k[b]
    o = window_attention_step(q, k, v, kc, vc, n, sinks=sinks)
    _close(o, want, TOL[dtype])
    assert torch.equal(kc, before)  # the one slot is changed and no other, none of a sequence that takes no part
    # a history put in whole leaves what single steps leave
    S = cap + 50
    hist = [_randn(1, S + 1, h, D, seed=20 + i, dtype=dtype) for i, h in enumerate((H, Hk, Hk))]
    kc1, vc1 = kc[:1].clone(), vc[:1].clone()
    fill_window_cache(hist[1][:, :S], hist[2][:, :S], kc1, vc1, sinks=sinks)
    o = window_attention_step(hist[0][:, S], hist[1][:, S], hist[2][:, S], kc1, vc1,
                              torch.tensor([S], dtype=torch.int32, device=DEV), sinks=sinks)
    whole = window_attention(*hist, window=cap - sinks, sinks=sinks)[:, S]
    _close(o, whole, TOL[dtype])


def test_window_step_cache_offsets_beyond_32_bits():
    """A cache whose last sequence starts past 2^31 elements."""
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    B, cap, Hk, D = 3, 1 << 22, 4, 64  # 2^30 elements a sequence
    base = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
    kc = torch.empty(B, cap, Hk, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    del base
    kc[2, :40], vc[2, :40] = _randn(40, Hk, D, seed=1, dtype=torch.bfloat16), _randn(40, Hk, D, seed=2, dtype=torch.bfloat16)
    q, k, v = (_randn(B, 4, D, seed=i, dtype=torch.bfloat16) for i in range(3, 6))
    n = torch.tensor([-1, -1, 40], dtype=torch.int32, device=DEV)
    o = window_attention_step(q, k, v, kc, vc, n, sinks=4)
    kk, vv = torch.cat([kc[2, :40], k[2:]]).double(), torch.cat([vc[2, :40], v[2:]]).double()
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[2].double(), kk) * D ** -0.5, -1)
    _close(o[2], torch.einsum("hn,nhd->hd", p, vv), TOL[torch.bfloat16])
    assert torch.equal(kc[2, 40], k[2]) and torch.equal(vc[2, 40], v[2])


def test_window_step_refusals():
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    q, k, v = (_randn(2, h, 16, seed=i) for i, h in enumerate((4, 2, 2)))
    kc, vc = (torch.zeros(2, 6, 2, 16, device=DEV) for _ in range(2))
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (dict(n=n.long()), dict(n=n[:1]), dict(kc=kc[:1]), dict(kc=kc.bfloat16()), dict(vc=vc[:, :5]),
                dict(q=q[:, :3]), dict(v=v[..., :8]), dict(sinks=6), dict(sinks=-1)):
        a = dict(dict(q=q, k=k, v=v, kc=kc, vc=vc, n=n, sinks=1), **bad)
        with pytest.raises(RuntimeError, match="window_attention_step"):
            window_attention_step(a["q"], a["k"], a["v"], a["kc"], a["vc"], a["n"], sinks=a["sinks"])


# ── gradient clipping ──────────────────────────────────────────────────────
def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


@pytest.mark.parametrize("sizes", [[1], [0, 3], [5, 0, 100000, 7, 16385], [384] * 200 + [70000], [3] * 2500])
@pytest.mark.parametrize("kinds", ["fp32", "bf16", "mixed", "fp64"])
def test_clip_grad_norm_in_place(sizes, kinds):
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm, grad_norm

    pick = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "fp64": [torch.float64],
            "mixed": [torch.float32, torch.bfloat16, torch.float64]}[kinds]
    flat = {d: _randn(sum(sizes) + 8, seed=3, dtype=d) for d in set(pick)}
    gs, off = [], 1  # views at odd offsets of one buffer
    for i, n in enumerate(sizes):
        gs.append(flat[pick[i % len(pick)]][off:off + n])
        off += n
    norm64 = _norm64(gs)
    assert abs(float(grad_norm(gs)) - norm64) <= 1e-6 * norm64
    for max_norm in (2.0 * norm64 + 1.0, 0.25 * norm64):
        want = [t.double() * min(1.0, max_norm / (norm64 + 1e-6)) for t in gs]
        got = clip_grad_norm(gs, max_norm)
        assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - norm64) <= 1e-6 * norm64
        for a, b in zip(gs, want):
            if a.numel():
                _close(a, b, 4e-3 if a.dtype == torch.bfloat16 else 1e-6)


@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                     (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
def test_clip_grad_norm_into_other_buffers(src, dst):
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm

    shapes = [(7, 9), (300, 77), (64, 1024), (5,), (0, 4), (40000,)]
    gs = [_randn(*s, seed=i, dtype=src) for i, s in enumerate(shapes)]
    flat = torch.full((sum(g.numel() for g in gs) + 1,), 7.0, dtype=dst, device=DEV)
    out = [v.view(s) for v, s in zip(flat[1:].split([g.numel() for g in gs]), shapes)]
    keep = [g.clone() for g in gs]
    n64 = _norm64(gs)
    for m in (0.1, 1e9):
        clip_grad_norm(gs, m, out=out)
        for g, k, o in zip(gs, keep, out):
            assert torch.equal(g, k)
            if g.numel():
                _close(o, g.double() * min(1.0, m / (n64 + 1e-6)), 4e-3 if dst == torch.bfloat16 else 1e-6)
    assert float(flat[0]) == 7.0


def test_clip_grad_norm_extremes_and_layouts():
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm, grad_norm

    big = [torch.full((1000,), 1e30, device=DEV), torch.full((10,), -1e30, device=DEV)]
    assert abs(float(grad_norm(big)) / (1e30 * math.sqrt(1010)) - 1) < 1e-6  # squares beyond fp32
    tiny = [torch.full((1000,), 1e-30, device=DEV)]
    assert abs(float(grad_norm(tiny)) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    bad = [torch.tensor([1.0, float("nan")], device=DEV), torch.ones(3, device=DEV)]
    assert math.isnan(float(clip_grad_norm(bad, 1.0))) and torch.isnan(bad[1]).all()
    inf = [torch.tensor([1.0, float("inf")], device=DEV), torch.ones(3, device=DEV)]
    assert math.isinf(float(clip_grad_norm(inf, 1.0))) and (inf[1] == 0).all()
    w = _randn(40, 30, seed=1)
    for view in (w.t(), w[:, ::2], w[3:17, 5:9]):
        v = view.clone(memory_format=torch.preserve_format) if view.is_contiguous() else view
        want = v.double() * 0.5 * _norm64([v]) / (_norm64([v]) + 1e-6)
        clip_grad_norm([v], 0.5 * _norm64([v]))
        _close(v, want, 1e-6)
    ref = [_randn(50, 20, seed=i).requires_grad_() for i in range(3)]
    for t in ref:
        t.grad = _randn(50, 20, seed=9)
    mine = [t.grad.clone() for t in ref]
    n0 = torch.nn.utils.clip_grad_norm_(ref, 0.7)
    n1 = clip_grad_norm(mine, 0.7)
    _close(n1, n0, 1e-6)
    for a, t in zip(mine, ref):
        _close(a, t.grad, 1e-6)


def test_clip_grad_norm_refusals_and_graph():
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm

    a, b = torch.ones(4, device=DEV), torch.ones(5, device=DEV)
    with pytest.raises(ValueError):
        clip_grad_norm([a], -1.0)
    with pytest.raises(ValueError):
        clip_grad_norm([a, b], 1.0, out=[a])
    with pytest.raises(ValueError):
        clip_grad_norm([a, None], 1.0, out=[a, b])
    for g, o in (([a], [b]), ([a], [a.double()]), ([a.half()], [a.half()]), ([a, b.cpu()], [a, b])):
        with pytest.raises(RuntimeError, match="clip_grad_norm"):
            clip_grad_norm(g, 1.0, out=o)
    g = [_randn(1000, seed=1), _randn(7, seed=2)]
    clip_grad_norm(g, 1e9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = clip_grad_norm(g, 3.0)
    g[0].copy_(_randn(1000, seed=3))
    want = _norm64(g)
    graph.replay()
    torch.cuda.synchronize()
    assert abs(float(n) - want) <= 1e-6 * want and abs(_norm64(g) - 3.0) <= 1e-5


# ── the operators together ─────────────────────────────────────────────────
@pytest.mark.parametrize("D,window,sinks,causal", [(128, 640, 16, False), (64, 512, 4, True), (96, 300, 0, True)])
def test_window_attention_many_blocks_against_fp32_kernels(D, window, sinks, causal):
    """Thousands of blocks, several rounds of the GPU: the tensor-core kernels against the CUDA-core ones in fp32
    (which the tests above hold to fp64), on the same bf16 values."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, S, H, Hk = 2, 8192, 8, 2
    q, k, v = (_randn(B, S, h, D, seed=i, dtype=torch.bfloat16) for i, h in enumerate((H, Hk, Hk)))
    do = _randn(B, S, H, D, seed=5, dtype=torch.bfloat16)
    L = torch.tensor([S, 3000], dtype=torch.int32, device=DEV)
    res = []
    for dt in (torch.bfloat16, torch.float32):
        ts = [t.to(dt).requires_grad_() for t in (q, k, v)]
        o = window_attention(*ts, window=window, sinks=sinks, causal=causal, lengths=L)
        res.append([o, *torch.autograd.grad(o, ts, do.to(dt))])
    for name, a, b in zip(("o", "dq", "dk", "dv"), *res):
        _close(a, b, TOL[torch.bfloat16], name)
    _ext.check_error_flag(DEV)


def test_sequence_model_on_the_gpu_follows_the_cpu():
    """One training pass and a cached forecast against the fp32 CPU forms of the same weights: BF16 products in two
    blocks, so a few times the rounding of one."""
    from tornado_gcm_b200.models import sequence

    torch.manual_seed(0)
    cpu = sequence.SequenceEmulator(20, 3, statics=3, d_model=128, num_heads=2, kv_heads=1, num_layers=2, d_ff=200,
                                    window=40, max_positions=512)
    torch.nn.init.normal_(cpu.head.weight, std=0.05)
    gpu = sequence.SequenceEmulator(20, 3, statics=3, d_model=128, num_heads=2, kv_heads=1, num_layers=2, d_ff=200,
                                    window=40, max_positions=512).to(DEV)
    gpu.load_state_dict(cpu.state_dict())
    states, static = sequence.synthetic_columns(3, 150, 20, 3)
    L = torch.tensor([150, 80, 0], dtype=torch.int32)
    a = cpu.loss(states, static, L)
    b = gpu.loss(states.to(DEV), static.to(DEV), L.to(DEV))
    a.backward()
    b.backward()
    assert abs(float(a) - float(b)) <= 1e-2 * float(a)
    for (n, p), r in zip(gpu.named_parameters(), cpu.parameters()):
        _close(p.grad.cpu(), r.grad, 5e-2, n)
    f = gpu.forecast(states[:, :100].to(DEV), static.to(DEV), steps=60)
    with torch.no_grad():
        whole = gpu(torch.cat([states[:, :100].to(DEV), f[:, :-1]], 1), static.to(DEV))[:, 99:]
    _close(f, whole, 1e-2)
    _ext.check_error_flag(DEV)


def test_sequence_example_on_the_gpu():
    from tornado_gcm_b200.models import sequence

    r = sequence.main(["--steps", "31", "--batch", "4", "--length", "300", "--features", "12", "--window", "64",
                       "--layers", "2", "--width", "128", "--forecast", "20"])
    assert r["losses"][-1] < 0.5 * r["losses"][0] and r["gap"] < 1e-2


def test_trainer_with_native_clipping():
    """The hybrid trainer's step with either clipping: the same loss and, after it, the same weights."""
    from tornado_gcm_b200.training.trainer import GCMTrainer

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.lin = torch.nn.Linear(6, 5)

        def loss(self, data0, targets, forcings):
            return 100.0 * (self.lin(data0["x"]) - targets[0]["x"]).square().mean()

    torch.manual_seed(0)
    nets = [Net().to(DEV) for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    data, tgt = {"x": torch.randn(32, 6)}, [{"x": torch.randn(32, 5)}]
    trs = [GCMTrainer(n, lr=1e-2, max_grad_norm=0.5, graph=True, native_clip=native) for n, native in zip(nets, (False, True))]
    for _ in range(4):
        losses = [float(t.train_step(data, tgt, {})) for t in trs]
        assert abs(losses[0] - losses[1]) <= 1e-5 * losses[0]
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        _close(a, b, 1e-5)


@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_gradients_of_rows_with_a_few_keys(D):
    """Two or three keys to a row: dq and dk are differences of nearly equal numbers, and keep bf16's accuracy."""
    from tornado_gcm_b200.ops.window_attention import window_attention

    B, S = 30, 9
    q, k, v = (_randn(B, S, h, D, seed=i, dtype=torch.bfloat16).requires_grad_() for i, h in enumerate((4, 2, 2)))
    do = _randn(B, S, 4, D, seed=5, dtype=torch.bfloat16)
    L = torch.tensor([1 + b % 9 for b in range(B)], dtype=torch.int32, device=DEV)
    grads = torch.autograd.grad(window_attention(q, k, v, window=2, sinks=1, causal=False, lengths=L), [q, k, v], do)
    r = [t.detach().double().requires_grad_() for t in (q, k, v)]
    o64 = _attn64(*r, _see(S, 2, 1, False, L, B), D ** -0.5)
    for n, a, b in zip(("dq", "dk", "dv"), grads, torch.autograd.grad(o64, r, do.double())):
        _close(a, b, 2.6e-3, n)  # the two roundings of dS and of the result, 2.4e-3, and no third
