"""The sequence operators' CPU forms and the model at their edges: ragged histories, given positions, long forecasts,
padding, values that are not finite, refusals (no GPU)."""

import math

import pytest
import torch

from tornado_gcm_b200.models import sequence
from tornado_gcm_b200.neural.sequence_layers import SequenceTransformer
from tornado_gcm_b200.ops.rotary import qk_norm_rotary, rotary_table
from tornado_gcm_b200.ops.window_attention import fill_window_cache, window_attention, window_attention_step


def _randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def _body(max_positions=64, window=5, **kw):
    torch.manual_seed(0)
    return SequenceTransformer(32, 2, 2, 48, window, kv_heads=1, sinks=2, max_positions=max_positions, **kw)


def _emulator(max_positions=64):
    torch.manual_seed(0)
    m = sequence.SequenceEmulator(5, 3, statics=2, d_model=32, num_heads=2, num_layers=1, d_ff=40, window=6,
                                  max_positions=max_positions)
    torch.nn.init.normal_(m.head.weight, std=0.1)
    return m


@pytest.mark.parametrize("S", [1, 2, 5, 7, 8, 20])
@pytest.mark.parametrize("window,sinks", [(5, 2), (1, 0), (4, 3)])
def test_fill_window_cache_of_ragged_histories(S, window, sinks):
    """What single steps of the valid tokens leave, in every slot; NaN behind the end, and slots never written keep."""
    lengths = [S, S - 1, S // 2, min(sinks, S), 0, -1, S + 3]
    B, cap = len(lengths), window + sinks
    k, v = _randn(B, S, 1, 6, seed=1), _randn(B, S, 1, 6, seed=2)
    for b, n in enumerate(lengths):
        k[b, max(n, 0):], v[b, max(n, 0):] = math.nan, math.nan
    got = [torch.full((B, cap, 1, 6), 7.0) for _ in range(2)]
    want = [t.clone() for t in got]
    fill_window_cache(k, v, *got, sinks=sinks, lengths=torch.tensor(lengths, dtype=torch.int32))
    for b, n in enumerate(lengths):
        for t in range(min(max(n, 0), S)):
            slot = t if t < cap else sinks + (t - sinks) % window
            want[0][b, slot], want[1][b, slot] = k[b, t], v[b, t]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError):
        fill_window_cache(k, v, *got, sinks=sinks, lengths=torch.tensor([1, 2], dtype=torch.int32))


@pytest.mark.parametrize("S", [6, 12, 30])  # the cache holds seven tokens
def test_steps_behind_a_ragged_history(S):
    m = _body()
    x = _randn(4, S + 9, 32, seed=3)
    L = [S, S - 4, 1, 0]
    padded = x[:, :S].clone()
    for b, n in enumerate(L):
        padded[b, n:] = 5.0
    with torch.no_grad():
        cache = m.new_cache(4)
        m(padded, torch.tensor(L, dtype=torch.int32), cache=cache)
        assert cache.lengths.tolist() == L
        got = torch.stack([m.step(x[:, S + t], cache) for t in range(9)], 1)
        for b, n in enumerate(L):
            whole = m(torch.cat([x[b:b + 1, :n], x[b:b + 1, S:]], 1))[:, n:]
            assert torch.allclose(got[b:b + 1], whole, atol=1e-5), b


def test_emulator_takes_a_ragged_history_into_a_cache():
    m = _emulator()
    states, static = sequence.synthetic_columns(3, 16, 5, 3)
    lengths = torch.tensor([12, 4, -1], dtype=torch.int32)
    with torch.no_grad():
        cache = m.body.new_cache(3)
        m(states[:, :12], static, lengths, cache=cache)
        assert cache.lengths.tolist() == [14, 6, -1]
        got = states[:, 12] + m.head(m.body.step(m.embed(states[:, 12]), cache))
        for b, n in enumerate([12, 4]):
            whole = m(torch.cat([states[b:b + 1, :n], states[b:b + 1, 12:13]], 1), static[b:b + 1])[:, -1]
            assert torch.allclose(got[b:b + 1], whole, atol=1e-5)


def test_steps_behind_a_history_at_given_positions():
    m = _body()
    x = _randn(2, 20, 32, seed=3)
    for pos in (torch.arange(20) + 17, torch.stack([torch.arange(20) + 3, torch.arange(20) + 40])):
        with torch.no_grad():
            whole = m(x, None, pos)
            cache = m.new_cache(2)
            m(x[:, :12], None, pos[..., :12], cache=cache)
            got = torch.stack([m.step(x[:, t], cache) for t in range(12, 20)], 1)
        assert torch.allclose(got, whole[:, 12:], atol=1e-5)
    # ragged: each sequence goes on behind its own last valid position, one without tokens at its first position
    pos = torch.stack([torch.arange(20) + 3, torch.arange(20) + 40])
    cache = m.new_cache(2)
    with torch.no_grad():
        m(x[:, :12], torch.tensor([5, 0], dtype=torch.int32), pos[:, :12], cache=cache)
        got = m.step(x[:, 12], cache)
        for b, n in enumerate((5, 0)):
            rows = torch.cat([x[b:b + 1, :n], x[b:b + 1, 12:13]], 1)
            assert torch.allclose(got[b:b + 1], m(rows, None, pos[b, :n + 1])[:, -1], atol=1e-5)
    # positions that do not follow on are given to the step
    pos = torch.arange(20) * 3
    cache = m.new_cache(2)
    with torch.no_grad():
        whole = m(x, None, pos)
        m(x[:, :12], None, pos[:12], cache=cache)
        got = torch.stack([m.step(x[:, t], cache, positions=pos[t].expand(2)) for t in range(12, 20)], 1)
    assert torch.allclose(got, whole[:, 12:], atol=1e-5)
    # a history without positions makes the cache count tokens again
    with torch.no_grad():
        m(x[:, :12], cache=cache)
        assert torch.allclose(m.step(x[:, 12], cache), m(x[:, :13])[:, -1], atol=1e-5)


def test_forecast_past_the_table_of_positions():
    states, static = sequence.synthetic_columns(2, 20, 5, 3)
    want = _emulator(256).forecast(states, static, steps=60)
    for rows in (4, 22, 40):  # short of the history, of the first step, of the last
        m = _emulator(rows)
        assert torch.equal(m.forecast(states, static, steps=60), want)
        assert torch.equal(m.forecast(states, static, steps=60), want)
    for steps in (0, -3):
        with pytest.raises(ValueError):
            _emulator().forecast(states, static, steps=steps)


def test_steps_past_the_table_of_positions_are_refused_until_it_grows():
    m = _body(max_positions=14)
    big = _body(max_positions=64)
    x = _randn(2, 30, 32, seed=3)
    cache = m.new_cache(2)
    with torch.no_grad():
        m(x[:, :12], cache=cache)
        for t in (12, 13):
            m.step(x[:, t], cache)
        before = [t.clone() for t in cache.k], cache.lengths.clone()
        with pytest.raises(IndexError, match="reserve"):
            m.step(x[:, 14], cache)
        assert all(torch.equal(a, b) for a, b in zip(cache.k, before[0])) and torch.equal(cache.lengths, before[1])
        m.reserve(30)
        got = torch.stack([m.step(x[:, t], cache) for t in range(14, 30)], 1)
        assert torch.allclose(got, big(x)[:, 14:], atol=1e-5)
        cache = m.new_cache(2)
        m(x[:, :3], None, torch.tensor([20, 25, 29]), cache=cache)
        with pytest.raises(IndexError, match="reserve"):
            m.step(x[:, 3], cache)
    table = m.layers[0].attn.table.clone()
    m.reserve(10)
    assert torch.equal(m.layers[0].attn.table, table)
    scaled = _body(max_positions=8, rotary_scaling="base", rotary_factor=4.0)
    scaled.reserve(50)
    assert torch.equal(scaled.layers[1].attn.table[:50], rotary_table(50, 16, scaling="base", factor=4.0))


def test_train_step_reads_the_error_flag_when_asked(monkeypatch):
    asked = []
    monkeypatch.setattr(sequence._ext, "check_error_flag", lambda device: asked.append(torch.device(device).type))
    m = _emulator()
    states, static = sequence.synthetic_columns(2, 10, 5, 3)
    opt = torch.optim.SGD(m.parameters(), lr=1e-3)
    sequence.train_step(m, opt, states, static)
    assert not asked
    sequence.train_step(m, opt, states, static, check_errors=True)
    m.forecast(states, static, steps=2)
    assert asked == ["cpu", "cpu"]


def test_the_step_has_no_gradient_and_says_so():
    base = [_randn(2, 2, 8, seed=i) for i in range(3)] + [torch.zeros(2, 6, 2, 8) for _ in range(2)]
    n = torch.zeros(2, dtype=torch.int32)
    for i in range(5):
        ts = [t.clone().requires_grad_() if j == i else t.clone() for j, t in enumerate(base)]
        with pytest.raises(RuntimeError, match="no gradient"):
            window_attention_step(*ts, n)
        with torch.no_grad():
            window_attention_step(*ts, n)
    # the layers' steps are outside autograd as a whole, not in part
    m = _body()
    x = _randn(2, 9, 32, seed=3).requires_grad_()
    cache = m.new_cache(2)
    m(x[:, :8], cache=cache)
    assert not any(t.requires_grad for t in cache.k + cache.v)
    assert not m.step(x[:, 8], cache).requires_grad
    layer = m.layers[0]
    assert not layer.step(x[:, 8], cache.k[0], cache.v[0], cache.lengths).requires_grad
    assert not layer.attn.step(x[:, 8], cache.k[0], cache.v[0], cache.lengths).requires_grad


def test_padding_of_the_model_may_hold_anything():
    m = _emulator()
    states, static = sequence.synthetic_columns(3, 16, 5, 3)
    L = torch.tensor([16, 9, 0], dtype=torch.int32)
    res = []
    for junk in (0.0, math.nan, math.inf):
        s = states.clone()
        s[1, 9:], s[2] = junk, junk
        m.zero_grad()
        loss = m.loss(s, static, L)
        loss.backward()
        res.append([loss.detach()] + [p.grad.clone() for p in m.parameters()])
    for other in res[1:]:
        assert all(torch.isfinite(b).all() and torch.equal(a, b) for a, b in zip(res[0], other))
    body = _body()
    x = _randn(2, 12, 32, seed=4)
    n = torch.tensor([12, 5], dtype=torch.int32)
    res = []
    for junk in (0.0, math.nan):
        body.zero_grad()
        y = x.clone()
        y[1, 5:] = junk
        out = body(y, n)
        (out[0].sum() + out[1, :5].square().sum()).backward()
        res.append([out.detach()[0], out.detach()[1, :5]] + [p.grad.clone() for p in body.parameters()])
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_with_keys_behind_the_end_that_hold_anything(causal):
    q, k, v = (_randn(2, 9, h, 4, seed=i, dtype=torch.float64) for i, h in enumerate((2, 1, 1)))
    lengths = torch.tensor([9, 4], dtype=torch.int32)
    res = []
    for junk in (0.0, math.nan, math.inf):
        ts = [q.clone(), k.clone(), v.clone()]
        ts[1][1, 4:], ts[2][1, 4:] = junk, junk
        ts = [t.requires_grad_() for t in ts]
        o = window_attention(*ts, window=3, sinks=1, causal=causal, lengths=lengths)
        res.append([o, *torch.autograd.grad(o.square().sum(), ts)])
    for other in res[1:]:
        assert all(torch.isfinite(b).all() and torch.equal(a, b) for a, b in zip(res[0], other))


def test_rows_whose_every_score_is_minus_infinity_give_zeros():
    q, k, v = (_randn(1, 8, 1, 4, seed=i) for i in range(3))
    k[..., 3] = 1.0
    q[:, 2] = 0.0
    want = window_attention(q, k, v, window=3)
    q[:, 2, :, 3] = -math.inf
    got = window_attention(q, k, v, window=3)
    assert (got[:, 2] == 0).all() and torch.equal(got[:, 3:], want[:, 3:]) and torch.equal(got[:, :2], want[:, :2])
    n = torch.full((1,), 7, dtype=torch.int32)
    assert (window_attention_step(q[:, 2], k[:, 7], v[:, 7], k.clone(), v.clone(), n) == 0).all()


def test_positions_outside_the_table_are_refused():
    q = _randn(1, 2, 1, 4, seed=1)
    table = rotary_table(8, 4)
    for pos in ([-1, 0], [0, 8]):
        with pytest.raises(IndexError):
            qk_norm_rotary(q, q, table, norm="none", positions=torch.tensor(pos))
    with pytest.raises(ValueError):
        qk_norm_rotary(q, q, table[:1], norm="none")


def test_the_step_computes_in_its_inputs_type():
    q, k, v = (_randn(2, h, 8, seed=i, dtype=torch.float64) for i, h in enumerate((4, 2, 2)))
    kc, vc = (_randn(2, 6, 2, 8, seed=i, dtype=torch.float64) for i in (5, 6))
    n = torch.tensor([3, 20], dtype=torch.int32)
    o = window_attention_step(q, k, v, kc, vc, n, sinks=1)
    for b, seen in enumerate((4, 6)):
        kk, vv = (t[b, :seen].repeat_interleave(2, 1) for t in (kc, vc))
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[b], kk) * 8 ** -0.5, -1)
        assert torch.allclose(o[b], torch.einsum("hn,nhd->hd", p, vv), rtol=0, atol=1e-14)


def test_caches_whose_sequences_share_memory_are_refused():
    q = _randn(3, 1, 8, seed=1)
    own, shared = torch.zeros(3, 6, 1, 8), torch.zeros(1, 6, 1, 8).expand(3, 6, 1, 8)
    n = torch.zeros(3, dtype=torch.int32)
    for kc, vc in ((shared, own), (own, shared)):
        with pytest.raises(RuntimeError, match="single memory location"):
            window_attention_step(q, q, q, kc, vc, n)
