"""The sequence operators that are timed, each in a plain form and as the framework's kernel.

Operators (all on one GPU):

* ``gated``: ``act(x Wgᵀ + bg) * (x Wuᵀ + bu)``, forward alone or with its gradients;
* ``qk``: the norm of every query and key head followed by the rotation of its first ``rotary`` values, forward
  alone or with its gradients;
* ``attn``: attention in a sliding window with the first ``sinks`` tokens always in sight, forward alone or with
  its gradients;
* ``step``: the same attention for one new token of every sequence, over a cache of ``sinks + window`` slots;
* ``clip``: the global norm of a list of gradients, and the clipped gradients in one flat fp32 buffer.

``run`` computes the plain form (elementary torch operations in fp32) while ``own`` is false and calls the
framework while it is true.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one grid point's worth of serving: a single token through a wide feed-forward, all of it weight traffic
        dict(name="gated one token", op="gated", tokens=1, d_in=1024, d_ff=4096, act="silu", bias=False, train=False),
        # training on the 128 x 64 grid of the 2.8 degree model at the towers' width, with a ragged hidden width
        dict(name="gated tower 2.8deg", op="gated", tokens=8192, d_in=384, d_ff=1000, act="gelu_tanh", bias=True,
             train=True),
        # the largest: two 2.8 degree grids through a wide transformer block
        dict(name="gated wide train", op="gated", tokens=16384, d_in=1024, d_ff=4096, act="silu", bias=False,
             train=True),
        # a small fp32 model over 37 levels, part of the head rotated in neighbouring pairs
        dict(name="qk levels fp32", op="qk", batch=96, seq=37, heads=6, kv_heads=6, head_dim=40, rotary=20,
             norm="layer", interleaved=True, dtype="fp32", train=True),
        # training on the 128 x 64 grid, shared key heads
        dict(name="qk grid train", op="qk", batch=2, seq=8192, heads=16, kv_heads=4, head_dim=64, rotary=64,
             norm="rms", interleaved=False, dtype="bf16", train=True),
        # a small fp32 model over a season of 6-hour steps
        dict(name="attn season fp32", op="attn", batch=2, seq=365, heads=4, kv_heads=2, head_dim=32, window=112,
             sinks=2, causal=True, ragged=False, dtype="fp32", train=True),
        # training on long sequences, shared key heads, a causal window and a few static tokens in front
        dict(name="attn causal train", op="attn", batch=2, seq=8192, heads=16, kv_heads=4, head_dim=64, window=512,
             sinks=4, causal=True, ragged=False, dtype="bf16", train=True),
        # a forward pass over the 256 x 128 grid's tokens, a band of rows on both sides, sequences of several lengths
        dict(name="attn band forward", op="attn", batch=2, seq=32768, heads=8, kv_heads=8, head_dim=128, window=640,
             sinks=16, causal=False, ragged=True, dtype="bf16", train=False),
        # a forecast of one sequence, one step
        dict(name="step one sequence", op="step", batch=1, heads=16, kv_heads=4, head_dim=64, window=512, sinks=4,
             dtype="bf16"),
        # an ensemble's step: many sequences, each with its own history
        dict(name="step ensemble", op="step", batch=256, heads=16, kv_heads=4, head_dim=64, window=1460, sinks=4,
             dtype="bf16"),
        # the gradients of a tower of width 384
        dict(name="clip tower", op="clip", layers=6, width=384, d_ff=1000, dtype="fp32"),
        # bf16 gradients of a wide model, widened to fp32 as they are clipped
        dict(name="clip wide bf16", op="clip", layers=24, width=1024, d_ff=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gated", "qk", "attn", "step", "clip"])
    if op == "gated":
        train = rng.random() < 0.5
        tokens = _log(rng, 16 if train else 1, 16384)
        odd = rng.random() < 0.2
        d_in = _log(rng, 64, 1024)
        d_ff = _log(rng, 64, 4096)
        if not odd:
            d_in, d_ff = (d_in + 7) // 8 * 8, (d_ff + 7) // 8 * 8
        return dict(op=op, tokens=tokens, d_in=d_in, d_ff=d_ff, act=rng.choice(["silu", "gelu_tanh", "gelu", "relu"]),
                    bias=rng.random() < 0.5, train=train)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    dtype = "fp32" if rng.random() < 0.2 else "bf16"
    head_dim = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128])
    if op == "qk":
        rotary = head_dim if rng.random() < 0.6 else max(2, head_dim // 4 * 2)
        tokens = _log(rng, 1, 2_000_000 // (heads * head_dim) * 8)
        batch = _log(rng, 1, min(64, tokens))
        return dict(op=op, batch=batch, seq=max(1, tokens // batch), heads=heads, kv_heads=kv, head_dim=head_dim,
                    rotary=rotary, norm=rng.choice(["layer", "rms", "none"]), interleaved=rng.random() < 0.4, dtype=dtype,
                    train=rng.random() < 0.5)
    if op == "attn":
        seq = _log(rng, 2, 1024 if dtype == "fp32" else 16384)
        window = _log(rng, 1, min(1024, seq))
        batch = max(1, min(_log(rng, 1, 64), 120_000_000 // (seq * (window + 32) * heads) or 1))
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv, head_dim=head_dim, window=window,
                    sinks=rng.choice([0, 0, 1, 4, 17]), causal=rng.random() < 0.6, ragged=rng.random() < 0.4,
                    dtype=dtype, train=rng.random() < 0.5)
    if op == "step":
        window = _log(rng, 16, 8192)
        batch = max(1, min(_log(rng, 1, 512), 90_000_000 // (window * kv * head_dim)))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv, head_dim=head_dim, window=window,
                    sinks=rng.choice([0, 1, 4, 32]), dtype=dtype)
    width = _log(rng, 32, 1024)
    return dict(op=op, layers=_log(rng, 1, 24), width=width, d_ff=_log(rng, width, 4 * width),
                dtype=rng.choice(["fp32", "bf16"]))


# ── inputs ─────────────────────────────────────────────────────────────────
def _lengths(case):
    """Valid tokens of each sequence: spread from the whole length down to a fraction of it."""
    B, S = case["batch"], case["seq"]
    return [S - b * S // B for b in range(B)]


def _history(case):
    """Tokens that each sequence of a step holds already: from an empty cache to one that has wrapped twice."""
    B, cap = case["batch"], case["window"] + case["sinks"]
    return [3 * cap] if B == 1 else [3 * cap * b // (B - 1) for b in range(B)]


def _clip_shapes(case):
    w, f = case["width"], case["d_ff"]
    layer = [(3 * w, w), (w, w), (f, w), (f, w), (w, f), (w,), (w,), (f,), (f,)]
    return layer * case["layers"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)

    st = dict(case=case)
    op = case["op"]
    if op == "gated":
        T, K, F = case["tokens"], case["d_in"], case["d_ff"]
        bf = torch.bfloat16
        st["x"] = randn(T, K, dtype=bf)
        st["w_gate"] = randn(F, K, dtype=bf, scale=K ** -0.5)
        st["w_up"] = randn(F, K, dtype=bf, scale=K ** -0.5)
        st["b_gate"] = randn(F, dtype=bf, scale=0.2) if case["bias"] else None
        st["b_up"] = randn(F, dtype=bf, scale=0.2) if case["bias"] else None
        if case["train"]:
            st["dh"] = randn(T, F, dtype=bf)
            for n in ("x", "w_gate", "w_up", "b_gate", "b_up"):
                if st[n] is not None:
                    st[n].requires_grad_()
    elif op == "qk":
        B, S, H, Hk, D, R = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim", "rotary"))
        dt = _DTYPES[case["dtype"]]
        # queries, keys and values come out of one projection: the heads are views of its rows
        rows = randn(B, S, (H + 2 * Hk) * D, dtype=dt)
        st["q"] = rows[..., :H * D].unflatten(-1, (H, D))
        st["k"] = rows[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
        st["q_weight"] = st["k_weight"] = st["q_bias"] = st["k_bias"] = None
        if case["norm"] != "none":
            st["q_weight"], st["k_weight"] = 1 + randn(D, scale=0.1), 1 + randn(D, scale=0.1)
        if case["norm"] == "layer":
            st["q_bias"], st["k_bias"] = randn(D, scale=0.1), randn(D, scale=0.1)
        P = S + 64
        freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        ang = torch.arange(P, dtype=torch.float64, device="cuda")[:, None] * freq
        st["table"] = torch.stack([ang.cos(), ang.sin()], -1).float()
        start = torch.randint(0, 65, (B, 1), generator=g, device="cuda", dtype=torch.int32)
        st["positions"] = start + torch.arange(S, device="cuda", dtype=torch.int32)
        if case["train"]:
            st["dq"], st["dk"] = randn(B, S, H, D, dtype=dt), randn(B, S, Hk, D, dtype=dt)
            st["q"], st["k"] = st["q"].detach().requires_grad_(), st["k"].detach().requires_grad_()
            for n in ("q_weight", "k_weight", "q_bias", "k_bias"):
                if st[n] is not None:
                    st[n].requires_grad_()
    elif op == "attn":
        B, S, H, Hk, D = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
        dt = _DTYPES[case["dtype"]]
        st["q"], st["k"], st["v"] = (randn(B, S, h, D, dtype=dt) for h in (H, Hk, Hk))
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        if case["train"]:
            st["do"] = randn(B, S, H, D, dtype=dt)
            for n in ("q", "k", "v"):
                st[n].requires_grad_()
    elif op == "step":
        B, H, Hk, D = (case[n] for n in ("batch", "heads", "kv_heads", "head_dim"))
        dt, cap = _DTYPES[case["dtype"]], case["window"] + case["sinks"]
        st["q"], st["k"], st["v"] = (randn(B, h, D, dtype=dt) for h in (H, Hk, Hk))
        st["k_cache"], st["v_cache"] = randn(B, cap, Hk, D, dtype=dt), randn(B, cap, Hk, D, dtype=dt)
        st["lengths"] = torch.tensor(_history(case), dtype=torch.int32, device="cuda")
    else:
        dt = _DTYPES[case["dtype"]]
        st["grads"] = [randn(*s, dtype=dt, scale=0.01) for s in _clip_shapes(case)]
        n = sum(t.numel() for t in st["grads"])
        st["flat"] = torch.zeros(n, device="cuda")
        st["out"] = [v.view_as(t) for v, t in zip(st["flat"].split([t.numel() for t in st["grads"]]), st["grads"])]
        st["max_norm"] = 1.0 if n > 10000 else 0.1
    return st


# ── one pass ───────────────────────────────────────────────────────────────
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    with torch.no_grad():
        return _PLAIN[op](state)


def _own_gated(st):
    from tornado_gcm_b200.ops.gated import gated_linear

    h = gated_linear(st["x"], st["w_gate"], st["w_up"], st["b_gate"], st["b_up"], activation=st["case"]["act"])
    if not st["case"]["train"]:
        return h
    names = [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if st[n] is not None]
    return dict(zip(["h"] + names, (h,) + torch.autograd.grad(h, [st[n] for n in names], st["dh"])))


def _own_qk(st):
    from tornado_gcm_b200.ops.rotary import qk_norm_rotary

    c = st["case"]
    q, k = qk_norm_rotary(st["q"], st["k"], st["table"], st["q_weight"], st["k_weight"], st["q_bias"], st["k_bias"],
                          norm=c["norm"], interleaved=c["interleaved"], positions=st["positions"])
    if not c["train"]:
        return q, k
    names = [n for n in ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias") if st[n] is not None]
    grads = torch.autograd.grad([q, k], [st[n] for n in names], [st["dq"], st["dk"]])
    return dict(zip(["yq", "yk"] + names, (q, k) + grads))


def _own_attn(st):
    from tornado_gcm_b200.ops.window_attention import window_attention

    c = st["case"]
    o = window_attention(st["q"], st["k"], st["v"], window=c["window"], sinks=c["sinks"], causal=c["causal"],
                         lengths=st["lengths"])
    if not c["train"]:
        return o
    return (o,) + torch.autograd.grad(o, [st["q"], st["k"], st["v"]], st["do"])


def _own_step(st):
    from tornado_gcm_b200.ops.window_attention import window_attention_step

    o = window_attention_step(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["lengths"],
                              sinks=st["case"]["sinks"])
    return o, st["k_cache"], st["v_cache"]


def _own_clip(st):
    from tornado_gcm_b200.ops.gradnorm import clip_grad_norm

    return clip_grad_norm(st["grads"], st["max_norm"], out=st["out"]), st["flat"]


_OWN = {"gated": _own_gated, "qk": _own_qk, "attn": _own_attn, "step": _own_step, "clip": _own_clip}


# ── the plain forms, in fp32 ───────────────────────────────────────────────
def _act(name, z):
    """The activation and its derivative."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    a = (2 / math.pi) ** 0.5
    t = torch.tanh(a * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)


def _plain_gated(st):
    c = st["case"]
    x, wg, wu = (st[n].float() for n in ("x", "w_gate", "w_up"))
    zg, zu = x @ wg.T, x @ wu.T
    if c["bias"]:
        zg, zu = zg + st["b_gate"].float(), zu + st["b_up"].float()
    a, da = _act(c["act"], zg)
    h = (a * zu).bfloat16()
    if not c["train"]:
        return h
    dh = st["dh"].float()
    dg, du = dh * zu * da, dh * a
    out = dict(h=h, x=dg @ wg + du @ wu, w_gate=dg.T @ x, w_up=du.T @ x)
    if c["bias"]:
        out.update(b_gate=dg.sum(0), b_up=du.sum(0))
    return {n: t.bfloat16() for n, t in out.items()}


def _rotate(x, cos, sin, interleaved, back=False):
    """Rotates the first ``2 * cos.shape[-1]`` values of every head."""
    r = cos.shape[-1]
    if back:
        sin = -sin
    if interleaved:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., 2 * r:]], -1)


def _plain_qk(st):
    c, out = st["case"], {}
    eps = 1e-5
    cs = st["table"][st["positions"].long()]
    cos, sin = cs[..., 0].unsqueeze(-2), cs[..., 1].unsqueeze(-2)
    for n in ("q", "k"):
        x = st[n].float()
        w, b = st[n + "_weight"], st[n + "_bias"]
        xc = x - x.mean(-1, keepdim=True) if c["norm"] == "layer" else x
        r = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + eps) if c["norm"] != "none" else torch.ones_like(x[..., :1])
        hat = xc * r
        y = hat if w is None else hat * w
        y = y if b is None else y + b
        out["y" + n] = _rotate(y, cos, sin, c["interleaved"]).to(st[n].dtype)
        if c["train"]:
            dy = _rotate(st["d" + n].float(), cos, sin, c["interleaved"], back=True)
            dhat = dy if w is None else dy * w
            if c["norm"] == "none":
                dx = dhat
            else:
                dx = dhat - hat * (dhat * hat).mean(-1, keepdim=True)
                if c["norm"] == "layer":
                    dx = dx - dhat.mean(-1, keepdim=True)
                dx = dx * r
            out[n] = dx.to(st[n].dtype)
            if w is not None:
                out[n + "_weight"] = (dy * hat).sum((0, 1, 2))
            if b is not None:
                out[n + "_bias"] = dy.sum((0, 1, 2))
    return out if c["train"] else (out["yq"], out["yk"])


def _plain_attn(st):
    """Blocks of ``window`` queries against the two or three blocks of keys that they can see, and the sinks."""
    c = st["case"]
    q, k, v = (st[n].float() for n in ("q", "k", "v"))
    B, S, H, D = q.shape
    Hk, N, n_s = k.shape[2], H // k.shape[2], min(c["sinks"], S)
    W = min(c["window"], S)
    nb = -(-S // W)
    span = 2 if c["causal"] else 3
    pad = torch.nn.functional.pad
    after = (nb + span - 2) * W - S
    kb, vb = (pad(t, (0, 0, 0, 0, W, after)).unfold(1, span * W, W) for t in (k, v))
    kb, vb = kb.transpose(-1, -2), vb.transpose(-1, -2)                       # (B, nb, Hk, span W, D)

    def blocks(t):                                                            # (B, nb, Hk, N W, D)
        t = pad(t, (0, 0, 0, 0, 0, nb * W - S)).reshape(B, nb, W, Hk, N, D)
        return t.permute(0, 1, 3, 4, 2, 5).reshape(B, nb, Hk, N * W, D)

    def unblocks(t):
        t = t.reshape(B, nb, Hk, N, W, D).permute(0, 1, 4, 2, 3, 5)
        return t.reshape(B, nb * W, H, D)[:, :S]

    ar = lambda n: torch.arange(n, device=q.device)  # noqa: E731
    ks, vs = (t[:, :n_s].transpose(1, 2).unsqueeze(1) for t in (k, v))        # (B, 1, Hk, sinks, D)
    qp = (ar(nb)[:, None] * W + ar(W)).reshape(nb, W, 1)
    kp = (ar(nb)[:, None] * W - W + ar(span * W)).reshape(nb, 1, span * W)
    far = (qp - kp) if c["causal"] else (qp - kp).abs()
    ok_w = (kp >= n_s) & (kp < S) & (far < W) & (far >= 0)
    ok_s = (qp >= ar(n_s)) if c["causal"] else (qp >= 0).expand(nb, W, n_s)
    L = torch.full((B,), S, device=q.device) if st["lengths"] is None else st["lengths"].long()
    ok_w = ok_w & (kp < L.reshape(B, 1, 1, 1))
    ok_s = ok_s & (ar(n_s) < L.reshape(B, 1, 1, 1))
    ok = torch.cat([ok_s, ok_w], -1).reshape(B, nb, 1, 1, W, n_s + span * W)
    qb = blocks(q)
    scale = D ** -0.5
    s = torch.cat([qb @ ks.transpose(-1, -2), qb @ kb.transpose(-1, -2)], -1) * scale
    s = s.reshape(B, nb, Hk, N, W, -1).masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    del s
    z = p.sum(-1, keepdim=True)
    p = (p / torch.where(z == 0, torch.ones_like(z), z)).reshape(B, nb, Hk, N * W, -1)
    o = unblocks(p[..., :n_s] @ vs + p[..., n_s:] @ vb).to(st["q"].dtype)
    if not c["train"]:
        return o
    do = blocks(st["do"].float())
    dp = torch.cat([do @ vs.transpose(-1, -2), do @ vb.transpose(-1, -2)], -1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    dq = unblocks(ds[..., :n_s] @ ks + ds[..., n_s:] @ kb)

    def keys(a, t):
        """Adds what every block of queries says about its keys at the keys' places."""
        at = (kp + W).reshape(-1)
        both = (a[..., n_s:].transpose(-1, -2) @ t).permute(0, 1, 3, 2, 4).reshape(B, -1, Hk, D)
        whole = torch.zeros(B, W + S + after, Hk, D, device=q.device).index_add_(1, at, both)[:, W:W + S]
        whole[:, :n_s] += (a[..., :n_s].transpose(-1, -2) @ t).sum(1).transpose(1, 2)
        return whole

    return o, dq.to(o.dtype), keys(ds, qb).to(o.dtype), keys(p, do).to(o.dtype)


def _plain_step(st):
    c = st["case"]
    B, H, D = st["q"].shape
    Hk, cap, W = st["k"].shape[1], st["k_cache"].shape[1], c["window"]
    at, b = st["lengths"].long(), torch.arange(B, device="cuda")
    slot = torch.where(at < cap, at, c["sinks"] + (at - c["sinks"]) % W)
    st["k_cache"][b, slot], st["v_cache"][b, slot] = st["k"], st["v"]
    k, v = (st[n].float().transpose(1, 2) for n in ("k_cache", "v_cache"))
    s = st["q"].float().reshape(B, Hk, H // Hk, D) @ k.transpose(-1, -2) * D ** -0.5
    seen = torch.arange(cap, device="cuda") <= at[:, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)) @ v
    return o.reshape(B, H, D).to(st["q"].dtype), st["k_cache"], st["v_cache"]


def _plain_clip(st):
    norm = torch.stack([t.float().square().sum() for t in st["grads"]]).sum().sqrt()
    coef = (st["max_norm"] / (norm + 1e-6)).clamp(max=1)
    return norm, torch.cat([t.float().reshape(-1) for t in st["grads"]], out=st["flat"]).mul_(coef)


_PLAIN = {"gated": _plain_gated, "qk": _plain_qk, "attn": _plain_attn, "step": _plain_step, "clip": _plain_clip}


# ── what a pass cannot do without ──────────────────────────────────────────
def _pairs(S, W, sinks, causal, L):
    """Query-key pairs in sight of each other, of one sequence with L valid tokens and S queries."""
    total = 0
    for p in range(S):
        lo, hi = p - W + 1, p if causal else p + W - 1
        lo, hi = max(lo, 0), min(hi, L - 1)
        n = max(0, hi - lo + 1)
        head = min(sinks, L, p + 1 if causal else L)  # sinks in sight, less those inside the window
        total += n + max(0, min(head, lo) if hi >= lo else head)
    return total


def work(case):
    op = case["op"]
    if op == "gated":
        T, K, F = case["tokens"], case["d_in"], case["d_ff"]
        b = 2 * F if case["bias"] else 0
        fwd = T * K + 2 * F * K + b + T * F
        return dict(bytes=2 * (fwd + (T * F + T * K + 2 * F * K + b if case["train"] else 0)),
                    flops=(12 if case["train"] else 4) * T * K * F)
    if op == "clip":
        n = sum(math.prod(s) for s in _clip_shapes(case))
        return dict(bytes=n * (4 + (2 if case["dtype"] == "bf16" else 4)), flops=3 * n)
    e = 2 if case["dtype"] == "bf16" else 4
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    if op == "qk":
        rows = case["batch"] * case["seq"] * (H + Hk)
        return dict(bytes=rows * D * e * (4 if case["train"] else 2) + case["seq"] * case["rotary"] * 4,
                    flops=rows * D * (30 if case["train"] else 12))
    if op == "step":
        cap = case["window"] + case["sinks"]
        seen = sum(min(n + 1, cap) for n in _history(case))
        return dict(bytes=e * D * (2 * Hk * seen + case["batch"] * (2 * H + 2 * Hk)), flops=4 * H * D * seen)
    B, S = case["batch"], case["seq"]
    Ls = _lengths(case) if case["ragged"] else [S] * B
    pairs = H * sum(_pairs(S, case["window"], case["sinks"], case["causal"], L) for L in set(Ls) for _ in range(Ls.count(L)))
    one = B * S * D * e
    return dict(bytes=one * (2 * H + 2 * Hk) + (one * (2 * H + 2 * Hk) if case["train"] else 0),
                flops=(14 if case["train"] else 4) * pairs * D)


# ── the definitions, in 64 bits ────────────────────────────────────────────
def exact(case, seed):
    st = prepare(case, seed)
    for n, t in st.items():
        if torch.is_tensor(t) and t.is_floating_point():
            st[n] = t.detach().double()
    return _EXACT[case["op"]](st, case)


def _through(fn, leaves, weights):
    """fn's outputs and the gradients of its leaves, by automatic differentiation in 64 bits."""
    leaves = [t.requires_grad_() for t in leaves]
    with torch.enable_grad():
        ys = fn()
    return [y.detach() for y in ys], torch.autograd.grad(ys, leaves, weights)


def _exact_gated(st, case):
    F = torch.nn.functional
    act = dict(relu=F.relu, silu=F.silu, gelu=F.gelu, gelu_tanh=lambda z: F.gelu(z, approximate="tanh"))[case["act"]]

    def f():
        return [act(F.linear(st["x"], st["w_gate"], st["b_gate"])) * F.linear(st["x"], st["w_up"], st["b_up"])]

    if not case["train"]:
        return f()[0]
    names = [n for n in ("x", "w_gate", "w_up", "b_gate", "b_up") if st[n] is not None]
    (h,), grads = _through(f, [st[n] for n in names], [st["dh"]])
    return dict(zip(["h"] + names, [h, *grads]))


def _exact_qk(st, case):
    F = torch.nn.functional
    D, R = case["head_dim"], case["rotary"]
    at = torch.arange(R // 2, device="cuda")
    first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + R // 2)
    turn = torch.complex(st["table"][..., 0], st["table"][..., 1])[st["positions"].long()].unsqueeze(2)

    def one(x, w, b):
        if case["norm"] == "layer":
            x = F.layer_norm(x, (D,), w, b, 1e-5)
        elif case["norm"] == "rms":
            x = w * x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def f():
        return [one(st["q"], st["q_weight"], st["q_bias"]), one(st["k"], st["k_weight"], st["k_bias"])]

    if not case["train"]:
        return tuple(f())
    names = [n for n in ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias") if st[n] is not None]
    ys, grads = _through(f, [st[n] for n in names], [st["dq"], st["dk"]])
    return dict(zip(["yq", "yk"] + names, [*ys, *grads]))


def _exact_attn(st, case):
    """Head by head over slabs of queries, every key of the sequence scored."""
    B, S, H, D = st["q"].shape
    N = H // st["k"].shape[2]
    outs = [torch.zeros_like(st["q"])]
    if case["train"]:
        outs += [torch.zeros_like(st[n]) for n in ("q", "k", "v")]
    j = torch.arange(S, device="cuda")
    slab = max(1, 2 ** 26 // S)
    for b in range(B):
        L = S if st["lengths"] is None else int(st["lengths"][b])
        for h in range(H):
            k, v = st["k"][b, :, h // N], st["v"][b, :, h // N]
            for i0 in range(0, S, slab):
                i = torch.arange(i0, min(S, i0 + slab), device="cuda")[:, None]
                near = (i - j < case["window"]) & ((j <= i) if case["causal"] else (j - i < case["window"]))
                see = (near | ((j < case["sinks"]) & ((j <= i) if case["causal"] else (j >= 0)))) & (j < L)
                q = st["q"][b, i0:i0 + slab, h]
                p = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(~see, -math.inf), -1)
                p = torch.nan_to_num(p, nan=0.0)
                o = p @ v
                outs[0][b, i0:i0 + slab, h] = o
                if case["train"]:
                    do = st["do"][b, i0:i0 + slab, h]
                    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(D)
                    outs[1][b, i0:i0 + slab, h] = ds @ k
                    outs[2][b, :, h // N] += ds.T @ q
                    outs[3][b, :, h // N] += p.T @ do
    return tuple(outs) if case["train"] else outs[0]


def _exact_step(st, case):
    B, H, D = st["q"].shape
    Hk, cap = st["k"].shape[1], st["k_cache"].shape[1]
    o = torch.zeros_like(st["q"])
    for b, n in enumerate(_history(case)):
        slot = n if n < cap else case["sinks"] + (n - case["sinks"]) % case["window"]
        st["k_cache"][b, slot], st["v_cache"][b, slot] = st["k"][b], st["v"][b]
        seen = min(n + 1, cap)
        k, v = (st[m][b, :seen].repeat_interleave(H // Hk, 1) for m in ("k_cache", "v_cache"))
        p = torch.softmax(torch.einsum("hd,nhd->hn", st["q"][b], k) / math.sqrt(D), -1)
        o[b] = torch.einsum("hn,nhd->hd", p, v)
    return o, st["k_cache"], st["v_cache"]


def _exact_clip(st, case):
    flat = torch.cat([t.double().flatten() for t in st["grads"]])
    norm = torch.linalg.vector_norm(flat)
    return norm, flat * min(1.0, st["max_norm"] / (float(norm) + 1e-6))


_EXACT = {"gated": _exact_gated, "qk": _exact_qk, "attn": _exact_attn, "step": _exact_step, "clip": _exact_clip}
