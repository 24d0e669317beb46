"""Cases of the token mixers of hybrid-attention models: the gated delta rule (chunked and single token), the causal
convolution in front of it, and the per-head norm + rotation of queries and keys.

Where ``own`` is false, ``run`` computes the plain form from elementary torch operations in 32 bits (exponents and
angles in 64, where their differences and far positions need it), rounded once at the end; where it is true, ``run``
makes the calls of ``loongforge_b200.ops``.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
BF16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # A packed row of chat samples: lengths around the 64-token chunk, a tensor-parallel shard of heads.
        {"name": "delta train ragged small", "op": "delta_train", "lens": "1,2,63,64,65,130,445", "hk": 2, "hv": 4,
         "dk": 128, "dv": 128},
        # One 4096-token row of pretraining with all heads of the 80B hybrid (16 key, 32 value heads).
        {"name": "delta train 4096", "op": "delta_train", "lens": "4096", "hk": 16, "hv": 32, "dk": 128, "dv": 128},
        # A long packed row of documents, the same heads.
        {"name": "delta train packed 16384", "op": "delta_train", "lens": "8192,4096,2048,1500,548", "hk": 16,
         "hv": 32, "dk": 128, "dv": 128},
        # Prefill of prompts that continue a state, a shard of the 27B hybrid's heads; outputs the state for decoding.
        {"name": "delta prefill with state", "op": "delta_prefill", "lens": "700,1024,333", "hk": 4, "hv": 12,
         "dk": 128, "dv": 128},
        # One conversation, one token: latency.
        {"name": "delta step 1", "op": "delta_step", "batch": 1, "slots": 4, "hk": 16, "hv": 32, "dk": 128, "dv": 128},
        # A busy server: 192 rows out of a pool of 256 states, the 27B hybrid's 48 value heads.
        {"name": "delta step 192", "op": "delta_step", "batch": 192, "slots": 256, "hk": 16, "hv": 48, "dk": 128,
         "dv": 128},
        # Convolution over q|k|v channels of the 0.8B hybrid (16 key and value heads), ragged packed row, with a bias.
        {"name": "conv train ragged", "op": "conv_train", "lens": "1,3,70,500,1027,446", "channels": 6144, "kernel": 4,
         "bias": True},
        # The 80B hybrid's channels over a long packed row.
        {"name": "conv train packed 16384", "op": "conv_train", "lens": "8192,4096,2048,1500,548", "channels": 8192,
         "kernel": 4, "bias": False},
        # Single tokens through the convolution's window.
        {"name": "conv step 1", "op": "conv_step", "batch": 1, "slots": 4, "channels": 8192, "kernel": 4,
         "bias": False},
        {"name": "conv step 192", "op": "conv_step", "batch": 192, "slots": 256, "channels": 10240, "kernel": 4,
         "bias": False},
        # 30B mixture of experts: 32 query heads in 4 groups of head dim 128, all of it rotated, positions of a packed row.
        {"name": "qk norm rope 128", "op": "qk", "tokens": 8192, "groups": 4, "rep": 8, "dim": 128, "rot": 128,
         "gated": False, "axes": 1, "interleaved": False, "offset": 0.0},
        # Vision-language hybrid: output-gated attention, head dim 256 with a quarter rotated, t/h/w positions, odd length.
        {"name": "qk norm rope 3 axes gated", "op": "qk", "tokens": 4099, "groups": 2, "rep": 16, "dim": 256, "rot": 64,
         "gated": True, "axes": 3, "interleaved": False, "offset": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total):
    """A text of sequence lengths that add up to `total`."""
    left, out = total, []
    for _ in range(rng.randint(0, 6)):
        n = _log(rng, 1, max(1, left))
        if n < left:
            out.append(n)
            left -= n
    return ",".join(str(n) for n in out + [left])


def draw(rng):
    op = rng.choice(["delta_train", "delta_train", "delta_prefill", "delta_step", "conv_train", "conv_step", "qk", "qk"])
    if op in ("delta_train", "delta_prefill"):
        hk = rng.choice([1, 2, 4, 8, 16])
        hv = hk * rng.choice([1, 2, 3])
        most = 16384 * 32 // hv // (1 if hv > 8 else 4)
        return {"op": op, "lens": _lens(rng, _log(rng, 1, min(8192, most))), "hk": hk, "hv": hv,
                "dk": rng.choice([64, 128, 128]), "dv": rng.choice([64, 128, 128])}
    if op == "delta_step":
        b, hk = _log(rng, 1, 192), rng.choice([1, 2, 4, 8, 16])
        return {"op": op, "batch": b, "slots": b + rng.randint(0, 64), "hk": hk, "hv": hk * rng.choice([1, 2, 3]),
                "dk": rng.choice([64, 128, 128]), "dv": rng.choice([64, 128, 128])}
    if op == "conv_train":
        return {"op": op, "lens": _lens(rng, _log(rng, 1, 16384)), "channels": 8 * _log(rng, 4, 1024),
                "kernel": rng.choice([2, 3, 4]), "bias": rng.random() < 0.5}
    if op == "conv_step":
        b = _log(rng, 1, 192)
        return {"op": op, "batch": b, "slots": b + rng.randint(0, 64), "channels": 8 * _log(rng, 4, 1280),
                "kernel": rng.choice([2, 3, 4]), "bias": rng.random() < 0.5}
    dim = rng.choice([64, 128, 256])
    axes = rng.choice([1, 2, 3])
    return {"op": "qk", "tokens": _log(rng, 1, 8192), "groups": rng.choice([1, 2, 4, 8]), "rep": rng.choice([1, 2, 4, 8]),
            "dim": dim, "rot": rng.choice([dim, dim // 2, dim // 4]), "gated": rng.random() < 0.5, "axes": axes,
            "interleaved": axes == 1 and rng.random() < 0.3, "offset": float(rng.choice([0, 1]))}


def _ints(text):
    return [int(n) for n in str(text).split(",")]


# ------------------------------------------------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp(max=20))))


def _gates(g, rows, hv):
    """Log decay and write strength as the layer makes them: a rate per head, a softplus of a projection; a sigmoid."""
    rate = _rand(g, hv) * 16 + 1e-3
    log_decay = -rate * _softplus(torch.randn(rows, hv, generator=g, device=DEV) + 1)
    beta = 1 / (1 + torch.exp(-torch.randn(rows, hv, generator=g, device=DEV)))
    return log_decay.contiguous(), beta.contiguous()


def _bounds(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"op": op}
    if op in ("delta_train", "delta_prefill", "delta_step"):
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        lens = [1] * case["batch"] if op == "delta_step" else _ints(case["lens"])
        T = sum(lens)
        # after the convolution and its SiLU: keys with a common mean, as in the model
        s["q"], s["k"] = (_silu(torch.randn(T, hk, dk, generator=g, device=DEV)).to(BF16) for _ in range(2))
        s["v"] = _silu(torch.randn(T, hv, dv, generator=g, device=DEV)).to(BF16)
        s["g"], s["beta"] = _gates(g, T, hv)
        s["lens"], s["cu"] = lens, _bounds(lens)
        if op == "delta_train":
            s["do"] = _randn(g, T, hv, dv)
        elif op == "delta_prefill":
            s["state"] = _randn(g, len(lens), hv, dk, dv, scale=0.1, dtype=torch.float32)
        else:
            s["state"] = _randn(g, case["slots"], hv, dk, dv, scale=0.1, dtype=torch.float32)
            s["slot"] = torch.randperm(case["slots"], generator=g, device=DEV)[:case["batch"]].to(torch.int32)
    elif op in ("conv_train", "conv_step"):
        C, K = case["channels"], case["kernel"]
        s["w"] = ((_rand(g, C, K) * 2 - 1) * K ** -0.5).to(BF16)
        s["b"] = _randn(g, C, scale=0.1) if case["bias"] else None
        if op == "conv_train":
            s["lens"] = _ints(case["lens"])
            s["cu"] = _bounds(s["lens"])
            s["x"], s["dy"] = _randn(g, sum(s["lens"]), C), _randn(g, sum(s["lens"]), C)
        else:
            s["x"] = _randn(g, case["batch"], C)
            s["state"] = _randn(g, case["slots"], C, K - 1)
            s["slot"] = torch.randperm(case["slots"], generator=g, device=DEV)[:case["batch"]].to(torch.int32)
    else:
        T, G, r, D, rot = case["tokens"], case["groups"], case["rep"], case["dim"], case["rot"]
        parts = 2 * r + 2 if case["gated"] else r + 2
        s["dims"] = (T, G, r, D, rot, case["gated"], case["interleaved"], case["offset"])
        s["qkv"] = _randn(g, T, G * parts * D)
        s["qw"], s["kw"] = (((_rand(g, D) - 0.5) * 0.4 + 1 - case["offset"]).to(BF16) for _ in range(2))
        s["dq"], s["dk"], s["dv"] = _randn(g, T, G * r, D), _randn(g, T, G, D), _randn(g, T, G, D)
        s["dgate"] = _randn(g, T, G, r, D) if case["gated"] else None
        half = rot // 2
        s["inv"] = (1e7 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(DEV, torch.float32)
        if case["axes"] == 1:  # positions restart at the packed row's sequence boundaries; a table of angles
            cut = max(1, int(T * 0.7))
            s["pos"] = torch.cat([torch.arange(cut), torch.arange(T - cut)]).to(DEV, torch.int32)
            s["table"] = (torch.arange(cut, device=DEV, dtype=torch.float32)[:, None] * s["inv"]).contiguous()
        else:  # an image in the middle of text: the axes part there, and text goes on behind the largest
            side = max(1, int(math.sqrt(T / 2)))
            n = min(T, side * side)
            lead = (T - n) // 2
            a = torch.arange(lead)
            grid = torch.stack([torch.zeros(n), torch.arange(n) // side, torch.arange(n) % side]).long() + lead
            tail = torch.arange(T - n - lead) + lead + side
            s["pos"] = torch.cat([a.expand(3, -1), grid, tail.expand(3, -1)], 1)[3 - case["axes"]:].to(DEV, torch.int32).contiguous()
            s["axis"] = (torch.arange(half) % case["axes"]).to(DEV, torch.int32)
    return s


# -------------------------------------------------------------------------------------------------------- plain forms


def _padded(lens, step):
    """Where token t lies when every sequence is padded to L, the longest length rounded up to `step`: [T]; and L."""
    L = -(-max(lens) // step) * step
    at = torch.arange(L, device=DEV) < torch.tensor(lens, device=DEV)[:, None]
    return at.reshape(-1).nonzero()[:, 0], L


def _spread(x, at, rows):
    return torch.zeros(rows, *x.shape[1:], device=DEV).index_copy(0, at, x)


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_delta(q, k, v, g, beta, lens, state):
    """Chunks of 64 tokens of all sequences at once: inside a chunk products of 64 x 64 matrices, from chunk to chunk the
    state, so that the loop over chunks is the recurrence itself. Float inputs; returns o [T, hv, dv] and the last states."""
    hk, hv, dk, dv, C = q.shape[1], v.shape[1], q.shape[2], v.shape[2], 64
    at, L = _padded(lens, C)
    N = len(lens)
    cut = lambda x: _spread(x, at, N * L).view(N, L // C, C, *x.shape[1:]).transpose(2, 3)  # noqa: E731
    q, k = _unit(q) * dk ** -0.5, _unit(k)
    if hv != hk:
        q, k = q.repeat_interleave(hv // hk, 1), k.repeat_interleave(hv // hk, 1)
    q, k, v, g, beta = cut(q), cut(k), cut(v), cut(g[..., None])[..., 0], cut(beta[..., None])  # [N, n, hv, C, ...]
    gc = g.double().cumsum(-1)
    low = torch.ones(C, C, device=DEV).tril() > 0
    decay = torch.exp((gc[..., :, None] - gc[..., None, :]).float().masked_fill(~low, -math.inf))
    m = (k @ k.transpose(-1, -2)) * decay * beta * torch.ones(C, C, device=DEV).tril(-1)
    # the inverse of I + m from blocks of doubled size: [[a, 0], [b, c]]^-1 = [[a^-1, 0], [-c^-1 b a^-1, c^-1]]
    inv, size = torch.ones_like(beta)[..., None], 1  # [..., block, size, size]
    while size < C:
        blocks = m.unflatten(-1, (-1, size)).unflatten(-3, (-1, size)).transpose(-2, -3)  # [..., row block, column block, ...]
        odd = torch.arange(0, C // size, 2, device=DEV)
        a, c = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        below = -c @ blocks[..., odd + 1, odd, :, :] @ a
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([below, c], -1)], -2)
        size *= 2
    inv = inv[..., 0, :, :]
    p = (q @ k.transpose(-1, -2)) * decay
    up, down = torch.exp(gc).float()[..., None], torch.exp(gc[..., -1:] - gc).float()[..., None]
    s = torch.zeros(N, hv, dk, dv, device=DEV) if state is None else state
    out = []
    for c in range(L // C):
        u = inv[:, c] @ (beta[:, c] * (v[:, c] - up[:, c] * (k[:, c] @ s)))
        out.append(up[:, c] * (q[:, c] @ s) + p[:, c] @ u)
        s = s * up[:, c, :, -1:] + (k[:, c] * down[:, c]).transpose(-1, -2) @ u
    o = torch.stack(out, 1).transpose(2, 3).reshape(N * L, hv, dv)
    return o.index_select(0, at), s


def _plain_conv(x, w, b, lens):
    K = w.shape[1]
    at, L = _padded(lens, 1)
    xp = _spread(x, at, len(lens) * L).view(len(lens), L, -1)
    xp = torch.cat([torch.zeros(len(lens), K - 1, x.shape[1], device=DEV), xp], 1)
    y = sum(xp[:, j:j + L] * w[:, j] for j in range(K))
    y = _silu(y if b is None else y + b)
    return y.reshape(-1, x.shape[1]).index_select(0, at)


def _plain_rot(x, ang, rot, interleaved):
    c, s = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    h = rot // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :h], x[..., h:rot])
    a, b = a * c - b * s, b * c + a * s
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _angles(s):
    """In 64 bits [T, rot/2]: the given table's rows, or position times frequency of each frequency's axis."""
    if "table" in s:
        return s["table"].double()[s["pos"].long()]
    return s["pos"].double()[s["axis"].long()].t() * s["inv"].double()


def _plain_qk(qkv, qw, kw, s):
    T, G, r, D, rot, gated, il, off = s["dims"]
    x = qkv.view(T, G, -1, D)
    n = lambda t, w: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * (w + off)  # noqa: E731
    ang = _angles(s)
    q = _plain_rot(n(x[:, :, :r].reshape(T, G * r, D), qw), ang, rot, il)
    k = _plain_rot(n(x[:, :, -2], kw), ang, rot, il)
    return (q, k, x[:, :, -1]) + ((x[:, :, r:2 * r],) if gated else ())


def _leaf(x):
    return None if x is None else x.float().requires_grad_()


def _bf(*ts):
    return [t.to(BF16) for t in ts if t is not None]


def _run_plain(s):
    op = s["op"]
    if op == "delta_train":
        x = [_leaf(s[n]) for n in ("q", "k", "v", "g", "beta")]
        o, _ = _plain_delta(*x, s["lens"], None)
        d = torch.autograd.grad(o, x, s["do"].float())
        return [o.detach().to(BF16)] + _bf(*d[:3]) + list(d[3:])
    if op == "delta_prefill":
        o, last = _plain_delta(s["q"].float(), s["k"].float(), s["v"].float(), s["g"], s["beta"], s["lens"], s["state"])
        return [o.to(BF16), last]
    if op == "delta_step":
        rep = s["v"].shape[1] // s["q"].shape[1]
        q = (_unit(s["q"].float()) * s["q"].shape[-1] ** -0.5).repeat_interleave(rep, 1)
        k = _unit(s["k"].float()).repeat_interleave(rep, 1)
        at = s["slot"].long()
        old = s["state"][at] * torch.exp(s["g"])[..., None, None]
        u = s["beta"][..., None] * (s["v"].float() - (k[..., None] * old).sum(-2))
        new = old + k[..., None] * u[..., None, :]
        s["state"][at] = new
        return [(q[..., None] * new).sum(-2).to(BF16), s["state"]]
    if op == "conv_train":
        x, w, b = _leaf(s["x"]), _leaf(s["w"]), _leaf(s["b"])
        y = _plain_conv(x, w, b, s["lens"])
        d = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"].float())
        return _bf(y.detach(), *d)
    if op == "conv_step":
        at = s["slot"].long()
        win = torch.cat([s["state"][at], s["x"][..., None]], -1)
        y = (win.float() * s["w"].float()).sum(-1)
        s["state"][at] = win[..., 1:]
        return [_silu(y if s["b"] is None else y + s["b"].float()).to(BF16), s["state"]]
    x, qw, kw = _leaf(s["qkv"]), _leaf(s["qw"]), _leaf(s["kw"])
    y = _plain_qk(x, qw, kw, s)
    up = [s[n].float() for n in ("dq", "dk", "dv", "dgate") if s[n] is not None]
    d = torch.autograd.grad(y, [x, qw, kw], up)
    return _bf(y[0].detach(), y[1].detach(), *d)


# ------------------------------------------------------------------------------------------------- the framework's calls


def _run_own(s):
    from loongforge_b200.ops import functional as OF
    from loongforge_b200.ops import linear_attn as LA

    op = s["op"]
    ask = lambda n: None if s[n] is None else s[n].detach().requires_grad_()  # noqa: E731
    if op == "delta_train":
        x = [ask(n) for n in ("q", "k", "v", "g", "beta")]
        o = LA.gated_delta_rule(*x, cu_seqlens=s["cu"])
        return [o.detach(), *torch.autograd.grad(o, x, s["do"])]
    if op == "delta_prefill":
        with torch.no_grad():
            return list(LA.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], cu_seqlens=s["cu"],
                                            initial_state=s["state"], output_final_state=True))
    if op == "delta_step":
        # the pool of states is updated in place, here as in the plain form: each pass goes on from the last one
        o = LA.gated_delta_rule_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], state_indices=s["slot"])
        return [o, s["state"]]
    if op == "conv_train":
        x, w, b = ask("x"), ask("w"), ask("b")
        y = LA.causal_conv1d(x, w, b, cu_seqlens=s["cu"], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"])]
    if op == "conv_step":
        y = LA.causal_conv1d_step(s["x"], s["state"], s["w"], s["b"], state_indices=s["slot"], activation="silu")
        return [y, s["state"]]
    T, G, r, D, rot, gated, il, off = s["dims"]
    x, qw, kw = ask("qkv"), ask("qw"), ask("kw")
    where = {"freqs": s["table"]} if "table" in s else {"inv_freq": s["inv"], "axis": s["axis"]}
    y = OF.qk_norm_rope(x, G, r, qw, kw, pos_ids=s["pos"], rot_dim=rot, interleaved=il, eps=1e-6, w_offset=off,
                        gated=gated, **where)
    up = [s[n] for n in ("dq", "dk", "dv", "dgate") if s[n] is not None]
    return [y[0].detach(), y[1].detach(), *torch.autograd.grad(y, [x, qw, kw], up)]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op in ("delta_train", "delta_prefill", "delta_step"):
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        rows = case["batch"] if op == "delta_step" else sum(_ints(case["lens"]))
        qk, vo, gates = rows * hk * dk * 2, rows * hv * dv * 2, rows * hv * 4
        if op == "delta_step":
            return {"bytes": 2 * qk + 2 * vo + 2 * gates + 8 * rows * hv * dk * dv, "flops": 7 * rows * hv * dk * dv}
        # per token and head: S^T k, S^T q and the outer product; the backward pass twice that
        flops = 6 * rows * hv * dk * dv
        if op == "delta_prefill":
            n = len(_ints(case["lens"]))
            return {"bytes": 2 * qk + 2 * vo + 2 * gates + 8 * n * hv * dk * dv, "flops": flops}
        return {"bytes": 4 * qk + 4 * vo + 4 * gates, "flops": 3 * flops}
    if op == "conv_train":
        n = sum(_ints(case["lens"])) * case["channels"]
        return {"bytes": 8 * n, "flops": n * (6 * case["kernel"] + 12)}
    if op == "conv_step":
        n, K = case["batch"] * case["channels"], case["kernel"]
        return {"bytes": 4 * n + 4 * n * (K - 1) + 2 * case["channels"] * K, "flops": n * (2 * K + 4)}
    T, G, r, D = case["tokens"], case["groups"], case["rep"], case["dim"]
    row = G * (2 * r + 2 if case["gated"] else r + 2) * D
    qk = G * (r + 1) * D
    # the packed row, q and k written; all upstream gradients read, the packed gradient written
    return {"bytes": 2 * T * (row + qk + row + row), "flops": 30 * T * qk}


# ------------------------------------------------------------------------------------------------------------- exact


def _exact_delta(s, train):
    """The recurrence token by token in 64 bits, all sequences side by side, and its reverse for the gradients; states
    are kept every 64 tokens and computed again from there. A step behind a sequence's end changes nothing."""
    lens, rep = s["lens"], s["v"].shape[1] // s["q"].shape[1]
    N, L, first = len(lens), max(lens), s["cu"].tolist()
    dk = s["q"].shape[-1]

    def lay(x):
        y = torch.zeros(L, N, *x.shape[1:], dtype=torch.float64, device=DEV)
        for n in range(N):
            y[:lens[n], n] = x[first[n]:first[n + 1]].double()
        return y

    def back(y):
        return torch.cat([y[:lens[n], n] for n in range(N)])

    qx, kx = lay(s["q"]), lay(s["k"])
    rq = 1 / torch.sqrt(qx.square().sum(-1, keepdim=True) + 1e-6)
    rk = 1 / torch.sqrt(kx.square().sum(-1, keepdim=True) + 1e-6)
    q = (qx * rq * dk ** -0.5).repeat_interleave(rep, 2)
    k = (kx * rk).repeat_interleave(rep, 2)
    v, a, beta = lay(s["v"]), torch.exp(lay(s["g"])), lay(s["beta"])
    S = s["state"].double() if s.get("state") is not None else torch.zeros(N, v.shape[2], dk, v.shape[3], dtype=torch.float64, device=DEV)
    o, marks = torch.empty_like(v), []

    def step(S, t):
        Sb = a[t][..., None, None] * S
        e = v[t] - (k[t].unsqueeze(-2) @ Sb).squeeze(-2)
        return Sb, e, Sb + k[t].unsqueeze(-1) * (beta[t][..., None] * e).unsqueeze(-2)

    for t in range(L):
        if train and t % 64 == 0:
            marks.append(S)
        S = step(S, t)[2]
        o[t] = (q[t].unsqueeze(-2) @ S).squeeze(-2)
    if not train:
        return [back(o), S]
    do = lay(s["do"])
    dq, dkk, dv, da, db = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(a), torch.zeros_like(beta)
    dS = torch.zeros_like(S)
    for c in range(len(marks) - 1, -1, -1):
        hi, kept, S = min(L, 64 * c + 64), [], marks[c]
        for t in range(64 * c, hi):
            Sb, e, S1 = step(S, t)
            kept.append((S, Sb, e, S1))
            S = S1
        for t in range(hi - 1, 64 * c - 1, -1):
            S0, Sb, e, S1 = kept.pop()
            dq[t] = (S1 @ do[t].unsqueeze(-1)).squeeze(-1)
            dS = dS + q[t].unsqueeze(-1) * do[t].unsqueeze(-2)
            du = (k[t].unsqueeze(-2) @ dS).squeeze(-2)
            db[t] = (du * e).sum(-1)
            de = beta[t][..., None] * du
            dv[t] = de
            dkk[t] = (dS @ (beta[t][..., None] * e).unsqueeze(-1) - Sb @ de.unsqueeze(-1)).squeeze(-1)
            dS = dS - k[t].unsqueeze(-1) * de.unsqueeze(-2)
            da[t] = (dS * S0).sum((-1, -2))
            dS = a[t][..., None, None] * dS
    fold = lambda d: d.unflatten(2, (-1, rep)).sum(3)  # noqa: E731
    dq, dkk = fold(dq) * dk ** -0.5, fold(dkk)
    dq = rq * (dq - qx * rq * rq * (dq * qx).sum(-1, keepdim=True))
    dkk = rk * (dkk - kx * rk * rk * (dkk * kx).sum(-1, keepdim=True))
    return [back(o), back(dq), back(dkk), back(dv), back(da * a), back(db)]


def _exact_conv(s):
    x, dy, w = s["x"].double(), s["dy"].double(), s["w"].double()
    K, first, ys, dxs = w.shape[1], s["cu"].tolist(), [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(w[:, 0])
    for lo, hi in zip(first, first[1:]):
        xs = torch.zeros(hi - lo + K - 1, x.shape[1], dtype=torch.float64, device=DEV)
        xs[K - 1:] = x[lo:hi]
        pre = torch.zeros_like(x[lo:hi]) if s["b"] is None else s["b"].double().expand(hi - lo, -1).clone()
        for j in range(K):
            pre += xs[j:j + hi - lo] * w[:, j]
        sig = 1 / (1 + torch.exp(-pre))
        ys.append(pre * sig)
        dp = dy[lo:hi] * sig * (1 + pre * (1 - sig))
        db += dp.sum(0)
        d = torch.zeros_like(xs)
        for j in range(K):
            dw[:, j] += (dp * xs[j:j + hi - lo]).sum(0)
            d[j:j + hi - lo] += dp * w[:, j]
        dxs.append(d[K - 1:])
    return [torch.cat(ys), torch.cat(dxs), dw] + ([] if s["b"] is None else [db])


def _exact_qk(s):
    T, G, r, D, rot, gated, il, off = s["dims"]
    x = s["qkv"].double().view(T, G, -1, D)
    ang = _angles(s)
    turn = torch.complex(torch.cos(ang), torch.sin(ang))[:, None, None]
    i = torch.arange(rot // 2, device=DEV)
    lo, hi = (2 * i, 2 * i + 1) if il else (i, i + rot // 2)

    def rotate(t, z):
        c = torch.complex(t[..., lo], t[..., hi]) * z
        y = t.clone()
        y[..., lo], y[..., hi] = c.real, c.imag
        return y

    dx, outs, dws = torch.zeros_like(x), [], []
    for sl, w, d in ((slice(0, r), s["qw"], s["dq"].view(T, G, r, D)), (slice(-2, -1), s["kw"], s["dk"].view(T, G, 1, D))):
        t, w = x[:, :, sl], w.double() + off
        n = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
        outs.append(rotate(t * n * w, turn).reshape(T, -1, D))
        d = rotate(d.double(), turn.conj())
        dws.append((d * t * n).sum((0, 1, 2)))
        d = d * w
        dx[:, :, sl] = n * d - t * n ** 3 * (d * t).mean(-1, keepdim=True)
    dx[:, :, -1] = s["dv"].double()
    if gated:
        dx[:, :, r:2 * r] = s["dgate"].double()
    return outs + [dx.view(T, -1)] + dws


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("delta_train", "delta_prefill"):
        # two loops over the longest sequence's tokens, whole states in 64 bits
        if max(s["lens"]) * (3 if op == "delta_train" else 1) > 40000 or len(s["lens"]) * max(s["lens"]) * s["v"].shape[1] > 3_000_000:
            return None
        return _exact_delta(s, op == "delta_train")
    if op == "delta_step":
        state = s["state"].double()
        s = {**s, "state": state[s["slot"].long()]}
        o, new = _exact_delta(s, False)
        state[s["slot"].long()] = new
        return [o, state]
    if op == "conv_train":
        return _exact_conv(s)
    if op == "conv_step":
        at, state = s["slot"].long(), s["state"].double()
        old, x, w = state[at], s["x"].double(), s["w"].double()
        y = x * w[:, -1] + (0 if s["b"] is None else s["b"].double())
        for j in range(old.shape[-1]):
            y = y + old[..., j] * w[:, j]
        state[at] = torch.cat([old[..., 1:], x[..., None]], -1)
        return [y / (1 + torch.exp(-y)), state]
    return _exact_qk(s)
