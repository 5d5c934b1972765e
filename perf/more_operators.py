"""The operators of a gated delta layer, as cases that can be timed and checked.

The layer is  projection -> norms of the heads' keys and queries -> gated delta rule -> group norm, gated -> projection,
and its operators here are

  delta       S_t = e^(g_t) S_(t-1) + beta_t k_t (v_t - e^(g_t) S_(t-1)' k_t)',  o_t = scale S_t' q_t, for every head's state
              S of N keys x P values; several value heads may share a head of queries and keys
  delta_bwd   its gradients with respect to q, k, v, g, beta and the state carried in
  norm        n = (x - mean) / sqrt(variance + eps) over each group of a token's channels, z = n w + b, and
              y = z silu(gate), or silu(z) without a gate, stored as it is or in 8 bits (e4m3) with a power-of-two scale for
              each block of 128 channels
  norm_bwd    the gradients of y with respect to x, w, b and the gate

`run` computes them by elementary torch operations in 32 bits (sums of g in 64), or, where `own` is true, by the calls
that a user of helix_amd makes. Widths are those of the layers that the scan's benchmark has: 64 heads of 64 with 128
keys in 8 groups, 80 heads of 64, 27 heads of 192.

Options of a case. delta: `seqs` sequences of `tokens` tokens, `qk_heads` heads of `keys` channels of q and k, `heads` of
`values` channels of v, storage type `store`, `carry`: a state is carried in, `packed`: q, k and v are column ranges of one
projected row per token. norm: `rows` tokens of `dim` channels in `groups`, `store`, `gate` or none, `fp8` output.
"""
import math

import torch

own = False

STORE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BLOCK = 128
CHUNK = 64


def _delta(seqs, tokens, qk_heads, heads, keys, values, store="bf16", carry=False, packed=True, op="delta"):
    return {"op": op, "seqs": seqs, "tokens": tokens, "qk_heads": qk_heads, "heads": heads, "keys": keys,
            "values": values, "store": store, "carry": carry, "packed": packed}


def _norm(rows, dim, groups, store="bf16", gate=True, fp8=False):
    return {"op": "norm", "rows": rows, "dim": dim, "groups": groups, "store": store, "gate": gate, "fp8": fp8}


def _norm_bwd(rows, dim, groups, store="bf16", gate=True):
    return {"op": "norm_bwd", "rows": rows, "dim": dim, "groups": groups, "store": store, "gate": gate}


def listed():
    cases = [
        # The next token of one conversation: latency.
        ("delta - one token", _delta(1, 1, 8, 64, 128, 64, carry=True)),
        # The next token of 64 conversations: every state is read and written.
        ("delta - 64 single tokens", _delta(64, 1, 8, 64, 128, 64, carry=True)),
        # A short user turn on a conversation's state.
        ("delta - turn of 67 tokens", _delta(1, 67, 8, 64, 128, 64, carry=True)),
        # A long prompt.
        ("delta - 8k prompt", _delta(1, 8192, 8, 64, 128, 64)),
        # A ragged batch in 32 bits, heads of their own queries and keys, states carried in.
        ("delta - ragged batch f32", _delta(3, 1003, 27, 27, 64, 192, store="f32", carry=True, packed=False)),
        # A training step on four sequences: the rule's gradients.
        ("delta backward - batch of 4", _delta(4, 2048, 8, 64, 128, 64, op="delta_bwd")),
        # A training step on short samples with few, odd heads.
        ("delta backward - ragged f16", _delta(2, 333, 5, 5, 40, 72, store="f16", carry=True, packed=False, op="delta_bwd")),
        # The next token of one conversation, before the layer's last projection in 8 bits: latency.
        ("norm - one token", _norm(1, 4096, 64, fp8=True)),
        # A long prompt, before the same projection.
        ("norm - 8k prompt", _norm(8192, 4096, 64, fp8=True)),
        # A ragged batch through a layer kept in 32 bits, without a gate or an 8-bit output.
        ("norm - ragged batch f32", _norm(2871, 5184, 27, store="f32", gate=False)),
        # A training step on eight sequences of an 80-head layer: the norm's gradients.
        ("norm backward - batch of 8", _norm_bwd(32768, 5120, 80)),
        # A training step on short samples with groups of an odd width.
        ("norm backward - ragged f16", _norm_bwd(1003, 2565, 27, store="f16")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, low, high):
    return _spread(rng, low, high) | 1


def draw(rng):
    op = rng.choice(["delta", "delta", "delta", "delta_bwd", "delta_bwd", "norm", "norm", "norm_bwd", "norm_bwd"])
    store = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_bwd"):
        rows = _spread(rng, 1, 32768)
        width = rng.choice([64, 64, 128, 192, 8 * _spread(rng, 1, 64), _odd(rng, 3, 1023)])
        groups = max(1, min(_spread(rng, 1, 128), 8192 // width))
        while rows * groups * width * (2 if store == "f32" else 1) > 32768 * 5120:
            rows = max(1, rows // 2)
        if op == "norm_bwd":
            return _norm_bwd(rows, groups * width, groups, store, rng.random() < 0.6)
        return _norm(rows, groups * width, groups, store, rng.random() < 0.6, rng.random() < 0.5)
    qk_heads = rng.choice([1, 2, 4, 8, _spread(rng, 1, 32)])
    heads = qk_heads * rng.choice([1, 1, 2, 3, 8])
    keys = rng.choice([64, 128, 128, 8 * _spread(rng, 1, 16), _odd(rng, 5, 127)])
    values = rng.choice([64, 64, 128, 192, 8 * _spread(rng, 1, 32), _odd(rng, 5, 255)])
    seqs = rng.choice([1, 1, 2, 3, 8, 64])
    tokens = rng.choice([_spread(rng, 1, 128), _spread(rng, 64, 8192), _spread(rng, 64, 8192)])
    if op == "delta":
        tokens = rng.choice([1, tokens, tokens])
    # At most what the listed ones cost: their states, their tokens, and chunks one after another.
    while seqs > 1 and seqs * heads * keys * values > 64 * 64 * 128 * 64:
        seqs //= 2
    while tokens > 1 and seqs * tokens * heads * keys * values * (2 if store == "f32" else 1) > 4 * 2048 * 64 * 128 * 64:
        tokens //= 2
    return _delta(seqs, tokens, qk_heads, heads, keys, values, store, rng.random() < 0.5, rng.random() < 0.5, op)


# ---- inputs --------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = STORE[case["store"]]
    if case["op"] in ("norm", "norm_bwd"):
        rows, dim, groups = case["rows"], case["dim"], case["groups"]
        # Heads of different sizes, as a state's outputs are.
        x = ((normal(rows, groups, dim // groups) + 0.2 * normal(groups, 1)) * torch.exp(0.5 * normal(groups, 1)))
        x = x.reshape(rows, dim).to(st)
        w, b = 1 + 0.2 * normal(dim), 0.1 * normal(dim)
        gate = normal(rows, dim).to(st) if case["gate"] else None
        state = {"op": case["op"], "groups": groups, "x": x, "w": w, "b": b, "gate": gate}
        if case["op"] == "norm":
            state["fp8"] = case["fp8"]
        else:
            h = x.unflatten(-1, (groups, -1)).double()
            mean = h.mean(-1)
            state["rstd"] = torch.rsqrt((h - mean[..., None]).square().mean(-1) + EPS).float()
            state["mean"] = mean.float()
            state["dy"] = normal(rows, dim).to(st)
        return state
    S, L, Hk, H, N, P = (case[k] for k in ("seqs", "tokens", "qk_heads", "heads", "keys", "values"))
    # Keys and queries of length one (but for their rounding), as a layer norms them.
    q, k = (torch.nn.functional.normalize(normal(S, L, Hk, N), dim=-1) for _ in range(2))
    v = normal(S, L, H, P)
    if case["packed"]:
        row = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(st)
        q, k, v = row.split([Hk * N, Hk * N, H * P], -1)
        q, k, v = q.unflatten(-1, (Hk, N)), k.unflatten(-1, (Hk, N)), v.unflatten(-1, (H, P))
    else:
        q, k, v = q.to(st), k.to(st), v.to(st)
    # Heads that forget within a few tokens and heads that remember thousands.
    rate = torch.exp(normal(H) * 1.5 - 2.5)
    g = -rate * torch.nn.functional.softplus(normal(S, L, H))
    beta = torch.sigmoid(normal(S, L, H))
    state = {"op": case["op"], "q": q, "k": k, "v": v, "g": g, "beta": beta,
             "s0": 0.3 * normal(S, H, N, P) if case["carry"] else None}
    if case["op"] == "delta_bwd":
        state["do"] = normal(S, L, H, P).to(st)
        state["ds"] = normal(S, H, N, P) if case["carry"] else None
    return state


# ---- plain forms ---------------------------------------------------------------

def _blocks(x, value=0.0):
    """x with its last dimension in blocks of 128, the last one filled up."""
    fill = -x.shape[-1] % BLOCK
    if fill:
        x = torch.nn.functional.pad(x, (0, fill), value=value)
    return x.unflatten(-1, (-1, BLOCK))


def _quantize(y):
    """y in e4m3 and the scales: the lowest power of two at which a block's largest magnitude is at most 448."""
    b = _blocks(y)
    mantissa, exponent = torch.frexp(b.abs().amax(-1))            # magnitude = mantissa 2^exponent, mantissa in [1/2, 1)
    exponent = exponent - 9 + (mantissa > 0.875).int()            # 448 = 0.875 * 2^9
    exponent = torch.where(mantissa == 0, -126, exponent.clamp(min=-126))
    one = torch.ones_like(mantissa)
    q = (b * torch.ldexp(one, -exponent)[..., None]).flatten(-2)[..., :y.shape[-1]]
    return q.to(torch.float8_e4m3fn), torch.ldexp(one, exponent).to(torch.float8_e8m0fnu)


def _chunks(x, heads, dtype=torch.float32):
    """x [S, L, h, ...] as [S heads, chunks, up to CHUNK tokens, ...], heads repeated where several share one, zeros past the
    last token."""
    x = x.to(dtype)
    size = min(CHUNK, x.shape[1])
    if x.shape[2] != heads:
        x = x.repeat_interleave(heads // x.shape[2], 2)
    x = x.transpose(1, 2).flatten(0, 1)
    fill = -x.shape[1] % size
    if fill:
        x = torch.cat([x, x.new_zeros(x.shape[0], fill, *x.shape[2:])], 1)
    return x.unflatten(1, (-1, size))


def _tokens(x, like):
    """What _chunks laid out, back to like's [S, L, h, ...]."""
    x = x.flatten(1, 2)[:, :like.shape[1]].unflatten(0, (like.shape[0], -1))
    return x.transpose(1, 2).contiguous()


def _parts(s):
    """Per chunk: q (scaled), k, v, beta; decays from the chunk's start and to its end, and between its tokens; the inverse
    of 1 + A, A[i, j] = beta_i decay_ij k_i k_j below the diagonal; and the products of q and k with their decays."""
    H = s["v"].shape[2]
    q, k, v = (_chunks(s[n], H) for n in ("q", "k", "v"))
    q = q * s["q"].shape[-1] ** -0.5
    beta, G = _chunks(s["beta"], H), _chunks(s["g"], H, torch.float64).cumsum(-1)
    size = G.shape[-1]
    low = torch.ones(size, size, device=q.device, dtype=torch.bool).tril()
    E = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], -torch.inf)).float()
    start, left = torch.exp(G).float(), torch.exp(G[..., -1:] - G).float()
    kt = k.transpose(-1, -2).contiguous()
    A = (beta[..., None] * E * (k @ kt)).tril(-1)
    T = torch.eye(size, device=q.device).expand_as(A).clone()
    for i in range(1, size):
        T[..., i:i + 1, :i] = -(A[..., i:i + 1, :i] @ T[..., :i, :i])
    return {"q": q, "k": k, "v": v, "beta": beta, "E": E, "start": start, "left": left, "A": A, "T": T, "P": E * (q @ kt)}


def _first_state(s):
    S, _, H, P = s["v"].shape
    if s["s0"] is None:
        return torch.zeros(S * H, s["q"].shape[-1], P, device=s["v"].device)
    return s["s0"].flatten(0, 1)


def _walk(p, state):
    """The states that the chunks start from, what each chunk's tokens bring (D) and the state after the last."""
    states, brought = [], []
    for c in range(p["k"].shape[1]):
        states.append(state)
        k = p["k"][:, c]
        rest = p["v"][:, c] - p["start"][:, c, :, None] * (k @ state)
        d = p["T"][:, c] @ (p["beta"][:, c, :, None] * rest)
        state = p["start"][:, c, -1, None, None] * state + (k * p["left"][:, c, :, None]).transpose(-1, -2).contiguous() @ d
        brought.append(d)
    return torch.stack(states, 1), torch.stack(brought, 1), state


def _delta_forward(s):
    p = _parts(s)
    states, d, last = _walk(p, _first_state(s))
    o = p["start"][..., None] * (p["q"] @ states) + p["P"] @ d
    S, _, H, _ = s["v"].shape
    return {"o": _tokens(o, s["v"]).to(s["v"].dtype), "s": last.unflatten(0, (S, H))}


def _shared(x, like):
    """Gradients of heads that share one of like's, added."""
    x = _tokens(x, like)
    return x.unflatten(2, (like.shape[2], -1)).sum(3)


def _delta_backward(s):
    p = _parts(s)
    S, L, H, P = s["v"].shape
    N = s["q"].shape[-1]
    states, d, _ = _walk(p, _first_state(s))
    do = _chunks(s["do"], H)
    ds = torch.zeros(S * H, N, P, device=do.device) if s["ds"] is None else s["ds"].flatten(0, 1)
    q, k, beta, start, left = p["q"], p["k"], p["beta"], p["start"], p["left"]
    ends, z = [], []
    for c in range(k.shape[1] - 1, -1, -1):
        ends.append(ds)
        dd = p["P"][:, c].transpose(-1, -2).contiguous() @ do[:, c] + (k[:, c] * left[:, c, :, None]) @ ds
        zc = p["T"][:, c].transpose(-1, -2).contiguous() @ dd
        z.append(zc)
        ds = (start[:, c, -1, None, None] * ds + (q[:, c] * start[:, c, :, None]).transpose(-1, -2).contiguous() @ do[:, c]
              - (k[:, c] * start[:, c, :, None]).transpose(-1, -2).contiguous() @ (beta[:, c, :, None] * zc))
    ends, z = torch.stack(ends[::-1], 1), torch.stack(z[::-1], 1)
    dr = beta[..., None] * z
    st, et, dt = (x.transpose(-1, -2).contiguous() for x in (states, ends, d))
    dP, dA = (do @ dt).tril(), -(z @ dt).tril(-1)
    out, back, last = do @ st, dr @ st, d @ et        # of q, of k through the chunk's start, of k to its end
    dp, da = dP * p["E"], dA * p["E"] * beta[..., None]
    dq = start[..., None] * out + dp @ k
    dk = (left[..., None] * last - start[..., None] * back + dp.transpose(-1, -2).contiguous() @ q + da @ k
          + da.transpose(-1, -2).contiguous() @ k)
    rest = p["v"] - start[..., None] * (k @ states)
    dbeta = (z * rest).sum(-1) + (dA * (p["E"] * (k @ k.transpose(-1, -2).contiguous())).tril(-1)).sum(-1)
    # What the sums of g from the chunk's start get; g_t gets those of t and after it.
    pairs, tail = dP * p["P"] + dA * p["A"], left * (k * last).sum(-1)
    dG = pairs.sum(-1) - pairs.sum(-2) + start * ((q * out).sum(-1) - (k * back).sum(-1)) - tail
    dG[..., -1] += tail.sum(-1) + start[..., -1] * (states * ends).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    t = s["v"].dtype
    return {"dq": (_shared(dq, s["q"]) * N ** -0.5).to(t), "dk": _shared(dk, s["k"]).to(t), "dv": _tokens(dr, s["v"]).to(t),
            "dg": _tokens(dg, s["g"]), "dbeta": _tokens(dbeta, s["g"]), "ds0": ds.unflatten(0, (S, H))}


def _norm_forward(s):
    h = s["x"].float().unflatten(-1, (s["groups"], -1))
    mean = h.mean(-1)
    h = h - mean[..., None]
    rstd = torch.rsqrt(h.square().mean(-1) + EPS)
    z = (h * rstd[..., None]).flatten(-2) * s["w"] + s["b"]
    a = z if s["gate"] is None else s["gate"].float()
    y = (a / (1 + torch.exp(-a))) if s["gate"] is None else z * (a / (1 + torch.exp(-a)))
    if s["fp8"]:
        q, scale = _quantize(y)
        return {"q": q, "scale": scale}
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _norm_backward(s):
    t = s["x"].dtype
    h = s["x"].float().unflatten(-1, (s["groups"], -1))
    n = ((h - s["mean"][..., None]) * s["rstd"][..., None]).flatten(-2)
    z, dy = n * s["w"] + s["b"], s["dy"].float()
    a = z if s["gate"] is None else s["gate"].float()
    sig = 1 / (1 + torch.exp(-a))
    slope = sig * (1 + a * (1 - sig))
    dz = dy * slope if s["gate"] is None else dy * (a * sig)
    dn = (dz * s["w"]).unflatten(-1, (s["groups"], -1))
    ng = n.unflatten(-1, (s["groups"], -1))
    dx = s["rstd"][..., None] * (dn - dn.mean(-1, keepdim=True) - ng * (dn * ng).mean(-1, keepdim=True))
    return {"dx": dx.flatten(-2).to(t), "dw": (dz * n).sum(0), "db": dz.sum(0),
            "dgate": None if s["gate"] is None else (dy * z * slope).to(t)}


def _run_own(s):
    if s["op"] in ("delta", "delta_bwd"):
        from helix_amd.delta import delta_rule, delta_rule_backward

        if s["op"] == "delta":
            o, last = delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["s0"])
            return {"o": o, "s": last}
        grads = delta_rule_backward(s["do"], s["q"], s["k"], s["v"], s["g"], s["beta"], s["s0"], s["ds"])
        return dict(zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), grads))
    from helix_amd.norm import group_norm, group_norm_backward, group_norm_fp8

    if s["op"] == "norm" and s["fp8"]:
        q, scale = group_norm_fp8(s["x"], s["w"], s["b"], s["gate"], groups=s["groups"], activation="silu", eps=EPS)
        return {"q": q, "scale": scale}
    if s["op"] == "norm":
        y, mean, rstd = group_norm(s["x"], s["w"], s["b"], s["gate"], groups=s["groups"], activation="silu", eps=EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    dx, dw, db, dgate = group_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["b"], s["gate"],
                                            groups=s["groups"], activation="silu")
    return {"dx": dx, "dw": dw, "db": db, "dgate": dgate}


def run(state):
    if own:
        return _run_own(state)
    return {"delta": _delta_forward, "delta_bwd": _delta_backward, "norm": _norm_forward,
            "norm_bwd": _norm_backward}[state["op"]](state)


def work(case):
    es = BYTES[case["store"]]
    if case["op"] in ("norm", "norm_bwd"):
        each, stats = case["rows"] * case["dim"], 8 * case["rows"] * case["groups"]
        if case["op"] == "norm_bwd":
            return {"bytes": es * each * (5 if case["gate"] else 3) + stats + 16 * case["dim"], "flops": 25 * each}
        nbytes = es * each * (2 if case["gate"] else 1) + 8 * case["dim"]
        if case["fp8"]:
            nbytes += each + case["rows"] * -(-case["dim"] // BLOCK)
        else:
            nbytes += es * each + stats
        return {"bytes": nbytes, "flops": 15 * each}
    S, L, Hk, H, N, P = (case[k] for k in ("seqs", "tokens", "qk_heads", "heads", "keys", "values"))
    rows, state = S * L * (2 * Hk * N + H * P) * es, 4 * S * H * N * P
    if case["op"] == "delta":
        nbytes = rows + S * L * H * (P * es + 8) + state * (2 if case["carry"] else 1)
        return {"bytes": nbytes, "flops": 7 * S * L * H * N * P}
    nbytes = 2 * rows + S * L * H * (P * es + 16) + state * (3 if case["carry"] else 1)
    return {"bytes": nbytes, "flops": 20 * S * L * H * N * P}


# ---- in 64 bits ----------------------------------------------------------------

def _step(S, k, v, decay, beta):
    """The state after one token, and what the token brought."""
    S = decay[..., None, None] * S
    d = beta[..., None] * (v - (S * k[..., None]).sum(-2))
    return S + k[..., None] * d[..., None, :], d


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_bwd"):
        groups = case["groups"]
        x = s["x"].double().view(case["rows"], groups, -1)
        sig = None if s["gate"] is None else torch.sigmoid(s["gate"].double())
        w, b = s["w"].double(), s["b"].double()
        if case["op"] == "norm":
            mean, var = x.mean(-1), x.var(-1, correction=0)
            n = ((x - mean[..., None]) / (var + EPS).sqrt()[..., None]).view(case["rows"], -1)
            z = n * w + b
            y = z * torch.sigmoid(z) if sig is None else z * sig * s["gate"].double()
            if not case["fp8"]:
                return {"y": y, "mean": mean, "rstd": (var + EPS) ** -0.5}
            # Block by block; the quotients as they are before they are rounded to 8 bits.
            scale = torch.empty(case["rows"], -(-case["dim"] // BLOCK), device="cuda", dtype=torch.float64)
            for i in range(scale.shape[1]):
                part = y[:, i * BLOCK:(i + 1) * BLOCK]
                scale[:, i] = torch.exp2(torch.ceil(torch.log2(part.abs().max(1).values / 448)).clamp(min=-126))
                part /= scale[:, i, None]
            return {"q": y, "scale": scale}
        mean, rstd = s["mean"].double()[..., None], s["rstd"].double()[..., None]
        n = ((x - mean) * rstd).view(case["rows"], -1)
        z, dy = n * w + b, s["dy"].double()
        if sig is None:
            sig = torch.sigmoid(z)
            dz, dgate = dy * (sig + z * sig * (1 - sig)), None
        else:
            gate = s["gate"].double()
            dz, dgate = dy * gate * sig, dy * z * (sig + gate * sig * (1 - sig))
        t = (dz * w).view_as(x)
        n3 = n.view_as(x)
        dx = (t - t.mean(-1, keepdim=True) - n3 * (t * n3).mean(-1, keepdim=True)) * rstd
        return {"dx": dx.view(case["rows"], -1), "dw": (dz * n).sum(0), "db": dz.sum(0), "dgate": dgate}
    # Token by token.
    S, L, Hk, H, N, P = (case[k] for k in ("seqs", "tokens", "qk_heads", "heads", "keys", "values"))
    share = H // Hk
    scale = N ** -0.5

    def head(x, t):
        return x[:, t].double().repeat_interleave(share, 1)

    decay, beta = torch.exp(s["g"].double()), s["beta"].double()
    now = torch.zeros(S, H, N, P, device="cuda", dtype=torch.float64) if s["s0"] is None else s["s0"].double()
    if case["op"] == "delta":
        o = torch.empty(S, L, H, P, device="cuda", dtype=torch.float64)
        for t in range(L):
            now, _ = _step(now, head(s["k"], t), s["v"][:, t].double(), decay[:, t], beta[:, t])
            o[:, t] = scale * (now * head(s["q"], t)[..., None]).sum(-2)
        return {"o": o, "s": now}
    kept = []     # the state before every 64th token
    for t in range(L):
        if t % 64 == 0:
            kept.append(now)
        now, _ = _step(now, head(s["k"], t), s["v"][:, t].double(), decay[:, t], beta[:, t])
    dS = torch.zeros_like(now) if s["ds"] is None else s["ds"].double()
    like = {"device": "cuda", "dtype": torch.float64}
    dq, dk, dv = torch.empty(S, L, Hk, N, **like), torch.empty(S, L, Hk, N, **like), torch.empty(S, L, H, P, **like)
    dg, dbeta = torch.empty(S, L, H, **like), torch.empty(S, L, H, **like)
    for start in range((L - 1) // 64 * 64, -1, -64):
        end = min(L, start + 64)
        before, now = [], kept[start // 64]
        for t in range(start, end):
            before.append(now)
            now, _ = _step(now, head(s["k"], t), s["v"][:, t].double(), decay[:, t], beta[:, t])
        for t in range(end - 1, start - 1, -1):
            q, k, v, do = head(s["q"], t), head(s["k"], t), s["v"][:, t].double(), s["do"][:, t].double()
            old = decay[:, t, :, None, None] * before[t - start]
            miss = v - (old * k[..., None]).sum(-2)
            d = beta[:, t, :, None] * miss
            new = old + k[..., None] * d[..., None, :]
            dq[:, t] = scale * (new * do[..., None, :]).sum(-1).view(S, Hk, share, N).sum(2)
            dS = dS + scale * q[..., None] * do[..., None, :]
            dd = (dS * k[..., None]).sum(-2)
            dmiss = beta[:, t, :, None] * dd
            dbeta[:, t], dv[:, t] = (dd * miss).sum(-1), dmiss
            each = (dS * d[..., None, :]).sum(-1) - (old * dmiss[..., None, :]).sum(-1)
            dk[:, t] = each.view(S, Hk, share, N).sum(2)
            dS = dS - k[..., None] * dmiss[..., None, :]
            dg[:, t] = (dS * old).sum((-1, -2))
            dS = decay[:, t, :, None, None] * dS
    return {"dq": dq, "dk": dk, "dv": dv, "dg": dg, "dbeta": dbeta, "ds0": dS}
