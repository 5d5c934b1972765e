"""The operators of a gated recurrent layer, as cases that can be timed and checked.

The layer is  residual + norm -> projection -> gated recurrence -> norm -> projection,  and its operators are

  norm        h = x + r;  y = h w / sqrt(mean(h^2) + eps), stored as it is or in 8 bits (e4m3) with a power-of-two
              scale for each block of 128 channels of a row
  norm_bwd    the gradients of y and h with respect to x (and r) and w
  matmul      C = A B^T with A and B in e4m3 and a power-of-two scale for each block of 128 along the products' sum
  scan        h_t = f_t h_(t-1) + (1 - f_t) v_t,  f_t = sigmoid(g_t), for every channel by itself
  scan_bwd    its gradients with respect to g, v and the state carried in

`run` computes them by elementary torch operations in 32 bits, or, where `own` is true, by the calls that a user of
helix_amd makes. Widths are those of the layers that the scan's benchmark has: 64 heads of 64 (2048 channels of the
model, 4096 inside, projections of 10304 columns), 80 heads of 64 (2560 and 5120) and 27 heads of 192 (5184).

Options of a case. norm: `rows` tokens of `dim` channels, storage type `store`, `residual` or none, `fp8` output or
one of the storage type. matmul: `m`, `n`, `k`, the output's type `store`. scan: `seqs` sequences of `tokens` tokens
of `dim` channels, `store`, `carry`: a state is carried in, `packed`: g and v are column ranges of one projected row
per token and not tensors of their own.
"""
import math

import torch

own = False

STORE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BLOCK = 128


def _norm(rows, dim, store="bf16", residual=True, fp8=True):
    return {"op": "norm", "rows": rows, "dim": dim, "store": store, "residual": residual, "fp8": fp8}


def _norm_bwd(rows, dim, store="bf16", residual=True):
    return {"op": "norm_bwd", "rows": rows, "dim": dim, "store": store, "residual": residual}


def _matmul(m, n, k, store="bf16"):
    return {"op": "matmul", "m": m, "n": n, "k": k, "store": store}


def _scan(seqs, tokens, dim, store="bf16", carry=False, packed=True, op="scan"):
    return {"op": op, "seqs": seqs, "tokens": tokens, "dim": dim, "store": store, "carry": carry, "packed": packed}


def listed():
    cases = [
        # The next token of one conversation, before the layer's first projection: latency.
        ("norm, one token", _norm(1, 2048)),
        # A long prompt, before the same projection.
        ("norm, 8k prompt", _norm(8192, 2048)),
        # A ragged batch through a layer kept in 32 bits, without a residual or an 8-bit output.
        ("norm, ragged batch, f32", _norm(2871, 5184, store="f32", residual=False, fp8=False)),
        # A training step on eight sequences: the norm's gradients, the residual's added.
        ("norm backward, batch of 8", _norm_bwd(32768, 2560)),
        # The next token of one conversation through the first projection: the weights are read once.
        ("projection, one token", _matmul(1, 10304, 2048)),
        # A short user turn through the last projection.
        ("projection, turn of 67 tokens", _matmul(67, 2048, 4096)),
        # A long prompt through the first projection.
        ("projection, 8k prompt", _matmul(8192, 10304, 2048)),
        # Batched prefill through the last projection of an 80-head layer.
        ("projection, batch of 8", _matmul(32768, 2560, 5120)),
        # The next token of 64 conversations through the recurrence.
        ("recurrence, 64 single tokens", _scan(64, 1, 4096, carry=True)),
        # A long prompt through the recurrence, g and v as the projection leaves them.
        ("recurrence, 8k prompt", _scan(1, 8192, 4096)),
        # A ragged batch in 32 bits, with states carried in.
        ("recurrence, ragged batch, f32", _scan(3, 1003, 5184, store="f32", carry=True, packed=False)),
        # A training step on eight sequences: the recurrence's gradients.
        ("recurrence backward, batch of 8", _scan(8, 4096, 5120, op="scan_bwd")),
    ]
    return [dict(case, name=name) for name, case in cases]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _odd(rng, low, high):
    return _spread(rng, low, high) | 1


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "matmul", "matmul", "matmul", "scan", "scan", "scan_bwd"])
    store = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_bwd"):
        rows = _spread(rng, 1, 32768)
        dim = rng.choice([_odd(rng, 128, 8192), 16 * _odd(rng, 8, 512), 2048, 2560, 4096, 5184])
        while rows * dim * (2 if store == "f32" else 1) > 32768 * 2560:
            rows = max(1, rows // 2)
        if op == "norm_bwd":
            return _norm_bwd(rows, dim, store, rng.random() < 0.7)
        return _norm(rows, dim, store, rng.random() < 0.7, rng.random() < 0.6)
    if op == "matmul":
        m = _spread(rng, 1, 32768)
        n = rng.choice([_odd(rng, 64, 10576), 8 * _odd(rng, 8, 1300), 2048, 2560, 4096, 5184, 10304, 10576])
        k = rng.choice([16 * _odd(rng, 8, 400), 128 * _odd(rng, 2, 50), 2048, 2560, 4096, 5120, 5184])
        while m * n * k > 32768 * 2560 * 5120:
            m //= 2
        return _matmul(m, n, k, store)
    seqs = rng.choice([1, 1, 2, 3, 8, 64, 256])
    tokens = rng.choice([1, 1, _spread(rng, 2, 256), _spread(rng, 64, 16384), _spread(rng, 64, 16384)])
    dim = rng.choice([_odd(rng, 64, 8192), 8 * _odd(rng, 8, 1024), 2048, 4096, 5120, 5184])
    while seqs * tokens * dim * (2 if store == "f32" else 1) > 8 * 4096 * 5120:
        seqs, tokens = max(1, seqs // 2), max(1, tokens // 2)
    return _scan(seqs, tokens, dim, store, rng.random() < 0.5, rng.random() < 0.6, op)


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


def _dequantize(q, scale, dtype=torch.float32):
    return (_blocks(q.to(dtype)) * scale.to(dtype)[..., None]).flatten(-2)[..., :q.shape[-1]]


def _linear(f, u):
    """y_t = f_t y_(t-1) + u_t along dimension 1 from y_(-1) = 0, by doubling the reach of each step."""
    d, length = 1, u.shape[1]
    while d < length:
        u = torch.cat([u[:, :d], u[:, d:] + f[:, d:] * u[:, :-d]], 1)
        if 2 * d < length:
            f = torch.cat([f[:, :d], f[:, d:] * f[:, :-d]], 1)
        d *= 2
    return u


def _plain_scan(g, v, h0):
    g, v = g.float(), v.float()
    f, u = torch.sigmoid(g), torch.sigmoid(-g) * v
    if h0 is not None:
        u[:, 0] += f[:, 0] * h0
    return _linear(f, u)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] in ("norm", "norm_bwd"):
        rows, dim, st = case["rows"], case["dim"], STORE[case["store"]]
        # A few channels carry much more than the others, as a residual stream's do.
        channel = torch.exp(0.5 * normal(dim)) * (1 + 15 * (torch.rand(dim, generator=gen, device="cuda") < 0.01))
        x = (normal(rows, dim) * channel).to(st)
        w = 1 + 0.2 * normal(dim)
        other = normal(rows, dim).to(st) if case["residual"] else None
        if case["op"] == "norm":
            return {"op": "norm", "fp8": case["fp8"], "x": x, "w": w, "residual": other}
        rstd = torch.rsqrt(x.float().square().mean(-1) + EPS)
        return {"op": "norm_bwd", "dy": normal(rows, dim).to(st), "h": x, "w": w, "rstd": rstd, "dh": other}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        a = normal(m, k) * torch.exp(0.5 * normal(k))
        a, a_scale = _quantize(a)
        b, b_scale = _quantize(normal(n, k) / math.sqrt(k))
        return {"op": "matmul", "a": a, "a_scale": a_scale, "b": b, "b_scale": b_scale, "store": STORE[case["store"]]}
    seqs, tokens, dim, st = case["seqs"], case["tokens"], case["dim"], STORE[case["store"]]
    # Gates of a trained layer: mostly open to the past, some nearly closed.
    if case["packed"]:
        row = torch.empty(seqs, tokens, 2 * dim, device="cuda", dtype=st)
        row[..., :dim] = 2 + 1.5 * normal(seqs, tokens, dim)
        row[..., dim:] = normal(seqs, tokens, dim)
        g, v = row[..., :dim], row[..., dim:]
    else:
        g, v = (2 + 1.5 * normal(seqs, tokens, dim)).to(st), normal(seqs, tokens, dim).to(st)
    h0 = 0.5 * normal(seqs, dim) if case["carry"] else None
    state = {"op": case["op"], "g": g, "v": v, "h0": h0}
    if case["op"] == "scan_bwd":
        state["h"] = _plain_scan(g, v, h0).to(st)
        state["dh"] = normal(seqs, tokens, dim).to(st)
        state["dh_last"] = normal(seqs, dim) if case["carry"] else None
    return state


def _run_own(s):
    from helix_amd.matmul import matmul_fp8
    from helix_amd.norm import rms_norm, rms_norm_backward, rms_norm_fp8
    from helix_amd.recurrence import gated_scan, gated_scan_backward

    if s["op"] == "norm" and s["fp8"]:
        q, scale, h = rms_norm_fp8(s["x"], s["w"], s["residual"], eps=EPS)
        return {"q": q, "scale": scale, "h": h if s["residual"] is not None else None}
    if s["op"] == "norm":
        y, h, rstd = rms_norm(s["x"], s["w"], s["residual"], eps=EPS)
        return {"y": y, "rstd": rstd, "h": h if s["residual"] is not None else None}
    if s["op"] == "norm_bwd":
        dx, dw = rms_norm_backward(s["dy"], s["h"], s["w"], s["rstd"], s["dh"])
        return {"dx": dx, "dw": dw}
    if s["op"] == "matmul":
        return {"c": matmul_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=s["store"])}
    if s["op"] == "scan":
        h, last = gated_scan(s["g"], s["v"], s["h0"])
        return {"h": h, "last": last}
    dg, dv, dh0 = gated_scan_backward(s["dh"], s["g"], s["v"], s["h"], s["h0"], s["dh_last"])
    return {"dg": dg, "dv": dv, "dh0": dh0}


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        st = s["x"].dtype
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        rstd = torch.rsqrt(h.square().mean(-1) + EPS)
        y = h * rstd[:, None] * s["w"]
        kept = h.to(st) if s["residual"] is not None else None
        if s["fp8"]:
            q, scale = _quantize(y)
            return {"q": q, "scale": scale, "h": kept}
        return {"y": y.to(st), "rstd": rstd, "h": kept}
    if s["op"] == "norm_bwd":
        n = s["h"].float() * s["rstd"][:, None]
        dy = s["dy"].float()
        t = dy * s["w"]
        dx = s["rstd"][:, None] * (t - n * (t * n).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        return {"dx": dx.to(s["h"].dtype), "dw": (dy * n).sum(0)}
    if s["op"] == "matmul":
        c = _dequantize(s["a"], s["a_scale"]) @ _dequantize(s["b"], s["b_scale"]).t()
        return {"c": c.to(s["store"])}
    if s["op"] == "scan":
        h = _plain_scan(s["g"], s["v"], s["h0"])
        return {"h": h.to(s["g"].dtype), "last": h[:, -1].contiguous()}
    # lambda_t = dh_t + f_(t+1) lambda_(t+1): the same recurrence from the last token back.
    g, v, dh = s["g"].float(), s["v"].float(), s["dh"].float()
    f, stay = torch.sigmoid(g), torch.sigmoid(-g)
    if s["dh_last"] is not None:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dh_last"][:, None]], 1)
    after = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], 1)
    lam = _linear(after.flip(1), dh.flip(1)).flip(1)
    h0 = torch.zeros_like(lam[:, 0]) if s["h0"] is None else s["h0"]
    before = torch.cat([h0[:, None], s["h"][:, :-1].float()], 1)
    st = s["g"].dtype
    return {"dg": (lam * (before - v) * f * stay).to(st), "dv": (lam * stay).to(st), "dh0": f[:, 0] * lam[:, 0]}


def work(case):
    es = BYTES[case["store"]]
    if case["op"] == "norm":
        each = case["rows"] * case["dim"]
        nbytes = es * each * (3 if case["residual"] else 1) + 4 * case["dim"]
        if case["fp8"]:
            nbytes += each + case["rows"] * -(-case["dim"] // BLOCK)
        else:
            nbytes += es * each + 4 * case["rows"]
        return {"bytes": nbytes, "flops": 6 * each}
    if case["op"] == "norm_bwd":
        each = case["rows"] * case["dim"]
        return {"bytes": es * each * (4 if case["residual"] else 3) + 4 * case["rows"] + 8 * case["dim"], "flops": 10 * each}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + -(-k // BLOCK)) + es * m * n, "flops": 2 * m * n * k}
    each, states = case["seqs"] * case["tokens"] * case["dim"], case["seqs"] * case["dim"]
    if case["op"] == "scan":
        return {"bytes": es * 3 * each + 4 * states * (2 if case["carry"] else 1), "flops": 8 * each}
    return {"bytes": es * 6 * each + 4 * states * (3 if case["carry"] else 1), "flops": 14 * each}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        root = (h.pow(2).sum(1) / case["dim"] + EPS).sqrt()
        y = h / root[:, None] * s["w"].double()
        kept = h if s["residual"] is not None else None
        if not case["fp8"]:
            return {"y": y, "rstd": 1 / root, "h": kept}
        # Block by block; the quotients as they are before they are rounded to 8 bits.
        scale = torch.empty(case["rows"], -(-case["dim"] // BLOCK), device="cuda", dtype=torch.float64)
        for b in range(scale.shape[1]):
            part = y[:, b * BLOCK:(b + 1) * BLOCK]
            top = part.abs().max(1).values
            scale[:, b] = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-126))
            part /= scale[:, b, None]
        return {"q": y, "scale": scale, "h": kept}
    if case["op"] == "norm_bwd":
        h, dy, rstd = s["h"].double(), s["dy"].double(), s["rstd"].double()[:, None]
        dot = (dy * s["w"].double() * h).sum(1, keepdim=True) / case["dim"]
        dx = dy * s["w"].double() * rstd - h * (dot * rstd ** 3)
        if s["dh"] is not None:
            dx += s["dh"].double()
        return {"dx": dx, "dw": (dy * h * rstd).sum(0)}
    if case["op"] == "matmul":
        c = torch.zeros(case["m"], case["n"], device="cuda", dtype=torch.float64)
        for b in range(s["a_scale"].shape[1]):
            cut = slice(b * BLOCK, (b + 1) * BLOCK)
            a = s["a"][:, cut].double() * s["a_scale"][:, b, None].double()
            c += a @ (s["b"][:, cut].double() * s["b_scale"][:, b, None].double()).T
        return {"c": c}
    f = 1 / (1 + torch.exp(-s["g"].double()))
    v = s["v"].double()
    seqs, tokens, dim = v.shape
    h0 = torch.zeros(seqs, dim, device="cuda", dtype=torch.float64) if s["h0"] is None else s["h0"].double()
    if case["op"] == "scan":
        now = h0
        for t in range(tokens):
            now = v[:, t] + f[:, t] * (now - v[:, t])
            v[:, t] = now
        return {"h": v, "last": now}
    lam = torch.zeros_like(h0) if s["dh_last"] is None else s["dh_last"].double()
    for t in range(tokens - 1, -1, -1):
        past = h0 if t == 0 else s["h"][:, t - 1].double()
        lam = lam + s["dh"][:, t].double()
        gain = lam * (past - v[:, t])
        v[:, t] = lam * (1 - f[:, t])
        lam = lam * f[:, t]
        f[:, t] = gain * f[:, t] * (1 - f[:, t])
    return {"dg": f, "dv": v, "dh0": lam}
