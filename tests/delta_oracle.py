"""Plain 64-bit forms of the gated delta rule and its gradients on the CPU, token by token, and the bounds that the
kernels' arithmetic stays in (E, U and TINY as in layer_oracle.py).

What an output is a sum of has a size by norms: o_t = scale S_t' q_t is scale |q_t| |column of S_t| at most, and so on
(`Sizes`). The kernels form it by at most four products in a row (K S, X R, K' D, the output's own), each of up to 128 + 64
terms that are right to E and summed in fp32 with as many roundings. Roundings that go up as often as down leave
sqrt(192) E of the size for one product, sqrt(4 192) E = 28 E for four, and what a state is off by is carried on by maps of
norm one at most (keys of length one, beta up to 2, decays up to 1): FP32 = 32 E of the size, in the 2-norm over a whole
output. Outputs of 16 bits are rounded once more, U of themselves, after products of two parts of operands, 2^-17 of the
size (well below U)."""
from __future__ import annotations

import torch

from layer_oracle import E, TINY, U, f64

FP32 = 32 * E


def _heads(x, H):
    """x [S, L, Hk, N] in 64 bits with a head for every value head."""
    return f64(x).repeat_interleave(H // x.shape[2], 2)


def forward(q, k, v, g, beta, s0, scale):
    """(o, the states before the first token and after every one [L + 1][S, H, N, P], what the tokens brought)."""
    S, L, H, P = v.shape
    q, k, v, a, beta = _heads(q, H), _heads(k, H), f64(v), torch.exp(f64(g)), f64(beta)
    now = torch.zeros(S, H, q.shape[-1], P, dtype=torch.float64) if s0 is None else f64(s0)
    states, brought, o = [now], [], torch.zeros(S, L, H, P, dtype=torch.float64)
    for t in range(L):
        old = a[:, t, :, None, None] * now
        d = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None] @ old).squeeze(-2))
        now = old + k[:, t, ..., None] * d[..., None, :]
        o[:, t] = scale * (q[:, t, :, None] @ now).squeeze(-2)
        states.append(now)
        brought.append(d)
    return o, states, brought


def backward(do, q, k, v, g, beta, s0, ds, scale):
    """((dq, dk, dv, dg, dbeta, ds0), their sizes as norms) in 64 bits."""
    S, L, H, P = v.shape
    Hk, N = q.shape[2:]
    _, states, brought = forward(q, k, v, g, beta, s0, scale)
    q, k, v, a, beta, do = _heads(q, H), _heads(k, H), f64(v), torch.exp(f64(g)), f64(beta), f64(do)
    dS = torch.zeros(S, H, N, P, dtype=torch.float64) if ds is None else f64(ds)
    dq, dk = torch.zeros(S, L, H, N, dtype=torch.float64), torch.zeros(S, L, H, N, dtype=torch.float64)
    dv, dg, db = torch.zeros_like(v), torch.zeros_like(beta), torch.zeros_like(beta)
    size = {n: torch.zeros(()) .double() for n in ("dq", "dk", "dv", "dg", "dbeta")}
    top = dS.square().sum()
    for t in range(L - 1, -1, -1):
        old, new, d = a[:, t, :, None, None] * states[t], states[t + 1], brought[t]
        miss = v[:, t] - (k[:, t, :, None] @ old).squeeze(-2)
        dq[:, t] = scale * (new * do[:, t, :, None]).sum(-1)
        dS = dS + scale * q[:, t, ..., None] * do[:, t, :, None]
        z = (dS * k[:, t, ..., None]).sum(-2)
        bz = beta[:, t, :, None] * z
        dv[:, t], db[:, t] = bz, (z * miss).sum(-1)
        dk[:, t] = (dS * d[..., None, :]).sum(-1) - (old * bz[..., None, :]).sum(-1)
        e, s = dS.square().sum((-1, -2)), torch.maximum(old.square().sum((-1, -2)), new.square().sum((-1, -2)))
        kk = k[:, t].square().sum(-1)
        size["dq"] += (scale ** 2 * s * do[:, t].square().sum(-1)).sum()
        size["dv"] += (beta[:, t].square() * kk * e).sum()
        size["dk"] += (e * d.square().sum(-1) + s * beta[:, t].square() * kk * e).sum()
        size["dbeta"] += (kk * e * (v[:, t].square().sum(-1) + kk * s)).sum()
        size["dg"] += (e * s).sum()
        dS = dS - k[:, t, ..., None] * bz[..., None, :]
        dg[:, t] = (dS * old).sum((-1, -2))
        dS = a[:, t, :, None, None] * dS
        top = torch.maximum(top, dS.square().sum())
    size["ds0"] = top
    share = H // Hk
    dq, dk = dq.unflatten(2, (Hk, share)).sum(3), dk.unflatten(2, (Hk, share)).sum(3)
    # The heads that share are added one after another in fp32. With terms of norm s each, size = s sqrt(share), the sum of
    # the first h has s sqrt(h), and its rounding E of that: together E s sqrt(1 + 2 + .. + share) = E size sqrt(share / 2),
    # beside the 32 E of the size that the terms are off by.
    for n in ("dq", "dk"):
        size[n] *= (1 + (share / 2) ** 0.5 / 32) ** 2   # (sizes are squares here)
    return (dq, dk, dv, dg, db, dS), {n: float(x) ** 0.5 for n, x in size.items()}


def forward_sizes(q, states, scale, H):
    """(of o, of s) as norms."""
    qs = _heads(q, H).square().sum(-1)
    o = sum(float((qs[:, t] * s.square().sum((-1, -2))).sum()) for t, s in enumerate(states[1:]))
    return scale * o ** 0.5, max(float(s.norm()) for s in states)


def amplification(k, g, beta, H):
    """By how much forming X may enlarge a relative error: the largest row of |T| (1 + M) |T| |beta| over the chunks of 64,
    T the inverse and M the magnitudes that the entries below its diagonal are sums of."""
    k, g, beta = _heads(k, H).transpose(1, 2), f64(g).transpose(1, 2), f64(beta).transpose(1, 2)
    worst = 1.0
    for t in range(0, k.shape[2], 64):
        kc, G, b = k[:, :, t:t + 64], g[:, :, t:t + 64].cumsum(-1), beta[:, :, t:t + 64]
        low = torch.ones(G.shape[-1], G.shape[-1]).tril(-1).bool()
        decay = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], -torch.inf))
        A = b[..., None] * decay * (kc @ kc.transpose(-1, -2))
        M = b[..., None].abs() * decay * (kc.abs() @ kc.abs().transpose(-1, -2))
        eye = torch.eye(G.shape[-1], dtype=torch.float64)
        T = torch.linalg.inv(eye + A).abs()
        worst = max(worst, float((T @ (eye + M) @ T * b[..., None, :].abs()).sum(-1).max()))
    return worst


def close(got, want, size, dtype, what, amp=1.0):
    """The 2-norm of the difference within FP32 amp of the size and, stored in `dtype`, its rounding of every element."""
    got = f64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = FP32 * amp * size + 1e-30
    if dtype != torch.float32:
        fine += U[dtype] * float(want.norm()) * (1 + FP32) + 2.0 ** -17 * size + TINY[dtype] * want.numel() ** 0.5
    off = float((got - want).norm())
    assert off <= fine, f"{what}: off by {off:.3g}, {off / fine:.3g} of the bound"
