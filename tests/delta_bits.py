"""Problems of the delta rule whose 16-bit results are small differences of large sums, so that an operand which has lost
bits shows in them, and bounds for every element (E, U and TINY as in layer_oracle.py).

A result is rounded once, U of itself. What it is a sum of, |a| + |b| = size, is right to a few roundings of fp32: the
products' own, those of the sums and of what is formed before (D = X R, its decays): sixteen at most, 16 E of the size. Here
the terms differ by 2^-13 of themselves or less, U of which is 2^-21, below 16 E 2 = 2^-19; an operand of two bf16 parts is
off by up to 2^-17 of itself."""
from __future__ import annotations

import torch

import delta_oracle as do_
from layer_oracle import E, TINY, U, f64


def within(got, want, size, dtype, what):
    off = (f64(got) - want).abs()
    fine = U[dtype] * want.abs() + 16 * E * size + TINY[dtype]
    assert (off <= fine).all(), f"{what}: {float((off / fine).max()):.3g} of the bound"


def one_way(S, L, H, N, dtype):
    """(q, k) along the first key."""
    x = torch.zeros(S, L, H, N)
    x[..., 0] = 1
    return x.to(dtype), x.to(dtype)


def uniform(gen, *shape):
    """In [1, 2)."""
    return 1 + torch.rand(*shape, generator=gen)


def of_states(L, dtype, seed, H=4, P=48):
    """Two rows of a state that nearly cancel: ((q, k, v, g, beta, s0, scale), the outputs' sizes)."""
    gen = torch.Generator().manual_seed(seed)
    q, k = one_way(1, L, H, 2, dtype)
    q[..., 1] = -1
    a = uniform(gen, 1, H, P)
    s0 = torch.stack([a, a * (1 + 2.0 ** -13 * (torch.rand(1, H, P, generator=gen) - 0.5))], 2)
    v, zero = torch.zeros(1, L, H, P).to(dtype), torch.zeros(1, L, H)
    return (q, k, v, zero, zero, s0, 1.0), f64(s0).sum(2)[:, None].expand(1, L, H, P)


def of_tokens(L, dtype, seed, H=64):
    """What two tokens brought, nearly cancelling in all outputs that follow."""
    gen = torch.Generator().manual_seed(seed)
    q, k = one_way(1, L, H, 2, dtype)
    q[..., 1] = -1
    k[:, 1, :, 0], k[:, 1, :, 1] = 0, 1
    v = torch.zeros(1, L, H, 1)
    v[:, :2] = uniform(gen, 1, 2, H, 1).to(dtype).float()
    beta = torch.zeros(1, L, H)
    beta[:, 0] = uniform(gen, 1, H) / 2
    beta[:, 1] = beta[:, 0] * v[:, 0, :, 0] / v[:, 1, :, 0] * (1 + 2.0 ** -13 * (torch.rand(1, H, generator=gen) - 0.5))
    size = (f64(beta[:, :2, :, None]) * f64(v[:, :2])).cumsum(1)
    size = torch.cat([size[:, :1], size[:, 1:].expand(1, L - 1, H, 1)], 1)
    return (q, k, v.to(dtype), torch.zeros(1, L, H), beta, None, 1.0), size


def of_dq(L, dtype, seed, H=64):
    """Gradients of queries from what two tokens with opposite keys brought: (do, problem, sizes)."""
    gen = torch.Generator().manual_seed(seed)
    q, k = one_way(1, L, H, 2, dtype)
    k[:, 1, :, 0] = -1
    k[:, 2:] = 0
    v, beta = torch.zeros(1, L, H, 1), torch.zeros(1, L, H)
    v[:, :2] = uniform(gen, 1, 2, H, 1).to(dtype).float()
    beta[:, 0] = uniform(gen, 1, H) / 2
    d = beta[:, 0] * v[:, 0, :, 0]
    beta[:, 1] = d / (v[:, 1, :, 0] + d) * (1 + 2.0 ** -13 * (torch.rand(1, H, generator=gen) - 0.5))
    do = uniform(gen, 1, L, H, 1).to(dtype)
    do[:, :2] = 0
    size = torch.zeros(1, L, H, 2, dtype=torch.float64)
    size[..., 0] = 2 * f64(do[..., 0]) * f64(d)
    return do, (q, k, v.to(dtype), torch.zeros(1, L, H), beta, None, 1.0), size


def of_dk(L, dtype, seed, H=64):
    """Gradients of the first key from two tokens whose opposite queries a decay brings together."""
    gen = torch.Generator().manual_seed(seed)
    q, k = one_way(1, L, H, 2, dtype)
    k[:, 1:] = 0
    q[:, 2, :, 0] = -1
    q[:, 3:] = 0
    v, beta, g = torch.zeros(1, L, H, 1), torch.zeros(1, L, H), torch.zeros(1, L, H)
    v[:, 0], beta[:, 0] = uniform(gen, 1, H, 1), uniform(gen, 1, H) / 2
    do = torch.zeros(1, L, H, 1)
    do[:, 1:3] = uniform(gen, 1, 2, H, 1).sort(1).values.to(dtype).float()
    g[:, 2] = torch.log(do[:, 1] / do[:, 2])[..., 0] + 2.0 ** -13 * (torch.rand(1, H, generator=gen) - 0.5)
    size = torch.zeros(1, L, H, 2, dtype=torch.float64)
    size[:, 0, :, 0] = 2 * f64(do[:, 1, :, 0]) * f64(beta[:, 0]) * f64(v.to(dtype)[:, 0, :, 0])
    size[..., 1] = 0
    return do.to(dtype), (q, k, v.to(dtype), g, beta, None, 1.0), size


def outputs(problem):
    return do_.forward(*problem)[0]


def ordinary(q, k, v, g, beta, s0, scale):
    """(o, the bounds' size) of any problem. A state's column is off by 28 E of its norm as often up as down
    (delta_oracle.py); no element by more than eight times that, 224 E = 14 times what `within` allows of a size."""
    o, states, _ = do_.forward(q, k, v, g, beta, s0, scale)
    col = torch.stack([s.norm(dim=2) for s in states]).max(0).values
    qs = do_._heads(q, v.shape[2]).norm(dim=-1)
    return o, 14 * abs(scale) * qs[..., None] * col[:, None]
