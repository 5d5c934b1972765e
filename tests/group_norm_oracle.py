"""Plain 64-bit forms of group_norm and its gradients on the CPU, and the bounds that fp32 arithmetic with one rounding
to the storage type stays in (E, U and TINY as in layer_oracle.py)."""
from __future__ import annotations

import torch

from layer_oracle import E, TINY, U, f64


def act(kind, u):
    """(a(u), a'(u))."""
    if kind is None:
        return u, torch.ones_like(u)
    s = torch.sigmoid(u)
    if kind == "sigmoid":
        return s, s * torch.sigmoid(-u)
    return u * s, s + u * s * torch.sigmoid(-u)


def forward(x, w, b, gate, groups, kind, eps):
    """(y, mean, rstd, z) in 64 bits."""
    h = f64(x).unflatten(-1, (groups, -1))
    mean = h.mean(-1)
    d = h - mean[..., None]
    rstd = 1 / (d.square().mean(-1) + eps).sqrt()
    z = (d * rstd[..., None]).flatten(-2) * f64(w) + (0 if b is None else f64(b))
    y = act(kind, z)[0] if gate is None else z * act(kind, f64(gate))[0]
    return y, mean, rstd, z


def forward_bound(x, w, b, gate, groups, kind, eps, y, mean, rstd, z):
    """(of y in its type, of mean, of rstd). A sum of a group is a tree over chains of at most width / 64 + 32 terms: c
    roundings in all. What the mean is off by is in every difference; the variance takes it and its own sum's c
    roundings, its root half of that. z gets n's error and three roundings; an activation is off by at most 10 E of
    itself (two by the hardware's exponential and reciprocal, the rest by roundings) and its slope is below 1.1."""
    h = f64(x).unflatten(-1, (groups, -1))
    c = E * (h.shape[-1] / 64 + 48)
    dm = c * h.abs().mean(-1)
    d = (h - mean[..., None]).abs()
    var = d.square().mean(-1)
    dd = dm[..., None] + E * d
    dr = rstd * (0.5 * (2 * (d * dd).mean(-1) + dd.square().mean(-1) + c * var) / (var + eps) + 4 * E)
    n = d * rstd[..., None]
    dn = (dd * (rstd + dr)[..., None] + d * dr[..., None] + 2 * E * n).flatten(-2)
    bias = 0 if b is None else f64(b).abs()
    dz = f64(w).abs() * dn + 3 * E * (f64(w).abs() * n.flatten(-2) + bias)
    if gate is None:
        off = (1.1 if kind else 1.0) * dz + 10 * E * y.abs()
    else:
        off = act(kind, f64(gate))[0].abs() * dz + 12 * E * y.abs()
    return off + (y.abs() + off) * U[x.dtype] + TINY[x.dtype], dm + 1e-37, dr + 1e-37


def backward(dy, x, w, mean, rstd, b, gate, groups, kind):
    """(dx, dweight, dbias, dgate or None) in 64 bits."""
    dim = x.shape[-1]
    r = f64(rstd)[..., None]
    n = ((f64(x).unflatten(-1, (groups, -1)) - f64(mean)[..., None]) * r)
    z = n.flatten(-2) * f64(w) + (0 if b is None else f64(b))
    a, slope = act(kind, z if gate is None else f64(gate))
    dz = f64(dy) * (slope if gate is None else a)
    t = (dz * f64(w)).unflatten(-1, (groups, -1))
    dx = r * (t - t.mean(-1, keepdim=True) - n * (t * n).mean(-1, keepdim=True))
    return (dx.flatten(-2), (dz * n.flatten(-2)).reshape(-1, dim).sum(0), dz.reshape(-1, dim).sum(0),
            None if gate is None else f64(dy) * z * slope)


def backward_bound(dy, x, w, mean, rstd, b, gate, groups, kind, dx, dgate):
    """mean and rstd are given: n is off by 2 E of |x| rstd + |mean| rstd (a difference of rounded values is exact but for
    its own rounding), z by that and three roundings, slopes and activations by 10 E of themselves and, without a gate,
    by z's error times a second derivative below 0.6. Sums over a group as in forward_bound, those over the rows have at
    most rows + 64 roundings."""
    dim, dt = x.shape[-1], x.dtype
    rows = x.numel() // dim
    r, aw = f64(rstd)[..., None], f64(w).abs()
    h = f64(x).unflatten(-1, (groups, -1))
    n = (h - f64(mean)[..., None]) * r
    dn = 3 * E * n.abs()
    bias = 0 if b is None else f64(b)
    z = n.flatten(-2) * f64(w) + bias
    dz_ = aw * dn.flatten(-2) + 3 * E * (aw * n.flatten(-2).abs() + (0 if b is None else bias.abs()))
    u = z if gate is None else f64(gate)
    a, slope = act(kind, u)
    parts = slope.abs() if kind is None else torch.sigmoid(u) * (1 + u.abs() * torch.sigmoid(-u))
    dslope = 14 * E * parts + (0.6 * dz_ if gate is None and kind else 0)
    ady = f64(dy).abs()
    size = ady * (parts if gate is None else a.abs())           # of dz
    ddz = ady * (dslope if gate is None else 12 * E * a.abs()) + E * size
    t, dt_ = (aw * size).unflatten(-1, (groups, -1)), (aw * (ddz + E * size)).unflatten(-1, (groups, -1))
    c = E * (h.shape[-1] / 64 + 48)
    mt, dmt = t.mean(-1, keepdim=True), dt_.mean(-1, keepdim=True) + c * t.mean(-1, keepdim=True)
    tn = t * n.abs()
    mn = tn.mean(-1, keepdim=True)
    dmn = (dt_ * n.abs() + t * dn).mean(-1, keepdim=True) + (c + E) * mn
    off = r * (dt_ + dmt + n.abs() * dmn + dn * mn + 4 * E * (t + mt + n.abs() * mn))
    off = off.flatten(-2)
    bx = off + (dx.abs() + off) * U[dt] + TINY[dt]
    rows_off = E * (rows + 64)
    bw = (ddz * n.flatten(-2).abs() + size * dn.flatten(-2)).reshape(-1, dim).sum(0)
    bw = bw + rows_off * (size * n.flatten(-2).abs()).reshape(-1, dim).sum(0) + 1e-37
    bb = ddz.reshape(-1, dim).sum(0) + rows_off * size.reshape(-1, dim).sum(0) + 1e-37
    if gate is None:
        return bx, bw, bb, None
    og = ady * (dz_ * parts + z.abs() * 16 * E * parts)
    return bx, bw, bb, og + (dgate.abs() + og) * U[dt] + TINY[dt]
