"""Norms into the storage type or 8 bits, and their backward passes.

rms_norm, of whole rows with the residual's addition:

    h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * weight

group_norm, of the groups of a row's channels (a head's outputs, say) with an activation a or a gate:

    z = (x - mean) * rstd * weight + bias,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = z * a(gate), or a(z)

A user's layer calls rms_norm_fp8 before a projection in 8 bits (helix_amd.matmul), and rms_norm and
rms_norm_backward where it trains. 8-bit rows are float8_e4m3fn with a float8_e8m0fnu scale, a power of two, for each
block of 128 channels (include/helix/helix_layer.h).
"""
from __future__ import annotations

import torch

from . import abi
from .layer import (FP8, FP8_BLOCK, FP8_SCALE, IO_DTYPES, device_index, empty, expect, io_code, packed, ptr, row_stride,
                    rows_like, run, scratch, stream_handle, under)


def _weight_code(weight: torch.Tensor, x: torch.Tensor) -> int:
    dtype = weight.dtype
    if dtype != torch.float32 and dtype != x.dtype:
        raise ValueError(f"weight must be float32 or {x.dtype}; got {dtype}")
    expect("weight", weight, dtype, x.shape[-1:], x)
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    return IO_DTYPES[dtype]


def fp8_rows(shape, device) -> tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised 8-bit rows and their scales; rows start at multiples of 16 bytes, those of the scales of 4, as
    matmul_fp8 wants them."""
    dim = shape[-1]
    blocks = -(-dim // FP8_BLOCK)
    pitch, s_pitch = -(-dim // 16) * 16, -(-blocks // 4) * 4
    lead = shape[:-1]
    q = torch.empty(*lead, pitch, dtype=FP8, device=device)
    scale = torch.empty(*lead, s_pitch, dtype=FP8_SCALE, device=device)
    return q if pitch == dim else q[..., :dim], scale if s_pitch == blocks else scale[..., :blocks]


def _norm(op, fn, x, weight, residual, eps, fp8, want_rstd, stream):
    index = device_index(op, x)
    io = io_code("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least 1")
    dim = x.shape[-1]
    w_code = 0
    if weight is not None:
        w_code = _weight_code(weight, x)
    ld_x = row_stride("x", x)
    ld_r = 0
    h = x
    y = q = scale = rstd = None
    with under(index, stream):
        if residual is not None:
            expect("residual", residual, x.dtype, x.shape, x)
            ld_r = row_stride("residual", residual)
            if weight is not None:
                h = rows_like(x)
        if fp8:
            q, scale = fp8_rows(x.shape, x.device)
        else:
            y = rows_like(x)
        if want_rstd:
            rstd = empty(x.shape[:-1], torch.float32, x.device)
    pitch = -(-dim // 16) * 16
    args = packed(abi.NORM_STRUCT.pack, x.numel() // dim, dim, io, w_code, eps, x.data_ptr(), ptr(residual), ptr(weight),
                  0 if h is x else h.data_ptr(), ptr(y), ptr(q), ptr(scale), ptr(rstd), ld_x, ld_r, dim, dim, pitch,
                  -(-dim // (4 * FP8_BLOCK)) * 4)
    run(fn, index, stream_handle(index, stream), args)
    return y, q, scale, h, rstd


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-5,
             stream: torch.cuda.Stream | None = None):
    """The norm of x [..., dim], or of x + residual, in x's type: returns (y, h, rstd).

    x and residual are float32, bfloat16 or float16, weight [dim] is float32 or x's type. h is x + residual rounded to
    x's type (x itself without a residual), rstd float32 [...]; rms_norm_backward takes both. The norm is that of the
    sum before it is rounded."""
    y, _, _, h, rstd = _norm("rms_norm", abi.lib().helix_norm_encode, x, weight, residual, eps, False, True, stream)
    return y, h, rstd


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-5,
                 stream: torch.cuda.Stream | None = None):
    """The norm of x [..., dim], or of x + residual, in 8 bits: returns (q, scale, h).

    q float8_e4m3fn [..., dim] and scale float8_e8m0fnu [..., ceil(dim / 128)] are what matmul_fp8 takes; h as in
    rms_norm."""
    _, q, scale, h, _ = _norm("rms_norm_fp8", abi.lib().helix_norm_encode, x, weight, residual, eps, True, False,
                              stream)
    return q, scale, h


def quantize_fp8(x: torch.Tensor, *, stream: torch.cuda.Stream | None = None):
    """x [..., dim] in 8 bits: returns (q, scale) as rms_norm_fp8 does. A projection's weights [n, k] are laid out with
    it once."""
    _, q, scale, _, _ = _norm("quantize_fp8", abi.lib().helix_quantize_fp8_encode, x, None, None, 0.0, True, False,
                              stream)
    return q, scale


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dh: torch.Tensor | None = None, *, stream: torch.cuda.Stream | None = None):
    """Gradients of rms_norm's y and h, from dy and dh (None: h is not used further): returns (dx, dweight).

    dx, in h's type, is the gradient of x and of residual alike; dweight is float32, and its sum over the rows is taken
    in an order that depends on the shape alone."""
    index = device_index("rms_norm_backward", h)
    io = io_code("h", h)
    if h.dim() < 1 or h.shape[-1] < 1:
        raise ValueError("h must have a last dimension of at least 1")
    dim = h.shape[-1]
    rows = h.numel() // dim
    expect("dy", dy, h.dtype, h.shape, h)
    expect("rstd", rstd, torch.float32, h.shape[:-1], h)
    if not rstd.is_contiguous():
        raise ValueError("rstd must be contiguous")
    ld_dh = 0
    if dh is not None:
        expect("dh", dh, h.dtype, h.shape, h)
        ld_dh = row_stride("dh", dh)
    w_code = _weight_code(weight, h)
    ld_dy, ld_h = row_stride("dy", dy), row_stride("h", h)
    with under(index, stream):
        dx = rows_like(h)
        dweight = torch.empty(dim, dtype=torch.float32, device=h.device)
    st = stream_handle(index, stream)

    def pack(buf, nbytes):
        return abi.NORM_BACKWARD_STRUCT.pack(rows, dim, io, w_code, 0, dy.data_ptr(), h.data_ptr(), weight.data_ptr(),
                                             rstd.data_ptr(), ptr(dh), dx.data_ptr(), dweight.data_ptr(), buf, nbytes,
                                             ld_dy, ld_h, ld_dh, dim)

    L = abi.lib()
    need = L.helix_norm_backward_scratch_size(packed(pack, 0, 0))
    buf = scratch(index, st, stream, need)
    run(L.helix_norm_backward_encode, index, st, pack(ptr(buf), need))
    return dx, dweight


ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}


def _groups(op, x, weight, bias, gate, groups, activation):
    """Checks, and what both passes tell the library of them: (device, io, rows, dim, codes, ld_gate)."""
    index = device_index(op, x)
    io = io_code("x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least 1")
    dim = x.shape[-1]
    if not isinstance(groups, int) or groups < 1 or dim % groups:
        raise ValueError(f"groups must divide the last dimension, {dim}; got {groups}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu' or 'sigmoid'; got {activation!r}")
    w_code = _weight_code(weight, x)
    if bias is not None:
        expect("bias", bias, weight.dtype, x.shape[-1:], x)
        if not bias.is_contiguous():
            raise ValueError("bias must be contiguous")
    ld_gate = 0
    if gate is not None:
        expect("gate", gate, x.dtype, x.shape, x)
        ld_gate = row_stride("gate", gate)
    return index, io, x.numel() // dim, dim, (groups, io, w_code, ACTIVATIONS[activation]), ld_gate


def _group_norm(op, x, weight, bias, gate, groups, activation, eps, fp8, stream):
    index, _, rows, dim, codes, ld_gate = _groups(op, x, weight, bias, gate, groups, activation)
    ld_x = row_stride("x", x)
    y = q = scale = mean = rstd = None
    with under(index, stream):
        if fp8:
            q, scale = fp8_rows(x.shape, x.device)
        else:
            y = rows_like(x)
            mean, rstd = (empty((*x.shape[:-1], groups), torch.float32, x.device) for _ in range(2))
    args = packed(abi.GROUP_NORM_STRUCT.pack, rows, dim, *codes, eps, x.data_ptr(), weight.data_ptr(), ptr(bias),
                  ptr(gate), ptr(y), ptr(q), ptr(scale), ptr(mean), ptr(rstd), ld_x, ld_gate, dim, -(-dim // 16) * 16,
                  -(-dim // (4 * FP8_BLOCK)) * 4)
    run(abi.lib().helix_group_norm_encode, index, stream_handle(index, stream), args)
    return y, mean, rstd, q, scale


def group_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, *, groups: int, activation: str | None = "silu", eps: float = 1e-5,
               stream: torch.cuda.Stream | None = None):
    """The norm of each of `groups` groups of neighbouring channels of x [..., dim], times the activation of gate or,
    without one, activated itself; in x's type: returns (y, mean, rstd).

    x and gate are float32, bfloat16 or float16 (one type), weight and bias [dim] float32 or x's type (one type).
    activation is "silu", "sigmoid" or None (the gate, or the norm, as it is). mean and rstd, float32 [..., groups],
    are what group_norm_backward takes."""
    return _group_norm("group_norm", x, weight, bias, gate, groups, activation, eps, False, stream)[:3]


def group_norm_fp8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                   gate: torch.Tensor | None = None, *, groups: int, activation: str | None = "silu",
                   eps: float = 1e-5, stream: torch.cuda.Stream | None = None):
    """group_norm in 8 bits: returns (q, scale) as rms_norm_fp8 does, what matmul_fp8 takes."""
    return _group_norm("group_norm_fp8", x, weight, bias, gate, groups, activation, eps, True, stream)[3:]


def group_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, bias: torch.Tensor | None = None, gate: torch.Tensor | None = None, *,
                        groups: int, activation: str | None = "silu", stream: torch.cuda.Stream | None = None):
    """Gradients of group_norm's y from dy: returns (dx, dweight, dbias, dgate).

    dx and dgate (None without a gate) have x's type; dweight and dbias (None without a bias) are float32, and their
    sums over the rows are taken in an order that depends on the shape alone. mean and rstd are what group_norm returned
    for x."""
    index, _, rows, dim, codes, ld_gate = _groups("group_norm_backward", x, weight, bias, gate, groups, activation)
    expect("dy", dy, x.dtype, x.shape, x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        expect(name, t, torch.float32, (*x.shape[:-1], groups), x)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    ld_dy, ld_x = row_stride("dy", dy), row_stride("x", x)
    with under(index, stream):
        dx = rows_like(x)
        dgate = None if gate is None else rows_like(x)
        dweight = torch.empty(dim, dtype=torch.float32, device=x.device)
        dbias = None if bias is None else torch.empty_like(dweight)
    st = stream_handle(index, stream)

    def pack(buf, nbytes):
        return abi.GROUP_NORM_BACKWARD_STRUCT.pack(rows, dim, *codes, 0, dy.data_ptr(), x.data_ptr(), weight.data_ptr(),
                                                   ptr(bias), ptr(gate), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                                                   ptr(dgate), dweight.data_ptr(), ptr(dbias), buf, nbytes, ld_dy, ld_x,
                                                   ld_gate, dim, dim)

    L = abi.lib()
    need = L.helix_group_norm_backward_scratch_size(packed(pack, 0, 0))
    buf = scratch(index, st, stream, need)
    run(L.helix_group_norm_backward_encode, index, st, pack(ptr(buf), need))
    return dx, dweight, dbias, dgate
