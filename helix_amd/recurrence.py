"""Gated linear recurrence per channel, and its backward pass (include/helix/helix_layer.h).

    f_t = sigmoid(g_t),  h_t = f_t h_(t-1) + (1 - f_t) v_t,  h_(-1) = h0

The state is float32 throughout. A token that is to leave the state as it is has g = +inf (and a finite v).
"""
from __future__ import annotations

import torch

from . import abi
from .layer import device_index, expect, io_code, ptr, run_with_scratch, stream_handle, under


def _strides(name: str, t: torch.Tensor) -> tuple[int, int]:
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: the channels must be contiguous")
    return t.stride(0), t.stride(1)


def _state(name: str, t: torch.Tensor | None, like: torch.Tensor) -> None:
    if t is None:
        return
    expect(name, t, torch.float32, (like.shape[0], like.shape[2]), like)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _shape(op: str, g: torch.Tensor) -> tuple[int, int, int, int, int]:
    index = device_index(op, g)
    if g.dim() != 3:
        raise ValueError("g must be [sequences, tokens, channels]")
    return (index, io_code("g", g), *g.shape)


def gated_scan(g: torch.Tensor, v: torch.Tensor, h0: torch.Tensor | None = None, *,
               stream: torch.cuda.Stream | None = None):
    """The recurrence over g and v [S, L, D]: returns (h, last).

    g and v are float32, bfloat16 or float16 (one type), of any token and sequence strides (column ranges of one
    projected row per token, say); h0 and last, the state before and after, are float32 [S, D] (h0 zeros when None).
    L = 1 is the step of a single token."""
    index, io, S, L, D = _shape("gated_scan", g)
    expect("v", v, g.dtype, g.shape, g)
    _state("h0", h0, g)
    with under(index, stream):
        h = torch.empty(S, L, D, dtype=g.dtype, device=g.device)
        last = torch.empty(S, D, dtype=torch.float32, device=g.device)
    st = stream_handle(index, stream)
    strides = (*_strides("g", g), *_strides("v", v), L * D, D)

    def pack(buf, nbytes):
        return abi.GATED_SCAN_STRUCT.pack(S, L, D, io, g.data_ptr(), v.data_ptr(), ptr(h0), h.data_ptr(),
                                          last.data_ptr(), buf, nbytes, *strides)

    lib = abi.lib()
    run_with_scratch(lib.helix_gated_scan_encode, lib.helix_gated_scan_scratch_size, index, st, stream, pack)
    return h, last


def gated_scan_backward(dh: torch.Tensor, g: torch.Tensor, v: torch.Tensor, h: torch.Tensor,
                        h0: torch.Tensor | None = None, dh_last: torch.Tensor | None = None, *,
                        stream: torch.cuda.Stream | None = None):
    """Gradients of gated_scan from dh [S, L, D] and dh_last [S, D] (None: last is not used further): returns
    (dg, dv, dh0), dg and dv of g's type and dh0 float32. h is what gated_scan returned for g, v and h0."""
    index, io, S, L, D = _shape("gated_scan_backward", g)
    for name, t in (("dh", dh), ("v", v), ("h", h)):
        expect(name, t, g.dtype, g.shape, g)
    _state("h0", h0, g)
    _state("dh_last", dh_last, g)
    with under(index, stream):
        dg = torch.empty(S, L, D, dtype=g.dtype, device=g.device)
        dv = torch.empty(S, L, D, dtype=g.dtype, device=g.device)
        dh0 = torch.empty(S, D, dtype=torch.float32, device=g.device)
    st = stream_handle(index, stream)
    strides = (*_strides("dh", dh), *_strides("g", g), *_strides("v", v), *_strides("h", h), L * D, D, L * D, D)

    def pack(buf, nbytes):
        return abi.GATED_SCAN_BACKWARD_STRUCT.pack(S, L, D, io, dh.data_ptr(), g.data_ptr(), v.data_ptr(), h.data_ptr(),
                                                   ptr(h0), ptr(dh_last), dg.data_ptr(), dv.data_ptr(), dh0.data_ptr(),
                                                   buf, nbytes, *strides)

    lib = abi.lib()
    run_with_scratch(lib.helix_gated_scan_backward_encode, lib.helix_gated_scan_backward_scratch_size, index, st, stream, pack)
    return dg, dv, dh0
