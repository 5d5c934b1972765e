"""Gated delta rule, a recurrence whose state is a matrix per head, and its backward pass (include/helix/helix_layer.h).

    S_t = e^(g_t) S_(t-1) + beta_t k_t (v_t - e^(g_t) S_(t-1)' k_t)',  o_t = scale S_t' q_t,  S_(-1) = s0

The state, keys x values, is float32 throughout. Keys are taken as they are: a layer norms them (and the queries) to
length one, rms_norm with a weight of keys ** -0.5, say. A token that is to leave the state as it is has g = 0, beta = 0 and
any finite q, k and v (0 times a NaN is a NaN: memory that nothing has written is no padding). g = -inf forgets all before.
"""
from __future__ import annotations

import torch

from . import abi
from .layer import device_index, expect, io_code, packed, ptr, run, run_with_scratch, scratch, stream_handle, under


def _tensor(name: str, t: torch.Tensor, dtype: torch.dtype, shape, like: torch.Tensor, inner: str) -> tuple[int, ...]:
    """Checks t, and returns its strides but the last dimension's, whose elements have to be neighbours."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != like.get_device():
        expect(name, t, dtype, shape, like)
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the {inner} must be contiguous")
    return strides[:-1]


def _state(name: str, t: torch.Tensor | None, like: torch.Tensor, shape) -> None:
    if t is None:
        return
    if t.dtype != torch.float32 or t.shape != shape or t.get_device() != like.get_device():
        expect(name, t, torch.float32, shape, like)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _inputs(op, q, k, v, g, beta, s0, scale):
    """Checks: (device, the sizes' fields of the arguments, the inputs' strides)."""
    index = device_index(op, q)
    io = io_code("q", q)
    if q.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be [sequences, tokens, heads, keys] and v [sequences, tokens, heads, values]")
    S, L, Hk, N = q.shape
    H, P = v.shape[2:]
    if N < 1 or P < 1:
        raise ValueError("heads must have at least one key and one value channel")
    if H % Hk if Hk else H:
        raise ValueError(f"the {Hk} heads of q and k must divide the {H} heads of v")
    dtype, gates = q.dtype, (S, L, H)
    strides = (*_tensor("q", q, dtype, q.shape, q, "channels"), *_tensor("k", k, dtype, q.shape, q, "channels"),
               *_tensor("v", v, dtype, (S, L, H, P), q, "channels"), *_tensor("g", g, torch.float32, gates, q, "heads"),
               *_tensor("beta", beta, torch.float32, gates, q, "heads"))
    _state("s0", s0, q, (S, H, N, P))
    return index, (S, L, Hk, H, N, P, io, N ** -0.5 if scale is None else scale), strides


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               s0: torch.Tensor | None = None, *, scale: float | None = None, stream: torch.cuda.Stream | None = None):
    """The rule over q and k [S, L, Hk, N], v [S, L, H, P], g and beta [S, L, H]: returns (o, s).

    q, k and v are float32, bfloat16 or float16 (one type), of any strides but the last (column ranges of one projected
    row per token, say); Hk divides H, and H / Hk neighbouring heads of v share a head of q and k. N is at most 128. g, the
    logarithm of the decay, and beta are float32. o [S, L, H, P] has v's type; s0 and s, the states before and after, are
    float32 [S, H, N, P] (s0 zeros when None). scale is N ** -0.5 when None. L = 1 is the step of a single token."""
    index, sizes, strides = _inputs("delta_rule", q, k, v, g, beta, s0, scale)
    S, L, _, H, N, P = sizes[:6]
    with under(index, stream):
        o = torch.empty(S, L, H, P, dtype=v.dtype, device=v.device)
        s = torch.empty(S, H, N, P, dtype=torch.float32, device=v.device)
    st = stream_handle(index, stream)

    def pack(buf, nbytes):
        return abi.DELTA_RULE_STRUCT.pack(*sizes, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                                          ptr(s0), o.data_ptr(), s.data_ptr(), buf, nbytes, *strides, L * H * P, H * P, P)

    lib = abi.lib()
    run_with_scratch(lib.helix_delta_rule_encode, lib.helix_delta_rule_scratch_size, index, st, stream, pack)
    return o, s


def delta_rule_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                        beta: torch.Tensor, s0: torch.Tensor | None = None, ds: torch.Tensor | None = None, *,
                        scale: float | None = None, stream: torch.cuda.Stream | None = None):
    """Gradients of delta_rule from do [S, L, H, P] and ds [S, H, N, P] (None: s is not used further): returns
    (dq, dk, dv, dg, dbeta, ds0), dq, dk and dv of q's type, the others float32. The inputs are delta_rule's; its states
    are formed again. dq and dk of a head that several heads of v share are the sums over them."""
    index, sizes, strides = _inputs("delta_rule_backward", q, k, v, g, beta, s0, scale)
    S, L, Hk, H, N, P = sizes[:6]
    strides = (*_tensor("do", do, q.dtype, (S, L, H, P), q, "channels"), *strides)
    _state("ds", ds, q, (S, H, N, P))
    with under(index, stream):
        dq, dk = ((torch.empty if H else torch.zeros)(S, L, Hk, N, dtype=q.dtype, device=q.device) for _ in range(2))
        dv = torch.empty(S, L, H, P, dtype=q.dtype, device=q.device)
        dg, dbeta = (torch.empty(S, L, H, dtype=torch.float32, device=q.device) for _ in range(2))
        ds0 = torch.empty(S, H, N, P, dtype=torch.float32, device=q.device)
    st = stream_handle(index, stream)

    def pack(buf, nbytes):
        return abi.DELTA_RULE_BACKWARD_STRUCT.pack(*sizes, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                   g.data_ptr(), beta.data_ptr(), ptr(s0), ptr(ds), dq.data_ptr(),
                                                   dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(),
                                                   ds0.data_ptr(), buf, nbytes, *strides)

    lib = abi.lib()
    need = lib.helix_delta_rule_backward_scratch_size(packed(pack, 0, 0))
    buf = scratch(index, st, stream, need)
    run(lib.helix_delta_rule_backward_encode, index, st, pack(ptr(buf), need))
    return dq, dk, dv, dg, dbeta, ds0
