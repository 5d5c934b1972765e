"""The group norm's C ABI without a GPU, and its 64-bit forms against automatic differentiation."""
import ctypes
import os
import subprocess

import pytest
import torch

import group_norm_oracle as go
import layer_oracle as lo
from helix_amd import abi
from helix_amd.desc import (HELIX_ERR_INVALID_ARG, HELIX_ERR_NO_DEVICE, HELIX_ERR_SCRATCH_TOO_SMALL,
                            HELIX_ERR_UNSUPPORTED_SHAPE, HELIX_OK)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 12   # an address that nothing reads


@pytest.fixture(scope="module")
def host():
    c = abi.Context(host_only=True)
    yield c
    c.close()


def call(host, name, args):
    return int(getattr(abi.lib(), name)(host.handle, None, args))


def test_packed_arguments_match_the_header(tmp_path):
    structs = {"helix_group_norm_args": abi.GROUP_NORM_STRUCT,
               "helix_group_norm_backward_args": abi.GROUP_NORM_BACKWARD_STRUCT}
    src = tmp_path / "sizes.c"
    src.write_text("#include <stdio.h>\n#include \"helix/helix_layer.h\"\nint main(void) {\n" +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));\n' for n in structs) + "return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {n: int(v) for n, v in out.items()} == {n: s.size for n, s in structs.items()}


def fwd(rows=4, dim=192, groups=3, io=2, w=0, act=1, eps=1e-5, x=P, weight=P, bias=0, gate=0, y=P, q=0, scale=0, mean=P,
        rstd=P, ld=256):
    return abi.GROUP_NORM_STRUCT.pack(rows, dim, groups, io, w, act, eps, x, weight, bias, gate, y, q, scale, mean, rstd,
                                      *[ld] * 5)


@pytest.mark.parametrize("change,status", [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(rows=0), HELIX_OK), (dict(rows=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(dim=0), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(groups=0), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(groups=5), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(dim=8193, groups=1, ld=8193), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(dim=8192, groups=1, ld=8192), HELIX_ERR_NO_DEVICE), (dict(io=3), HELIX_ERR_INVALID_ARG),
    (dict(w=1), HELIX_ERR_INVALID_ARG), (dict(act=3), HELIX_ERR_INVALID_ARG), (dict(act=-1), HELIX_ERR_INVALID_ARG),
    (dict(eps=float("inf")), HELIX_ERR_INVALID_ARG), (dict(eps=-1.0), HELIX_ERR_INVALID_ARG),
    (dict(x=0), HELIX_ERR_INVALID_ARG), (dict(x=P + 1), HELIX_ERR_INVALID_ARG), (dict(weight=0), HELIX_ERR_INVALID_ARG),
    (dict(bias=P + 2), HELIX_ERR_INVALID_ARG), (dict(gate=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(y=0), HELIX_ERR_INVALID_ARG), (dict(q=P, scale=P), HELIX_ERR_INVALID_ARG),
    (dict(y=0, q=P), HELIX_ERR_INVALID_ARG), (dict(y=0, q=P, scale=P), HELIX_ERR_NO_DEVICE),
    (dict(y=0, q=P, scale=P, dim=19200, groups=200, ld=19200), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(y=0, q=P, scale=P, dim=25600, groups=200, ld=25600), HELIX_ERR_NO_DEVICE),
    (dict(ld=100), HELIX_ERR_INVALID_ARG), (dict(ld=-256), HELIX_ERR_INVALID_ARG), (dict(mean=P + 2), HELIX_ERR_INVALID_ARG),
])
def test_checks(host, change, status):
    assert call(host, "helix_group_norm_encode", fwd(**change)) == status


def bwd(rows=40, dim=192, groups=3, io=2, w=0, act=1, res=0, dy=P, x=P, weight=P, bias=0, gate=P, mean=P, rstd=P, dx=P,
        dgate=P, dw=P, db=P, scratch=P, nbytes=1 << 30, ld=256):
    return abi.GROUP_NORM_BACKWARD_STRUCT.pack(rows, dim, groups, io, w, act, res, dy, x, weight, bias, gate, mean, rstd, dx,
                                               dgate, dw, db, scratch, nbytes, *[ld] * 5)


@pytest.mark.parametrize("change,status", [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(rows=0, dw=0, db=0), HELIX_OK), (dict(rows=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(groups=7), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(io=-1), HELIX_ERR_INVALID_ARG), (dict(w=1), HELIX_ERR_INVALID_ARG),
    (dict(act=9), HELIX_ERR_INVALID_ARG), (dict(res=1), HELIX_ERR_INVALID_ARG), (dict(dy=0), HELIX_ERR_INVALID_ARG),
    (dict(x=0), HELIX_ERR_INVALID_ARG), (dict(mean=0), HELIX_ERR_INVALID_ARG), (dict(rstd=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(dx=0), HELIX_ERR_INVALID_ARG), (dict(dgate=0), HELIX_ERR_INVALID_ARG), (dict(gate=0), HELIX_ERR_INVALID_ARG),
    (dict(gate=0, dgate=0), HELIX_ERR_NO_DEVICE), (dict(ld=100), HELIX_ERR_INVALID_ARG), (dict(dw=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(scratch=0), HELIX_ERR_SCRATCH_TOO_SMALL), (dict(nbytes=16), HELIX_ERR_SCRATCH_TOO_SMALL),
    (dict(scratch=P + 4), HELIX_ERR_INVALID_ARG), (dict(dw=0, db=0, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
])
def test_backward_checks(host, change, status):
    assert call(host, "helix_group_norm_backward_encode", bwd(**change)) == status


def test_scratch_covers_every_part():
    # Parts of a launch times row slots times both sums, whatever the shape.
    size = abi.lib().helix_group_norm_backward_scratch_size
    for rows in (1, 3, 64, 1000, 32768, 1 << 22):
        for dim, groups in ((64, 1), (192, 3), (5120, 80), (8192, 1), (2565, 27), (5, 5)):
            assert size(bwd(rows=rows, dim=dim, groups=groups)) % (8 * dim) == 0
            assert size(bwd(rows=rows, dim=dim, groups=groups)) >= 8 * dim


@pytest.mark.parametrize("kind", [None, "silu", "sigmoid"])
@pytest.mark.parametrize("gated", [False, True])
def test_oracle_gradients_by_differentiation(kind, gated):
    torch.manual_seed(0)
    x, w, b, gate = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((5, 12), (12,), (12,), (5, 12)))
    h = x.unflatten(-1, (3, 4))
    mean = h.mean(-1)
    rstd = ((h - mean[..., None]).square().mean(-1) + 1e-5).rsqrt()
    z = ((h - mean[..., None]) * rstd[..., None]).flatten(-2) * w + b
    u = gate if gated else z
    a = u if kind is None else torch.sigmoid(u) * (u if kind == "silu" else 1)
    y = z * a if gated else a
    assert torch.allclose(go.forward(x, w, b, gate if gated else None, 3, kind, 1e-5)[0], y, rtol=1e-13, atol=1e-13)
    dy = torch.randn(5, 12, dtype=torch.float64)
    want = torch.autograd.grad((y * dy).sum(), (x, w, b) + ((gate,) if gated else ()))
    got = go.backward(dy, x, w, mean, rstd, b, gate if gated else None, 3, kind)
    for g, v in zip(got, want):
        assert torch.allclose(g, v, rtol=1e-11, atol=1e-12)


def test_the_checks_see_a_mistake():
    # Planted in the 64-bit side: a neighbour's group, a lost bias, the gate's slope in place of its value.
    torch.manual_seed(1)
    x, w, b, gate, dy = (torch.randn(*s) for s in ((6, 96), (96,), (96,), (6, 96), (6, 96)))
    y, mean, rstd, z = go.forward(x, w, b, gate, 3, "silu", 1e-5)
    by = go.forward_bound(x, w, b, gate, 3, "silu", 1e-5, y, mean, rstd, z)[0]
    lo.within(y.float(), y, by)
    for bad in (go.forward(x.roll(1, -1), w, b, gate, 3, "silu", 1e-5), go.forward(x, w, None, gate, 3, "silu", 1e-5),
                go.forward(x, w, b, gate, 3, "sigmoid", 1e-5)):
        with pytest.raises(AssertionError):
            lo.within(bad[0].float(), y, by)
    args = (dy, x, w, mean.float(), rstd.float(), b, gate, 3, "silu")
    got = go.backward(*args)
    bounds = go.backward_bound(*args, got[0], got[3])
    for g, c in zip(got, bounds):
        lo.within(g.float(), g, c)
        with pytest.raises(AssertionError):
            lo.within((g * (1 + 1e-4 + 2 ** -7)).float(), g, c)
