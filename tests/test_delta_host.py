"""The delta rule's C ABI without a GPU, and its 64-bit forms against automatic differentiation."""
import os
import subprocess

import pytest
import torch

import delta_oracle as do_
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
    structs = {"helix_delta_rule_args": abi.DELTA_RULE_STRUCT,
               "helix_delta_rule_backward_args": abi.DELTA_RULE_BACKWARD_STRUCT}
    src = tmp_path / "sizes.c"
    src.write_text("#include <stdio.h>\n#include \"helix/helix_layer.h\"\nint main(void) {\n" +
                   "".join(f'printf("{n} %zu\\n", sizeof({n}));\n' for n in structs) + "return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {n: int(v) for n, v in out.items()} == {n: s.size for n, s in structs.items()}


def args(S=2, L=100, Hk=2, H=4, N=64, V=32, io=2, scale=0.125, q=P, k=P, v=P, g=P, beta=P, s0=0, o=P, s=P, scratch=P,
         nbytes=1 << 40, tok=128, seq=12800, head=64, tok_g=4, tok_o=128, head_o=32, seq_o=12800):
    return abi.DELTA_RULE_STRUCT.pack(S, L, Hk, H, N, V, io, scale, q, k, v, g, beta, s0, o, s, scratch, nbytes, seq, tok, head,
                                      seq, tok, head, seq, tok, 32, 400, tok_g, 400, tok_g, seq_o, tok_o, head_o)


def bwd(S=2, L=100, Hk=2, H=4, N=64, V=32, io=2, scale=0.125, d_o=P, q=P, k=P, v=P, g=P, beta=P, s0=0, ds=0, dq=P, dk=P,
        dv=P, dg=P, db=P, ds0=P, scratch=P, nbytes=1 << 40, tok=128, seq=12800):
    return abi.DELTA_RULE_BACKWARD_STRUCT.pack(S, L, Hk, H, N, V, io, scale, d_o, q, k, v, g, beta, s0, ds, dq, dk, dv, dg, db,
                                               ds0, scratch, nbytes, *[seq, tok, 32] * 4, 400, 4, 400, 4)


BOTH = [
    (dict(), HELIX_ERR_NO_DEVICE), (dict(S=0), HELIX_OK), (dict(H=0), HELIX_OK), (dict(S=-1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(L=-1), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(Hk=3), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(Hk=0), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(N=0), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(N=129), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(V=0), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(V=(1 << 16) + 1), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(io=3), HELIX_ERR_INVALID_ARG),
    (dict(scale=float("nan")), HELIX_ERR_INVALID_ARG), (dict(q=0), HELIX_ERR_INVALID_ARG), (dict(k=P + 1), HELIX_ERR_INVALID_ARG),
    (dict(v=0), HELIX_ERR_INVALID_ARG), (dict(g=0), HELIX_ERR_INVALID_ARG), (dict(beta=P + 2), HELIX_ERR_INVALID_ARG),
    (dict(s0=P + 2), HELIX_ERR_INVALID_ARG), (dict(tok=-1), HELIX_ERR_INVALID_ARG), (dict(seq=-1), HELIX_ERR_INVALID_ARG),
    (dict(tok=1 << 24), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(scratch=0), HELIX_ERR_SCRATCH_TOO_SMALL),
    (dict(nbytes=16), HELIX_ERR_SCRATCH_TOO_SMALL), (dict(scratch=P + 4), HELIX_ERR_INVALID_ARG),
    (dict(S=1 << 28, Hk=1 << 28, H=1 << 28), HELIX_ERR_UNSUPPORTED_SHAPE), (dict(S=1 << 16, H=1 << 15, Hk=1), HELIX_ERR_UNSUPPORTED_SHAPE),
    (dict(tok=0, seq=0), HELIX_ERR_NO_DEVICE),   # inputs may be one row, read for every token
]


@pytest.mark.parametrize("change,status", BOTH + [
    (dict(o=0), HELIX_ERR_INVALID_ARG), (dict(s=0), HELIX_ERR_INVALID_ARG), (dict(s=P + 2), HELIX_ERR_INVALID_ARG),
    (dict(tok_o=127), HELIX_ERR_INVALID_ARG), (dict(seq_o=12799), HELIX_ERR_INVALID_ARG), (dict(head_o=31), HELIX_ERR_INVALID_ARG),
    (dict(head_o=3200, tok_o=32), HELIX_ERR_NO_DEVICE),   # heads outside tokens
    (dict(L=1, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE), (dict(L=6, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
    (dict(L=0, q=0, k=0, v=0, g=0, beta=0, o=0, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
])
def test_checks(host, change, status):
    assert call(host, "helix_delta_rule_encode", args(**change)) == status


@pytest.mark.parametrize("change,status", BOTH + [
    (dict(d_o=0), HELIX_ERR_INVALID_ARG), (dict(ds=P + 1), HELIX_ERR_INVALID_ARG), (dict(dq=0), HELIX_ERR_INVALID_ARG),
    (dict(dk=P + 1), HELIX_ERR_INVALID_ARG), (dict(dv=0), HELIX_ERR_INVALID_ARG), (dict(dg=0), HELIX_ERR_INVALID_ARG),
    (dict(db=P + 2), HELIX_ERR_INVALID_ARG), (dict(ds0=0), HELIX_ERR_INVALID_ARG),
    (dict(L=0, q=0, k=0, v=0, g=0, beta=0, d_o=0, dq=0, dk=0, dv=0, dg=0, db=0, scratch=0, nbytes=0), HELIX_ERR_NO_DEVICE),
])
def test_backward_checks(host, change, status):
    assert call(host, "helix_delta_rule_backward_encode", bwd(**change)) == status


def test_scratch_stays_bounded():
    # Long calls go in segments of a bounded scratch (and a state each, backward), of a chunk of every sequence at least.
    L = abi.lib()
    for size, make, most in ((L.helix_delta_rule_scratch_size, args, 1 << 30),
                             (L.helix_delta_rule_backward_scratch_size, bwd, 3 << 30)):
        small = size(make(S=1, L=64, Hk=1, H=1))
        assert 0 < small < 1 << 20
        assert size(make(S=1, L=65, Hk=1, H=1)) > small
        assert size(make(S=4, L=1 << 18, Hk=8, H=64, N=128, V=64)) <= most
        assert size(make(S=4, L=1 << 18, Hk=8, H=64, N=128, V=64)) > most // 3


@pytest.mark.parametrize("sizes", [dict(S=1 << 28, Hk=1 << 28, H=1 << 28), dict(S=1 << 16, H=1 << 15), dict(N=1 << 30, V=1 << 30),
                                   dict(N=129), dict(V=-1), dict(S=-1, H=-1), dict(L=-(1 << 31)), dict(Hk=-1, H=0)])
def test_scratch_of_sizes_that_are_refused(sizes):
    # A size for every argument; what a call then refuses needs none.
    L = abi.lib()
    assert L.helix_delta_rule_scratch_size(args(**sizes)) == 0 and L.helix_delta_rule_backward_scratch_size(bwd(**sizes)) == 0


def test_oracle_gradients_by_differentiation():
    torch.manual_seed(0)
    S, L, Hk, H, N, V = 2, 9, 2, 4, 5, 3
    shapes = ((S, L, Hk, N), (S, L, Hk, N), (S, L, H, V), (S, L, H), (S, L, H), (S, H, N, V))
    q, k, v, g, beta, s0 = (0.5 * torch.randn(*s, dtype=torch.float64) for s in shapes)
    ins = [t.requires_grad_(True) for t in (q, k, v, -g.abs(), torch.sigmoid(beta), s0)]
    q, k, v, g, beta, s0 = ins
    out, s = [], s0
    for t in range(L):
        qt, kt = (x[:, t].repeat_interleave(2, 1) for x in (q, k))
        s = torch.exp(g[:, t])[..., None, None] * s
        d = beta[:, t, :, None] * (v[:, t] - torch.einsum("shn,shnp->shp", kt, s))
        s = s + kt[..., None] * d[..., None, :]
        out.append(0.3 * torch.einsum("shn,shnp->shp", qt, s))
    o = torch.stack(out, 1)
    got, states, _ = do_.forward(q, k, v, g, beta, s0, 0.3)
    assert torch.allclose(got, o, rtol=1e-13, atol=1e-14) and torch.allclose(states[-1], s, rtol=1e-13, atol=1e-14)
    do, ds = torch.randn_like(o), torch.randn_like(s)
    want = torch.autograd.grad((o * do).sum() + (s * ds).sum(), ins)
    grads, _ = do_.backward(do, *ins, ds, 0.3)
    for a, b in zip(grads, want):
        assert torch.allclose(a, b, rtol=1e-11, atol=1e-12)


def test_the_checks_see_a_mistake():
    # Planted in the 64-bit side: operands of two parts for three, a token's decay left out, beta of a neighbour.
    torch.manual_seed(1)
    S, L, H, N, V = 1, 150, 2, 32, 24
    q, k = (torch.nn.functional.normalize(torch.randn(S, L, H, N), dim=-1) for _ in range(2))
    v, g, beta = torch.randn(S, L, H, V), -torch.rand(S, L, H), torch.rand(S, L, H)
    o, states, _ = do_.forward(q, k, v, g, beta, None, N ** -0.5)
    so, ss = do_.forward_sizes(q, states, N ** -0.5, H)
    do_.close(o.float(), o, so, torch.float32, "o")
    do_.close(states[-1].float(), states[-1], ss, torch.float32, "s")
    g2 = g.clone()
    g2[0, 70, 0] = 0
    for bad in (do_.forward(q, k, v, g2, beta, None, N ** -0.5), do_.forward(q, k, v, g, beta.roll(1, 1), None, N ** -0.5),
                do_.forward(q, k * (1 + 2 ** -15), v, g, beta, None, N ** -0.5)):
        with pytest.raises(AssertionError):
            do_.close(bad[0].float(), o, so, torch.float32, "o")
            do_.close(bad[1][-1].float(), states[-1], ss, torch.float32, "s")
