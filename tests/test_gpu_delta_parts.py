"""Calls of the delta rule that go in parts (sequences, or heads of one, after one another in the same scratch) and segments: the
same bits as calls of those sequences and heads alone."""
import pytest
import torch

from helix_amd import abi
from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu

NAMES = ("dq", "dk", "dv", "dg", "dbeta", "ds0")


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def problem(S, L, Hk, H, N, P, dtype, seed=0, carry=True):
    q, k = (normal(S, L, Hk, N, seed=seed + i, dtype=dtype) / N ** 0.5 for i in range(2))
    v = normal(S, L, H, P, seed=seed + 2, dtype=dtype)
    g, beta = -torch.rand(S, L, H, device="cuda"), torch.rand(S, L, H, device="cuda")
    return [q, k, v, g, beta, 0.3 * normal(S, H, N, P, seed=seed + 3) if carry else None]


def of(p, seqs, heads, share):
    """The sequences and heads [from, to) of a problem, as views."""
    (a, b), (c, d) = seqs, heads
    qk = slice(c // share, -(-d // share))
    q, k, v, g, beta, s0 = p
    g, beta = (t[a:b, :, c:d].contiguous() for t in (g, beta))
    return [q[a:b, :, qk], k[a:b, :, qk], v[a:b, :, c:d], g, beta, None if s0 is None else s0[a:b, c:d].contiguous()]


def backward_scratch(S, L, Hk, H, N, P, dtype):
    io = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    return abi.lib().helix_delta_rule_backward_scratch_size(
        abi.DELTA_RULE_BACKWARD_STRUCT.pack(S, L, Hk, H, N, P, io, 1.0, *[0] * 32))


# (Columns of the state in blocks of 16 on both sides, or of 32 on both.)
@pytest.mark.parametrize("S,L,Hk,H,N,P,dtype,some", [
    (700, 200, 4, 64, 16, 16, torch.bfloat16, [((0, 1), (0, 64)), ((381, 384), (0, 64)), ((699, 700), (0, 64))]),   # sequences
    (2, 200, 2000, 16000, 16, 12, torch.float16, [((0, 1), (0, 80)), ((1, 2), (6144, 6208)), ((1, 2), (15992, 16000))]),   # heads of one
    (3, 16000, 100, 300, 16, 16, torch.bfloat16, [((0, 1), (0, 3)), ((2, 3), (147, 153)), ((2, 3), (297, 300))]),   # and in segments
    (24, 2048, 8, 64, 64, 64, torch.bfloat16, [((0, 4), (0, 64)), ((20, 24), (0, 64))]),
    (20, 1000, 8, 64, 64, 64, torch.float32, [((0, 4), (0, 64)), ((16, 20), (0, 64))]),
])
def test_backward_in_parts(gpu, S, L, Hk, H, N, P, dtype, some):
    p = problem(S, L, Hk, H, N, P, dtype, seed=1)
    d, ds = normal(S, L, H, P, seed=9, dtype=dtype), normal(S, H, N, P, seed=10)
    each = 3 * 18432 + 768 + 8 * N * P + 512 * P + 768 + 20480 * Hk // H
    assert S * H * -(-L // 64) * each > 2 << 30 and backward_scratch(S, L, Hk, H, N, P, dtype) <= 3 << 30
    grads = delta_rule_backward(d, *p, ds)
    share = H // Hk
    for seqs, heads in some:
        (a, b), (c, e) = seqs, heads
        one = delta_rule_backward(d[a:b, :, c:e], *of(p, seqs, heads, share), ds[a:b, c:e].contiguous())
        for n, x, y in zip(NAMES, one, grads):
            y = y[a:b, c:e] if n == "ds0" else y[a:b, :, c // share:e // share] if n in ("dq", "dk") else y[a:b, :, c:e]
            assert torch.equal(x, y), (n, seqs, heads)


@pytest.mark.parametrize("S,L,Hk,H,N,P,dtype,some", [
    (40000, 70, 1, 1, 16, 8, torch.bfloat16, [((0, 3), (0, 1)), ((19999, 20002), (0, 1)), ((39997, 40000), (0, 1))]),   # sequences
    (2, 200, 20000, 40000, 8, 12, torch.float16, [((0, 1), (0, 4)), ((1, 2), (19996, 20004)), ((1, 2), (39998, 40000))]),   # heads
    (1, 70, 1, 40000, 40, 8, torch.float32, [((0, 1), (0, 5)), ((0, 1), (19996, 20004)), ((0, 1), (39999, 40000))]),   # of one query head
    (2, 130, 3, 90000, 16, 4, torch.bfloat16, [((0, 1), (14997, 15003)), ((1, 2), (29997, 30000)), ((1, 2), (44998, 45006)), ((1, 2), (89993, 90000))]),
])
def test_forward_in_parts(gpu, S, L, Hk, H, N, P, dtype, some):
    p = problem(S, L, Hk, H, N, P, dtype, seed=20)
    o, s = delta_rule(*p)
    for seqs, heads in some:
        (a, b), (c, d) = seqs, heads
        o1, s1 = delta_rule(*of(p, seqs, heads, H // Hk))
        assert torch.equal(o1, o[a:b, :, c:d]) and torch.equal(s1, s[a:b, c:d])


# Token by token: 2^24 - 1 workgroups a launch.
@pytest.mark.parametrize("S,L,Hk,H,P", [((1 << 24) + 5, 3, 1, 1, 2), (1, 1, (1 << 24) + 6, (1 << 24) + 6, 1), (1, 1, 1, (1 << 24) + 6, 1),
                                        (1 << 17, 2, 1, 1, (1 << 13) + 1)])
def test_steps_of_more_than_one_launch(gpu, S, L, Hk, H, P):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of GPU memory")
    p = problem(S, L, Hk, H, 1, P, torch.bfloat16, seed=30)
    o, s = delta_rule(*p)
    seqs, heads = (S, H // 2) if S == 1 else (S // 2, H)
    for first in (True, False):
        at = ((0, seqs) if first else (S - seqs, S)) if S > 1 else (0, 1), ((0, heads) if first else (H - heads, H)) if S == 1 else (0, H)
        (a, b), (c, d) = at
        o1, s1 = delta_rule(*of(p, *at, H // Hk))
        assert torch.equal(o1, o[a:b, :, c:d]) and torch.equal(s1, s[a:b, c:d])
