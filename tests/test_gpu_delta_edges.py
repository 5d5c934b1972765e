"""The delta rule where a call leaves little to do or values are at the ends of their types."""
import pytest
import torch

import delta_oracle as do_
import layer_oracle as lo
from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
def test_query_heads_without_value_heads(gpu, dtype):
    # Their gradients are sums over no heads: zeros, whatever the memory held.
    q = torch.full((2, 70, 3, 40), float("nan"), device="cuda", dtype=dtype)
    v, g = torch.empty(2, 70, 0, 8, device="cuda", dtype=dtype), torch.empty(2, 70, 0, device="cuda")
    for _ in range(3):
        stale = [torch.full_like(q, float("nan")) for _ in range(8)]
        del stale
        dq, dk, dv, dg, dbeta, ds0 = delta_rule_backward(v, q, q, v, g, g)
        assert (dq == 0).all() and (dk == 0).all()
        assert dv.shape == v.shape and dg.shape == dbeta.shape == g.shape and ds0.shape == (2, 0, 40, 8)


def problem(S, L, Hk, H, N, P, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.nn.functional.normalize(torch.randn(S, L, Hk, N, generator=gen), dim=-1).to(dtype).cuda() for _ in range(2))
    v = torch.randn(S, L, H, P, generator=gen).to(dtype).cuda()
    g, beta = (torch.rand(S, L, H, generator=gen).cuda() for _ in range(2))
    return q, k, v, -g, beta, 0.3 * torch.randn(S, H, N, P, generator=gen).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,n", [(6, 3), (20, 11), (64, 63), (150, 70), (150, 128)])
@pytest.mark.parametrize("fill", ["lowest", "largest"])
def test_masked_tokens_of_the_lowest_value(gpu, fill, L, n, dtype):
    # Tokens with g = 0 and beta = 0 bring nothing, whatever finite v they have: the type's ends are.
    q, k, v, g, beta, s0 = problem(2, L, 1, 2, 40, 24, dtype, L)
    g[:, n:], beta[:, n:] = 0, 0
    v2 = v.clone()
    v2[:, n:] = torch.finfo(dtype).min if fill == "lowest" else torch.finfo(dtype).max
    v[:, n:] = 0
    o, s = delta_rule(q, k, v, g, beta, s0)
    o2, s2 = delta_rule(q, k, v2, g, beta, s0)
    assert o2.isfinite().all() and torch.equal(o2, o) and torch.equal(s2, s)
    do, ds = torch.randn_like(v), torch.randn_like(s0)
    do[:, n:] = 0
    for name, a, b in zip(("dq", "dk", "dv", "dg", "ds0"), *((x[0], x[1], x[2], x[3], x[5]) for x in (
            delta_rule_backward(do, q, k, t, g, beta, s0, ds) for t in (v, v2)))):
        assert a.isfinite().all() and torch.equal(a, b), name


# In fp32 the ends of the type are not a bf16 number: an operand's first part must not round to infinity.
@pytest.mark.parametrize("L", [5, 70])
def test_values_at_the_end_of_fp32(gpu, L):
    q, k, v, g, beta, _ = problem(1, L, 1, 1, 8, 16, torch.float32, 3)
    top = torch.finfo(torch.float32).max
    v[:, 2, :, :8] = top * (1 - torch.arange(8, device="cuda") * 2.0 ** -12)
    v[:, 3:] = 0
    beta[:, 2] = 1e-3
    sc = 8 ** -0.5
    want, states, _ = do_.forward(q, k, v, g, beta, None, sc)
    so, ss = do_.forward_sizes(q, states, sc, 1)
    o, s = delta_rule(q, k, v, g, beta)
    do_.close(o, want, so, torch.float32, "o")
    do_.close(s, states[-1], ss, torch.float32, "s")
    # q and k as large, the other of them small.
    big, small = q.clone(), k * 1e-38
    big[:, 1:3] = top * q[:, 1:3].sign()
    o, s = delta_rule(big, small, 1e30 * torch.ones_like(v), torch.zeros_like(g), beta)
    assert o.isfinite().all() and s.isfinite().all()
    want, states, _ = do_.forward(big, small, 1e30 * torch.ones_like(v), torch.zeros_like(g), beta, None, sc)
    so, _ = do_.forward_sizes(big, states, sc, 1)
    # Keys of 1e-38 are at the other end: a bf16 part is right to half of its least, 2^-134, so that an element of k is off by
    # that much in itself and o_t = scale sum over j of (q_t . k_j) d_j by scale |q_t| sqrt(8) 2^-134 sum |d_j|, where
    # |d_j| = beta_j 1e30 sqrt(16) (what earlier keys take from it is below 1e-38 of that). In the 2-norm over all t:
    d = lo.f64(beta)[0, :, 0].cumsum(0) * 1e30 * 4
    least = float((sc * lo.f64(big)[0, :, 0].norm(dim=-1) * 8 ** 0.5 * 2.0 ** -134 * d).norm())
    off = float((lo.f64(o) - want).norm())
    assert off <= do_.FP32 * so + least, (off, do_.FP32 * so, least)


@pytest.mark.parametrize("N", [8, 72])
@pytest.mark.parametrize("L", [5, 70])
def test_gradients_of_outputs_at_the_end_of_fp32(gpu, L, N):
    # With scale 1 and no decay, what multiplies the queries is at the end too. (Small q and v: all that follows stays finite.)
    q, k, v, g, beta, _ = problem(1, L, 1, 1, N, 16, torch.float32, 5)
    q, v, g = 1e-3 * q, 1e-2 * v, torch.zeros_like(g)
    do = torch.zeros_like(v)
    do[:, 2, :, :8] = torch.finfo(torch.float32).max * (1 - torch.arange(8, device="cuda") * 2.0 ** -12)
    want, size = do_.backward(do, q, k, v, g, beta, None, None, 1.0)
    got = delta_rule_backward(do, q, k, v, g, beta, scale=1.0)
    for n, a, b in zip(("dq", "dk", "dv", "dg", "dbeta", "ds0"), got, want):
        assert a.isfinite().all(), n
        # (In units of 2^100, whose squares a norm can add.)
        do_.close(a.double() * 2.0 ** -100, b * 2.0 ** -100, size[n] * 2.0 ** -100, torch.float32, n)
