"""The delta rule's gradients from a gradient of its outputs in any layout: the same bits as from a dense copy."""
import pytest
import torch

from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def layouts(S, L, H, P, dtype, seed):
    """d_o [S, L, H, P] as a user's program may have it."""
    yield normal(S, L, H, P, seed=seed, dtype=dtype).transpose(0, 1).contiguous().transpose(0, 1)          # sequences inside tokens
    yield normal(S, H, L, P, seed=seed + 1, dtype=dtype).transpose(1, 2)                                   # heads outside tokens
    yield normal(S, L, 2 * H * P + 3, seed=seed + 2, dtype=dtype)[..., 3:H * P + 3].unflatten(-1, (H, P))  # columns of a wider row
    yield normal(S, L, H, P + 1, seed=seed + 3, dtype=dtype)[..., 1:]                                      # unaligned, odd strides
    yield normal(1, 1, 1, P, seed=seed + 4, dtype=dtype).expand(S, L, H, P)                                # one row for all
    yield normal(S, 1, H, P, seed=seed + 5, dtype=dtype).expand(S, L, H, P)
    yield normal(S, 2 * L, H, P, seed=seed + 6, dtype=dtype)[:, ::2]                                       # every other token


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("S,L,Hk,H,N,P", [(2, 5, 1, 2, 24, 40), (2, 150, 2, 6, 40, 33), (3, 130, 1, 2, 128, 64), (1, 70, 64, 256, 16, 32)])
def test_gradients_of_outputs_in_any_layout(gpu, S, L, Hk, H, N, P, dtype):
    q, k = (normal(S, L, Hk, N, seed=i, dtype=dtype) / N ** 0.5 for i in (1, 2))
    v, g, beta = normal(S, L, H, P, seed=3, dtype=dtype), -torch.rand(S, L, H, device="cuda"), torch.rand(S, L, H, device="cuda")
    s0, ds = normal(S, H, N, P, seed=4), normal(S, H, N, P, seed=5)
    for do in layouts(S, L, H, P, dtype, 10):
        assert do.shape == v.shape
        want = delta_rule_backward(do.contiguous(), q, k, v, g, beta, s0, ds)
        got = delta_rule_backward(do, q, k, v, g, beta, s0, ds)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("L,tok,seq", [(300, (1 << 23) + 24, 64), (3, 200, (1 << 31) + 72), (70, 200, (1 << 31) + 72)])
def test_gradients_of_outputs_past_32_bits(gpu, L, tok, seq):
    S, H, N, P = 2, 2, 24, 32
    q, k = (normal(S, L, 1, N, seed=i, dtype=torch.bfloat16) / 5 for i in (1, 2))
    v, g, beta = normal(S, L, H, P, seed=3, dtype=torch.bfloat16), -torch.rand(S, L, H, device="cuda"), torch.rand(S, L, H, device="cuda")
    do = torch.empty((S - 1) * seq + L * tok, dtype=torch.bfloat16, device="cuda").as_strided((S, L, H, P), (seq, tok, P, 1), 0)
    do.copy_(normal(S, L, H, P, seed=4, dtype=torch.bfloat16))
    want = delta_rule_backward(do.contiguous(), q, k, v, g, beta)
    assert all(torch.equal(a, b) for a, b in zip(delta_rule_backward(do, q, k, v, g, beta), want))


@pytest.mark.parametrize("L,tok", [(5, (1 << 31) + 8), (300, (1 << 23) + 8)])
def test_gates_past_32_bits(gpu, L, tok):
    # Gates whose tokens lie gigabytes apart.
    S, H, N, P = 2, 3, 24, 32
    q, k = (normal(S, L, 1, N, seed=i, dtype=torch.bfloat16) / 5 for i in (1, 2))
    v, do = (normal(S, L, H, P, seed=i, dtype=torch.bfloat16) for i in (3, 4))
    g, beta = -torch.rand(S, L, H, device="cuda"), torch.rand(S, L, H, device="cuda")
    want = (*delta_rule(q, k, v, g, beta), *delta_rule_backward(do, q, k, v, g, beta))
    buf = torch.empty((L - 1) * tok + 64, device="cuda")
    far = [buf.as_strided((S, L, H), (8, tok, 1), at) for at in (0, 32)]
    for x, y in zip(far, (g, beta)):
        x.copy_(y)
    got = (*delta_rule(q, k, v, *far), *delta_rule_backward(do, q, k, v, *far))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
