"""The delta rule's 16-bit results keep fp32's accuracy before they are rounded, token by token and in chunks: every element
against the 64-bit forms (delta_bits.py)."""
import pytest
import torch

import delta_bits as db
import delta_oracle as do_
from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def on_gpu(problem):
    return [None if t is None else t.cuda() for t in problem[:6]]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("L", [4, 20, 64, 70])
@pytest.mark.parametrize("make", [db.of_states, db.of_tokens])
def test_outputs_that_cancel(gpu, make, L, dtype):
    for seed in range(3):
        problem, size = make(L, dtype, seed)
        o, _ = delta_rule(*on_gpu(problem), scale=problem[6])
        db.within(o, db.outputs(problem), size, dtype, "o")


# A walk of one column block and of two, 64 keys and 128.
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("H,N,P", [(2, 64, 32), (2, 128, 32), (256, 64, 32), (256, 128, 32)])
def test_states_that_cancel_in_wide_heads(gpu, H, N, P, dtype):
    problem, size = db.of_states(20, dtype, 5, H, P)
    q, k, v, g, beta, s0, scale = problem
    q, k = (torch.nn.functional.pad(t, (0, N - 2)) for t in (q, k))
    s0 = torch.nn.functional.pad(s0, (0, 0, 0, N - 2))
    o, _ = delta_rule(*on_gpu((q, k, v, g, beta, s0)), scale=scale)
    db.within(o, do_.forward(q, k, v, g, beta, s0, scale)[0], size, dtype, "o")


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("L", [4, 64, 70])
@pytest.mark.parametrize("make,name,at", [(db.of_dq, "dq", 0), (db.of_dk, "dk", 1)])
def test_gradients_that_cancel(gpu, make, name, at, L, dtype):
    for seed in range(3):
        do, problem, size = make(L, dtype, seed)
        got = delta_rule_backward(do.cuda(), *on_gpu(problem), scale=problem[6])[at]
        db.within(got, do_.backward(do, *problem[:6], None, problem[6])[0][at], size, dtype, name)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("L", [3, 16, 100, 200])
@pytest.mark.parametrize("N,P", [(64, 48), (128, 64), (37, 21)])
def test_every_element_of_ordinary_outputs(gpu, N, P, L, dtype):
    gen = torch.Generator().manual_seed(L + N)
    q, k = (torch.nn.functional.normalize(torch.randn(2, L, 2, N, generator=gen), dim=-1).to(dtype) for _ in range(2))
    v = torch.randn(2, L, 4, P, generator=gen).to(dtype)
    g, beta = -0.3 * torch.rand(2, L, 4, generator=gen), torch.rand(2, L, 4, generator=gen)
    problem = (q, k, v, g, beta, 0.3 * torch.randn(2, 4, N, P, generator=gen), N ** -0.5)
    want, size = db.ordinary(*problem)
    db.within(delta_rule(*on_gpu(problem))[0], want, size, dtype, "o")
