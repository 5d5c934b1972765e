"""examples/delta_layer.py: the norms, the projections, the delta rule and the group norm together, served and trained."""
import importlib.util
import os

import pytest
import torch

from helix_amd.norm import quantize_fp8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "delta_layer.py")
    spec = importlib.util.spec_from_file_location("delta_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def normal(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def plain(w, p, x, residual, state=None):
    """The layer without roundings, token by token and differentiable; p: w_in, w_out, both norms, log_rate and bias."""
    r = x + residual
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-5) * p[2]
    qk, v, gate, a, b = w.split(y @ p[0].T)
    q, k = torch.nn.functional.normalize(qk, dim=-1).repeat_interleave(w.heads // w.qk_heads, -2).split(w.heads, -2)
    decay, beta = torch.exp(-torch.exp(p[4]) * torch.nn.functional.softplus(a + p[5])), torch.sigmoid(b)
    S = torch.zeros(x.shape[0], w.heads, w.keys, w.values, dtype=x.dtype, device=x.device) if state is None else state
    o = []
    for t in range(x.shape[1]):
        S = decay[:, t, :, None, None] * S
        d = beta[:, t, :, None] * (v[:, t] - (S * k[:, t, ..., None]).sum(-2))
        S = S + k[:, t, ..., None] * d[..., None, :]
        o.append(w.keys ** -0.5 * (S * q[:, t, ..., None]).sum(-2))
    o = torch.stack(o, 1)
    d = o - o.mean(-1, keepdim=True)
    n = (d * torch.rsqrt(d.square().mean(-1, keepdim=True) + 1e-5)).flatten(-2) * p[3]
    return (n * torch.nn.functional.silu(gate)) @ p[1].T, r


def dequantized(t):
    q, s = quantize_fp8(t)
    return q.double() * s.double().repeat_interleave(128, -1)[..., :t.shape[-1]]


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# Values in 8 bits are within 2^-4 of themselves (half a step of three bits): the input's and the group norm's, and the first
# are in the heads' variance twice, once for each of v and the keys that it is corrected by.
@pytest.mark.parametrize("S,L,dim,heads,qk,keys,values", [(1, 300, 256, 4, 2, 64, 64), (3, 5, 200, 6, 2, 40, 24),
                                                          (4, 1, 512, 8, 1, 128, 64)])
def test_served_against_plain(gpu, layer, S, L, dim, heads, qk, keys, values):
    w = layer.Weights(dim, heads, qk, keys, values, seed=1)
    x, residual = normal(S, L, dim, seed=2, dtype=torch.bfloat16), normal(S, L, dim, seed=3, dtype=torch.bfloat16)
    state = 0.3 * normal(S, heads, keys, values, seed=4)
    out, r, _ = layer.Served(w)(x, residual, state)
    exact = [dequantized(w.w_in), dequantized(w.w_out), *(t.double() for t in w.parameters()[2:])]
    want, want_r = plain(w, exact, x.double(), residual.double(), state.double())
    assert relative(out, want) < 4 * 2.0 ** -4
    assert relative(r, want_r) < 2.0 ** -8


# A value at the border of two codes may take the other one where another kernel's sum rounds otherwise: a step, 2^-3 at
# most, of some of them.
def test_tokens_one_by_one(gpu, layer):
    served = layer.Served(layer.Weights(256, 8, 2, seed=5))
    x = normal(2, 150, 256, seed=6, dtype=torch.bfloat16)
    whole, _, last = served(x)
    out, _, state = served(x[:, :140].contiguous())
    outs = [out]
    for t in range(140, 150):
        out, _, state = served(x[:, t:t + 1].contiguous(), None, state)
        outs.append(out)
    assert relative(torch.cat(outs, 1), whole.double()) < 2.0 ** -4
    assert relative(state, last.double()) < 2.0 ** -4


@pytest.mark.parametrize("S", [1, 5])
def test_captured_tokens_equal_the_eager_ones(gpu, layer, S):
    served = layer.Served(layer.Weights(256, 8, 2, seed=7))
    x, r = normal(S, 30, 256, seed=8, dtype=torch.bfloat16), normal(S, 30, 256, seed=9, dtype=torch.bfloat16)
    _, _, state = served(x[:, :20].contiguous(), r[:, :20].contiguous())
    decoder = layer.Decoder(served, state)
    for t in range(20, 30):
        out, left, state = served(x[:, t:t + 1], r[:, t:t + 1], state)
        got, got_left = decoder(x[:, t:t + 1], r[:, t:t + 1])
        assert torch.equal(got, out) and torch.equal(got_left, left) and torch.equal(decoder.state, state)


# Every operation's error in float32 is a few 2^-24 of sums of up to 256 terms, those of the recurrence of 2 80 tokens more:
# 1e-4 holds them all.
def test_gradients(gpu, layer):
    w = layer.Weights(96, 4, 2, 24, 20, dtype=torch.float32, seed=10)
    x, residual = (normal(2, 80, 96, seed=11 + i).requires_grad_() for i in range(2))
    dout, dr = normal(2, 80, 96, seed=13), normal(2, 80, 96, seed=14)
    for p in w.parameters():
        p.requires_grad_(True)
    leaves = [x, residual, *w.parameters()]
    got = torch.autograd.grad(layer.train_forward(w, x, residual), leaves, (dout, dr))
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(plain(w, exact[2:], exact[0], exact[1]), exact, (dout.double(), dr.double()))
    for g, e in zip(got, want):
        assert relative(g, e) < 1e-4


def test_training_runs(gpu, layer):
    w = layer.Weights(128, 4, 2, 64, 32, seed=15)
    x, target = normal(2, 64, 128, seed=16, dtype=torch.bfloat16), normal(2, 64, 128, seed=17, dtype=torch.bfloat16)
    before = [p.clone() for p in w.parameters()]
    losses = layer.train(w, x, target, 2, lr=0.02)
    assert all(v == v and v < float("inf") for v in losses)
    assert all(p.isfinite().all() and not torch.equal(p, b) for p, b in zip(w.parameters(), before))
