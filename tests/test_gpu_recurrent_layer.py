"""examples/recurrent_layer.py: the layer operators together, served and trained."""
import importlib.util
import os

import pytest
import torch

from helix_amd.norm import quantize_fp8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "recurrent_layer.py")
    spec = importlib.util.spec_from_file_location("recurrent_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def normal(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def plain(w, x, residual, state=None):
    """The layer without roundings, differentiable."""
    r = x + residual
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 1e-5) * w[2]
    g, v = (y @ w[0].T).chunk(2, -1)
    f = torch.sigmoid(g)
    hs, h = [], torch.zeros_like(v[:, 0]) if state is None else state
    for t in range(x.shape[1]):
        h = f[:, t] * h + (1 - f[:, t]) * v[:, t]
        hs.append(h)
    h = torch.stack(hs, 1)
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * w[3]
    return y @ w[1].T, r


def dequantized(t):
    q, s = quantize_fp8(t)
    return q.double() * s.double().repeat_interleave(128, -1)[..., :t.shape[-1]]


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# Values in 8 bits are within 2^-4 of themselves (half a step of three bits), and there are two layers of them.
@pytest.mark.parametrize("S,L,dim,inner", [(1, 300, 256, 384), (3, 5, 200, 130), (4, 1, 512, 256)])
def test_served_against_plain(gpu, layer, S, L, dim, inner):
    w = layer.Weights(dim, inner, seed=1)
    x, residual = normal(S, L, dim, seed=2, dtype=torch.bfloat16), normal(S, L, dim, seed=3, dtype=torch.bfloat16)
    state = normal(S, inner, seed=4)
    out, r, _ = layer.Served(w)(x, residual, state)
    exact = [dequantized(w.w_in), dequantized(w.w_out), w.norm_in.double(), w.norm_out.double()]
    want, want_r = plain(exact, x.double(), residual.double(), state.double())
    assert relative(out, want) < 2 * 2.0 ** -4
    assert relative(r, want_r) < 2.0 ** -8


# A value at the border of two codes may take the other one where another kernel's sum rounds otherwise: a step, 2^-3 at
# most, of some of them.
def test_tokens_one_by_one(gpu, layer):
    w = layer.Weights(256, 384, seed=5)
    served = layer.Served(w)
    x = normal(2, 150, 256, seed=6, dtype=torch.bfloat16)
    whole, _, last = served(x)
    out, _, state = served(x[:, :140].contiguous())
    outs = [out]
    for t in range(140, 150):
        out, _, state = served(x[:, t:t + 1].contiguous(), None, state)
        outs.append(out)
    assert relative(torch.cat(outs, 1), whole.double()) < 2.0 ** -4
    assert relative(state, last.double()) < 2.0 ** -4


# Every operation's error in float32 is a few 2^-24 of sums of up to 384 terms: 1e-4 holds them all.
def test_gradients(gpu, layer):
    w = layer.Weights(96, 130, dtype=torch.float32, seed=7)
    x, residual = (normal(2, 40, 96, seed=8 + i).requires_grad_() for i in range(2))
    dout, dr = normal(2, 40, 96, seed=10), normal(2, 40, 96, seed=11)
    for p in w.parameters():
        p.requires_grad_(True)
    leaves = [x, residual, *w.parameters()]
    got = torch.autograd.grad(layer.train_forward(w, x, residual), leaves, (dout, dr))
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = torch.autograd.grad(plain(exact[2:], exact[0], exact[1]), exact, (dout.double(), dr.double()))
    for g, e in zip(got, want):
        assert relative(g, e) < 1e-4


def test_training_lowers_the_loss(gpu, layer):
    w = layer.Weights(128, 256, seed=12)
    x, target = normal(2, 64, 128, seed=13, dtype=torch.bfloat16), normal(2, 64, 128, seed=14, dtype=torch.bfloat16)
    losses = layer.train(w, x, target, 5, lr=0.02)
    assert losses[-1] < losses[0]
