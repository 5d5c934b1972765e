"""A gated delta layer from the layer operators: served in 8 bits, trained in the storage type.

    r = residual + x                                         rms_norm_fp8(x, norm_in, residual) -> 8 bits, r
    q, k, v, gate, a, b = norm(r) W_in                       matmul_fp8, one projected row per token
    q, k of length one                                       rms_norm with a weight of keys ** -0.5
    g = -e^rate softplus(a + bias), beta = sigmoid(b)          decays and gains of the value heads
    S_t = e^g S_(t-1) + beta k (v - e^g S_(t-1)' k)', o = S_t' q     delta_rule, the state carried from call to call
    out = (norm of o's heads, gated) W_out                   group_norm_fp8, matmul_fp8

    python examples/delta_layer.py [--dim 2048] [--heads 64] [--qk-heads 8] [--prompt 8192] [--tokens 64]

serves a prompt and then single tokens, and takes a few training steps. Random weights and inputs.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path[:0] = [os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."), os.path.dirname(os.path.abspath(__file__))]

from helix_amd.delta import delta_rule, delta_rule_backward  # noqa: E402
from helix_amd.matmul import matmul_fp8  # noqa: E402
from helix_amd.norm import group_norm, group_norm_backward, group_norm_fp8, quantize_fp8, rms_norm, rms_norm_fp8  # noqa: E402
from recurrent_layer import Norm  # noqa: E402


class Weights:
    """Of one layer: w_in (rows of q, k, v, gate, a and b), w_out [dim, heads values], both norms', and the decays'."""

    def __init__(self, dim: int, heads: int, qk_heads: int, keys: int = 128, values: int = 64, dtype=torch.bfloat16,
                 device="cuda", seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)

        self.heads, self.qk_heads, self.keys, self.values = heads, qk_heads, keys, values
        self.parts = [2 * qk_heads * keys, heads * values, heads * values, heads, heads]
        self.w_in = normal(sum(self.parts), dim, scale=dim ** -0.5)
        self.w_out = normal(dim, heads * values, scale=(heads * values) ** -0.5)
        self.norm_in = torch.ones(dim, device=device)
        self.norm_out = torch.ones(heads * values, device=device)
        self.log_rate = torch.randn(heads, generator=g, device=device) - 2.5
        self.bias = 0.5 * torch.randn(heads, generator=g, device=device)
        self.length_one = torch.full((keys,), keys ** -0.5, device=device)

    def parameters(self):
        return [self.w_in, self.w_out, self.norm_in, self.norm_out, self.log_rate, self.bias]

    def split(self, row):
        """(q and k as [..., 2 qk_heads, keys], v, gate, a, b) of projected rows."""
        qk, v, gate, a, b = row.split(self.parts, -1)
        return qk.unflatten(-1, (2 * self.qk_heads, self.keys)), v.unflatten(-1, (self.heads, self.values)), gate, a, b

    def gates(self, a, b):
        g = -torch.exp(self.log_rate) * torch.nn.functional.softplus(a.float() + self.bias)
        return g, torch.sigmoid(b.float())


class Served:
    """The layer in 8 bits. Its projections are laid out once; every call takes and returns the state."""

    def __init__(self, w: Weights):
        self.w = w
        self.w_in, self.w_out = quantize_fp8(w.w_in), quantize_fp8(w.w_out)

    def __call__(self, x, residual=None, state=None):
        """x, residual [sequences, tokens, dim], state [sequences, heads, keys, values] (None: a fresh sequence): returns
        (out, residual, state) for the next layer and the next call. One token per sequence is the step of a decoder."""
        w = self.w
        q, scale, residual = rms_norm_fp8(x, w.norm_in, residual)
        qk, v, gate, a, b = w.split(matmul_fp8(q, scale, *self.w_in, out_dtype=x.dtype))
        qk = rms_norm(qk.contiguous(), w.length_one, eps=1e-6)[0]
        g, beta = w.gates(a, b)
        o, state = delta_rule(qk[..., :w.qk_heads, :], qk[..., w.qk_heads:, :], v, g, beta, state)
        q, scale = group_norm_fp8(o.flatten(-2), w.norm_out, None, gate, groups=w.heads)
        return matmul_fp8(q, scale, *self.w_out, out_dtype=x.dtype), residual, state


class Decoder:
    """Single tokens through a captured step: a replay takes the state that the one before left."""

    def __init__(self, layer: Served, state, dtype=torch.bfloat16):
        dim = layer.w.norm_in.shape[0]
        self.state = state.clone()
        self.x, self.residual = (torch.zeros(state.shape[0], 1, dim, dtype=dtype, device=state.device) for _ in range(2))
        layer(self.x, self.residual, self.state)   # (what a first call does once is not captured)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out, self.left, after = layer(self.x, self.residual, self.state)
            self.state.copy_(after)

    def __call__(self, x, residual=None):
        """x, residual [sequences, 1, dim]: (out, residual) in memory that the next call writes again."""
        self.x.copy_(x)
        if residual is None:
            self.residual.zero_()
        else:
            self.residual.copy_(residual)
        self.graph.replay()
        return self.out, self.left


class Delta(torch.autograd.Function):
    """delta_rule from a state of zeros: o."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta):
        o, _ = delta_rule(q, k, v, g, beta)
        ctx.save_for_backward(q, k, v, g, beta)
        return o

    @staticmethod
    def backward(ctx, do):
        return delta_rule_backward(do.contiguous(), *ctx.saved_tensors)[:5]


class GroupNorm(torch.autograd.Function):
    """group_norm with a gate: y."""

    @staticmethod
    def forward(ctx, x, weight, gate, groups):
        y, mean, rstd = group_norm(x, weight, None, gate, groups=groups)
        ctx.save_for_backward(x, weight, mean, rstd, gate)
        ctx.groups = groups
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd, gate = ctx.saved_tensors
        dx, dweight, _, dgate = group_norm_backward(dy.contiguous(), x, weight, mean, rstd, None, gate, groups=ctx.groups)
        return dx, dweight.to(weight.dtype), dgate, None


def train_forward(w: Weights, x, residual):
    """(out, residual), with gradients for the weights and both inputs."""
    y, residual = Norm.apply(x, w.norm_in, residual)
    qk, v, gate, a, b = w.split(y @ w.w_in.T)
    q, k = torch.nn.functional.normalize(qk.float(), dim=-1).to(x.dtype).split(w.qk_heads, -2)
    g, beta = w.gates(a, b)
    o = Delta.apply(q, k, v, g, beta)
    return GroupNorm.apply(o.flatten(-2), w.norm_out, gate, w.heads) @ w.w_out.T, residual


def train(w: Weights, x, target, steps: int, lr: float = 0.05) -> list[float]:
    """Steps of plain gradient descent towards target: the loss before each."""
    for p in w.parameters():
        p.requires_grad_(True)
    losses = []
    for _ in range(steps):
        out, residual = train_forward(w, x, torch.zeros_like(x))
        loss = ((out + residual).float() - target.float()).square().mean()
        losses.append(loss.item())
        grads = torch.autograd.grad(loss, w.parameters())
        with torch.no_grad():
            for p, g in zip(w.parameters(), grads):
                p -= lr * g / (g.float().square().mean().sqrt() + 1e-12) * p.float().square().mean().sqrt()
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--dim", type=int, default=2048)
    ap.add_argument("--heads", type=int, default=64)
    ap.add_argument("--qk-heads", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--train-steps", type=int, default=4)
    a = ap.parse_args()
    w = Weights(a.dim, a.heads, a.qk_heads)
    layer = Served(w)
    x = torch.randn(1, a.prompt + a.tokens, a.dim, device="cuda").to(torch.bfloat16)

    def clock(f, n):
        f()
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            f()
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n * 1e6

    out, _, state = layer(x[:, :a.prompt])
    print(f"prompt of {a.prompt}: {clock(lambda: layer(x[:, :a.prompt]), 20):.0f} us a layer")
    token = x[:, :1].contiguous()
    print(f"one token: {clock(lambda: layer(token, token, state), 200):.0f} us a layer")
    print(f"one token, captured, the state carried: {clock(Decoder(layer, state).graph.replay, 200):.0f} us a layer")
    decoder = Decoder(layer, state)
    steps, captured = [], []
    for t in range(a.prompt, a.prompt + a.tokens):
        out, _, state = layer(x[:, t:t + 1], None, state)
        steps.append(out)
        captured.append(decoder(x[:, t:t + 1])[0].clone())
    if steps:
        whole = layer(x)[0][:, a.prompt:].float()
        error = (torch.cat(steps, 1).float() - whole).norm() / whole.norm()
        print(f"{a.tokens} tokens one by one against all at once: {error.item():.2e}")
        print(f"captured and eager tokens are equal: {torch.equal(torch.cat(captured, 1), torch.cat(steps, 1))}")
    part = x[:, :min(a.prompt, 1024)]
    losses = train(w, part, torch.randn_like(part), a.train_steps)
    print("training loss: " + ", ".join(f"{v:.4f}" for v in losses))


if __name__ == "__main__":
    main()
