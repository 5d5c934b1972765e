"""A gated recurrent layer from the layer operators: served in 8 bits, trained in the storage type.

    r  = residual + x                      rms_norm_fp8(x, w1, residual) -> 8 bits, r
    g, v = norm(r) W_in                    matmul_fp8 against [2 inner, dim]
    h_t = f h_(t-1) + (1 - f) v, f = sigmoid(g)    gated_scan, the state carried from call to call
    out = norm(h) W_out                    rms_norm_fp8(h, w2), matmul_fp8 against [dim, inner]

    python examples/recurrent_layer.py [--dim 2048] [--inner 4096] [--prompt 8192] [--tokens 64]

serves a prompt and then single tokens, and takes a few training steps. Random weights and inputs.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from helix_amd.matmul import matmul_fp8  # noqa: E402
from helix_amd.norm import quantize_fp8, rms_norm, rms_norm_backward, rms_norm_fp8  # noqa: E402
from helix_amd.recurrence import gated_scan, gated_scan_backward  # noqa: E402


class Weights:
    """Of one layer: w_in [2 inner, dim] (the gates' rows first), w_out [dim, inner], and both norms'."""

    def __init__(self, dim: int, inner: int, dtype=torch.bfloat16, device="cuda", seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)

        self.w_in = normal(2 * inner, dim, scale=dim ** -0.5)
        self.w_out = normal(dim, inner, scale=inner ** -0.5)
        self.norm_in = torch.ones(dim, device=device)
        self.norm_out = torch.ones(inner, device=device)

    def parameters(self):
        return [self.w_in, self.w_out, self.norm_in, self.norm_out]


class Served:
    """The layer in 8 bits. Its projections are laid out once; every call takes and returns the state."""

    def __init__(self, w: Weights):
        self.inner = w.w_out.shape[1]
        self.w_in, self.w_out = quantize_fp8(w.w_in), quantize_fp8(w.w_out)
        self.norm_in, self.norm_out = w.norm_in, w.norm_out

    def __call__(self, x, residual=None, state=None):
        """x, residual [sequences, tokens, dim], state [sequences, inner] (None: a fresh sequence): returns (out,
        residual, state) for the next layer and the next call. One token per sequence is the step of a decoder."""
        q, scale, residual = rms_norm_fp8(x, self.norm_in, residual)
        gv = matmul_fp8(q, scale, *self.w_in, out_dtype=x.dtype)
        h, state = gated_scan(gv[..., :self.inner], gv[..., self.inner:], state)
        q, scale, _ = rms_norm_fp8(h, self.norm_out)
        return matmul_fp8(q, scale, *self.w_out, out_dtype=x.dtype), residual, state


class Decoder:
    """Single tokens through a captured step: a replay takes the state that the one before left."""

    def __init__(self, layer: Served, state, dtype=torch.bfloat16):
        dim = layer.norm_in.shape[0]
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


class Norm(torch.autograd.Function):
    """rms_norm of x + residual: (y, h)."""

    @staticmethod
    def forward(ctx, x, weight, residual):
        y, h, rstd = rms_norm(x, weight, residual)
        ctx.save_for_backward(h, weight, rstd)
        ctx.set_materialize_grads(False)
        ctx.added = residual is not None
        return (y, h) if ctx.added else (y, None)

    @staticmethod
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        dy = torch.zeros_like(h) if dy is None else dy.contiguous()
        dx, dweight = rms_norm_backward(dy, h, weight, rstd, None if dh is None else dh.contiguous())
        return dx, dweight.to(weight.dtype), dx if ctx.added else None


class Recurrence(torch.autograd.Function):
    """gated_scan from a state of zeros over gv = [g, v]: h. g and v are read where the projection left them."""

    @staticmethod
    def forward(ctx, gv):
        g, v = gv.chunk(2, -1)
        h, _ = gated_scan(g, v)
        ctx.save_for_backward(gv, h)
        return h

    @staticmethod
    def backward(ctx, dh):
        gv, h = ctx.saved_tensors
        dg, dv, _ = gated_scan_backward(dh.contiguous(), *gv.chunk(2, -1), h)
        return torch.cat((dg, dv), -1)


def train_forward(w: Weights, x, residual):
    """(out, residual), with gradients for the weights and both inputs."""
    y, residual = Norm.apply(x, w.norm_in, residual)
    h = Recurrence.apply(y @ w.w_in.T)
    y, _ = Norm.apply(h, w.norm_out, None)
    return y @ w.w_out.T, residual


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
    ap.add_argument("--inner", type=int, default=4096)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--train-steps", type=int, default=4)
    a = ap.parse_args()
    w = Weights(a.dim, a.inner)
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
    whole = layer(x)[0][:, a.prompt:].float()
    if steps:
        error = (torch.cat(steps, 1).float() - whole).norm() / whole.norm()
        print(f"{a.tokens} tokens one by one against all at once: {error.item():.2e}")
        print(f"captured and eager tokens are equal: {torch.equal(torch.cat(captured, 1), torch.cat(steps, 1))}")
    losses = train(w, x[:, :min(a.prompt, 1024)], torch.randn_like(x[:, :min(a.prompt, 1024)]), a.train_steps)
    print("training loss: " + ", ".join(f"{v:.4f}" for v in losses))


if __name__ == "__main__":
    main()
