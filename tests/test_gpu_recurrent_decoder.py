"""examples/recurrent_layer.py: tokens through the captured step, which carries its state, against the eager ones."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "recurrent_layer.py")
    spec = importlib.util.spec_from_file_location("recurrent_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("S,dim,inner", [(1, 256, 384), (5, 200, 130), (20, 2048, 4096)])
@pytest.mark.parametrize("residual", [False, True])
def test_captured_tokens_equal_the_eager_ones(gpu, layer, S, dim, inner, residual):
    served = layer.Served(layer.Weights(dim, inner, seed=1))
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(S, 30, dim, generator=gen, device="cuda").bfloat16()
    r = torch.randn(S, 30, dim, generator=gen, device="cuda").bfloat16() if residual else torch.zeros_like(x)
    _, _, state = served(x[:, :20].contiguous(), r[:, :20].contiguous())
    decoder = layer.Decoder(served, state)
    for t in range(20, 30):
        out, left, state = served(x[:, t:t + 1], r[:, t:t + 1], state)
        got, got_left = decoder(x[:, t:t + 1], r[:, t:t + 1] if residual else None)
        assert torch.equal(got, out) and torch.equal(got_left, left) and torch.equal(decoder.state, state)
