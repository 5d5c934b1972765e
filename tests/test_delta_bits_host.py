"""The checks of every element of the delta rule's 16-bit outputs (delta_bits.py) see what loses bits: planted in the 64-bit
forms, on the CPU."""
import pytest
import torch

import delta_bits as db
import delta_oracle as do_
from layer_oracle import f64

HALVES = [torch.float16, torch.bfloat16]


def parts(x, n):
    """x as the sum of n bf16 parts."""
    left, out = f64(x), 0
    for _ in range(n):
        part = left.to(torch.bfloat16).double()
        out, left = out + part, left - part
    return out


def truncated(x, dtype):
    """x cut, not rounded, to dtype."""
    y = x.float().to(dtype)
    over = f64(y).abs() > x.abs()
    return torch.where(over, (y.view(torch.int16) - 1).view(dtype), y)


@pytest.mark.parametrize("dtype", HALVES)
def test_three_parts_and_one_rounding_pass(dtype):
    for make in (db.of_states, db.of_tokens):
        problem, size = make(20, dtype, 1)
        want = db.outputs(problem)
        db.within(want.float().to(dtype), want, size, dtype, make.__name__)
        q, k, v, g, beta, s0, scale = problem
        if s0 is not None:
            got = do_.forward(q, k, v, g, beta, parts(s0, 3), scale)[0]
            db.within(got.float().to(dtype), want, size, dtype, make.__name__)
    for make, at in ((db.of_dq, 0), (db.of_dk, 1)):
        do, problem, size = make(20, dtype, 2)
        want = do_.backward(do, *problem[:6], None, problem[6])[0][at]
        assert 0 < float(want.abs().max()) < 2.0 ** -11 * float(size.max())
        db.within(want.float().to(dtype), want, size, dtype, make.__name__)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("n", [1, 2])
def test_fewer_parts_are_seen(dtype, n):
    problem, size = db.of_states(20, dtype, 3)
    q, k, v, g, beta, s0, scale = problem
    with pytest.raises(AssertionError):
        db.within(do_.forward(q, k, v, g, beta, parts(s0, n), scale)[0].float().to(dtype), db.outputs(problem), size, dtype, "o")
    # D, in an output's sum of what the tokens brought.
    problem, size = db.of_tokens(20, dtype, 4)
    want, _, brought = do_.forward(*problem)
    lost = want.clone()
    lost[:, 2:] += sum(problem[0][:, 2:, :, i, None].double() * (parts(brought[i], n) - brought[i])[:, None] for i in range(2))
    with pytest.raises(AssertionError):
        db.within(lost.float().to(dtype), want, size, dtype, "o")
    # What multiplies the keys in dq, and the queries in dk.
    do, problem, size = db.of_dq(20, dtype, 5)
    want = do_.backward(do, *problem[:6], None, 1.0)[0][0]
    d = do_.forward(*problem)[2]
    m = [f64(do)[..., 0] * d[i][:, None, :, 0] for i in range(2)]
    off = (parts(m[0], n) - m[0]) - (parts(m[1], n) - m[1])
    got = want.clone()
    got[:, 2:, :, 0] += off[:, 2:]
    with pytest.raises(AssertionError):
        db.within(got.float().to(dtype), want, size, dtype, "dq")
    do, problem, size = db.of_dk(20, dtype, 6)
    want = do_.backward(do, *problem[:6], None, 1.0)[0][1]
    d, decay = do_.forward(*problem)[2], torch.exp(f64(problem[3][:, 2]))
    m = [f64(do)[:, 1, :, 0] * d[0][..., 0], f64(do)[:, 2, :, 0] * decay * d[0][..., 0]]
    got = want.clone()
    got[:, 0, :, 0] += (parts(m[0], n) - m[0]) - (parts(m[1], n) - m[1])
    with pytest.raises(AssertionError):
        db.within(got.float().to(dtype), want, size, dtype, "dk")


@pytest.mark.parametrize("dtype", HALVES)
def test_cutting_for_rounding_is_seen(dtype):
    gen = torch.Generator().manual_seed(7)
    q, k = (torch.nn.functional.normalize(torch.randn(1, 70, 2, 24, generator=gen), dim=-1).to(dtype) for _ in range(2))
    v, g, beta = torch.randn(1, 70, 2, 16, generator=gen).to(dtype), -torch.rand(1, 70, 2, generator=gen), torch.rand(1, 70, 2, generator=gen)
    want, size = db.ordinary(q, k, v, g, beta, None, 24 ** -0.5)
    db.within(want.float().to(dtype), want, size, dtype, "o")
    with pytest.raises(AssertionError):
        db.within(truncated(want, dtype), want, size, dtype, "o")
