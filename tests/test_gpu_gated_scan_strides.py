"""helix_amd.recurrence on rows that are the same memory for several tokens: what lies past a sequence's ends, where a
run of tokens goes on over them, must not enter."""
import pytest
import torch

import layer_oracle as lo
from helix_amd.recurrence import gated_scan, gated_scan_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def check_backward(dh, g, v, h, h0, dh_last):
    want = lo.scan_backward(dh, g, v, h, h0, dh_last)
    bounds = lo.scan_backward_bound(dh, g, v, h, h0, dh_last, want[0], want[1])
    got = gated_scan_backward(dh, g, v, h, h0, dh_last)
    for name, a, b, c in zip(("dg", "dv", "dh0"), got, want, bounds):
        lo.within(a, b, c, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 16, 17, 31, 33, 64, 65, 150, 513, 1030])
@pytest.mark.parametrize("D", [72, 129])
def test_gradient_of_a_sum_over_tokens(gpu, L, D, dtype):
    # dh of h.sum(1) and of h.sum((0, 1)): token and sequence strides of 0.
    g, v, h0 = (2 + normal(2, L, D, seed=1)).to(dtype), normal(2, L, D, seed=2, dtype=dtype), normal(2, D, seed=3)
    h, _ = gated_scan(g, v, h0)
    check_backward(normal(2, 1, D, seed=4, dtype=dtype).expand(2, L, D), g, v, h, h0, normal(2, D, seed=5))
    check_backward(normal(1, 1, D, seed=6, dtype=dtype).expand(2, L, D), g, v, h, None, None)


@pytest.mark.parametrize("L", [17, 43, 150, 300])
def test_rows_that_overlap(gpu, L):
    # Tokens 8 elements apart, 96 of each: all inputs but h are windows of one line.
    line = normal(8 * L + 400, seed=7)
    window = [line.as_strided((1, L, 96), (0, 8, 1), o) for o in (0, 101, 203)]
    h0 = normal(1, 96, seed=8)
    h64, last64 = lo.scan(window[0], window[1], h0)
    bh, bl = lo.scan_bound(window[0], window[1], h0, h64)
    h, last = gated_scan(window[0], window[1], h0)
    lo.within(h, h64, bh, "h")
    lo.within(last, last64, bl, "last")
    check_backward(window[2], window[0], window[1], h, h0, normal(1, 96, seed=9))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [17, 150])
def test_one_value_for_all_tokens(gpu, L, dtype):
    # v the same at every token, infinite in one channel: infinite from the first token on, and no NaN after the last.
    g, v = normal(1, L, 70, seed=10, dtype=dtype), normal(1, 1, 70, seed=11, dtype=dtype)
    v[0, 0, 9] = float("inf")
    h, last = gated_scan(g, v.expand(1, L, 70))
    assert (h[0, :, 9] == float("inf")).all() and last[0, 9] == float("inf")
    keep = torch.arange(70, device="cuda") != 9
    g, v = g[..., keep], v[..., keep]
    h64, last64 = lo.scan(g, v.expand(1, L, 69), None)
    bh, bl = lo.scan_bound(g, v.expand(1, L, 69), None, h64)
    lo.within(h[..., keep], h64, bh, "h")
    lo.within(last[..., keep], last64, bl, "last")


@pytest.mark.parametrize("L", [5, 17, 100])
def test_one_state_for_all_tokens(gpu, L):
    # h as one row for all tokens: before the first token there is h0, or nothing, and not that row.
    g, v, dh = normal(1, L, 64, seed=12), normal(1, L, 64, seed=13), normal(1, L, 64, seed=14)
    row = normal(1, 1, 64, seed=15).expand(1, L, 64)
    check_backward(dh, g, v, row, None, None)
    check_backward(dh, g, v, row, normal(1, 64, seed=16), None)
