"""The layer operators on more rows, sequences and columns than one launch can count threads for (2^32): the same bits as in
pieces that it can."""
import pytest
import torch

from helix_amd.matmul import matmul_fp8
from helix_amd.norm import quantize_fp8, rms_norm, rms_norm_backward
from helix_amd.recurrence import gated_scan, gated_scan_backward

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


@pytest.fixture(autouse=True)
def memory(gpu):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of GPU memory")
    yield
    torch.cuda.empty_cache()


def test_norm_of_many_narrow_rows(gpu):
    # A wave a row: 2^26 - 4 of them a launch.
    rows, dim = (1 << 26) + 1029, 2
    x, r = normal(rows, dim, seed=1, dtype=torch.bfloat16), normal(rows, dim, seed=2, dtype=torch.bfloat16)
    w = 1 + normal(dim, seed=3)
    whole = rms_norm(x, w, r)
    half = rows // 2
    for part in (slice(0, half), slice(half, rows)):
        for a, b in zip(whole, rms_norm(x[part], w, r[part])):
            assert torch.equal(a[part], b)
    # The gradients go through the rows part by part, and as many as there are.
    dx, dw = rms_norm_backward(r, whole[1], w, whole[2])
    dx2, dw2 = rms_norm_backward(r[half:], whole[1][half:], w, whole[2][half:])
    assert torch.equal(dx[half:], dx2) and torch.isfinite(dw).all() and torch.isfinite(dw2).all()


def test_norm_of_many_wide_rows(gpu):
    # A workgroup a row: 2^24 - 1 of them a launch. One row for all to read, 35 GB to write.
    rows, dim = (1 << 24) + 3, 2049
    x = normal(1, dim, seed=4, dtype=torch.bfloat16)
    q, scale = quantize_fp8(x.expand(rows, dim))
    one, one_scale = quantize_fp8(x)
    for at in range(0, rows, 1 << 20):
        assert (q.view(torch.uint8)[at:at + (1 << 20)] == one.view(torch.uint8)).all(), at
    assert (scale.view(torch.uint8) == one_scale.view(torch.uint8)).all()


@pytest.mark.parametrize("S,L", [((1 << 24) + 5, 17), ((1 << 22) + 3, 260)])
def test_recurrence_of_many_sequences(gpu, S, L):
    g, v, h0 = (normal(S, L, 1, seed=s, dtype=torch.float16) for s in (5, 6, 7))
    h0 = h0[:, 0].float()
    h, last = gated_scan(g, v, h0)
    grads = gated_scan_backward(v, g, v, h, h0, last)
    half = S // 2
    for part in (slice(0, half), slice(half, S)):
        h2, last2 = gated_scan(g[part], v[part], h0[part])
        assert torch.equal(h[part], h2) and torch.equal(last[part], last2)
        for a, b in zip(grads, gated_scan_backward(v[part], g[part], v[part], h2, h0[part], last2)):
            assert torch.equal(a[part], b)


@pytest.mark.parametrize("m,n", [(1, (1 << 28) + 37), (17, (1 << 27) + 37)])
def test_product_with_many_columns(gpu, m, n):
    # 16 columns a workgroup, of four or eight waves.
    gen = torch.Generator(device="cuda").manual_seed(8)
    a, sa = quantize_fp8(normal(m, 16, seed=9))
    b = torch.randint(0, 0x70, (n, 16), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    sb = torch.randint(120, 130, (n, 1), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu)
    c = matmul_fp8(a, sa, b, sb)
    third = n // 3 // 16 * 16
    for part in (slice(0, third), slice(third, 2 * third), slice(2 * third, n)):
        assert torch.equal(c[:, part], matmul_fp8(a, sa, b[part], sb[part]))
