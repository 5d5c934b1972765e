"""helix_amd.matmul on the GPU against the 64-bit form of layer_oracle.py."""
import pytest
import torch

import layer_oracle as lo
from helix_amd.abi import HelixError
from helix_amd.matmul import matmul_fp8
from helix_amd.norm import fp8_rows, quantize_fp8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def operands(m, n, k, seed=0):
    # Columns of unequal size, so that a scale of the wrong block or row shows.
    a = normal(m, k, seed=seed) * torch.exp(normal(k, seed=seed + 1)) * torch.exp(normal(m, 1, seed=seed + 2))
    b = normal(n, k, seed=seed + 3) * torch.exp(normal(n, 1, seed=seed + 4)) / k ** 0.5
    return (*quantize_fp8(a), *quantize_fp8(b))


def check(a, sa, b, sb, dtype=torch.bfloat16, out=None):
    c = matmul_fp8(a, sa, b, sb, out_dtype=dtype, out=out)
    a2, sa2 = a.reshape(-1, a.shape[-1]), sa.reshape(-1, sa.shape[-1])
    want, size = lo.matmul(a2, sa2, b, sb)
    lo.within(c.reshape(-1, c.shape[-1]), want, lo.matmul_bound(want, size, a.shape[-1], c.dtype), "c")
    return c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 15, 16, 100, 128, 129, 256, 400, 640, 1024, 2047, 2048])
@pytest.mark.parametrize("m,n", [(1, 33), (5, 130), (67, 70)])
def test_depths(gpu, m, n, k, dtype):
    check(*operands(m, n, k, seed=k), dtype)


# Rows from one token to several tiles of every size, with and without a ragged edge.
@pytest.mark.parametrize("m", [1, 2, 8, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256, 257, 384, 511, 700])
@pytest.mark.parametrize("n,k", [(1, 256), (16, 384), (100, 512), (257, 272), (640, 1280)])
def test_rows(gpu, m, n, k):
    check(*operands(m, n, k, seed=m))


@pytest.mark.parametrize("m,n,k", [(1, 10304, 2048), (3, 2048, 4096), (16, 5184, 2000), (67, 2048, 4096),
                                   (300, 4104, 656), (1024, 1024, 512), (1500, 2600, 384), (2048, 2047, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_larger(gpu, m, n, k, dtype):
    check(*operands(m, n, k, seed=1), dtype)


@pytest.mark.parametrize("m,n,k", [(40, 2048, 4096), (67, 2560, 5120), (100, 130, 9000), (150, 640, 2900)])
def test_sum_in_parts(gpu, m, n, k):
    check(*operands(m, n, k, seed=8), torch.float16)
    a, sa, b, sb = operands(m, n, k, seed=9)
    assert torch.equal(check(a, sa, b, sb), matmul_fp8(a, sa, b, sb))


# More tiles than workgroups run at once, a last band of one row of tiles, rows and columns past the last tile.
@pytest.mark.parametrize("m,n,k,dtype", [(4400, 4200, 600, torch.bfloat16), (2060, 8210, 704, torch.float16),
                                         (700, 1003, 640, torch.bfloat16), (4500, 4300, 1200, torch.bfloat16)])
def test_many_tiles(gpu, m, n, k, dtype):
    check(*operands(m, n, k, seed=11), dtype)


def test_scales_of_any_alignment(gpu):
    # Rows of five scale bytes, one after the other, and from an odd address.
    m, n, k = 400, 300, 600
    a, sa, b, sb = operands(m, n, k, seed=10)
    want = check(a, sa, b, sb)
    flat = torch.empty((m + n) * 5 + 1, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    ta, tb = flat[1:1 + 5 * m].view(m, 5), flat[1 + 5 * m:].view(n, 5)
    ta.copy_(sa)
    tb.copy_(sb)
    assert torch.equal(matmul_fp8(a, ta, b, tb), want)
    assert torch.equal(matmul_fp8(a, sa, b, tb), want) and torch.equal(matmul_fp8(a, ta, b, sb), want)


def test_leading_dimensions_strides_and_out(gpu):
    m, n, k = 70, 90, 200
    a, sa, b, sb = operands(m, n, k, seed=2)
    wide_a, wide_b = (torch.full((r, 512), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for r in (m, n))
    wide_a[:, 16:16 + k] = a
    wide_b[:, 208:208 + k] = b
    wide_s = torch.full((m + n, 9), 255, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    wide_s[:m, 3:5] = sa
    wide_s[m:, 5:7] = sb
    want = matmul_fp8(a, sa, b, sb)
    # NaNs on either side of the rows and scales, and past the end of a row.
    va, vb, vsa, vsb = wide_a[:, 16:16 + k], wide_b[:, 208:208 + k], wide_s[:m, 3:5], wide_s[m:, 5:7]
    assert torch.equal(matmul_fp8(va, vsa, vb, vsb), want)
    out = torch.full((m, 2 * n + 1), 7.0, dtype=torch.bfloat16, device="cuda")
    got = matmul_fp8(va, vsa, vb, vsb, out=out[:, n:2 * n])
    assert got.data_ptr() == out[:, n:].data_ptr() and torch.equal(out[:, n:2 * n], want)
    assert (out[:, :n] == 7).all() and (out[:, 2 * n] == 7).all()
    lead = matmul_fp8(a.view(7, 10, k) if a.is_contiguous() else a.unflatten(0, (7, 10)), sa.view(7, 10, -1), b, sb)
    assert lead.shape == (7, 10, n) and torch.equal(lead.view(m, n), want)


@pytest.mark.parametrize("m", [3, 200])
def test_rows_far_apart(gpu, m):
    # Rows of both operands, their scales and the result reach past 2^32 bytes.
    k, n = 300, 70
    a, sa, b, sb = operands(m, n, k, seed=6)

    def spread(t, rows):
        ld = (1 << 33) // rows // 256 * 256
        far = torch.empty(rows, ld // t.element_size(), device="cuda", dtype=torch.uint8 if t.element_size() == 1 else t.dtype)
        view = far.view(t.dtype)[:, :t.shape[1]]
        view.copy_(t)
        return view

    want = matmul_fp8(a, sa, b, sb)
    out = spread(want, m)
    out.zero_()
    got = matmul_fp8(spread(a, m), spread(sa, m), spread(b, n), spread(sb, n), out=out)
    assert torch.equal(got, want)


def test_every_code_and_wide_scales(gpu):
    # All finite codes, in every place of a block, against ones; scales up to the range's ends.
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes = codes[(codes & 0x7f) != 0x7f]
    a, sa = fp8_rows((254, 256), "cuda")
    a.view(torch.uint8).copy_(torch.stack([codes.roll(r)[torch.arange(256, device="cuda") % 254] for r in range(254)]))
    sa.view(torch.uint8)[:, 0] = 127
    sa.view(torch.uint8)[:, 1] = torch.arange(254, device="cuda", dtype=torch.uint8) // 8 + 110
    b, sb = fp8_rows((20, 256), "cuda")
    b.view(torch.uint8).fill_(0x38)   # 1.0
    sb.view(torch.uint8).fill_(127)
    sb.view(torch.uint8)[5] = 1
    sb.view(torch.uint8)[6] = 200
    check(a, sa, b, sb, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 300), (40, 300), (300, 300), (300, 700), (50, 3000)])
def test_nan_stays_in_its_row(gpu, m, k, dtype):
    a, sa, b, sb = operands(m, 140, k, seed=3)
    want = matmul_fp8(a, sa, b, sb, out_dtype=dtype)
    a.view(torch.uint8)[0, 299] = 0x7f
    sb.view(torch.uint8)[7, 1] = 255
    got = matmul_fp8(a, sa, b, sb, out_dtype=dtype)
    assert torch.isnan(got[0]).all() and torch.isnan(got[:, 7]).all()
    keep = torch.arange(140, device="cuda") != 7
    assert torch.equal(got[1:, keep], want[1:, keep])


def test_empty(gpu):
    a, sa, b, sb = operands(4, 8, 128)
    assert matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 8)
    assert matmul_fp8(a, sa, b[:0], sb[:0]).shape == (4, 0)


@pytest.mark.parametrize("m", [1, 40, 200, 600])
def test_other_stream_and_graph(gpu, m):
    a, sa, b, sb = operands(m, 300, 2048, seed=4)
    want = matmul_fp8(a, sa, b, sb)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = matmul_fp8(a, sa, b, sb, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = matmul_fp8(a, sa, b, sb)
    for k in range(3):
        a2, sa2, _, _ = operands(m, 300, 2048, seed=5 + k)
        a.copy_(a2)
        sa.copy_(sa2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.clone(), matmul_fp8(a, sa, b, sb))


def test_refusals(gpu):
    a, sa, b, sb = operands(4, 8, 256)
    f = a.float()
    for bad in (dict(a=f), dict(b=f), dict(a_scale=sa.float()), dict(a_scale=sa[:, :1]), dict(b_scale=sb[:7]),
                dict(b=b[:, :128]), dict(a=a.cpu()), dict(out_dtype=torch.float64),
                dict(out=torch.empty(4, 9, device="cuda")), dict(a=a[:, ::2])):
        with pytest.raises(ValueError):
            matmul_fp8(**{"a": a, "a_scale": sa, "b": b, "b_scale": sb, **bad})
    tight = torch.zeros(4, 100, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    shifted = torch.zeros(4, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 8:108]
    s = sa[:, :1]
    for bad in (tight, shifted):
        with pytest.raises(HelixError):
            matmul_fp8(bad, s, b[:, :100], sb[:, :1])
