"""helix_amd.matmul where every result is known to the bit: whole numbers, whose products the matrix instruction does not
cut and whose sums are exact in fp32. A lost, doubled or misplaced element is seen at any depth and in any type."""
import pytest
import torch

from helix_amd.matmul import matmul_fp8
from helix_amd.norm import fp8_rows

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
# Few rows, sums in parts, tiles of every size, more tiles than run at once; whole and ragged depths.
SHAPES = [(1, 300, 2047), (16, 5184, 2000), (40, 130, 9000), (67, 2560, 5120), (130, 140, 2047), (150, 640, 2900), (300, 260, 2048),
          (300, 4104, 656), (700, 1003, 640), (1000, 900, 3333), (4400, 4200, 600), (2060, 8210, 704)]


def rows(values, low):
    """8-bit rows of these whole numbers, the scale of block b of row i 2^(low + (i + b) % 2); and what they stand for."""
    q, scale = fp8_rows(values.shape, "cuda")
    q.copy_(values.to(torch.float8_e4m3fn))
    i, b = (torch.arange(s, device="cuda") for s in scale.shape)
    e = low + (i[:, None] + b) % 2
    scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))
    return q, scale, values.double() * torch.exp2(e.double()).repeat_interleave(128, 1)[:, :values.shape[1]]


def exact(x, y):
    return x @ y.T.contiguous()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_few_terms(gpu, m, n, k, dtype):
    # Up to 64 terms of 1, 2 or 4: sums up to 256, exact in every type. With rows enough each place of a sum counts in some.
    gen = torch.Generator(device="cuda").manual_seed(m)
    at = torch.rand(m, k, generator=gen, device="cuda").argsort(1)[:, :64]
    a = torch.zeros(m, k, device="cuda").scatter_(1, at, 1.0)
    a *= torch.randint(0, 2, (m, k), generator=gen, device="cuda") * 2 - 1
    b = (torch.randint(0, 2, (n, k), generator=gen, device="cuda") * 2 - 1).float()
    qa, sa, x = rows(a, 0)
    qb, sb, y = rows(b, 0)
    want = exact(x, y)
    assert want.abs().max() <= 256
    assert torch.equal(matmul_fp8(qa, sa, qb, sb, out_dtype=dtype).double(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_all_terms(gpu, m, n, k, dtype):
    # Whole numbers up to 3 everywhere: the sum is rounded once, to nearest even.
    gen = torch.Generator(device="cuda").manual_seed(n)
    a, b = (torch.randint(-3, 4, (r, k), generator=gen, device="cuda").float() for r in (m, n))
    qa, sa, x = rows(a, -1)
    qb, sb, y = rows(b, 0)
    want = exact(x, y)
    assert torch.equal(matmul_fp8(qa, sa, qb, sb, out_dtype=dtype), want.float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 512), (40, 700), (300, 700), (300, 256), (2000, 1024)])
def test_wide_scales(gpu, m, k, dtype):
    # Exponents of a and b far apart, and at the ends of their range, whose sum is near zero.
    gen = torch.Generator(device="cuda").manual_seed(k)
    a, b = (torch.randint(-3, 4, (r, k), generator=gen, device="cuda").float() for r in (m, 150))
    qa, sa, x = rows(a, 0)
    qb, sb, y = rows(b, 0)
    want = exact(x, y)
    for e in (1, 60, 126, -60, -126):
        ta, tb = sa.clone(), sb.clone()
        ta.view(torch.uint8).add_(e if e > 0 else 256 + e)
        tb.view(torch.uint8).sub_(e if e > 0 else 256 + e)
        assert torch.equal(matmul_fp8(qa, ta, qb, tb, out_dtype=dtype), want.float().to(dtype)), e
