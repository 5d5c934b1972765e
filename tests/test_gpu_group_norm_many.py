"""group_norm on more groups than one launch has units or threads for: the same bits as in pieces."""
import pytest
import torch

from helix_amd.norm import group_norm, group_norm_backward, group_norm_fp8

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


@pytest.fixture(autouse=True)
def memory(gpu):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of GPU memory")
    yield
    torch.cuda.empty_cache()


# Four lanes a group: 64 of them a workgroup, 2^30 a launch; a wave a group: 2^26; a workgroup: 2^24.
@pytest.mark.parametrize("rows,groups,width", [((1 << 21) + 5, 512, 2), ((1 << 26) + 7, 1, 300), ((1 << 23) + 3, 2, 1030)])
def test_forward(gpu, rows, groups, width):
    dim = groups * width
    few = dim * rows > 1 << 32
    x = normal(1 if few else rows, dim, seed=1, dtype=torch.bfloat16)
    if few:
        x = x.expand(rows, dim)   # (one row for all to read)
    w, b = 1 + normal(dim, seed=2), normal(dim, seed=3)
    y, mean, rstd = group_norm(x, w, b, groups=groups)
    step = rows // 3
    for at in (0, step, 2 * step, rows - step):
        part = slice(at, at + step)
        y1, mean1, rstd1 = group_norm(x[part], w, b, groups=groups)
        assert torch.equal(y[part], y1) and torch.equal(mean[part], mean1) and torch.equal(rstd[part], rstd1)
        del y1, mean1, rstd1


@pytest.mark.parametrize("rows,groups,width", [((1 << 19) + 3, 2048, 32), ((1 << 24) + 5, 5, 30)])
def test_eight_bits(gpu, rows, groups, width):
    dim = groups * width
    x = normal(1, dim, seed=4, dtype=torch.bfloat16).expand(rows, dim)
    w = 1 + normal(dim, seed=5)
    gate = normal(1, dim, seed=6, dtype=torch.bfloat16).expand(rows, dim)
    q, scale = group_norm_fp8(x, w, None, gate, groups=groups)
    one, one_scale = group_norm_fp8(x[:1], w, None, gate[:1], groups=groups)
    for at in range(0, rows, 1 << 17):
        assert (q.view(torch.uint8)[at:at + (1 << 17)] == one.view(torch.uint8)).all(), at
    assert (scale.view(torch.uint8) == one_scale.view(torch.uint8)).all()


def test_backward_of_many_rows(gpu):
    # The gradients go through the rows part by part, and as many as there are: no launch of it is cut.
    rows, groups, width = (1 << 21) + 5, 512, 2
    dim = groups * width
    x, dy = normal(rows, dim, seed=7, dtype=torch.bfloat16), normal(1, dim, seed=8, dtype=torch.bfloat16).expand(rows, dim)
    w = 1 + normal(dim, seed=9)
    _, mean, rstd = group_norm(x, w, groups=groups)
    dx, dw, _, _ = group_norm_backward(dy, x, w, mean, rstd, groups=groups)
    step = rows // 3
    for at in (0, rows - step):
        part = slice(at, at + step)
        dx1, dw1, _, _ = group_norm_backward(dy[part], x[part], w, mean[part], rstd[part], groups=groups)
        assert torch.equal(dx[part], dx1) and torch.isfinite(dw1).all()
    assert torch.isfinite(dw).all()
