"""Sizes and values that the C structs of the layer operators cannot hold: refused as any other wrong argument."""
import pytest
import torch

from helix_amd.matmul import matmul_fp8
from helix_amd.norm import quantize_fp8, rms_norm, rms_norm_backward, rms_norm_fp8
from helix_amd.recurrence import gated_scan, gated_scan_backward

pytestmark = pytest.mark.gpu

MANY = (1 << 31) + 8


@pytest.mark.parametrize("eps", [1e39, -1e300])
def test_eps(gpu, eps):
    x, w = torch.ones(2, 8, device="cuda"), torch.ones(8, device="cuda")
    for norm in (rms_norm, rms_norm_fp8):
        with pytest.raises(ValueError, match="out of range"):
            norm(x, w, eps=eps)


def test_sizes(gpu):
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of GPU memory")
    wide = torch.empty(MANY, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="out of range"):
        rms_norm(wide, wide)
    with pytest.raises(ValueError, match="out of range"):
        rms_norm_backward(wide, wide, wide, torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="out of range"):
        quantize_fp8(wide)
    tokens = wide.view(1, MANY, 1)
    with pytest.raises(ValueError, match="out of range"):
        gated_scan(tokens, tokens)
    with pytest.raises(ValueError, match="out of range"):
        gated_scan_backward(tokens, tokens, tokens, tokens)
    a, sa = quantize_fp8(torch.ones(1, 16, device="cuda"))
    with pytest.raises(ValueError, match="out of range"):
        matmul_fp8(a, sa, a.expand(MANY, 16), sa.expand(MANY, 1))
    with pytest.raises(ValueError, match="out of range"):
        matmul_fp8(a.expand(MANY, 16), sa.expand(MANY, 1), a, sa)
