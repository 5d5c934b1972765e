"""The delta rule where a call leaves little to do or values are at the ends of their types."""
import pytest
import torch

import delta_oracle as do_
from helix_amd.delta import delta_rule, delta_rule_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
def test_query_heads_without_value_heads(gpu, dtype):
    # Their gradients are sums over no heads: zeros, whatever the memory held.
    q = torch.full((2, 70, 3, 40), float("nan"), device="cuda", dtype=dtype)
    v, g = torch.empty(2, 70, 0, 8, device="cuda", dtype=dtype), torch.empty(2, 70, 0, device="cuda")
    for _ in range(3):
        stale = [torch.full_like(q, float("nan")) for _ in range(8)]
        del stale
        dq, dk, dv, dg, dbeta, ds0 = delta_rule_backward(v, q, q, v, g, g)
        assert (dq == 0).all() and (dk == 0).all()
        assert dv.shape == v.shape and dg.shape == dbeta.shape == g.shape and ds0.shape == (2, 0, 40, 8)
