"""A layer whose weight is frozen keeps no gradient of an earlier pass."""
import pytest
import torch

from rtp_b200.module.collectives import allign_grad
from rtp_b200.module.linear import ColumnParallelLinear, RowParallelLinear
from rtp_b200.parallel import fused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("frozen", [0, 1])
def test_no_stale_gradient(frozen):
    torch.manual_seed(0)
    kw = dict(bias=False, device="cuda", dtype=torch.bfloat16)
    layers = [ColumnParallelLinear(64, 2 * 128, packed_parts=2, **kw), RowParallelLinear(128, 64, **kw)]
    x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
    for step in range(2):
        for m in layers:
            m.linear.weight.grad = None
        y = fused.gated_mlp(*layers, x)
        y.float().pow(2).sum().backward()
        for m in layers:
            allign_grad(m)
        if step == 0:
            assert all(m.linear.weight.grad is not None for m in layers)
            layers[frozen].linear.weight.requires_grad_(False)
            with torch.no_grad():
                x.mul_(2)
    assert layers[frozen].linear.weight.grad is None and layers[1 - frozen].linear.weight.grad is not None
