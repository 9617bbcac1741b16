"""Gated feed-forward block: plain evaluation and refusals, without a GPU."""
import pytest
import torch

from rtp_b200.ops import functional as FO
from rtp_b200.ops import mlp


def test_plain():
    g = torch.Generator().manual_seed(0)
    x, wgu, wd = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 3, 5), (14, 5), (4, 7)))
    a, b = x @ wgu[:7].t(), x @ wgu[7:].t()
    want = (a / (1 + (-a).exp()) * b) @ wd.t()
    torch.testing.assert_close(FO.gated_mlp(x, wgu, wd), want, rtol=1e-12, atol=1e-13)
    torch.testing.assert_close(FO.gated_mlp(x[0, 0], wgu, wd), want[0, 0], rtol=1e-12, atol=1e-13)
    assert FO.gated_mlp(x[:, :0], wgu, wd).shape == (2, 0, 4)


def test_gradients_by_differences():
    leaves = [torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((3, 4), (6, 4), (2, 3))]
    assert torch.autograd.gradcheck(FO.gated_mlp, leaves)


@pytest.mark.parametrize("over", [
    dict(x=torch.zeros(())), dict(x=torch.zeros(3, 8)), dict(w_gate_up=torch.zeros(64)), dict(w_gate_up=torch.zeros(30, 16)),
    dict(w_down=torch.zeros(16)), dict(w_down=torch.zeros(16, 24)), dict(x=torch.zeros(3, 16, dtype=torch.float64)),
    dict(w_down=torch.zeros(16, 32, dtype=torch.bfloat16)),
    dict(x=torch.zeros(3, 16, dtype=torch.int32), w_gate_up=torch.zeros(64, 16, dtype=torch.int32), w_down=torch.zeros(16, 32, dtype=torch.int32)),
])
def test_refusals(over):
    args = {**dict(x=torch.zeros(3, 16), w_gate_up=torch.zeros(64, 16), w_down=torch.zeros(16, 32)), **over}
    with pytest.raises(ValueError):
        FO.gated_mlp(**args)


def test_kernel_front_end_refuses_cpu_tensors():
    with pytest.raises(ValueError):
        mlp.gated_mlp(torch.zeros(3, 16).bfloat16(), torch.zeros(64, 16).bfloat16(), torch.zeros(16, 32).bfloat16())
