"""An input that a layer would rebuild in backward is kept where it or what it was made from has been changed since: the gradient is that of
the values that the forward saw, bit by bit."""
import pytest
import torch

from rtp_b200.module.linear import ColumnParallelLinear
from rtp_b200.ops import functional as FO
from rtp_b200.rotated_tensor_parallel import RotatedTensorParallel

pytestmark = pytest.mark.gpu


def consumers():
    torch.manual_seed(0)
    mk = lambda *s: (torch.randn(*s, device="cuda") * 0.1).bfloat16()
    wgu, wd = mk(256, 64).requires_grad_(), mk(64, 128)
    layer = ColumnParallelLinear(64, 128, bias=False, device="cuda", dtype=torch.bfloat16)
    wrapped = RotatedTensorParallel(torch.nn.Linear(64, 128, bias=False, device="cuda", dtype=torch.bfloat16))
    return {"block": (lambda h: FO.gated_mlp(h, wgu, wd), wgu), "layer": (layer, layer.linear.weight),
            "wrapped": (wrapped, next(wrapped.parameters()))}


@pytest.mark.parametrize("name", ["block", "layer", "wrapped"])
@pytest.mark.parametrize("what", ["nothing", "source", "source's view", "output", "weight"])
def test_changed_before_the_call(name, what):
    call, w = consumers()[name]
    buf = torch.randn(40, 64, device="cuda").bfloat16()
    scale = torch.ones(64, device="cuda", dtype=torch.bfloat16)

    def gradient(rebuilt):
        b, s = buf.clone(), scale.clone()
        h = FO.rms_norm(b, s) if what == "weight" else FO.gelu(b)
        assert FO.recompute_tag(h) is not None
        if what == "output":
            h = h.mul_(2) if rebuilt else h * 2
        if not rebuilt:
            h = h.clone()                              # no tag
        elif what == "source":
            b.normal_()
        elif what == "source's view":
            b[3:5].zero_()
        elif what == "weight":
            s.mul_(3)
        return torch.autograd.grad(call(h).float().sum(), w)[0]

    assert torch.equal(gradient(True), gradient(False))


@pytest.mark.parametrize("name", ["block", "layer", "wrapped"])
def test_changed_after_the_call(name):
    """Autograd keeps the sources and sees the change."""
    call, w = consumers()[name]
    b = torch.randn(40, 64, device="cuda").bfloat16()
    y = call(FO.gelu(b))
    b.zero_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.float().sum(), w)
