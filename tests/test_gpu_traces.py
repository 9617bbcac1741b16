"""Forward-mode derivatives are refused, and traces hold the launches of the decoder block's operators."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from rtp_b200.ops import functional as FO, rotary as R

pytestmark = pytest.mark.gpu
NAMES = ["rotary", "window", "mlp", "packed"]


def calls():
    g = torch.Generator("cuda").manual_seed(0)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    f, pos, t, wgu, wd = R.rotary_frequencies(64, device="cuda"), torch.arange(6, device="cuda"), mk(1, 6, 2, 64), mk(128, 64), mk(64, 64)
    return {
        "rotary": (lambda a: FO.rotary(a, None, pos, f)[0], t),
        "window": (lambda a: FO.window_attention(a, t, t, 4), mk(1, 6, 2, 64)),      # x apart from k and v: a trace knows tensors by identity
        "mlp": (lambda a: FO.gated_mlp(a, wgu, wd), mk(8, 64)),
        "packed": (lambda a: FO.rotary_window_attention(a, pos, f, 2, 2, window=4), mk(1, 6, 6 * 64)),
    }


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    call, x = calls()[name]
    with fw.dual_level(), pytest.raises(NotImplementedError):
        call(fw.make_dual(x, torch.ones_like(x)))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_traces_hold_the_launch(name, grad):
    call, x = calls()[name]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, (x,), check_trace=False)
        other = torch.randn_like(x).requires_grad_(grad)
        got, want = traced(other), call(other)
        assert torch.equal(got, want)
        if grad:
            d = torch.randn_like(want)
            assert torch.equal(torch.autograd.grad(got, other, d)[0], torch.autograd.grad(want, other, d)[0])


def test_inference_mode():
    for call, x in calls().values():
        want = call(x)
        with torch.inference_mode():
            assert torch.equal(call(x), want)
