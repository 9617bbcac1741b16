"""Forward-mode derivatives and traces of operators whose kernels autograd does not see, without a GPU: the launches are replaced by numpy."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from rtp_b200.ops import _lib, flash, functional as FO, mlp, rotary as R

POS, FREQS = torch.arange(6), R.rotary_frequencies(64)


def unseen(t, factor):
    """factor * t, made where neither autograd nor a trace sees it."""
    return None if t is None else torch.from_numpy(t.detach().numpy() * factor)


@pytest.fixture
def launches(monkeypatch):
    monkeypatch.setattr(R, "_rotate", lambda q, k, *a: (unseen(q, 2.0), unseen(k, 2.0)))
    monkeypatch.setattr(flash, "_window_fwd", lambda q, k, v, *a: (q, k, v, unseen(q, 3.0), torch.zeros(2)))
    monkeypatch.setattr(mlp, "gated_fwd", lambda x, *a: (unseen(x, 5.0), torch.zeros(2), torch.zeros(2)))
    monkeypatch.setattr(FO, "use_kernels", lambda t: True)
    for m in (R, mlp):
        monkeypatch.setattr(m, "kernel_takes", lambda *a: True)


def calls():
    g = torch.Generator().manual_seed(0)
    t = torch.randn(1, 6, 2, 64, generator=g)
    return {
        "rotary": (lambda a: FO.rotary(a, None, POS, FREQS)[0], t, 2.0),
        "mlp": (lambda a: FO.gated_mlp(a, torch.zeros(16, 64), torch.zeros(64, 8)), torch.randn(8, 64, generator=g), 5.0),
        "packed": (lambda a: FO.rotary_window_attention(a, POS, FREQS, 2, 2)[..., :64], torch.randn(1, 6, 6 * 64, generator=g), 6.0),
    }


NAMES = ["rotary", "mlp", "packed"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(launches, name):
    call, x, _ = calls()[name]
    with fw.dual_level(), pytest.raises(NotImplementedError):
        call(fw.make_dual(x, torch.ones_like(x)))
    call(x)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_traces_hold_the_launch(launches, name, grad):
    call, x, factor = calls()[name]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, (x,), check_trace=False)
    other = torch.randn_like(x)
    want = other * factor if name != "packed" else other[..., :64] * factor
    assert torch.equal(traced(other), want)


def test_through_autograd():
    a, b = torch.zeros(2), torch.zeros(2, requires_grad=True)
    assert not _lib.through_autograd(a, None) and _lib.through_autograd(a, b)
    with torch.no_grad():
        assert not _lib.through_autograd(b)
        with fw.dual_level():
            assert _lib.through_autograd(a)
    assert not _lib.through_autograd(a)


@pytest.mark.filterwarnings("ignore")
def test_traces_hold_no_tags():
    """A tag would make the traced graph's backward rebuild an input from the tensors that it was traced with."""
    seen = []

    def f(x):
        y = FO._tag(x * 2, "gelu", x)
        seen.append(FO.recompute_tag(y))
        return y
    torch.jit.trace(f, (torch.zeros(3),), check_trace=False)
    f(torch.zeros(3))
    assert seen[0] is None and seen[1] is not None
