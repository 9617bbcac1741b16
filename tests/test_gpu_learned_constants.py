"""Frequencies, a magnitude or a scale that want a gradient get it where the kernels have none.

Against central differences of the 64-bit evaluation: the inputs are fp32 or bf16 and the operators' sums are in fp32, whose error beside
the magnitudes of the summed terms is far below 1e-3 (bf16 results enter no gradient here but through the incoming one, which is 1)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from rtp_b200.ops import flash, functional as FO, rotary as R

pytestmark = pytest.mark.gpu


def close(got, f, at):
    """The gradient of f at `at`, element by element, beside differences in 64 bits."""
    at = at.detach().double()
    for i in range(at.numel()):
        step = torch.zeros_like(at).flatten()
        step[i] = 1e-6
        step = step.view(at.shape)
        want = float((f(at + step) - f(at - step)) / 2e-6)
        assert abs(float(got.flatten()[i]) - want) <= 1e-3 * (1 + abs(want))


def turned(x, pos, freqs, magnitude):
    n = freqs.shape[0]
    z = torch.complex(x[..., :n], x[..., n:2 * n]) * (magnitude * torch.exp(1j * pos.double()[None, :, None, None] * freqs))
    return torch.cat([z.real, z.imag, x[..., 2 * n:]], -1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_frequencies_and_magnitude(dtype):
    g = torch.Generator("cuda").manual_seed(0)
    q = torch.randn(2, 5, 2, 16, device="cuda", generator=g).to(dtype)
    pos = torch.arange(5, device="cuda")
    f = R.rotary_frequencies(8, theta=10.0, device="cuda").requires_grad_()
    m = torch.tensor(1.25, device="cuda", requires_grad=True)
    y, _ = FO.rotary(q, None, pos, f, magnitude=m)
    df, dm = torch.autograd.grad(y.float().sum(), (f, m))
    x = q.double()
    close(df, lambda v: turned(x, pos, v, 1.25).sum(), f)
    close(dm, lambda v: turned(x, pos, f.detach(), v).sum(), m)
    with torch.no_grad():
        assert torch.equal(FO.rotary(q, None, pos, f, magnitude=m)[0], FO.rotary(q, None, pos, f.detach(), magnitude=1.25)[0])


def test_frequencies_of_the_packed_form():
    g = torch.Generator("cuda").manual_seed(1)
    qkv = torch.randn(1, 9, 4 * 64, device="cuda", generator=g).bfloat16().requires_grad_()
    f = R.rotary_frequencies(64, device="cuda").requires_grad_()
    pos = torch.arange(9, device="cuda")
    o = FO.rotary_window_attention(qkv, pos, f, 2, 1, window=4)
    df, dx = torch.autograd.grad(o.float().sum(), (f, qkv))
    assert bool(df.abs().sum() > 0) and bool(dx.abs().sum() > 0) and df.shape == f.shape


def test_scale():
    g = torch.Generator("cuda").manual_seed(2)
    q, k, v = (torch.randn(1, 7, 2, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    s = torch.tensor(0.2, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(FO.window_attention(q, k, v, 3, sinks=1, sm_scale=s).float().sum(), s)
    a = torch.arange(7, device="cuda")
    hidden = (a > a[:, None]) | ((a[:, None] - a >= 3) & (a >= 1))

    def f(scale):
        p = (torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * scale).masked_fill(hidden, float("-inf")).softmax(-1)
        return torch.einsum("bhij,bjhd->bihd", p, v.double()).sum()
    close(d, f, s)


def test_the_kernels_refuse_them():
    q = torch.randn(1, 5, 2, 64, device="cuda").bfloat16()
    f, pos, one = R.rotary_frequencies(64, device="cuda"), torch.arange(5, device="cuda"), torch.ones((), device="cuda", requires_grad=True)
    for kw in (dict(freqs=f.clone().requires_grad_()), dict(freqs=f, magnitude=one)):
        with pytest.raises(ValueError):
            R.rotary(q, None, pos, **kw)
    with pytest.raises(ValueError):
        flash.window_attention(q, q, q, 3, sm_scale=one)


def test_forward_mode():
    """A derivative along a constant, beside its gradient summed over the same output."""
    q = torch.randn(1, 5, 2, 64, device="cuda").bfloat16()
    f, pos = R.rotary_frequencies(64, theta=10.0, device="cuda"), torch.arange(5, device="cuda")
    calls = [(lambda c: FO.rotary(q.float(), None, pos, f, magnitude=c)[0], torch.tensor(1.25, device="cuda")),
             (lambda c: FO.rotary(q.float(), None, pos, c)[0], f),
             (lambda c: FO.window_attention(q, q, q, 3, sm_scale=c), torch.tensor(0.2, device="cuda"))]
    for call, at in calls:
        along = torch.ones_like(at)
        with fw.dual_level():
            tangent = fw.unpack_dual(call(fw.make_dual(at, along))).tangent
        assert tangent is not None
        leaf = at.clone().requires_grad_()
        (g,) = torch.autograd.grad(call(leaf).float().sum(), leaf)
        # bf16 outputs have a tangent rounded to bf16 each: half a step of the 640 of them
        assert abs(float(tangent.float().sum() - g.sum())) <= 2.0 ** -8 * float(tangent.float().abs().sum()) + 1e-4
