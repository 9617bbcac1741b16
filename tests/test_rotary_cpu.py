"""Rotary positions: plain evaluation, frequencies and refusals, without a GPU."""
import math

import pytest
import torch

from rtp_b200.ops import functional as FO
from rtp_b200.ops import rotary as R


def _by_complex_numbers(x, positions, freqs, layout, magnitude):
    n = freqs.shape[0]
    i = torch.arange(n)
    one, two = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    pos = positions if positions.dim() == 2 else positions[None]
    turn = magnitude * torch.exp(1j * pos.double()[:, :, None, None] * freqs)
    y = x.double().clone()
    z = torch.complex(y[..., one], y[..., two]) * turn
    y[..., one], y[..., two] = z.real, z.imag
    return y


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(8, 8), (10, 4), (64, 32)])
@pytest.mark.parametrize("per_batch", [False, True])
def test_plain_against_complex_numbers(layout, hd, rot, per_batch):
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn(2, 5, 3, hd, generator=g, dtype=torch.float64), torch.randn(2, 5, 1, hd, generator=g, dtype=torch.float64)
    pos = torch.randint(-100, 10 ** 6, (2, 5) if per_batch else (5,), generator=g)
    f = R.rotary_frequencies(rot)
    a, b = FO.rotary(q, k, pos, f, layout=layout, magnitude=1.25)
    # 64-bit angles up to 1e6 are off by 1e6 * 2^-53 = 1.1e-10 rad on either side
    torch.testing.assert_close(a, _by_complex_numbers(q, pos, f, layout, 1.25), rtol=0, atol=2e-9)
    torch.testing.assert_close(b, _by_complex_numbers(k, pos, f, layout, 1.25), rtol=0, atol=2e-9)


def test_agrees_with_the_model_tables():
    from rtp_b200.models.llama import apply_rope, rope_tables
    x = torch.randn(2, 7, 3, 16)
    cos, sin = rope_tables(7, 16, 10000.0, "cpu")
    y, none = FO.rotary(x, None, torch.arange(7), R.rotary_frequencies(16), layout="interleaved")
    assert none is None
    torch.testing.assert_close(y, apply_rope(x, cos, sin), rtol=1e-5, atol=1e-5)


def test_frequencies():
    f = R.rotary_frequencies(8, theta=100.0)
    assert f.dtype == torch.float64
    torch.testing.assert_close(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    torch.testing.assert_close(R.rotary_frequencies(8, theta=100.0, scaling="linear", factor=4.0), f / 4)
    n = R.rotary_frequencies(8, theta=100.0, scaling="ntk", factor=4.0)
    torch.testing.assert_close(n[0], f[0])
    torch.testing.assert_close(n[-1], f[-1] / 4)                     # the slowest pair is squeezed by the whole factor
    y = R.rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    full = R.rotary_frequencies(128)
    turns = 4096 * full / (2 * math.pi)
    torch.testing.assert_close(y[turns >= 32], full[turns >= 32])
    torch.testing.assert_close(y[turns <= 1], full[turns <= 1] / 8)
    assert bool(((y <= full) & (y >= full / 8)).all())
    assert R.rotary_magnitude("yarn", 8.0) == pytest.approx(0.1 * math.log(8) + 1)
    assert R.rotary_magnitude("linear", 8.0) == 1.0 and R.rotary_magnitude("yarn", 0.5) == 1.0


def test_gradients_by_differences():
    q, k = torch.randn(1, 3, 2, 8, dtype=torch.float64, requires_grad=True), torch.randn(1, 3, 1, 8, dtype=torch.float64, requires_grad=True)
    f, pos = R.rotary_frequencies(4), torch.tensor([[3, 900, 0]])
    for layout in R.LAYOUTS:
        assert torch.autograd.gradcheck(lambda a, b: FO.rotary(a, b, pos, f, layout=layout, magnitude=0.7), (q, k))


def _args(**over):
    d = dict(q=torch.zeros(2, 4, 3, 16), k=torch.zeros(2, 4, 1, 16), positions=torch.arange(4), freqs=R.rotary_frequencies(16), layout="half")
    return {**d, **over}


@pytest.mark.parametrize("over", [
    dict(layout="other"), dict(q=torch.zeros(2, 4, 16)), dict(q=torch.zeros(2, 4, 3, 16, dtype=torch.int32)),
    dict(k=torch.zeros(2, 5, 1, 16)), dict(k=torch.zeros(2, 4, 1, 8)), dict(k=torch.zeros(2, 4, 1, 16, dtype=torch.float64)),
    dict(positions=torch.arange(4.0)), dict(positions=torch.arange(5)), dict(positions=torch.zeros(3, 4, dtype=torch.int64)),
    dict(positions=torch.zeros(2, 4, 1, dtype=torch.int64)),
    dict(freqs=R.rotary_frequencies(16).float()), dict(freqs=R.rotary_frequencies(18)), dict(freqs=torch.zeros(0, dtype=torch.float64)),
])
def test_refusals(over):
    with pytest.raises(ValueError):
        FO.rotary(**_args(**over))


def test_frequency_refusals():
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"), dict(rotary_dim=8, theta=0.0),
                dict(rotary_dim=8, scaling="linear", factor=0.0), dict(rotary_dim=8, scaling="yarn", beta_fast=1.0)):
        with pytest.raises(ValueError):
            R.rotary_frequencies(**bad)


def test_kernel_front_end_refuses_cpu_tensors():
    with pytest.raises(ValueError):
        R.rotary(**_args())


def test_arguments_as_they_lie_in_memory():
    """The kernels' argument structures, packed: their sizes, and each field of the windowed attention's."""
    from rtp_b200.ops import _lib, flash
    import ctypes as C
    assert len(R._PACK(*range(21), *range(3), 1.0, *range(10))) == 4 * 8 + 16 * 8 + 8 + 16 + 8 + 4 + 10 * 4 + 4
    refs = [[100 * r + i for i in range(8)] for r in range(8)]
    a = _lib.WindowArgs.from_buffer_copy(flash._PACK(*sum(refs, []), 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 0.5, 0.25, 14, 15, 16, 17, 18, 19, 20, 21, 22))
    f = a.f
    for name, want in zip(("q", "k", "v", "o", "dout", "dq", "dk", "dv"), refs):
        assert [getattr(getattr(f, name), n) or 0 for n, _ in _lib.FlashRef._fields_] == want
    names = [n for n, _ in _lib.FlashArgs._fields_][8:]
    assert [getattr(f, n) for n in names] == [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 0.5, 0.25, 14, 15, 16, 17]
    assert (a.kv_heads, a.window, a.sinks, a.scratch, a.scratch_bytes) == (18, 19, 20, 21, 22)
    assert C.sizeof(a) == 536
