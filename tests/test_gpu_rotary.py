"""Rotary positions on the GPU against complex multiplication in 64 bits.

Tolerance: the reduced angle is rounded once (2^-25 of half a turn: 9.4e-8 rad), sine and cosine are within two units of their last
place (1.2e-7), a product and a sum round three times (1.8e-7): 4e-7 of m (|a| + |b|) with room for the 64-bit angle at positions up
to 10^6 (1e-10 rad).  The result is rounded to its type: half a step, finfo.eps / 2 of its value."""
import pytest
import torch

from rtp_b200.ops import functional as FO
from rtp_b200.ops import rotary as R

pytestmark = pytest.mark.gpu


def turned(x, positions, freqs, layout, magnitude=1.0, inverse=False):
    """(the rotated x, the tolerance of each element) in 64 bits."""
    n = freqs.shape[0]
    i = torch.arange(n, device=x.device)
    one, two = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    pos = positions if positions.dim() == 2 else positions[None]
    turn = magnitude * torch.exp((-1j if inverse else 1j) * pos.double()[:, :, None, None] * freqs)
    y = x.double().clone()
    tol = torch.zeros_like(y)
    z = torch.complex(y[..., one], y[..., two]) * turn
    slack = 4e-7 * magnitude * (y[..., one].abs() + y[..., two].abs())
    tol[..., one], tol[..., two] = slack, slack
    y[..., one], y[..., two] = z.real, z.imag
    return y, tol + y.abs() * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).tiny


def close(got, want):
    y, tol = want
    bad = (got.double() - y).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - y).abs() / tol).max()):.2f} tolerances"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 32), (80, 40), (96, 12), (10, 6), (256, 256), (2, 2)])
def test_forward_and_backward(dtype, layout, hd, rot):
    g = torch.Generator("cuda").manual_seed(hd + rot)
    B, S, H, Hk = 3, 37, 5, 2
    q = torch.randn(B, S, H, hd, device="cuda", generator=g).to(dtype).requires_grad_()
    k = torch.randn(B, S, Hk, hd, device="cuda", generator=g).to(dtype).requires_grad_()
    dq, dk = (torch.randn(t.shape, device="cuda", generator=g).to(dtype) for t in (q, k))
    pos = torch.randint(-1000, 10 ** 6, (B, S), device="cuda", generator=g)
    f = R.rotary_frequencies(rot, device="cuda")
    a, b = FO.rotary(q, k, pos, f, layout=layout, magnitude=1.125)
    close(a, turned(q.detach(), pos, f, layout, 1.125))
    close(b, turned(k.detach(), pos, f, layout, 1.125))
    ga, gb = torch.autograd.grad((a, b), (q, k), (dq, dk))
    close(ga, turned(dq, pos, f, layout, 1.125, inverse=True))
    close(gb, turned(dk, pos, f, layout, 1.125, inverse=True))
    # gradient against a difference of the (linear) map: <dq, R q> = <R^T dq, q>
    a, x = a.detach(), q.detach()
    lhs, rhs = (dq.double() * a.double()).sum(), (ga.double() * x.double()).sum()
    scale = (dq.double().abs() * a.double().abs()).sum() + (ga.double().abs() * x.double().abs()).sum()
    assert abs(float(lhs - rhs)) <= float(scale) * (torch.finfo(dtype).eps / 2 + 1e-6)


@pytest.mark.parametrize("B,S,H,Hk", [(1, 1, 1, 1), (1, 1, 40, 8), (7, 1, 3, 3), (1, 1000, 1, 1), (2, 333, 40, 40), (5, 64, 2, 1)])
def test_sizes(B, S, H, Hk):
    g = torch.Generator("cuda").manual_seed(S)
    q = torch.randn(B, S, H, 64, device="cuda", generator=g).bfloat16()
    k = torch.randn(B, S, Hk, 64, device="cuda", generator=g).bfloat16()
    pos = torch.arange(S, device="cuda", dtype=torch.int32)
    f = R.rotary_frequencies(64, scaling="yarn", factor=4.0, device="cuda")
    a, b = FO.rotary(q, k, pos, f)
    close(a, turned(q, pos, f, "half"))
    close(b, turned(k, pos, f, "half"))
    assert a.is_contiguous() and b.is_contiguous()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_views_and_odd_addresses(layout):
    g = torch.Generator("cuda").manual_seed(1)
    f = R.rotary_frequencies(48, device="cuda")
    pos = torch.randint(0, 5000, (1, 21), device="cuda", generator=g)
    packed = torch.randn(4, 21, 9, 64, device="cuda", generator=g).bfloat16()
    cases = [(packed[:, :, :5], packed[:, :, 5:7]),                                    # parts of one projection
             (packed.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :3], packed[:, :, 3:4]),      # [S, B] order beside [B, S]
             (packed.transpose(2, 3).contiguous().transpose(2, 3)[:, :, :2], packed[:, :, 2:3]),      # head_dim not innermost
             (packed[:1, :, :2].expand(4, 21, 2, 64), packed[..., :1, :].expand(4, 21, 3, 64))]       # broadcast views
    flat = torch.randn(4 * 21 * 2 * 64 + 8, device="cuda", generator=g).bfloat16()
    for off in (1, 2, 4):                                                              # addresses of 2, 4 and 8 bytes' alignment
        cases.append((flat[off:off + 4 * 21 * 2 * 64].view(4, 21, 2, 64), packed[:, :, :1]))
    for q, k in cases:
        a, b = FO.rotary(q, k, pos, f, layout=layout)
        close(a, turned(q, pos, f, layout))
        close(b, turned(k, pos, f, layout))


def test_far_positions():
    q = torch.randn(1, 4, 2, 128, device="cuda")
    pos = torch.tensor([2 ** 31 + 7, 2 ** 24 + 1, -(2 ** 31) - 9, 10 ** 9], device="cuda")
    f = R.rotary_frequencies(128, device="cuda")
    y, tol = turned(q, pos, f, "half")
    # the 64-bit angle itself: 2^31 * 2^-53 on either side, three roundings here
    a, _ = FO.rotary(q, None, pos, f)
    close(a, (y, tol + 4 * 2.0 ** 31 * 2.0 ** -53 * 2 * q.double().abs().amax()))


def test_empty_one_sided_and_partial_gradients():
    f = R.rotary_frequencies(64, device="cuda")
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64), (2, 3, 0, 64)):
        a, b = FO.rotary(torch.empty(shape, device="cuda"), None, torch.arange(shape[1], device="cuda"), f)
        assert a.shape == shape and b is None
    q = torch.randn(2, 3, 2, 64, device="cuda", requires_grad=True)
    k = torch.randn(2, 3, 1, 64, device="cuda")
    pos = torch.arange(3, device="cuda")
    a, b = FO.rotary(q, k, pos, f)
    (g,) = torch.autograd.grad(a, q, torch.ones_like(a))                  # b unused, k without gradient
    close(g, turned(torch.ones_like(a), pos, f, "half", inverse=True))
    (g,) = torch.autograd.grad(FO.rotary(q, None, pos, f)[0], q, torch.ones_like(a).expand_as(a))
    close(g, turned(torch.ones_like(a), pos, f, "half", inverse=True))


def test_second_gradient():
    q = torch.randn(1, 3, 1, 8, device="cuda", requires_grad=True)
    d = torch.randn(1, 3, 1, 8, device="cuda", requires_grad=True)
    f, pos = R.rotary_frequencies(8, device="cuda"), torch.tensor([5, 0, 77], device="cuda")
    a, _ = FO.rotary(q, None, pos, f)
    (g,) = torch.autograd.grad(a, q, d, create_graph=True)
    (gg,) = torch.autograd.grad(g, d, torch.ones_like(g))
    close(gg, turned(torch.ones_like(g), pos, f, "half"))


def test_stream_and_graph():
    f, pos = R.rotary_frequencies(64, device="cuda"), torch.arange(50, device="cuda")
    q = torch.randn(2, 50, 4, 64, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, _ = FO.rotary(q, None, pos, f)
    torch.cuda.current_stream().wait_stream(s)
    close(a, turned(q, pos, f, "half"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b, _ = FO.rotary(q, None, pos, f)
    q.normal_()
    pos += 1000
    graph.replay()
    close(b, turned(q, pos, f, "half"))


def test_special_values_stay_in_their_pairs():
    q = torch.ones(1, 2, 2, 64, device="cuda").bfloat16()
    q[0, 0, 1, 3] = float("nan")
    q[0, 1, 0, 40] = float("inf")                                          # behind the rotated part
    a, _ = FO.rotary(q, None, torch.arange(2, device="cuda"), R.rotary_frequencies(16, device="cuda"))
    bad = torch.zeros_like(a, dtype=torch.bool)
    bad[0, 0, 1, [3, 11]] = True
    bad[0, 1, 0, 40] = True
    assert bool((torch.isfinite(a) == ~bad).all()) and bool(torch.isinf(a[0, 1, 0, 40]))
