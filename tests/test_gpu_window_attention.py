"""Windowed attention with sinks on the tcgen05 kernels against dense attention in 64 bits.

Tolerances are worst cases of the roundings that the kernels make (u = 2^-8, half a step of bf16 relative to the value):
  o   probabilities rounded for P V, the result rounded:                       u (P |V| + |o|)
  dV  probabilities rounded for P^T dO, the result rounded:                    u (P^T |dO| + |dV|)
  dS  = P (dP - delta), rounded: u |dS|; delta is made from the rounded o:     + P (|dO| . error of o)
  dQ  = scale dS K, dK = scale dS^T Q, rounded:                                scale (error of dS) |K| + u |dQ|, likewise dK
and 2e-4 of the sums of magnitudes for what happens in fp32 (scores of up to 128 products, exponentials, sums)."""
import pytest
import torch

from rtp_b200.ops import flash
from rtp_b200.ops import functional as FO

pytestmark = pytest.mark.gpu
U, F32 = 2.0 ** -8, 2e-4


def hidden(Sq, Sk, window, sinks):
    p, j = torch.arange(Sk - Sq, Sk, device="cuda")[:, None], torch.arange(Sk, device="cuda")
    return (j > p) | ((j <= p - window) & (j >= sinks))


def reference(q, k, v, do, window, sinks, scale):
    """[(value, tolerance)] of o, dq, dk, dv in 64 bits."""
    B, Sq, H, hd = q.shape
    Sk, Hk = k.shape[1:3]
    G = H // Hk
    Q, K, V, D = (t.double().transpose(1, 2) for t in (q, k, v, do))
    K, V = (t.repeat_interleave(G, dim=1) for t in (K, V))
    P = (Q @ K.transpose(2, 3) * scale).masked_fill_(hidden(Sq, Sk, window, sinks), float("-inf")).softmax(-1)
    o = P @ V
    eo = (U + F32) * (P @ V.abs()) + U * o.abs()
    dP, delta = D @ V.transpose(2, 3), (D * o).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    eS = (U + F32) * dS.abs() + P * ((D.abs() * eo).sum(-1, keepdim=True) + F32 * (D.abs() @ V.abs().transpose(2, 3) + (D * o).abs().sum(-1, keepdim=True)))
    dq, eq = scale * (dS @ K), abs(scale) * (eS @ K.abs())
    dk, ek = scale * (dS.transpose(2, 3) @ Q), abs(scale) * (eS.transpose(2, 3) @ Q.abs())
    dv, ev = P.transpose(2, 3) @ D, (U + F32) * (P.transpose(2, 3) @ D.abs())
    fold = lambda t: t.view(B, Hk, G, Sk, hd).sum(2)
    dk, ek, dv, ev = (fold(t) for t in (dk, ek, dv, ev))
    out = [(o, eo), (dq, eq + U * dq.abs()), (dk, ek + U * dk.abs()), (dv, ev + U * dv.abs())]
    return [tuple(t.transpose(1, 2) for t in pair) for pair in out]


def close(name, got, want):
    y, tol = want
    assert got.shape == y.shape
    err = (got.double() - y).abs()
    bad = ~(err <= tol + 1e-12)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst "
                                 f"{float((err / (tol + 1e-12)).max()):.2f} tolerances")


def tensors(B, Sq, Sk, H, Hk, hd, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    return mk(B, Sq, H, hd), mk(B, Sk, Hk, hd), mk(B, Sk, Hk, hd), mk(B, Sq, H, hd)


def check(q, k, v, do, window, sinks, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = FO.window_attention(*leaves, window, sinks=sinks, sm_scale=scale)
    grads = torch.autograd.grad(o, leaves, do)
    want = reference(q, k, v, do, window, sinks, q.shape[3] ** -0.5 if scale is None else scale)
    for name, got, w in zip(("o", "dq", "dk", "dv"), (o.detach(), *grads), want):
        close(name, got, w)
    with torch.no_grad():
        assert torch.equal(FO.window_attention(*leaves, window, sinks=sinks, sm_scale=scale), o)


SIZES = [(1, 1), (2, 2), (127, 127), (128, 128), (129, 129), (257, 257), (640, 640), (1, 2), (1, 1000), (130, 300), (500, 1500)]
WINDOWS = [(1, 0), (1, 1), (2, 0), (5, 4), (127, 128), (128, 0), (129, 130), (300, 1), (10 ** 9, 0), (64, 1000)]


@pytest.mark.parametrize("Sq,Sk", SIZES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("hd", [64, 128])
def test_sizes_and_windows(Sq, Sk, window, sinks, hd):
    B, H, Hk = (2, 3, 3) if window % 2 else (1, 4, 2)
    check(*tensors(B, Sq, Sk, H, Hk, hd, Sq + window), window, sinks)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk,window,sinks", [
    (4, 1500, 1500, 16, 16, 200, 4),        # more work than SMs in both directions
    (3, 1537, 1537, 12, 4, 200, 1),
    (1, 2300, 2300, 8, 1, 256, 130),        # one key head for all, two blocks of sinks
    (2, 1000, 1900, 10, 2, 700, 64),
    (1, 4096, 4096, 2, 1, 64, 4),           # the sinks' queries in pieces
    (1, 4000, 4000, 1, 1, 1, 129),
])
def test_large(B, Sq, Sk, H, Hk, window, sinks, hd):
    check(*tensors(B, Sq, Sk, H, Hk, hd), window, sinks)


def test_pieces_of_sinks_are_taken():
    from rtp_b200.ops import _lib
    import ctypes as C
    q, k, v, _ = tensors(1, 4096, 4096, 2, 1, 64)
    a = flash._window_args(q, k, v, q, None, 64, 4, 1.0)
    assert _lib.lib().rtp_window_bwd_scratch(C.byref(a)) > 0


@pytest.mark.parametrize("scale", [0.3, 1.0, 1e-3])
def test_scales(scale):
    check(*tensors(2, 300, 300, 4, 2, 64), 100, 3, scale)


@pytest.mark.parametrize("hd", [64, 128])
def test_views(hd):
    B, S, H, Hk = 2, 200, 4, 2
    g = torch.Generator("cuda").manual_seed(3)
    packed = torch.randn(B, S, H + 2 * Hk, hd, device="cuda", generator=g).bfloat16()
    q, k, v = packed[:, :, :H], packed[:, :, H:H + Hk], packed[:, :, H + Hk:]
    do = torch.randn(B, S, H, hd, device="cuda", generator=g).bfloat16()
    check(q, k, v, do, 70, 2)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    seq_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    dim_last_but_one = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    check(heads_first(q), seq_first(k), dim_last_but_one(v), heads_first(do), 70, 2)
    check(seq_first(q), heads_first(k), seq_first(v), seq_first(do), 70, 2)
    check(q[:1].expand(B, S, H, hd), k[:, :, :1].expand(B, S, Hk, hd), v[:1].expand(B, S, Hk, hd), do[:, :1].expand(B, S, H, hd), 70, 2)
    odd = torch.empty(B * S * H * hd + 1, dtype=torch.bfloat16, device="cuda")[1:].view(B, S, H, hd)
    check(odd.copy_(q), k, v, do, 70, 2)


def test_broadcast_leaf_gets_the_sum():
    q, k, v, do = tensors(3, 150, 150, 2, 1, 64)
    leaf = k[:1].clone().requires_grad_()
    o = FO.window_attention(q, leaf.expand(3, -1, -1, -1), v, 40, sinks=1)
    (g,) = torch.autograd.grad(o, leaf, do)
    y, tol = reference(q, leaf.detach().expand(3, -1, -1, -1), v, do, 40, 1, 64 ** -0.5)[2]
    close("dk", g, (y.sum(0, keepdim=True), tol.sum(0, keepdim=True) * (1 + 3 * U) + 3 * U * y.abs().sum(0, keepdim=True)))


def test_gradients_of_some_inputs():
    q, k, v, do = tensors(1, 130, 260, 4, 2, 64)
    want = reference(q, k, v, do, 50, 2, 64 ** -0.5)
    for n in range(3):
        leaves = [t.detach().requires_grad_(i == n) for i, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(FO.window_attention(*leaves, 50, sinks=2), leaves[n], do)
        close("qkv"[n], g, want[1 + n])


def test_difference_of_the_loss():
    """Gradients against a symmetric difference of sum(o * do) along a direction, the forward in 64 bits."""
    q, k, v, do = tensors(1, 200, 200, 2, 1, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(FO.window_attention(*leaves, 60, sinks=2), leaves, do)
    g = torch.Generator("cuda").manual_seed(9)
    steps = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64) for t in (q, k, v)]
    h = 1e-5

    def loss(s):
        return (reference(*(t.double() + s * d for t, d in zip((q, k, v), steps)), do, 60, 2, 64 ** -0.5)[0][0] * do.double()).sum()

    diff = float((loss(h) - loss(-h)) / (2 * h))
    along = sum(float((a.double() * d).sum()) for a, d in zip(grads, steps))
    # what the gradients may be off along this direction, and 1e-6 for the difference itself
    tol = sum(float((w[1] * d.abs()).sum()) for w, d in zip(reference(q, k, v, do, 60, 2, 64 ** -0.5)[1:], steps))
    assert abs(diff - along) <= tol + 1e-6 * abs(diff)


def test_same_bits_twice():
    q, k, v, do = tensors(1, 4096, 4096, 4, 1, 128)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = FO.window_attention(*leaves, 64, sinks=4)
        runs.append((o, *torch.autograd.grad(o, leaves, do)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_other_stream_and_graph():
    q, k, v, do = tensors(2, 2500, 2500, 2, 1, 64)
    want = reference(q, k, v, do, 64, 4, 64 ** -0.5)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def step():
        o = FO.window_attention(*leaves, 64, sinks=4)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        close(name, a, w)
    # two graphs, whose workspaces are their own, replayed side by side
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    with torch.no_grad():
        for t in (*leaves, do):
            t.copy_(torch.randn_like(t))
    want = reference(*(t.detach() for t in leaves), do, 64, 4, 64 ** -0.5)
    streams = [torch.cuda.Stream() for _ in graphs]
    for g, st in zip(graphs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
            close(name, a, w)


def test_second_gradient_is_refused():
    q, k, v, _ = tensors(1, 10, 10, 1, 1, 64)
    q.requires_grad_()
    (g,) = torch.autograd.grad(FO.window_attention(q, k, v, 4).float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_refusals_on_the_gpu():
    q, k, v, _ = tensors(1, 10, 10, 2, 2, 64)
    for bad in ((q.float(), k.float(), v.float()), (q[..., :32], k[..., :32], v[..., :32]), (q[:0], k[:0], v[:0])):
        with pytest.raises(ValueError):
            flash.window_attention(*bad, 4)
    for scale in (0.0, -0.5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            FO.window_attention(q, k, v, 4, sm_scale=scale)
    # those run in PyTorch operations behind the public entry point
    assert FO.window_attention(q.float(), k.float(), v.float(), 4).dtype == torch.float32
    assert FO.window_attention(q[..., :32], k[..., :32], v[..., :32], 4).shape == (1, 10, 2, 32)
    assert FO.window_attention(q[:0], k[:0], v[:0], 4).shape == (0, 10, 2, 64)
    assert FO.window_attention(q[:, :0], k, v, 4).shape == (1, 0, 2, 64)


def test_status_word_stays_clear():
    from rtp_b200.ops import _lib
    check(*tensors(1, 300, 300, 2, 2, 128), 100, 1)
    _lib.check_status("cuda:0")


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
def test_hidden_keys_that_are_not_finite(bad, hd):
    """They have no weight, whatever their scores: the output keeps its bits."""
    for Sq, Sk, window, sinks in ((1, 300, 20, 2), (40, 300, 20, 2), (40, 300, 150, 0)):
        q, k, v, _ = tensors(2, Sq, Sk, 4, 2, hd, Sk)
        seen = ~hidden(Sq, Sk, window, sinks).all(0)
        assert not bool(seen.all())
        want = FO.window_attention(q, k, v, window, sinks=sinks)
        k[:, ~seen] = bad
        assert torch.equal(FO.window_attention(q, k, v, window, sinks=sinks), want)
        assert bool(want.isfinite().all())


def test_visible_values_that_are_not_finite_reach_the_output():
    """A NaN in a query, a visible key or a visible value is one in the outputs and gradients that depend on it."""
    for n in range(3):
        q, k, v, do = tensors(1, 260, 260, 2, 1, 64, n)
        (q, k, v)[n][0, 200, 0, 5] = float("nan")
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = FO.window_attention(*leaves, 50, sinks=1)
        grads = torch.autograd.grad(o, leaves, do)
        rows = o.isnan().any(-1)[0]                                       # [queries, heads]
        if n == 0:
            assert bool(rows[200, 0]) and int(rows.sum()) == 1
        else:
            assert bool(rows[200:250].all()) and not bool(rows[:128].any())
        # dV = P^T dO does not depend on V
        assert [bool(g.isnan().any()) for g in grads] == [True, True, n < 2]
