"""Gated feed-forward block on the GEMM kernel against 64 bits.

Tolerances are worst cases: u = 2^-8 of a value for each rounding to bf16 (gate, up, their product, the gradients of the three, the
results), 1e-4 of the sum of magnitudes for a product's sums in fp32, and what those make of the steps behind them, with
|silu'| <= 1.1 and |silu''| <= 0.5."""
import pytest
import torch
import torch.nn.functional as F

from rtp_b200.ops import functional as FO
from rtp_b200.ops import mlp

pytestmark = pytest.mark.gpu
U, A, CROSS = 2.0 ** -8, 1e-4, 1.03        # CROSS: products of two of these errors


def reference(x, wgu, wd, dy):
    """[(value, tolerance)] of y, dx, dwgu, dwd in 64 bits."""
    x, wgu, wd, dy = (t.double() for t in (x, wgu, wd, dy))
    n = wd.shape[1]

    def product(a, ea, b, eb=None):         # a b^T with errors of a and b, sums in fp32, before the rounding of the result
        e = ea @ b.abs().t() + A * (a.abs() @ b.abs().t())
        return a @ b.t(), e if eb is None else e + a.abs() @ eb.t()

    zero = torch.zeros_like
    gu, egu = product(x, zero(x), wgu)
    egu = egu + U * gu.abs()
    g, u, eg, eu = gu[:, :n], gu[:, n:], egu[:, :n], egu[:, n:]
    s = torch.sigmoid(g)
    silu, d1 = g * s, s + g * s * (1 - s)
    h = silu * u
    eh = CROSS * (1.1 * eg * u.abs() + silu.abs() * eu + 1.1 * eg * eu) + (U + 1e-5) * h.abs()
    y, ey = product(h, eh, wd)
    dh, edh = product(dy, zero(dy), wd.t())
    edh = edh + U * dh.abs()
    dg, du = dh * u * d1, dh * silu
    edg = CROSS * (1.1 * (edh * u.abs() + dh.abs() * eu) + 0.5 * dh.abs() * u.abs() * eg) + (U + 1e-5) * dg.abs()
    edu = CROSS * (edh * silu.abs() + 1.1 * dh.abs() * eg) + (U + 1e-5) * du.abs()
    dgu, edgu = torch.cat([dg, du], 1), torch.cat([edg, edu], 1)
    dx, edx = product(dgu, edgu, wgu.t())
    dwgu, ewgu = product(dgu.t(), edgu.t(), x.t())
    dwd, ewd = product(dy.t(), zero(dy.t()), h.t(), eh.t())
    return [(v, e + U * v.abs()) for v, e in ((y, ey), (dx, edx), (dwgu, ewgu), (dwd, ewd))]


def close(name, got, want):
    y, tol = want
    err = (got.double().reshape(y.shape) - y).abs()
    bad = ~(err <= tol + 1e-12)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst "
                                 f"{float((err / (tol + 1e-12)).max()):.2f} tolerances")


def tensors(T, D, n, O, seed=0, scale=None):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return (mk(T, D).bfloat16(), (mk(2 * n, D) * (D ** -0.5 if scale is None else scale)).bfloat16(), (mk(O, n) * n ** -0.5).bfloat16(),
            mk(T, O).bfloat16())


def check(x, wgu, wd, dy):
    leaves = [t.detach().requires_grad_() for t in (x, wgu, wd)]
    y = FO.gated_mlp(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want = reference(x.reshape(-1, x.shape[-1]), wgu, wd, dy.reshape(-1, dy.shape[-1]))
    for name, got, w in zip(("y", "dx", "dwgu", "dwd"), (y.detach(), *grads), want):
        close(name, got, w)
    with torch.no_grad():
        assert torch.equal(FO.gated_mlp(*leaves), y)


@pytest.mark.parametrize("T,D,n,O", [
    (1, 8, 8, 8), (1, 64, 64, 64), (2, 200, 40, 16), (8, 2048, 8192, 2048), (1, 5120, 64, 8), (127, 64, 136, 264), (128, 128, 128, 128),
    (129, 136, 72, 200), (300, 1032, 2744, 1032), (1000, 256, 1000, 256), (513, 2048, 1024, 512), (2500, 512, 4096, 512), (700, 8, 1536, 8),
    (64, 1536, 2000, 136),
])
def test_sizes(T, D, n, O):
    check(*tensors(T, D, n, O, T))


@pytest.mark.parametrize("pair", [0, 1])
def test_both_tile_kinds(pair):
    from rtp_b200.ops import _lib
    _lib.lib().rtp_set_pair_mode(pair)
    try:
        for shape in ((8, 64, 64, 64), (300, 520, 776, 264), (1024, 512, 2048, 512)):
            check(*tensors(*shape, seed=pair))
    finally:
        _lib.lib().rtp_set_pair_mode(-1)


@pytest.mark.parametrize("scale", [0.0, 1e-3, 3.0])
def test_small_and_saturated_gates(scale):
    check(*tensors(200, 128, 264, 128, 1, scale))


@pytest.mark.parametrize("n", [1000, 704])
def test_bits_of_the_separate_launches(n):
    """`whole`: the fused launches round where the separate ones do and add up in their order."""
    from rtp_b200.ops.gemm import gemm
    x, wgu, wd, dy = tensors(300, 256, n, 264)
    y, kept, _ = mlp.gated_fwd(x, wgu, wd, True, True)
    gx, gg, gd = torch.empty_like(x), torch.empty_like(wgu), torch.empty_like(wd)
    mlp.gated_bwd(x, dy, wgu, wd, kept, None, gx, gg, gd, True)
    with torch.no_grad():
        gu = gemm(x, wgu)
        assert torch.equal(gu, kept)
    gu.requires_grad_()
    h = FO.swiglu_packed(gu)
    with torch.no_grad():
        assert torch.equal(gemm(h, wd), y)
        dh = gemm(dy, wd, b_mn=True)
        assert torch.equal(gemm(dy, h, a_mn=True, b_mn=True), gd)
    (dgu,) = torch.autograd.grad(h, gu, dh)
    with torch.no_grad():
        assert torch.equal(gemm(dgu, wgu, b_mn=True), gx)
        assert torch.equal(gemm(dgu, x, a_mn=True, b_mn=True), gg)


@pytest.mark.parametrize("T,D,n,O", [(8, 512, 2048, 512), (300, 256, 1000, 264), (9000, 128, 264, 128)])
def test_the_product_is_rounded_once(T, D, n, O):
    """y and the down projection's gradient have the error of a product rounded to bf16 once, not of rounded gates too."""
    x, wgu, wd, dy = tensors(T, D, n, O, 5)
    leaves = [t.detach().requires_grad_() for t in (x, wgu, wd)]
    y = FO.gated_mlp(*leaves)
    (gd,) = torch.autograd.grad(y, leaves[2], dy)
    x, wgu, wd, dy = (t.double() for t in (x, wgu, wd, dy))
    gu, egu = x @ wgu.t(), A * (x.abs() @ wgu.abs().t())
    g, u, eg, eu = gu[:, :n], gu[:, n:], egu[:, :n], egu[:, n:]
    h = g * torch.sigmoid(g) * u
    eh = CROSS * (1.1 * eg * u.abs() + (g * torch.sigmoid(g)).abs() * eu + 1.1 * eg * eu) + (U + 1e-5) * h.abs()
    for name, got, a, ea, b in (("y", y.detach(), h, eh, wd), ("dwd", gd, dy.t(), 0 * dy.t(), h.t())):
        want = a @ b.t()
        e = ea @ b.abs().t() + A * (a.abs() @ b.abs().t()) + (a.abs() @ eh if name == "dwd" else 0)
        close(name, got, (want, e + U * want.abs()))


def test_views():
    x, wgu, wd, dy = tensors(2 * 3 * 50, 128, 200, 64)
    check(x.view(2, 3, 50, 128), wgu, wd, dy.view(2, 3, 50, 64))
    check(x.view(2, 150, 128).transpose(0, 1), wgu, wd, dy.view(150, 2, 64))
    wide = torch.randn(300, 256, device="cuda").bfloat16()
    check(wide[:, 128:], wgu, wd, dy)                                     # rows further apart than they are long
    check(wide[:, 3:131], wgu, wd, dy)                                    # odd address
    check(x.t().contiguous().t(), wgu.t().contiguous().t(), wd.t().contiguous().t(), dy[:1].expand(300, 64))
    check(x[:1].expand(300, 128), wgu, wd, dy)
    odd = torch.empty(400 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(400, 128).copy_(wgu)
    check(x, odd, wd, dy)
    check(x[:, :120], torch.randn(400, 256, device="cuda").bfloat16()[:, :120], wd, dy)


def test_gradients_of_some_inputs():
    x, wgu, wd, dy = tensors(200, 128, 264, 128)
    want = reference(x, wgu, wd, dy)
    for n in range(3):
        leaves = [t.detach().requires_grad_(i == n) for i, t in enumerate((x, wgu, wd))]
        (g,) = torch.autograd.grad(FO.gated_mlp(*leaves), leaves[n], dy)
        close(("dx", "dwgu", "dwd")[n], g, want[1 + n])


def test_difference_of_the_loss():
    x, wgu, wd, dy = tensors(60, 64, 136, 72)
    leaves = [t.detach().requires_grad_() for t in (x, wgu, wd)]
    grads = torch.autograd.grad(FO.gated_mlp(*leaves), leaves, dy)
    g = torch.Generator("cuda").manual_seed(5)
    steps = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64) for t in leaves]
    eps = 1e-5

    def loss(s):
        return (reference(*(t.detach().double() + s * d for t, d in zip(leaves, steps)), dy)[0][0] * dy.double()).sum()

    diff = float((loss(eps) - loss(-eps)) / (2 * eps))
    along = sum(float((a.double() * d).sum()) for a, d in zip(grads, steps))
    tol = sum(float((w[1] * d.abs()).sum()) for w, d in zip(reference(x, wgu, wd, dy)[1:], steps))
    assert abs(diff - along) <= tol + 1e-6 * abs(diff)


def test_recomputed_input():
    """An input that its norm can make again is not kept, and gives the same gradients."""
    x, wgu, wd, dy = tensors(150, 128, 264, 128)
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x.requires_grad_()
    wgu.requires_grad_()
    tagged = FO.rms_norm(x, w)
    assert FO.recompute_tag(tagged) is not None
    a = torch.autograd.grad(FO.gated_mlp(tagged, wgu, wd), (x, w, wgu), dy)
    old = FO.set_activation_recompute(False)
    try:
        plain = FO.rms_norm(x, w)
        assert FO.recompute_tag(plain) is None
        b = torch.autograd.grad(FO.gated_mlp(plain, wgu, wd), (x, w, wgu), dy)
    finally:
        FO.set_activation_recompute(old)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_other_stream_and_graphs():
    x, wgu, wd, dy = tensors(8, 256, 2048, 256)                           # few rows: slices, whose workspace is the call's own
    leaves = [t.requires_grad_() for t in (x, wgu, wd)]

    def step():
        y = FO.gated_mlp(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    names = ("y", "dx", "dwgu", "dwd")
    want = reference(*(t.detach() for t in leaves), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    for n, a, w in zip(names, got, want):
        close(n, a, w)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    with torch.no_grad():
        for t in (x, dy):
            t.copy_(torch.randn_like(t))
    want = reference(*(t.detach() for t in leaves), dy)
    for g in graphs:
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        for n, a, w in zip(names, got, want):
            close(n, a, w)


def test_values_that_are_not_finite_stay_in_their_rows():
    x, wgu, wd, _ = tensors(300, 128, 264, 128)
    x[7, 3] = float("nan")
    x[200, 5] = float("inf")
    y = FO.gated_mlp(x, wgu, wd)
    bad = ~torch.isfinite(y).all(dim=1)
    assert bad.nonzero().flatten().tolist() == [7, 200]


def test_slices_are_taken_for_few_rows():
    L = mlp._L()
    import ctypes as C
    a = mlp.GatedFwd(T=8, D=2048, F=8192, O=2048)
    assert L.rtp_gated_fwd_scratch(C.byref(a)) > 0
    a = mlp.GatedFwd(T=4096, D=2048, F=8192, O=2048)
    assert L.rtp_gated_fwd_scratch(C.byref(a)) == 0


def test_refusals_on_the_gpu():
    x, wgu, wd, _ = tensors(4, 64, 64, 64)
    for bad in ((x.float(), wgu.float(), wd.float()), (x[:0], wgu, wd), (x[:, :60], wgu[:, :60], wd), (x, wgu[:120], wd[:, :60])):
        with pytest.raises(ValueError):
            mlp.gated_mlp(*bad)
        assert FO.gated_mlp(*bad).shape == (bad[0].shape[0], 64)          # in PyTorch operations behind the public entry point
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(FO.gated_mlp(x.requires_grad_(), wgu, wd).sum(), x, create_graph=True)[0]
        g.sum().backward()


@pytest.mark.parametrize("T,D,n", [(8192, 64, 64), (8200, 128, 200), (9000, 256, 264), (8191, 64, 64)])
def test_small_weights_over_many_rows(T, D, n):
    """Their gradients fall into slices from 8192 rows on."""
    import ctypes as C
    both = mlp.GatedBwd(T=T, D=D, F=n, O=D, dw_gu=1, dw_d=1)
    assert (mlp._L().rtp_gated_bwd_scratch(C.byref(both)) > 0) == (T >= 8192)
    check(*tensors(T, D, n, D, n))


@pytest.mark.parametrize("T,D,n", [(8, 2048, 8192), (300, 256, 1000), (9000, 128, 264), (1000, 512, 1024)])
def test_layers_give_the_same_bits(T, D, n):
    """A packed projection, the activation and a down projection as rotated layers of one rank, fused and one by one."""
    from rtp_b200.module.linear import ColumnParallelLinear, RowParallelLinear
    from rtp_b200.parallel import engine, fused
    torch.manual_seed(T)
    kw = dict(bias=False, device="cuda", dtype=torch.bfloat16)
    up, down = ColumnParallelLinear(D, 2 * n, packed_parts=2, **kw), RowParallelLinear(n, D, **kw)
    x, _, _, dy = tensors(T, D, 8, D)
    leaves = [x.requires_grad_(), up.linear.weight, down.linear.weight]
    y = fused.gated_mlp(up, down, x)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    y = down(FO.swiglu_packed(up(x)))
    want = [y, *torch.autograd.grad(y, leaves, dy)]
    engine.check_all()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
