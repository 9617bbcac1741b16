"""Rotary positions, windowed attention and the gated feed-forward block as a decoder runs them: the packed form of the first two
against 64 bits and against the operators one by one, and the Llama-shaped model with them.

Tolerance of the packed output, u = 2^-8: q' and k' are rounded to bf16 (u of their values, and 4e-7 of the terms of a turn), so a
score is off by e = scale (|dq'| |k'| + |q'| |dk'| + |dq'| |dk'|) and a probability by a factor within exp(+-2 max e); the
probabilities are rounded for P V and the result is rounded; 2e-4 of the sums of magnitudes for what happens in fp32."""
import copy
import math

import pytest
import torch

from rtp_b200.models.llama import Llama, LlamaConfig
from rtp_b200.ops import functional as FO
from rtp_b200.ops import rotary as R
from rtp_b200.parallel import engine
from rtp_b200.parallel.context import set_backend

pytestmark = pytest.mark.gpu
U, F32 = 2.0 ** -8, 2e-4


def with_tolerance(qkv, pos, f, H, Hk, layout, magnitude, window, sinks):
    B, S, W = qkv.shape
    hd = W // (H + 2 * Hk)
    t = qkv.double().view(B, S, H + 2 * Hk, hd)
    n = f.shape[0]
    i = torch.arange(n, device="cuda")
    one, two = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    turn = magnitude * torch.exp(1j * (pos if pos.dim() == 2 else pos[None]).double()[:, :, None, None] * f)

    def turned(x):
        z = torch.complex(x[..., one], x[..., two]) * turn
        y, e = x.clone(), torch.zeros_like(x)
        y[..., one], y[..., two] = z.real, z.imag
        e[..., one] = e[..., two] = 4e-7 * magnitude * (x[..., one].abs() + x[..., two].abs())
        return y, e + U * y.abs()

    (q, eq), (k, ek) = turned(t[:, :, :H]), turned(t[:, :, H:H + Hk])
    k, ek, v = (x.repeat_interleave(H // Hk, dim=2).transpose(1, 2) for x in (k, ek, t[:, :, H + Hk:]))
    q, eq = q.transpose(1, 2), eq.transpose(1, 2)
    a = torch.arange(S, device="cuda")
    hidden = (a > a[:, None]) | ((a[:, None] - a >= window) & (a >= sinks))
    scale = hd ** -0.5
    p = (q @ k.transpose(2, 3) * scale).masked_fill(hidden, -math.inf).softmax(-1)
    e = (eq @ k.abs().transpose(2, 3) + (q.abs() + eq) @ ek.transpose(2, 3)) * scale
    spread = torch.expm1(2 * e.masked_fill(hidden, 0.0).amax(-1, keepdim=True))
    o = p @ v
    tol = (p * (spread + (U + F32) * (1 + spread))) @ v.abs()
    tol = tol + U * (o.abs() + tol)
    return [x.transpose(1, 2).reshape(B, S, H * hd) for x in (o, tol)]


CASES = [(1, 1, 1, 1, None, 0), (2, 129, 4, 2, 40, 3), (3, 257, 3, 3, None, 0), (2, 700, 6, 1, 128, 130), (1, 2000, 4, 4, 1, 1)]


def packed(B, S, H, Hk, hd, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    qkv = torch.randn(B, S, (H + 2 * Hk) * hd, device="cuda", generator=g).bfloat16()
    do = torch.randn(B, S, H * hd, device="cuda", generator=g).bfloat16()
    pos = torch.randint(0, 100000, (B, 1), device="cuda", generator=g) + torch.arange(S, device="cuda")
    return qkv, do, pos


@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (128, 32)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,S,H,Hk,window,sinks", CASES)
def test_packed(B, S, H, Hk, window, sinks, layout, hd, rot):
    qkv, do, pos = packed(B, S, H, Hk, hd, S)
    f = R.rotary_frequencies(rot, scaling="yarn", factor=4.0, device="cuda")
    m = R.rotary_magnitude("yarn", 4.0)
    leaf = qkv.clone().requires_grad_()
    o = FO.rotary_window_attention(leaf, pos, f, H, Hk, layout=layout, magnitude=m, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, leaf, do)
    want, tol = with_tolerance(qkv, pos, f, H, Hk, layout, m, window or S, sinks)
    err = (o.detach().double() - want).abs()
    assert bool((err <= tol + 1e-12).all()), f"worst {float((err / (tol + 1e-12)).max()):.2f} tolerances"
    # the operators one by one, whose gradients are tested on their own, give the same bits
    parts = qkv.clone().requires_grad_()
    q, k, v = parts.view(B, S, H + 2 * Hk, hd).split((H, Hk, Hk), dim=2)
    q, k = FO.rotary(q, k, pos, f, layout=layout, magnitude=m)
    o2 = FO.window_attention(q, k, v, window or S, sinks=sinks).reshape(B, S, H * hd)
    assert torch.equal(o, o2)
    assert torch.equal(g, torch.autograd.grad(o2, parts, do)[0])
    with torch.no_grad():
        assert torch.equal(FO.rotary_window_attention(leaf, pos, f, H, Hk, layout=layout, magnitude=m, window=window, sinks=sinks), o)


def test_packed_other_inputs():
    """A projection that is not contiguous, another type, another head size and a gradient of odd strides."""
    qkv, do, pos = packed(2, 50, 4, 2, 64)
    f = R.rotary_frequencies(64, device="cuda")
    call = lambda t: FO.rotary_window_attention(t, pos, f, 4, 2, window=20, sinks=1)
    want = call(qkv)
    assert torch.equal(call(torch.cat([qkv, qkv], -1)[..., :qkv.shape[-1]]), want)
    leaf = qkv.clone().requires_grad_()
    strided = do.transpose(1, 2).contiguous().transpose(1, 2)
    a, b = torch.autograd.grad(call(leaf), leaf, do)[0], torch.autograd.grad(call(leaf), leaf, strided)[0]
    assert torch.equal(a, b)
    one = do[:, :1, :1].expand_as(do)
    assert torch.equal(torch.autograd.grad(call(leaf), leaf, one)[0], torch.autograd.grad(call(leaf), leaf, one.contiguous())[0])
    assert call(qkv.float()).dtype == torch.float32
    small = FO.rotary_window_attention(qkv, pos, R.rotary_frequencies(32, device="cuda"), 8, 4, window=20)      # heads of 32
    assert small.shape == (2, 50, 256)


OPTIONS = [dict(window=40, sinks=3), dict(rope_layout="half"),
           dict(window=100, sinks=1, rope_layout="half", rotary_dim=32, rope_scaling="yarn", rope_factor=8.0, rope_original_length=64)]


def models(options, **size):
    torch.manual_seed(0)
    cfg = dict(vocab_size=1024, d_model=256, n_layers=2, n_heads=4, d_ff=512, max_seq_len=128)
    return Llama(LlamaConfig(**{**cfg, **size}, **options)).to("cuda", torch.bfloat16)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("heads", [2, 4])
def test_model_against_fp32(options, heads):
    """The bounds of the model without these options: 3e-2 of the loss, 15 % and a cosine of 0.985 for each gradient."""
    model = models(options, n_heads=heads)
    ref = copy.deepcopy(model).float()
    ids = torch.randint(0, 1024, (2, 129), device="cuda")
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()
    set_backend("functional")
    try:
        loss_ref = ref(x, y)
        loss_ref.backward()
    finally:
        set_backend("auto")
    loss = model(x, y)
    loss.backward()
    engine.check_all()
    assert abs(loss.item() - loss_ref.item()) < 3e-2
    want = dict(ref.named_parameters())
    for n, p in model.named_parameters():
        a, b = p.grad.double().flatten(), want[n].grad.double().flatten()
        assert float((a - b).norm() / b.norm()) < 0.15 and float(a @ b / (a.norm() * b.norm())) > 0.985, n


def test_model_takes_the_gated_block():
    """One launch for gate, up and their product, the same loss as layer by layer, and hooks on a layer are still called."""
    from rtp_b200.ops import mlp
    model = models({})
    ids = torch.randint(0, 1024, (2, 129), device="cuda")
    x, y = ids[:, :-1].contiguous(), ids[:, 1:].contiguous()
    calls, inner = [], mlp.gated_fwd
    mlp.gated_fwd = lambda *a: calls.append(1) or inner(*a)
    try:
        loss = model(x, y)
        assert len(calls) == 2
        seen = []
        handles = [b.down.register_forward_hook(lambda m, i, o: seen.append(i[0].shape)) for b in model.blocks]
        assert torch.equal(model(x, y), loss) and len(calls) == 2 and seen == [(2, 128, 512)] * 2
        for h in handles:
            h.remove()
        old = FO.set_activation_recompute(False)
        try:
            assert torch.equal(model(x, y), loss) and len(calls) == 2
        finally:
            FO.set_activation_recompute(old)
        with torch.no_grad():
            assert torch.equal(model(x, y), loss) and len(calls) == 4
    finally:
        mlp.gated_fwd = inner


def test_flat_gradients_of_the_gated_block():
    from rtp_b200.module.collectives import allign_grad
    model = models({})
    ids = torch.randint(0, 1024, (2, 129), device="cuda")
    model(ids[:, :-1], ids[:, 1:].contiguous()).backward()
    for b in model.blocks:
        for layer in (b.gate_up, b.down):
            g = layer.linear.weight.grad.clone()
            allign_grad(layer)
            assert torch.equal(layer.linear.weight.grad, g)
            assert layer.linear.weight.grad.data_ptr() == layer._last_flat_grad.data_ptr()


def test_input_changed_in_place_is_not_made_again():
    g = torch.Generator("cuda").manual_seed(0)
    x, w = torch.randn(40, 64, device="cuda", generator=g).bfloat16().requires_grad_(), torch.ones(64, device="cuda", dtype=torch.bfloat16)
    wgu = (torch.randn(256, 64, device="cuda", generator=g) * 0.1).bfloat16().requires_grad_()
    wd = (torch.randn(64, 128, device="cuda", generator=g) * 0.1).bfloat16()

    def grad(make, change):
        h = make()
        with torch.no_grad():
            h = change(h)
        return torch.autograd.grad(FO.gated_mlp(h, wgu, wd).float().sum(), wgu)[0]

    assert torch.equal(grad(lambda: FO.gelu(x), lambda h: h.mul_(2)), grad(lambda: FO.gelu(x), lambda h: h * 2))
    with pytest.raises(RuntimeError):          # a view, which autograd guards
        grad(lambda: FO.rms_norm(x, w, 1e-5), lambda h: h.mul_(2))


@pytest.mark.parametrize("options", [{}, OPTIONS[0], OPTIONS[2]])
def test_model_in_a_graph(options):
    """A captured training step, replayed on other tokens, gives what an eager one gives; sums with atomics (embedding, norms) aside."""
    model = models(options)
    ids = torch.randint(0, 1024, (3, 2, 129), device="cuda")
    x, y = ids[0, :, :-1].contiguous(), ids[0, :, 1:].contiguous()

    def step():
        loss = model(x, y)
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            model.zero_grad(set_to_none=True)
            step()
    torch.cuda.current_stream().wait_stream(side)
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for n in (1, 2):
        x.copy_(ids[n, :, :-1])
        y.copy_(ids[n, :, 1:])
        for p in model.parameters():
            p.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [p.grad.clone() for p in model.parameters()]
        again = copy.deepcopy(model)
        again.zero_grad(set_to_none=True)
        want = again(x, y)
        want.backward()
        assert torch.equal(loss, want.detach())
        for (name, p), g in zip(again.named_parameters(), got):
            if "embedding" not in name and p.dim() > 1:
                assert torch.equal(p.grad, g), name
