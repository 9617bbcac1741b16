"""Gradients of the gated feed-forward block where a rounding too many can be told from half a step."""
import pytest
import torch

from rtp_b200.ops import functional as FO
from test_gpu_gated_mlp import A, U, close, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,n,O", [(64, 72, 64), (200, 136, 72), (264, 1000, 256), (1032, 2744, 264)])
def test_the_gradient_of_the_product_is_not_rounded(D, n, O):
    """Rows of x with a single one: gate and up are weights, exact in bf16, and an element of dwgu is one of dg or du, which are then rounded
    once: by half a step of their value, beside 1e-4 of the terms of dy Wd and 1e-5 of the factors behind it in fp32."""
    _, wgu, wd, _ = tensors(1, D, n, O, 7, 1.0)
    dy = tensors(D, 8, 8, O, 8)[3]
    x = torch.eye(D, device="cuda").bfloat16()
    leaf = wgu.clone().requires_grad_()
    (got,) = torch.autograd.grad(FO.gated_mlp(x, leaf, wd), leaf, dy)
    g, u, dy, wd = wgu[:n].double().t(), wgu[n:].double().t(), dy.double(), wd.double()
    s = torch.sigmoid(g)
    dh, edh = dy @ wd, A * (dy.abs() @ wd.abs())
    for at, factor, scale in ((slice(0, n), u * (s + g * s * (1 - s)), u.abs()), (slice(n, 2 * n), g * s, (g * s).abs())):
        want = dh * factor
        e = edh * factor.abs() + 1e-5 * dh.abs() * scale
        close("dwgu", got[at].t(), (want, e + U * (want.abs() + e)))
