"""Windowed attention whose visible scores are all -inf (keys of the type's lowest value): 0 / 0, as in a dense softmax, not zeros."""
import pytest
import torch

from rtp_b200.ops import functional as FO
from test_gpu_window_attention import hidden, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,Sq,Sk,H,window,sinks", [(1, 3, 3, 1, 1, 0), (1, 3, 3, 1, 2, 1), (2, 1, 400, 2, 200, 0), (2, 300, 300, 2, 1, 0), (4, 1500, 1500, 8, 100, 0)])
def test_rows_without_a_finite_score(B, Sq, Sk, H, window, sinks, hd):
    q, k, v, do = tensors(B, Sq, Sk, H, H, hd)
    q = q.abs() + 1
    low = torch.arange(Sk, device="cuda") < max(2, Sk // 2)
    k[:, low] = torch.finfo(torch.bfloat16).min
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = FO.window_attention(*leaves, window, sinks=sinks)
    seen = ~hidden(Sq, Sk, window, sinks)
    none = ~(seen & ~low).any(1)                       # rows that see low keys alone
    assert bool(o[:, none].isnan().all()) and bool(o[:, ~none].isfinite().all())
    dv = torch.autograd.grad(o, leaves[2], do)[0]
    touched = seen[none].any(0) if bool(none.any()) else torch.zeros_like(low)
    assert bool(dv[:, touched].isnan().all())


@pytest.mark.parametrize("hd", [64, 128])
def test_a_finite_score_beside_them(hd):
    """Keys of -inf beside a finite one have no weight."""
    q, k, v, _ = tensors(2, 300, 300, 2, 2, hd)
    q = q.abs() + 1
    k[:, 1::2] = torch.finfo(torch.bfloat16).min
    o = FO.window_attention(q, k, v, 8, sinks=2)
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * hd ** -0.5
    p = s.masked_fill(hidden(300, 300, 8, 2), float("-inf")).softmax(-1)
    # P rounded for the product, and the result: half a step of bf16 each, and 2e-4 for what happens in fp32
    want, sums = (torch.einsum("bhij,bjhd->bihd", p, t) for t in (v.double(), v.double().abs()))
    assert bool(((o.double() - want).abs() <= (2.0 ** -8 + 2e-4) * sums + 2.0 ** -8 * want.abs() + 1e-12).all())
