"""Launches that the gated feed-forward block counts: two products forward; one of dy Wd and one of the gradients backward; one more for each
product in slices."""
import pytest
import torch

from rtp_b200.ops import _lib, functional as FO, mlp
from test_gpu_gated_mlp import tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,D,n,forward,backward", [
    (300, 128, 264, 2, 2),
    (8, 2048, 8192, 3, 3),            # few rows: the down projection in slices, and the input gradient
    (8200, 64, 64, 2, 4),             # both weight gradients in slices
])
def test_counted(T, D, n, forward, backward):
    x, wgu, wd, dy = tensors(T, D, n, D)
    leaves = [t.requires_grad_() for t in (x, wgu, wd)]
    before = _lib.launches
    y = FO.gated_mlp(*leaves)
    assert _lib.launches - before == forward
    before = _lib.launches
    torch.autograd.grad(y, leaves, dy)
    assert _lib.launches - before == backward


def test_gradients_of_nothing():
    """dy Wd alone."""
    x, wgu, wd, dy = tensors(300, 128, 264, 128)
    _, gu, h = mlp.gated_fwd(x, wgu, wd, True)
    before = _lib.launches
    mlp.gated_bwd(x, dy, wgu, wd, gu, h, None, None, None)
    assert _lib.launches - before == 1
