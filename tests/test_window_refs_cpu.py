"""How views reach the windowed attention kernels, without a GPU."""
import pytest
import torch

from rtp_b200.ops import flash


def fields(t):
    return dict(zip(("ptr", "sb", "ss", "width", "col_base", "heads", "gstride", "hstride"), flash._ref(t)))


def test_a_single_head_of_any_stride():
    """The head stride of one head is any number: here 2^33 elements."""
    t = torch.empty_strided((1, 4, 1, 64), (2 ** 34, 64, 2 ** 33, 1), device="meta")
    f = fields(t)
    assert f["width"] == 64 and f["hstride"] == 0 and f["heads"] == 1
    flash._PACK(*flash._ref(t) * 8, 0, 0, *range(6), 0, 0, 0, 0, 0, 1.0, 0.0, 0, 0, 0, 0, *range(5))


@pytest.mark.parametrize("H", [2, 5])
def test_several_heads(H):
    t = torch.empty_strided((2, 4, H, 64), (4096, 64, 512, 1), device="meta")
    f = fields(t)
    assert f["hstride"] == 512 and f["width"] == (H - 1) * 512 + 64
