"""Windowed attention where its work is dealt out in other ways: backward over several groups of heads, of which the last is smaller, and
forward with two row tiles a CTA over two and more blocks of sinks.  Tolerances as derived in the reference's module."""
import pytest
import torch

from test_gpu_window_attention import check, tensors

pytestmark = pytest.mark.gpu


def pairs_of_a_group(Sq, Sk, window, qpk, hd, pairs):
    """(batch, key head) pairs whose gradients run side by side: as many as read 32 MB."""
    return min(max((32 << 20) // (4 * (min(Sq, window) * qpk + min(Sk, window)) * hd), 1), pairs)


@pytest.mark.parametrize("B,Sq,Sk,H,Hk,window,sinks", [
    (3, 2600, 2600, 8, 1, 2500, 3),
    (2, 2000, 2600, 24, 2, 1900, 140),
    (5, 2600, 2600, 8, 1, 2500, 0),
])
def test_groups_of_heads(B, Sq, Sk, H, Hk, window, sinks):
    pairs = B * Hk
    group = pairs_of_a_group(Sq, Sk, window, H // Hk, 128, pairs)
    assert group < pairs
    check(*tensors(B, Sq, Sk, H, Hk, 128), window, sinks)


def test_a_smaller_last_group_is_among_them():
    assert 3 % pairs_of_a_group(2600, 2600, 2500, 8, 128, 3) and 5 % pairs_of_a_group(2600, 2600, 2500, 8, 128, 5)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk,window,sinks", [
    (2, 2300, 2300, 8, 8, 256, 130),
    (4, 2300, 2300, 8, 2, 256, 300),        # more CTAs than SMs
    (2, 2000, 2400, 8, 8, 300, 200),
])
def test_two_row_tiles_over_blocks_of_sinks(B, Sq, Sk, H, Hk, window, sinks, hd):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-Sq // 128) * B * H > sms and sinks > 128
    check(*tensors(B, Sq, Sk, H, Hk, hd), window, sinks)
