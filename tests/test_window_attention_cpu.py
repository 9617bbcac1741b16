"""Windowed attention with sinks: plain evaluation against a loop over queries, and refusals, without a GPU."""
import math

import pytest
import torch

from rtp_b200.ops import flash
from rtp_b200.ops import functional as FO


def by_loops(q, k, v, window, sinks, scale):
    B, Sq, H, hd = q.shape
    Sk, G = k.shape[1], H // k.shape[2]
    o = torch.zeros_like(q)
    for i in range(Sq):
        p = i + Sk - Sq
        seen = [j for j in range(Sk) if j <= p and (j > p - window or j < sinks)]
        for h in range(H):
            s = torch.einsum("bd,bjd->bj", q[:, i, h], k[:, seen, h // G]) * scale
            o[:, i, h] = torch.einsum("bj,bjd->bd", s.softmax(-1), v[:, seen, h // G])
    return o


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (9, 9), (1, 9), (4, 9)])
@pytest.mark.parametrize("window", [1, 3, 100])
@pytest.mark.parametrize("sinks", [0, 2, 20])
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 2), (3, 1)])
def test_plain(Sq, Sk, window, sinks, H, Hk):
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, Sq, H, 8, generator=g, dtype=torch.float64)
    k, v = (torch.randn(2, Sk, Hk, 8, generator=g, dtype=torch.float64) for _ in range(2))
    # sums of at most 9 weights of 64-bit numbers near one
    torch.testing.assert_close(FO.window_attention(q, k, v, window, sinks), by_loops(q, k, v, window, sinks, 8 ** -0.5), rtol=0, atol=1e-14)
    torch.testing.assert_close(FO.window_attention(q, k, v, window, sinks, sm_scale=-0.7), by_loops(q, k, v, window, sinks, -0.7), rtol=0,
                               atol=1e-14)


def test_whole_window_is_causal_attention():
    q, k, v = (torch.randn(1, 12, 2, 16) for _ in range(3))
    torch.testing.assert_close(FO.window_attention(q, k, v, 12), FO.causal_attention(q, k, v), rtol=1e-5, atol=1e-6)


def test_gradients_by_differences():
    q = torch.randn(1, 4, 4, 4, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(1, 6, 2, 4, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda *a: FO.window_attention(*a, 2, sinks=1), (q, k, v))


def _args(**over):
    d = dict(q=torch.zeros(2, 4, 6, 64), k=torch.zeros(2, 5, 2, 64), v=torch.zeros(2, 5, 2, 64), window=3, sinks=1)
    return {**d, **over}


@pytest.mark.parametrize("over", [
    dict(q=torch.zeros(2, 4, 64)), dict(k=torch.zeros(2, 5, 64)), dict(v=torch.zeros(2, 4, 2, 64)), dict(q=torch.zeros(1, 4, 6, 64)),
    dict(q=torch.zeros(2, 4, 6, 128)), dict(q=torch.zeros(2, 4, 5, 64)), dict(q=torch.zeros(2, 6, 6, 64)),
    dict(q=torch.zeros(2, 4, 6, 64, dtype=torch.float64)), dict(v=torch.zeros(2, 5, 2, 64, dtype=torch.bfloat16)),
    dict(window=0), dict(window=-1), dict(window=2.0), dict(window=True), dict(window=None), dict(sinks=-1), dict(sinks=1.5),
    dict(k=torch.zeros(2, 5, 0, 64), v=torch.zeros(2, 5, 0, 64)),
    dict(q=torch.zeros(2, 4, 6, 64, dtype=torch.int32), k=torch.zeros(2, 5, 2, 64, dtype=torch.int32), v=torch.zeros(2, 5, 2, 64, dtype=torch.int32)),
])
def test_refusals(over):
    with pytest.raises(ValueError):
        FO.window_attention(**_args(**over))


def test_kernel_front_end_refuses_what_the_kernels_do_not_take():
    with pytest.raises(ValueError):
        flash.window_attention(**_args())


def _blocks_seen(Sq, Sk, window, sinks, tile):
    seen = set()
    for i in range(tile * 128, min(tile * 128 + 128, Sq)):
        p = i + Sk - Sq
        seen.update(range(max(0, p - window + 1) // 128, p // 128 + 1))
        if min(sinks, p + 1):
            seen.update(range((min(sinks, p + 1) - 1) // 128 + 1))
    return seen


@pytest.mark.parametrize("Sq,Sk,window,sinks", [(1, 1, 1, 0), (700, 700, 1, 0), (700, 700, 130, 4), (300, 1500, 200, 0), (300, 1500, 200, 140),
                                                (1000, 1000, 5000, 7), (129, 1280, 128, 128), (500, 2000, 129, 1)])
def test_blocks_that_no_query_sees(Sq, Sk, window, sinks):
    """The rule by which the front-end zeroes gradients of keys that the launch does not write."""
    seen = set().union(*(_blocks_seen(Sq, Sk, window, sinks, t) for t in range(math.ceil(Sq / 128))))
    unseen = max(0, Sk - Sq - window + 1) // 128 > -(-min(sinks, Sk) // 128)
    assert unseen == (len(seen) < math.ceil(Sk / 128))
