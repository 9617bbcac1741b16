"""Rotary attention over a window on a packed projection, and the Llama-shaped model's options that use it, without a GPU."""
import copy
import math

import pytest
import torch

from _dist import run_distributed
from rtp_b200.models.llama import Llama, LlamaConfig
from rtp_b200.ops import functional as FO
from rtp_b200.ops import rotary as R
from test_models_cpu import _compare

SMALL = dict(vocab_size=64, d_model=32, n_layers=2, n_heads=4, d_ff=64, max_seq_len=16)
OPTIONS = [dict(window=3, sinks=1), dict(window=100), dict(rope_layout="half"), dict(rotary_dim=4, rope_scaling="linear", rope_factor=4.0),
           dict(window=5, sinks=2, rope_layout="half", rotary_dim=6, rope_scaling="yarn", rope_factor=8.0, rope_original_length=64),
           dict(rope_scaling="ntk", rope_factor=2.0)]


def dense(qkv, pos, f, H, Hk, layout, magnitude, window, sinks):
    """In 64 bits, from a dense matrix of scores."""
    B, S, W = qkv.shape
    hd = W // (H + 2 * Hk)
    t = qkv.double().view(B, S, H + 2 * Hk, hd)
    q, k, v = t[:, :, :H], t[:, :, H:H + Hk], t[:, :, H + Hk:]
    n = f.shape[0]
    i = torch.arange(n)
    one, two = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    turn = magnitude * torch.exp(1j * (pos if pos.dim() == 2 else pos[None]).double()[:, :, None, None] * f)

    def turned(x):
        z = torch.complex(x[..., one], x[..., two]) * turn
        y = x.clone()
        y[..., one], y[..., two] = z.real, z.imag
        return y

    q, k = turned(q), turned(k).repeat_interleave(H // Hk, dim=2)
    v = v.repeat_interleave(H // Hk, dim=2)
    a = torch.arange(S)
    hidden = (a > a[:, None]) | ((a[:, None] - a >= window) & (a >= sinks))
    p = (torch.einsum("bihd,bjhd->bhij", q, k) * hd ** -0.5).masked_fill(hidden, -math.inf).softmax(-1)
    return torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, S, H * hd)


@pytest.mark.parametrize("S", [1, 2, 9])
@pytest.mark.parametrize("H,Hk", [(2, 2), (4, 1)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (2, 2)])
def test_packed_plain(S, H, Hk, layout, window, sinks):
    g = torch.Generator().manual_seed(S)
    qkv = torch.randn(2, S, (H + 2 * Hk) * 8, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 1000, (2, S), generator=g)
    f = R.rotary_frequencies(6)
    got = FO.rotary_window_attention(qkv, pos, f, H, Hk, layout=layout, magnitude=1.25, window=window, sinks=sinks)
    # sums of at most nine 64-bit numbers near one, angles up to 1000 off by 1e-13
    torch.testing.assert_close(got, dense(qkv, pos, f, H, Hk, layout, 1.25, window or S, sinks), rtol=0, atol=1e-11)


def test_packed_gradients_by_differences():
    qkv = torch.randn(1, 5, 4 * 4, dtype=torch.float64, requires_grad=True)
    f = R.rotary_frequencies(4)
    assert torch.autograd.gradcheck(lambda t: FO.rotary_window_attention(t, torch.arange(5), f, 2, 1, window=2, sinks=1), (qkv,))


@pytest.mark.parametrize("over", [
    dict(qkv=torch.zeros(10, 32)), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(heads=1, kv_heads=2, qkv=torch.zeros(2, 5, 40)),
    dict(positions=torch.arange(4)), dict(positions=torch.arange(5).float()), dict(freqs=torch.ones(5, dtype=torch.float64)),
    dict(freqs=torch.ones(2)), dict(layout="pairs"), dict(window=0), dict(window=1.5), dict(sinks=-1),
])
def test_packed_refusals(over):
    args = dict(qkv=torch.zeros(2, 5, 32), positions=torch.arange(5), freqs=R.rotary_frequencies(8), heads=2, kv_heads=1)
    with pytest.raises(ValueError):
        FO.rotary_window_attention(**{**args, **over})


def test_empty_batches():
    f = R.rotary_frequencies(8)
    assert FO.rotary_window_attention(torch.zeros(0, 5, 32), torch.arange(5), f, 2, 1).shape == (0, 5, 16)
    assert FO.rotary_window_attention(torch.zeros(2, 0, 32), torch.arange(0), f, 2, 1).shape == (2, 0, 16)


@pytest.mark.parametrize("options", OPTIONS)
def test_far_tokens_matter_only_inside_the_window(options):
    """A token outside every window does not move the last logits; without a window each one does."""
    torch.manual_seed(0)
    model = Llama(LlamaConfig(**{**SMALL, "n_layers": 1, "init_std": 0.3}, **options)).double()
    ids = torch.randint(0, 64, (2, 14))
    moved = ids.clone()
    moved[:, 5] = (moved[:, 5] + 1) % 64
    same = torch.equal(model(ids)[:, -1], model(moved)[:, -1])
    assert same == (0 < options.get("window", 0) < 9)
    first = ids.clone()
    first[:, 0] = (first[:, 0] + 1) % 64
    assert torch.equal(model(ids)[:, -1], model(first)[:, -1]) == (0 < options.get("window", 0) < 14 and not options.get("sinks", 0))


def test_options_at_their_defaults_leave_the_model_as_it_was():
    torch.manual_seed(0)
    plain = Llama(LlamaConfig(**SMALL)).double()
    other = copy.deepcopy(plain)
    other.cfg.window = 100                          # more than the sequence, by the other path
    for b in other.blocks:
        b.cfg = other.cfg
    assert plain.cfg.table_rope and not other.cfg.table_rope
    ids = torch.randint(0, 64, (2, 14))
    # the tables' angles are in 32 bits
    torch.testing.assert_close(plain(ids), other(ids), rtol=0, atol=1e-5)


def test_bad_options_are_refused():
    ids = torch.zeros(1, 4, dtype=torch.long)
    for bad in (dict(rope_scaling="cubic"), dict(rope_layout="pairs"), dict(rotary_dim=3), dict(rotary_dim=10), dict(sinks=2), dict(window=-1),
                dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            Llama(LlamaConfig(**SMALL, **bad))(ids)


def _ring(rank, world):
    for o in (OPTIONS[0], OPTIONS[4]):
        _compare(rank, world, lambda g: Llama(LlamaConfig(**SMALL, **o), group=g))


def test_options_on_a_ring():
    run_distributed(_ring, 2)
