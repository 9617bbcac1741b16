"""Which layers the gated feed-forward block's kernels may stand in for, without a GPU: the conditions on device and type are taken as met."""
import pytest
import torch
from torch import nn

from rtp_b200.models.llama import Llama, LlamaConfig
from rtp_b200.module.linear import ColumnParallelLinear, RowParallelLinear
from rtp_b200.ops import mlp
from rtp_b200.parallel import fused

SMALL = dict(vocab_size=64, d_model=32, n_layers=1, n_heads=4, d_ff=64, max_seq_len=16)


@pytest.fixture
def on_kernels(monkeypatch):
    """Every call is one for the kernels; they answer with this text."""
    monkeypatch.setattr(fused, "use_fused", lambda *a: True)
    monkeypatch.setattr(mlp, "kernel_takes", lambda *a: True)
    monkeypatch.setattr(mlp, "gated_mlp", lambda *a, **kw: "kernels")


def layers(down=RowParallelLinear, up=ColumnParallelLinear):
    return up(32, 128, bias=False, packed_parts=2), down(64, 32, bias=False), torch.zeros(3, 32)


class Doubled(RowParallelLinear):
    def forward(self, x):
        return 2 * super().forward(x)


class DoubledUp(ColumnParallelLinear):
    def forward(self, x):
        return 2 * super().forward(x)


def test_plain_layers_are_taken(on_kernels):
    assert fused.gated_mlp(*layers()) == "kernels"


def test_layers_with_their_own_forward_are_called(on_kernels, monkeypatch):
    assert fused.gated_mlp(*layers(down=Doubled)) is None
    assert fused.gated_mlp(*layers(up=DoubledUp)) is None
    for n in (0, 1):
        args = layers()
        args[n].forward = lambda x: x
        assert fused.gated_mlp(*args) is None
        del args[n].forward
        assert fused.gated_mlp(*args) == "kernels"
    args = layers()
    monkeypatch.setattr(RowParallelLinear, "forward", lambda self, x: x)
    assert fused.gated_mlp(*args) is None


def test_layers_of_another_kind_are_called(on_kernels):
    up, down, x = layers()
    for other in (nn.Sequential(down), nn.Linear(64, 32, bias=False), up):
        assert fused.gated_mlp(up, other, x) is None
    for other in (nn.Sequential(up), nn.Linear(32, 128, bias=False), down):
        assert fused.gated_mlp(other, down, x) is None


def test_hooks_and_the_in_place_mode(on_kernels):
    for n in (0, 1):
        args = layers()
        for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
            handle = getattr(args[n], register)(lambda *a: None)
            assert fused.gated_mlp(*args) is None
            handle.remove()
        handle = nn.modules.module.register_module_forward_hook(lambda *a: None)
        assert fused.gated_mlp(*args) is None
        handle.remove()
        assert fused.gated_mlp(*args) == "kernels"
        args[n].inplace = True
        assert fused.gated_mlp(*args) is None


def test_weights_that_left_the_shard(on_kernels):
    """The layers read the flat shard."""
    for n in (0, 1):
        args = layers()
        args[n].linear.weight.data = args[n].linear.weight.data.clone()
        assert fused.gated_mlp(*args) is None


@pytest.mark.parametrize("wrap", [lambda m: nn.Sequential(m), lambda m: nn.Linear(m.in_features, m.out_features, bias=False)])
def test_model_with_other_layers_runs(wrap):
    torch.manual_seed(0)
    model = Llama(LlamaConfig(**SMALL))
    ids = torch.randint(0, 64, (2, 9))
    block = model.blocks[0]
    want = model(ids)
    block.gate_up, block.down = wrap(block.gate_up), wrap(block.down)
    got = model(ids)
    assert got.shape == want.shape
    if isinstance(block.down, nn.Sequential):
        assert torch.equal(got, want)
