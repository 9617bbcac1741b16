"""A block of the Llama-shaped model called by itself."""
import pytest
import torch

from rtp_b200.models.llama import Llama, LlamaConfig, rope_tables
from rtp_b200.ops import rotary as R

SMALL = dict(vocab_size=64, d_model=32, n_layers=1, n_heads=4, d_ff=64, max_seq_len=16)


@pytest.mark.parametrize("options", [{}, dict(window=3, sinks=1)])
def test_tables_by_name(options):
    torch.manual_seed(0)
    block = Llama(LlamaConfig(**SMALL, **options)).blocks[0]
    x = torch.randn(2, 9, 32)
    a, b = (torch.arange(9), R.rotary_frequencies(8)) if options else rope_tables(9, 8, 10000.0, "cpu")
    assert torch.equal(block(x, cos=a, sin=b), block(x, a, b))
