"""``engine.check_all`` reads what kernels outside a ring report as well."""
import pytest
import torch

from rtp_b200.ops import _lib
from rtp_b200.parallel import engine


def test_words_outside_a_ring(monkeypatch):
    words = {("cuda", 0): torch.zeros(1, dtype=torch.int64), ("cuda", 1): torch.zeros(1, dtype=torch.int64)}
    monkeypatch.setattr(_lib, "_status_words", words)
    monkeypatch.setattr(engine, "_engines", {})
    engine.check_all()
    for w in words.values():
        w.fill_(1)
        with pytest.raises(_lib.RotationTimeout, match="timed out"):
            engine.check_all()
        assert int(w) == 0
        engine.check_all()
