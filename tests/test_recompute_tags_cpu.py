"""When a tagged tensor may be rebuilt from its sources."""
import torch

from rtp_b200.ops import functional as FO


def tagged():
    x, w = torch.randn(4), torch.randn(4)
    return FO._tag(x * 2, "norm", x, w, None, 1e-5, True), x, w


def test_untouched():
    y, x, w = tagged()
    kind, srcs = FO.recompute_tag(y)
    assert kind == "norm" and srcs[0] is x and srcs[1] is w and srcs[2:] == (None, 1e-5, True)
    assert FO.recompute_tag(x) is None


def test_changed_in_place():
    for n in range(3):
        t = tagged()
        t[n].add_(1)
        assert FO.recompute_tag(t[0]) is None
        t = tagged()
        t[n][1:].zero_()                       # through a view
        assert FO.recompute_tag(t[0]) is None


def test_changed_before():
    x = torch.randn(4)
    x.mul_(2)
    y = x * 2
    y.add_(1)
    assert FO.recompute_tag(FO._tag(y, "gelu", x)) is not None


def test_sources_without_versions():
    with torch.inference_mode():
        x = torch.randn(4)
    y = FO._tag(x * 2, "gelu", x)
    assert FO.recompute_tag(y) is None
