"""Arguments that rotary positions refuse, the same on the GPU as without one."""
import pytest
import torch

from rtp_b200.ops import functional as FO, rotary as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("over", [
    dict(q=torch.zeros(2, 4, 16)), dict(q=torch.zeros(16)), dict(q=torch.zeros(())), dict(k=torch.zeros(2, 4, 16)), dict(layout="other"),
    dict(q=torch.zeros(2, 4, 3, 16, dtype=torch.int32)), dict(k=torch.zeros(2, 5, 1, 16)), dict(k=torch.zeros(2, 4, 1, 8)),
    dict(k=torch.zeros(2, 4, 1, 16, dtype=torch.float64)), dict(positions=torch.arange(4.0)), dict(positions=torch.arange(5)),
    dict(positions=torch.zeros(3, 4, dtype=torch.int64)), dict(freqs=torch.ones(8)), dict(freqs=torch.ones(9, dtype=torch.float64)),
    dict(freqs=torch.ones(0, dtype=torch.float64)),
])
@pytest.mark.parametrize("entry", [FO.rotary, R.rotary])
def test_refusals(over, entry):
    args = {**dict(q=torch.zeros(2, 4, 3, 16), k=torch.zeros(2, 4, 1, 16), positions=torch.arange(4), freqs=R.rotary_frequencies(16), layout="half"),
            **over}
    with pytest.raises(ValueError):
        entry(**{n: t.cuda() if torch.is_tensor(t) else t for n, t in args.items()})


def test_tensors_on_two_devices():
    q, f = torch.zeros(2, 4, 3, 16, device="cuda"), R.rotary_frequencies(16, device="cuda")
    for bad in (dict(positions=torch.arange(4), freqs=f), dict(positions=torch.arange(4, device="cuda"), freqs=f.cpu())):
        with pytest.raises(ValueError):
            FO.rotary(q, None, **bad)
