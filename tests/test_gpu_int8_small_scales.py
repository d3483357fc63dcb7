"""The int8 quantiser next to its smallest scale, where half of a scale is not a number of fp32."""
import pytest
import torch

from test_gpu_int8 import quantised

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low,high", [(0.5, 1.0), (1.0, 2.0), (2.0, 4.0), (4.0, 64.0)])
def test_ties_and_their_neighbours(device, low, high):
    """fp32 rows whose scale is `low` to `high` times the smallest: every tie of the row's scale, and what lies one step of fp32
    beside it."""
    import prime_moe
    gen = torch.Generator().manual_seed(int(2 * low))
    peaks = ((low + (high - low) * torch.rand((64,), generator=gen, dtype=torch.float64)) * 127 * 2.0 ** -126).float()
    peaks[0] = float.fromhex("0x1.b39616p-119")
    scale = quantised(peaks[:, None])[1].double()
    ties = ((torch.arange(-127, 127, dtype=torch.float64) + 0.5) * scale[:, None]).float()
    big = torch.full_like(ties, 1.0)
    x = torch.cat([peaks[:, None], ties, torch.nextafter(ties, big), torch.nextafter(ties, -big), torch.zeros((64, 5))], 1)
    x = torch.clamp(x, -peaks[:, None], peaks[:, None])
    x[0, -2:] = torch.tensor([float.fromhex("0x1.b70420p-127"), float.fromhex("0x1.80239ap-124")])
    want, ws = quantised(x)  # on the CPU, in 64 bits
    q, s = prime_moe.quantize_int8(x.to(device))
    assert torch.equal(s.cpu(), ws)
    bad = q.cpu() != want
    assert not bad.any(), (int(bad.sum()), [(float(x[i, j]).hex(), float(s[i]).hex(), int(q[i, j]), int(want[i, j])) for i, j in bad.nonzero()[:4].tolist()])
