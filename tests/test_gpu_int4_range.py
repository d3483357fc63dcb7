"""Weights of 4 bits at the ends of what their types hold: scales and rows near the largest and the smallest numbers."""
import pytest
import torch

import int4_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


# ---- back to 16 bits


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_dequantize_with_every_size_of_scale(device, dtype, group):
    """value * scale, rounded once, for scales from the smallest to the largest number of the type; zeros stay zeros."""
    import prime_moe
    least, most = (2.0 ** -24, 65504.0) if dtype == F16 else (2.0 ** -126, torch.finfo(BF16).max)
    scales = [least * 4.0 ** i for i in range(200) if least * 4.0 ** i < most] + [most, most / 2, most / 7, most / 23, most / 24, most / 25]
    rows = (len(scales) + 15) // 16 * 16
    scale = torch.tensor((scales * 16)[:rows], dtype=torch.float64).to(dtype)[:, None].expand(rows, 256 // group).contiguous().to(device)
    values = (torch.arange(rows * 256).reshape(rows, 256) % 16 - 8).to(torch.int8).to(device)
    got = prime_moe.dequantize_int4(*prime_moe.pack_int4(values, scale))
    want = R.weights(values, scale).to(dtype)
    assert torch.equal(got, want)
    assert (got[values == 0] == 0).all() and torch.isfinite(got[values.abs() == 1]).all()


def test_quantized_weights_near_the_largest_come_back(device):
    import prime_moe
    w = torch.zeros((16, 128), device=device)
    w[3, :4] = torch.tensor([3.3e38, -3.3e38, 1e38, 5e37])
    w[9, 1] = -2e38
    q, s = prime_moe.quantize_int4(w, 128, BF16)
    got = prime_moe.dequantize_int4(q, s)
    assert torch.equal(got, R.weights(*R.quantize(w, 128, BF16)).to(BF16))
    assert torch.isfinite(got).all() and (got[w == 0] == 0).all() and got[3, 0] > 3e38
