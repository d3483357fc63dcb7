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


# ---- products


def spread(shape, low, high, gen, dtype, device):
    """Numbers of both signs whose sizes are spread from 2^low to 2^high over their logarithm."""
    size = torch.exp2(torch.rand(shape, generator=gen, dtype=torch.float64) * (high - low) + low)
    return torch.where(torch.rand(shape, generator=gen) < 0.5, -size, size).to(dtype).to(device)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (1, 4096, 256), (3, 48, 640), (16, 528, 512), (33, 64, 256), (70, 272, 1152)])
def test_rows_near_the_largest_number(device, M, N, K, group):
    """bf16 rows up to the type's end, scales that bring the products back: nothing on the way is infinite."""
    import prime_moe
    gen = torch.Generator().manual_seed(M + N + group)
    values = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(device)
    scale = ((torch.rand((N, K // group), generator=gen) + 0.5) * 2.0 ** -100).to(BF16).to(device)
    x = spread((M, K), 120, 127.9, gen, BF16, device)
    x[0, :32] = torch.finfo(BF16).max  # a sum of the same sign throughout
    y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
    R.check(y, *R.mm(x, values[None], scale[None], [M]), K, group)


def test_groups_of_the_largest_number(device):
    """Every x the largest of bf16 or its negative, of one sign, or as the weights' signs: the sums are the largest there can be."""
    import prime_moe
    most = torch.finfo(BF16).max
    for group in (32, 64, 128):
        values = torch.tensor([7, -8], dtype=torch.int8, device=device).repeat(16, 128)
        x = torch.full((4, 256), most, dtype=BF16, device=device)
        x[1], x[2, 1::2], x[3, ::2] = -most, -most, -most
        scale = torch.full((16, 256 // group), 2.0 ** -120, dtype=BF16, device=device)
        y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
        assert torch.equal(y, R.mm(x, values[None], scale[None], [4])[0].to(BF16))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_of_the_smallest_numbers(device, group):
    """Multiples of the least subnormal, 2^-133, and scales that bring them up: sums of a group are multiples of 2^-145, which fp32 holds,
    and with scales that are powers of two every sum has 24 bits at most, so that the output is the exact one, rounded once."""
    import prime_moe
    gen = torch.Generator().manual_seed(group)
    for M, N, K in ((1, 64, 1024), (7, 160, 384), (40, 48, 640)):
        values = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(device)
        scale = (2.0 ** torch.randint(40, 44, (N, K // group), generator=gen)).to(BF16).to(device)
        x = (torch.randint(-8, 9, (M, K), generator=gen).double() * 2.0 ** -133).to(BF16).to(device)
        y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
        assert (y != 0).any()
        assert torch.equal(y, R.mm(x, values[None], scale[None], [M])[0].to(BF16))


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("size", [-124, -118, -112, -104])
def test_outputs_of_the_smallest_numbers(device, size, group):
    """Each of the K / group + 8 sums that make an output may be rounded by half of 2^-137, beside what int4_ref.check allows."""
    import prime_moe
    gen = torch.Generator().manual_seed(group - size)
    M, N, K = 5, 64, 1024
    values = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(device)
    scale = ((torch.rand((N, K // group), generator=gen) + 0.5) * 2.0 ** (size // 2)).to(BF16).to(device)
    x = (torch.randn((M, K), generator=gen).double() * 2.0 ** (size - size // 2 - 7)).to(BF16).to(device)
    y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
    ref, m = R.mm(x, values[None], scale[None], [M])
    sums = R.sums_bound(m, K, group) + (K / group + 8) * 2.0 ** -138
    assert ((y.double() - ref).abs() <= sums + 2.0 ** -8 * (ref.abs() + sums) + 2.0 ** -134).all() and (y != 0).any()


@pytest.mark.parametrize("T", [1, 2, 5, 16])
@pytest.mark.parametrize("group", [32, 128])
def test_layer_of_4_bits_with_large_rows(device, T, group):
    """bf16: x near the type's end, or an activation near it (the up half alone is large, so that the gate's curve stays one)."""
    import prime_moe
    from layer_ref import Layer
    K, H, E = 256, 128, 3
    gen = torch.Generator().manual_seed(T + group)
    v1 = torch.randint(-8, 8, (E, 2 * H, K), generator=gen, dtype=torch.int8).to(device)
    v2 = torch.randint(-8, 8, (E, K, H), generator=gen, dtype=torch.int8).to(device)
    s1 = ((torch.rand((E, 2 * H, K // group), generator=gen) + 0.5) * 2.0 ** -7).to(BF16).to(device)
    s2 = ((torch.rand((E, K, H // group), generator=gen) + 0.5) * 2.0 ** -7).to(BF16).to(device)
    base = spread((T, K), -2, 3, gen, BF16, device)
    gate = torch.zeros((E, K), dtype=BF16, device=device)
    bias = torch.tensor([0.5, 0.25, 0.0], device=device)
    for size, up, down in ((2.0 ** 124, 1.0, 1.0), (1.0, 2.0 ** 118, 2.0 ** -118)):
        x, a1, a2 = base * size, s1 * (2.0 ** 5 / size if size > 1 else 1.0), s2 * down
        a1[:, H:] *= up
        ones = lambda v, s: 55 * R.weights(torch.ones_like(v), s).abs()
        ref = Layer(x, gate, R.weights(v1, a1), R.weights(v2, a2), E, bias, ones(v1, a1), ones(v2, a2), 2 * group + K / group + 30, 2 * group + H / group + 30)
        ref.check(*prime_moe.moe_layer_int4(x, gate, *prime_moe.pack_int4(v1, a1), *prime_moe.pack_int4(v2, a2), E, bias))
