"""Weights of 4 bits on the GPU: the quantiser and its inverse, products with them, against the definitions in 64 bits."""
import numpy as np
import pytest
import torch

import int4_ref as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---- quantiser


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("shape", [(16, 128), (48, 640), (2, 3, 32, 384), (32, 1152), (16, None)])
def test_quantize(device, shape, dtype, scale_dtype, group):
    import prime_moe
    shape = tuple(d or group for d in shape)
    gen = torch.Generator().manual_seed(shape[-1] + group)
    w = (torch.randn(shape, generator=gen) * torch.randn((*shape[:-1], 1), generator=gen).exp()).to(dtype).to(device)
    q, s = prime_moe.quantize_int4(w, group, scale_dtype)
    values, scale = R.quantize(w, group, scale_dtype)
    back = R.unpack(q, s, shape[-1])
    assert torch.equal(back[1], scale.cpu()) and torch.equal(back[0], values.cpu())
    # the layout is pack_int4's, the padding of the last tile included
    pq, ps = prime_moe.pack_int4(values, scale)
    assert torch.equal(q, pq) and torch.equal(s, ps)
    # and back: one rounding of an exact product (8 x 2^8 or 8 x 2^11 steps fit fp32)
    got = prime_moe.dequantize_int4(q, s, shape[-1])
    assert got.shape == w.shape and torch.equal(got, R.weights(values, scale).to(scale_dtype))


def test_quantize_borders(device):
    """Values half way between two integers go to the even one; zeros; the smallest scales; what is not finite."""
    import prime_moe
    w = torch.zeros((16, 128), device=device)
    w[0, :15] = torch.tensor([7, 6.5, 5.5, 4.5, 3.5, 2.5, 1.5, .5, -.5, -1.5, -2.5, -3.5, -4.5, -5.5, -6.5])
    w[1, :4] = torch.tensor([7.0, 3.5 + 2 ** -20, 3.5 - 2 ** -20, -7.0])
    w[2, 5] = float("inf")
    w[3, 7] = float("nan")
    w[4, 0] = -float("inf")
    w[5, :3] = torch.tensor([2.0 ** -140, -(2.0 ** -149), 2.0 ** -126])
    w[6, :4] = torch.tensor([2.0 ** -24, 10 * 2.0 ** -24, -10 * 2.0 ** -24, 3 * 2.0 ** -24])
    w[7, 0] = 7 * 65504.0
    w[8, 0] = 7 * 65536.0   # a scale beyond float16
    w[9, :2] = torch.tensor([3.4e38, -3.4e38])
    for scale_dtype in (BF16, F16):
        for group in (32, 64, 128):
            q, s = prime_moe.quantize_int4(w, group, scale_dtype)
            values, scale = R.quantize(w, group, scale_dtype)
            got = R.unpack(q, s, 128)
            assert torch.equal(got[0], values.cpu())
            assert torch.equal(got[1].nan_to_num(nan=-1.0), scale.cpu().nan_to_num(nan=-1.0))
            assert torch.isnan(got[1][2:5, 0]).all() and not torch.isnan(got[1][:2]).any()
            assert values[0, :15].tolist() == [7, 6, 6, 4, 4, 2, 2, 0, 0, -2, -2, -4, -4, -6, -6]
            assert torch.isnan(prime_moe.dequantize_int4(q, s)[2, :group]).all()


def test_empty(device):
    import prime_moe
    q, s = prime_moe.quantize_int4(torch.zeros((0, 16, 64), device=device, dtype=BF16), 64)
    assert q.shape == (0, 1, 1, 1024) and prime_moe.dequantize_int4(q, s, 64).shape == (0, 16, 64)
    q, s = prime_moe.quantize_int4(torch.zeros((2, 16, 64), device=device, dtype=BF16), 64)
    x = torch.zeros((0, 64), device=device, dtype=BF16)
    assert prime_moe.grouped_mm_int4(x, q, s, torch.zeros((2,), dtype=torch.int32, device=device)).shape == (0, 16)


# ---- products


def operands(shape, group, dtype, gen, device):
    values = torch.randint(-8, 8, shape, generator=gen, dtype=torch.int8)
    scale = ((torch.rand((*shape[:-1], shape[-1] // group), generator=gen) + 0.5) * 0.2 * shape[-1] ** -0.5).to(dtype)
    return values.to(device), scale.to(device)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 97])
@pytest.mark.parametrize("N,K", [(16, None), (48, 640), (528, 1024), (4096, 2048), (64, 7168)])
def test_dense(device, M, N, K, dtype, group):
    import prime_moe
    K = K or group
    gen = torch.Generator().manual_seed(M + N + K)
    values, scale = operands((N, K), group, dtype, gen, device)
    x = torch.randn((M, K), generator=gen).to(dtype).to(device)
    y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
    assert y.shape == (M, N) and y.dtype == dtype
    R.check(y, *R.mm(x, values[None], scale[None], [M]), K, group)


@pytest.mark.parametrize("counts,behind", [([1], 0), ([0, 3, 0], 0), ([15, 16, 17, 1, 0, 2], 7), ([32, 33, 31], 0), ([0, 70], 130), ([0], 4), ([0, 0, 0], 33)])
@pytest.mark.parametrize("N,K,group", [(16, 32, 32), (48, 192, 64), (272, 1152, 128), (1536, 2048, 32)])
def test_grouped(device, counts, behind, N, K, group):
    import prime_moe
    for dtype in (BF16, F16):
        gen = torch.Generator().manual_seed(N + K + len(counts))
        ends = np.cumsum(counts).tolist()
        M, E = ends[-1] + behind, len(counts)
        values, scale = operands((E, N, K), group, dtype, gen, device)
        x = torch.randn((M, K), generator=gen).to(dtype).to(device)
        x[ends[-1]:] = float("nan")  # rows of no expert reach nothing
        q, s = prime_moe.pack_int4(values, scale)
        y = prime_moe.grouped_mm_int4(x, q, s, torch.tensor(ends, dtype=torch.int32, device=device))
        R.check(y, *R.mm(x, values, scale, ends), K, group)
        assert (y[ends[-1]:] == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sums_of_integers_are_exact(device, dtype, group):
    """Small integers and scales that are powers of two: every sum is a multiple of 2^-4 below 2^20 and fits fp32 whatever the order, so
    that the output is the exact one, rounded once."""
    import prime_moe
    gen = torch.Generator().manual_seed(group)
    for M, N, K in ((1, 64, 1024), (7, 160, 384), (16, 1024, 512), (40, 48, 1152)):
        values = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(device)
        scale = (2.0 ** torch.randint(-4, 1, (N, K // group), generator=gen)).to(dtype).to(device)
        x = torch.randint(-8, 9, (M, K), generator=gen).to(dtype).to(device)
        y = prime_moe.grouped_mm_int4(x, *prime_moe.pack_int4(values, scale))
        assert torch.equal(y, R.mm(x, values[None], scale[None], [M])[0].to(dtype))


def test_one_weight_at_a_time(device):
    """x = unit vectors: every column of every row comes back, so that no two places are mixed up."""
    import prime_moe
    N, K, group = 48, 256, 32
    gen = torch.Generator().manual_seed(3)
    values = torch.randint(-8, 8, (N, K), generator=gen, dtype=torch.int8).to(device)
    scale = (torch.arange(N * K // group).view(N, -1) % 61 + 1).to(BF16).to(device)
    y = prime_moe.grouped_mm_int4(torch.eye(K, device=device, dtype=BF16), *prime_moe.pack_int4(values, scale))
    assert torch.equal(y.t(), R.weights(values, scale).to(BF16))


def test_strides_and_slices(device):
    """Rows further apart than they are long, a matrix out of a stack, NaN between the rows and behind the last."""
    import prime_moe
    gen = torch.Generator().manual_seed(5)
    N, K, M = 64, 160, 21
    values, scale = operands((3, N, K), 32, BF16, gen, device)
    q, s = prime_moe.pack_int4(values, scale)
    wide = torch.full((M, K + 24), float("nan"), dtype=BF16, device=device)
    wide[:, :K] = torch.randn((M, K), generator=gen).to(device)
    x = wide[:, :K]
    R.check(prime_moe.grouped_mm_int4(x, q[1], s[1]), *R.mm(x, values[1:2], scale[1:2], [M]), K, 32)
    assert torch.equal(prime_moe.grouped_mm_int4(x, q[1], s[1]), prime_moe.grouped_mm_int4(x.contiguous(), q[1], s[1]))


def test_rows_that_are_not_finite_stay_alone(device):
    import prime_moe
    gen = torch.Generator().manual_seed(6)
    N, K, M = 64, 256, 20
    values, scale = operands((N, K), 64, BF16, gen, device)
    q, s = prime_moe.pack_int4(values, scale)
    x = torch.randn((M, K), generator=gen).to(BF16).to(device)
    want = prime_moe.grouped_mm_int4(x, q, s)
    x[3, 17], x[18, 255] = float("inf"), float("nan")
    y = prime_moe.grouped_mm_int4(x, q, s)
    assert torch.isnan(y[[3, 18]]).all()
    rest = [i for i in range(M) if i not in (3, 18)]
    assert torch.equal(y[rest], want[rest])


def test_float16_reaches_its_range(device):
    """Small values of float16, which are subnormal, count; sums beyond the type become infinite, not NaN."""
    import prime_moe
    values = torch.full((16, 128), 7, dtype=torch.int8, device=device)
    x = torch.full((1, 128), 2.0 ** -24, dtype=F16, device=device)
    q, s = prime_moe.pack_int4(values, torch.ones((16, 1), dtype=F16, device=device))
    assert torch.equal(prime_moe.grouped_mm_int4(x, q, s), torch.full((1, 16), 7 * 128 * 2.0 ** -24, dtype=F16, device=device))
    x.fill_(60000.0)
    assert (prime_moe.grouped_mm_int4(x, q, s) == float("inf")).all()
    q, s = prime_moe.pack_int4(values, torch.full((16, 1), 2.0 ** -24, dtype=F16, device=device))
    x.fill_(1024.0)
    assert torch.equal(prime_moe.grouped_mm_int4(x, q, s), torch.full((1, 16), 7 * 128 * 2.0 ** -14, dtype=F16, device=device))


def test_offsets_out_of_order_stay_inside(device):
    """Unspecified outputs, but of a call that ends, and the next one is right."""
    import prime_moe
    gen = torch.Generator().manual_seed(8)
    values, scale = operands((4, 32, 128), 128, BF16, gen, device)
    q, s = prime_moe.pack_int4(values, scale)
    x = torch.randn((40, 128), generator=gen).to(BF16).to(device)
    for bad in ([40, 10, 30, 5], [-7, 100, 2 ** 30, -2 ** 31], [5, 5, 4, 40]):
        assert prime_moe.grouped_mm_int4(x, q, s, torch.tensor(bad, dtype=torch.int32, device=device)).shape == (40, 32)
    ends = [10, 10, 25, 40]
    R.check(prime_moe.grouped_mm_int4(x, q, s, torch.tensor(ends, dtype=torch.int32, device=device)), *R.mm(x, values, scale, ends), 128, 128)


def test_the_same_bits_every_time_and_in_a_graph(device):
    import prime_moe
    gen = torch.Generator().manual_seed(9)
    values, scale = operands((8, 256, 512), 64, BF16, gen, device)
    q, s = prime_moe.pack_int4(values, scale)
    x = torch.randn((24, 512), generator=gen).to(BF16).to(device)
    o = torch.tensor([3, 3, 10, 11, 11, 20, 24, 24], dtype=torch.int32, device=device)
    w = torch.randn((64, 512), generator=gen).to(BF16).to(device)

    def step():
        return (prime_moe.grouped_mm_int4(x, q, s, o), *prime_moe.quantize_int4(w, 64))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        x.copy_(torch.randn((24, 512), generator=gen).to(BF16)) if turn else None
        want = [t.clone() for t in step()]
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_another_stream(device):
    import prime_moe
    gen = torch.Generator().manual_seed(10)
    values, scale = operands((512, 1024), 128, F16, gen, device)
    q, s = prime_moe.pack_int4(values, scale)
    x = torch.randn((3, 1024), generator=gen).to(F16).to(device)
    want = prime_moe.grouped_mm_int4(x, q, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(4):
        with torch.cuda.stream(streams[turn % 2]):
            got.append(prime_moe.grouped_mm_int4(x, q, s))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_int4_experts_and_their_unpacked_form_agree(device):
    """As they are used together: a layer's weights quantised, decoded with in 4 bits, and unpacked for a prefill."""
    import prime_moe
    gen = torch.Generator().manual_seed(11)
    E, N, K, top_k = 8, 96, 256, 2
    w = (torch.randn((E, N, K), generator=gen) * K ** -0.5).to(BF16).to(device)
    q, s = prime_moe.quantize_int4(w, 32)
    for tokens in (3, 200):
        logits = torch.randn((tokens, E), generator=gen).to(device)
        x = torch.randn((tokens, K), generator=gen).to(BF16).to(device)
        _, _, order, experts, total = prime_moe.route(logits, top_k, block_m=1)
        offsets = prime_moe.expert_offsets(experts, total, E)
        rows = x[order.long() // top_k]
        values, scale = R.quantize(w, 32, BF16)
        ref, m = R.mm(rows, values, scale, offsets.tolist())
        R.check(prime_moe.grouped_mm_int4(rows, q, s, offsets), ref, m, K, 32)
        # (the unpacked weights are rounded to bfloat16: 2^-9 of a magnitude of 8 scales)
        y = prime_moe.grouped_mm(rows, prime_moe.dequantize_int4(q, s), offsets)
        assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 8 * 2.0 ** -9 * 1.01 * m + 1e-6).all()


def test_weights_behind_4_gb(device):
    """The last of many matrices, and the last rows of a matrix of more than 2^32 values: products, quantiser, inverse."""
    import prime_moe
    E, N, K, group = 260, 8192, 4096, 128
    gen = torch.Generator().manual_seed(3)
    values, scale = operands((1, N, K), group, BF16, gen, device)
    x = torch.randn((3, K), generator=gen).to(BF16).to(device)
    q, s = prime_moe.pack_int4(values, scale)
    many_q = torch.zeros((E, *q.shape[1:]), dtype=torch.uint8, device=device)
    many_s = torch.zeros((E, *s.shape[1:]), dtype=BF16, device=device)
    assert many_q.numel() > 1 << 32
    many_q[-1], many_s[-1] = q[0], s[0]
    ends = torch.tensor([0] * (E - 1) + [3], dtype=torch.int32, device=device)
    R.check(prime_moe.grouped_mm_int4(x, many_q, many_s, ends), *R.mm(x, values, scale, [3]), K, group)
    del many_q, many_s
    w = torch.zeros((132, N, K), dtype=BF16, device=device)
    assert w.numel() > 1 << 32
    w[-1] = torch.randn((N, K), generator=gen).to(BF16).to(device)
    q, s = prime_moe.quantize_int4(w, group)
    one = prime_moe.quantize_int4(w[-1], group)
    assert torch.equal(q[-1], one[0]) and torch.equal(s[-1], one[1])
    back = prime_moe.dequantize_int4(q, s)
    assert torch.equal(back[-1], prime_moe.dequantize_int4(*one)) and (back[0] == 0).all()
