"""The product of 8-bit integers and its quantiser on the GPU against exact integers and 64 bits."""
import numpy as np
import pytest
import torch

import grouped_ref as R
from test_gpu_grouped import cus  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def ints(shape, gen, device, lo=-128):
    return torch.randint(lo, 128, shape, generator=gen, dtype=torch.int8).to(device)


def check(got, ref):
    """fp32: the sum, and each product with a scale, is rounded (2^-24 each); then once to the output's type."""
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bound = (half + 3.01 * 2.0 ** -24) * ref.abs() + tiny
    bad = (got.double() - ref).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("counts,behind", [([1], 0), ([0, 3, 0], 0), ([63, 64, 65, 1, 0, 2], 7), ([255, 256, 257], 0), ([130, 31], 300), ([0], 4), ([700], 0)])
@pytest.mark.parametrize("N,K", [(8, 16), (24, 128), (256, 256), (264, 144), (520, 1008)])
def test_grouped(device, cus, counts, behind, N, K):
    import prime_moe
    gen = torch.Generator().manual_seed(N + K + len(counts))
    ends = np.cumsum(counts).tolist()
    M, E = ends[-1] + behind, len(counts)
    x, w = ints((M, K), gen, device), ints((E, N, K), gen, device)
    xs, ws = (torch.rand((M,), generator=gen) * 0.01 + 0.005).to(device), (torch.randn((E, N), generator=gen) * 0.02).to(device)
    off = torch.tensor(ends, dtype=torch.int32, device=device)
    ref = R.mm_int8(x, w, xs, ws, ends)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        y = prime_moe.grouped_mm_int8(x, w, xs, ws, off, dtype)
        assert y.dtype == dtype
        check(y, ref)
        assert (y[ends[-1]:] == 0).all()


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 127, 255, 256, 300, 1025])
@pytest.mark.parametrize("N,K", [(8, 16), (136, 400), (512, 2048)])
def test_dense(device, cus, M, N, K):
    import prime_moe
    gen = torch.Generator().manual_seed(M)
    x, w = ints((M, K), gen, device), ints((N, K), gen, device)
    xs, ws = torch.rand((M,), generator=gen).to(device), torch.rand((N,), generator=gen).to(device)
    ref = R.mm_int8(x, w[None], xs, ws[None], [M])
    for dtype in (torch.bfloat16, torch.float32):
        check(prime_moe.grouped_mm_int8(x, w, xs, ws, out_dtype=dtype), ref)


def test_sums_are_exact(device, cus):
    """The largest sums there are, and sums that an accumulator of 24 bits would round."""
    import prime_moe
    one = lambda n: torch.ones((n,), device=device)
    K = 131056
    x = torch.full((2, K), -128, dtype=torch.int8, device=device)
    x[1] = 127
    w = torch.full((8, K), -128, dtype=torch.int8, device=device)
    y = prime_moe.grouped_mm_int8(x, w, one(2), one(8), out_dtype=torch.float32)
    assert (y[0] == float(K * 16384)).all() and (y[1].double() == float(np.float32(-K * 127 * 128))).all()
    # 2^24 + 1 - 2^24: the large terms cancel
    K = 2048
    x = torch.zeros((1, K), dtype=torch.int8, device=device)
    x[:, :1024] = 127
    x[:, 1024] = 1
    x[:, 1025:] = 127
    w = torch.ones((8, K), dtype=torch.int8, device=device) * 127
    w[:, 1024] = 1
    w[:, 1025:] = -127
    y = prime_moe.grouped_mm_int8(x, w, one(1), one(8), out_dtype=torch.float32)
    assert (y == float(1024 * 16129 + 1 - 1023 * 16129)).all()


def test_strides_and_empty(device, cus):
    import prime_moe
    gen = torch.Generator().manual_seed(3)
    x, w = ints((70, 256), gen, device)[:, 16:-48], ints((3, 40, 320), gen, device)[:, :, 32:224]
    xs, ws = torch.rand((70,), generator=gen).to(device), torch.rand((3, 40), generator=gen).to(device)
    off = torch.tensor([10, 10, 66], dtype=torch.int32, device=device)
    check(prime_moe.grouped_mm_int8(x, w, xs, ws, off, torch.float32), R.mm_int8(x, w, xs, ws, [10, 10, 66]))
    check(prime_moe.grouped_mm_int8(x, w[1], xs, ws[1], None, torch.float32), R.mm_int8(x, w[1:2], xs, ws[1:2], [70]))
    assert prime_moe.grouped_mm_int8(x[:0], w[1], xs[:0], ws[1]).shape == (0, 40)
    # a row whose scale is NaN is NaN, and no other
    xs[5] = xs[67] = float("nan")  # (row 67 belongs to no group)
    y = prime_moe.grouped_mm_int8(x, w, xs, ws, off)
    assert torch.isnan(y[5]).all() and torch.isfinite(y[:5]).all() and torch.isfinite(y[6:]).all() and (y[66:] == 0).all()


def test_weights_beyond_32_bit_offsets(device, cus):
    import prime_moe
    gen = torch.Generator(device=device).manual_seed(4)
    E, N, K = 5, 32768, 32768
    w = torch.randint(-128, 128, (E, N, K), dtype=torch.int8, device=device, generator=gen)
    x = torch.randint(-128, 128, (9, K), dtype=torch.int8, device=device, generator=gen)
    ends = [2, 2, 4, 5, 9]
    ws = torch.rand((E, N), device=device, generator=gen)
    y = prime_moe.grouped_mm_int8(x, w, torch.ones((9,), device=device), ws, torch.tensor(ends, dtype=torch.int32, device=device), torch.float32)
    cols = torch.tensor([0, 1, 255, 256, N - 257, N - 1], device=device)
    check(y[:, cols], R.mm_int8(x, w[:, cols], torch.ones((9,), device=device), ws[:, cols], ends))


# ------------------------------------------------------------------------------- quantiser

def quantised(x):
    """The scale is one fp32 product (which 64 bits hold exactly, and round once), the quotient is taken in 64 bits."""
    c = float(np.float32(1.0) / np.float32(127.0))
    scale = torch.maximum((x.double().abs().amax(-1) * c).to(torch.float32), torch.tensor(2.0 ** -126, device=x.device))
    return torch.round(x.double() / scale.double()[..., None]).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 8), (3, 16), (64, 7168), (5, 40000), (4100, 2048), (4097, 2056), (4096, 4096), (2, 3, 264), (72,), (0, 64)])
def test_quantizer(device, dtype, shape):
    import prime_moe
    gen = torch.Generator(device=device).manual_seed(sum(shape))
    x = (torch.randn(shape, device=device, generator=gen) * torch.randn(shape[:-1] + (1,), device=device, generator=gen).exp()).to(dtype)
    q, scale = prime_moe.quantize_int8(x)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and q.shape == x.shape and scale.shape == x.shape[:-1]
    want, ws = quantised(x)
    assert torch.equal(scale, ws) and torch.equal(q, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantizer_at_borders(device, dtype):
    """Ties, their neighbours, zeros, the smallest and the largest numbers."""
    import prime_moe
    info = torch.finfo(dtype)
    rows = []
    for peak in (127.0, 63.5, 2.0 ** -10 * 127, 1.0, 3.0):
        k = torch.arange(-128, 128, dtype=torch.float64)
        r = ((k + 0.5) * (peak / 127)).to(dtype)
        rows += [r.clamp(-peak, peak)]
        rows += [torch.nextafter(r.float(), torch.full_like(r.float(), 1e30)).to(dtype).clamp(-peak, peak)]
        rows[-1][0] = rows[-2][0] = peak
    tiny = torch.zeros((256,), dtype=dtype)
    rows += [tiny.clone(), tiny.clone(), tiny.clone(), tiny.clone(), -tiny]
    rows[-4][:3] = torch.tensor([info.smallest_normal, -info.smallest_normal * 0.5, info.smallest_normal * info.eps], dtype=dtype)
    rows[-3][:2] = torch.tensor([info.max, -info.max], dtype=dtype)
    rows[-2][7] = info.smallest_normal * info.eps
    x = torch.stack(rows).to(device)
    q, scale = prime_moe.quantize_int8(x)
    want, ws = quantised(x)
    assert torch.equal(scale, ws) and torch.equal(q, want)


def test_quantizer_strides_and_rows_that_are_not_finite(device):
    import prime_moe
    gen = torch.Generator().manual_seed(5)
    x = torch.randn((40, 96), generator=gen).to(torch.bfloat16).to(device)
    q, scale = prime_moe.quantize_int8(x[:, 8:72])
    want, ws = quantised(x[:, 8:72])
    assert torch.equal(scale, ws) and torch.equal(q, want)
    x[3, 5], x[4, 95], x[5, 0] = float("nan"), float("inf"), float("-inf")
    q, scale = prime_moe.quantize_int8(x)
    good = [i for i in range(40) if i not in (3, 4, 5)]
    want, ws = quantised(x[good])
    assert torch.isnan(scale[3:6]).all() and (q[3:6] == 0).all()
    assert torch.equal(scale[good], ws) and torch.equal(q[good], want)


def test_captured(device):
    import prime_moe
    gen = torch.Generator().manual_seed(6)
    x = torch.randn((50, 256), generator=gen).to(torch.bfloat16).to(device)
    w, ws = ints((264, 256), gen, device), torch.rand((264,), generator=gen).to(device)
    fn = lambda: prime_moe.grouped_mm_int8(*(lambda q: (q[0], w, q[1], ws))(prime_moe.quantize_int8(x)))
    fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    for _ in range(3):
        x.copy_(torch.randn((50, 256), generator=gen).to(torch.bfloat16))
        graph.replay()
        assert torch.equal(out, fn())
