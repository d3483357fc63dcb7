"""Ragged expert products on the GPU against 64 bits: sizes, layouts, strides, groups without rows, what lies next to the
operands, gradients, graphs, streams."""
import numpy as np
import pytest
import torch

import grouped_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(params=[0, 8], ids=["whole device", "8 CUs"])
def cus(request):
    """Launches sized for the device, and for one of eight CUs: small cases then take the kernels of large ones, and many tiles
    follow each other in a workgroup."""
    from prime_moe import _native
    _native.load().pmoe_set_compute_units(request.param)
    yield request.param
    _native.load().pmoe_set_compute_units(0)


def make(shape, gen, dtype, device, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype).to(device)


def ends_tensor(ends, device):
    return torch.tensor(ends, dtype=torch.int32, device=device)


# counts of the groups; rows behind them
RAGGED = [
    ([1], 0),
    ([0, 0, 3, 0], 0),
    ([63, 64, 65, 1, 0, 2], 7),
    ([255, 0, 256, 257], 0),
    ([129, 193, 31, 32, 33], 300),
    ([513, 1], 1),
    ([0, 0], 5),
    ([700], 0),
    ([17, 0, 15, 16, 48], 3),
    ([2, 1, 1, 0, 5, 3], 0),
]


@pytest.mark.parametrize("counts,behind", RAGGED)
@pytest.mark.parametrize("N,K", [(8, 8), (24, 64), (256, 128), (264, 72), (520, 1000), (128, 136)])
@pytest.mark.parametrize("across", [False, True])
def test_forward(device, cus, counts, behind, N, K, across):
    import prime_moe
    gen = torch.Generator().manual_seed(N * 1000 + K + len(counts))
    ends = np.cumsum(counts).tolist()
    for dtype in DTYPES:
        x = make((ends[-1] + behind, K), gen, dtype, device)
        w = make((len(counts), N, K), gen, dtype, device, K ** -0.5)
        if across:
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        y = prime_moe.grouped_mm(x, w, ends_tensor(ends, device))
        ref, mags = R.mm(x, w, ends)
        R.check(y, ref, mags, K)
        assert (y[ends[-1]:] == 0).all()


# on eight CUs and two tiles of columns: tiles of 64 rows up to 256 rows, of 128 up to 512, of 256 beyond
@pytest.mark.parametrize("counts,behind", [([256], 0), ([257], 0), ([512], 3), ([513], 0), ([1100], 260), ([64, 0, 63, 65], 0),
                                           ([65, 64, 65], 0), ([128, 128, 129], 0), ([300, 212], 0)])
@pytest.mark.parametrize("across", [False, True])
def test_heights_of_tiles(device, cus, counts, behind, across):
    import prime_moe
    gen = torch.Generator().manual_seed(len(counts) + counts[0])
    ends, N, K = np.cumsum(counts).tolist(), 512, 256
    x = make((ends[-1] + behind, K), gen, torch.bfloat16, device)
    w = make((len(counts), N, K), gen, torch.bfloat16, device, K ** -0.5)
    y = prime_moe.grouped_mm(x, w.transpose(1, 2).contiguous().transpose(1, 2) if across else w, ends_tensor(ends, device))
    ref, mags = R.mm(x, w, ends)
    R.check(y, ref, mags, K)
    assert (y[ends[-1]:] == 0).all()


@pytest.mark.parametrize("counts,behind", RAGGED)
@pytest.mark.parametrize("N,K", [(8, 8), (24, 64), (256, 128), (264, 72), (520, 1000), (1032, 264)])
def test_weight_gradient(device, cus, counts, behind, N, K):
    import prime_moe
    gen = torch.Generator().manual_seed(N * 1000 + K + len(counts))
    ends = np.cumsum(counts).tolist()
    for dtype in DTYPES:
        dy = make((ends[-1] + behind, N), gen, dtype, device)
        x = make((ends[-1] + behind, K), gen, dtype, device)
        dw = prime_moe.grouped_mm_wgrad(dy, x, ends_tensor(ends, device))
        ref, mags = R.wgrad(dy, x, ends)
        R.check(dw, ref, mags, max(counts))
        for g, c in enumerate(counts):
            if c == 0:
                assert (dw[g] == 0).all()


@pytest.mark.parametrize("E,total", [(1, 5), (7, 100), (64, 4000), (257, 300), (1000, 2500), (1024, 1024)])
def test_many_groups(device, cus, E, total):
    import prime_moe
    gen = torch.Generator().manual_seed(E)
    ends = R.sized(total, E, gen)
    x, w = make((total + 3, 80), gen, torch.bfloat16, device), make((E, 48, 80), gen, torch.bfloat16, device)
    off = ends_tensor(ends, device)
    ref, mags = R.mm(x, w, ends)
    R.check(prime_moe.grouped_mm(x, w, off), ref, mags, 80)
    dy = make((total + 3, 48), gen, torch.bfloat16, device)
    ref, mags = R.wgrad(dy, x, ends)
    R.check(prime_moe.grouped_mm_wgrad(dy, x, off), ref, mags, total)


def test_no_rows(device):
    import prime_moe
    off = torch.zeros((3,), dtype=torch.int32, device=device)
    x, w = torch.empty((0, 64), dtype=torch.bfloat16, device=device), torch.ones((3, 32, 64), dtype=torch.bfloat16, device=device)
    assert prime_moe.grouped_mm(x, w, off).shape == (0, 32)
    dw = prime_moe.grouped_mm_wgrad(torch.empty((0, 32), dtype=torch.bfloat16, device=device), x, off)
    assert dw.shape == (3, 32, 64) and (dw == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_lies_next_to_the_operands_does_not_count(device, cus, dtype):
    """NaNs between the rows of strided operands, in rows behind the last group and in the rows of other groups."""
    import prime_moe
    gen = torch.Generator().manual_seed(5)
    N, K, counts, behind = 72, 200, [33, 0, 70, 5], 21
    ends = np.cumsum(counts).tolist()
    M = ends[-1] + behind
    nan = float("nan")

    def inside(shape, pad, fill=nan):
        t = torch.full(shape[:-1] + (shape[-1] + 2 * pad,), fill, dtype=dtype, device=device)
        t[..., pad:-pad] = make(shape, gen, dtype, device)
        return t[..., pad:-pad]

    x, w, dy = inside((M, K), 8), inside((len(counts), N, K), 16), inside((M, N), 24)
    wt = inside((len(counts), K, N), 8).transpose(1, 2)
    x[ends[-1]:] = nan
    dy[ends[-1]:] = nan
    off = ends_tensor(ends, device)
    for weights in (w, wt):
        ref, mags = R.mm(x, weights, ends)
        y = prime_moe.grouped_mm(x, weights, off)
        R.check(y, ref, mags, K)
        assert (y[ends[-1]:] == 0).all()
    ref, mags = R.wgrad(dy, x, ends)
    R.check(prime_moe.grouped_mm_wgrad(dy, x, off), ref, mags, 70)
    # a group of NaNs and infinities next to the others
    x[33:103] = nan
    x[40] = float("inf")
    w[1] = nan  # of an expert without rows
    y = prime_moe.grouped_mm(x, w, off)
    ref, mags = R.mm(x[:33], w, [33])
    R.check(y[:33], ref, mags, K)
    assert not torch.isfinite(y[33:103].float()).any()
    assert torch.isfinite(y[103:].float()).all()
    dw = prime_moe.grouped_mm_wgrad(dy, x, off)
    assert torch.isfinite(dw[[0, 1, 3]].float()).all() and not torch.isfinite(dw[2].float()).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients(device, dtype):
    """autograd against the formulas in 64 bits, for gradients of any strides, and against differences of the function."""
    import prime_moe
    gen = torch.Generator().manual_seed(6)
    N, K, counts, behind = 136, 328, [65, 0, 130, 1, 64], 9
    ends = np.cumsum(counts).tolist()
    M, E = ends[-1] + behind, len(counts)
    off = ends_tensor(ends, device)
    x = make((M, K), gen, dtype, device).requires_grad_()
    w = make((E, N, K), gen, dtype, device, K ** -0.5).requires_grad_()
    y = prime_moe.grouped_mm(x, w, off)
    full = make((M, N + 8), gen, dtype, device)
    grads = {"contiguous": make((M, N), gen, dtype, device), "rows apart": full[:, 8:], "odd": full[:, 3:-5],
             "across": make((N, M), gen, dtype, device).t(), "expanded": torch.ones((), dtype=dtype, device=device).expand(M, N)}
    for name, dy in grads.items():
        dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        ref, mags = R.mm(dy, w.detach().transpose(1, 2), ends)
        R.check(dx, ref, mags, N)
        assert (dx[ends[-1]:] == 0).all(), name
        ref, mags = R.wgrad(dy, x.detach(), ends)
        R.check(dw, ref, mags, max(counts))
    # one of the two only
    assert torch.equal(torch.autograd.grad(y, x, grads["contiguous"], retain_graph=True)[0],
                       prime_moe.grouped_mm(grads["contiguous"], w.detach().transpose(1, 2), off))
    # differences: the product is linear in either argument, so f(x + d) - f(x - d) = 2 df(d) up to the roundings of its outputs
    dy = grads["contiguous"]
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for arg, grad in ((x, dx), (w, dw)):
        d = torch.randn(arg.shape, generator=gen).sign().to(dtype).to(device) * 2.0 ** -4
        up, down = (arg.detach() + d), (arg.detach() - d)
        with torch.no_grad():
            f = [prime_moe.grouped_mm(a if arg is x else x, a if arg is w else w, off).double() for a in (up, down)]
        moved = (up.double() - down.double())
        have, want = ((f[0] - f[1]) * dy.double()).sum(), (moved * grad.double()).sum()
        half = torch.finfo(dtype).eps / 2
        sums = (max(K, N, M) + 2) * 2.0 ** -23
        mags = ((R.mm(x.detach(), w.detach(), ends)[1] + 1.0) * dy.double().abs()).sum()
        allowed = (half + sums) * (((f[0].abs() + f[1].abs()) * dy.double().abs()).sum() + (moved.abs() * grad.double().abs()).sum()) + sums * 4 * mags
        assert abs(float(have - want)) <= float(allowed)


def test_gradients_of_gradients(device):
    import prime_moe
    gen = torch.Generator().manual_seed(7)
    ends, N, K = [5, 5, 40], 24, 32
    off = ends_tensor(ends, device)
    x, w, dy = (make(s, gen, torch.float16, device, 0.5).requires_grad_() for s in ((43, K), (3, N, K), (43, N)))
    dx, dw = torch.autograd.grad(prime_moe.grouped_mm(x, w, off), (x, w), dy, create_graph=True)
    gx, gw = make((43, K), gen, torch.float16, device), make((3, N, K), gen, torch.float16, device)
    # <gx, dx> is bilinear in (dy, w), <gw, dw> in (dy, x)
    got = torch.autograd.grad((dx, dw), (dy, w, x), (gx, gw))
    a, am = R.mm(gx, w.detach(), ends)
    b, bm = R.mm(x.detach(), gw, ends)
    refs = [((a, am), (b, bm)), (R.wgrad(dy.detach(), gx, ends),), (R.mm(dy.detach(), gw.transpose(1, 2), ends),)]
    for g, parts in zip(got, refs):
        ref, mags = sum(p[0] for p in parts), sum(p[1] for p in parts)
        # each part is rounded to fp16 once, and so is their sum
        half = 2.0 ** -11
        bound = 64 * 2.0 ** -23 * mags + half * (sum(p[0].abs() for p in parts) + 2 * ref.abs()) * 1.01 + 2.0 ** -23
        assert ((g.double() - ref).abs() <= bound).all()


def test_gradients_of_shared_and_absent_operands(device):
    """One matrix for all experts (expanded), rows without an expert, no rows at all."""
    import prime_moe
    gen = torch.Generator().manual_seed(17)
    ends, N, K = [40, 40, 100], 40, 72
    off = ends_tensor(ends, device)
    w = make((N, K), gen, torch.bfloat16, device, 0.2).requires_grad_()
    x, dy = make((110, K), gen, torch.bfloat16, device).requires_grad_(), make((110, N), gen, torch.bfloat16, device)
    y = prime_moe.grouped_mm(x, w.expand(3, N, K), off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref, mags = R.mm(dy, w.detach().t().expand(3, K, N), ends)
    R.check(dx, ref, mags, N)
    parts, mags = R.wgrad(dy, x.detach(), ends)
    # each expert's part is rounded to bf16, then the sum of two (torch adds them in fp32 and rounds once)
    bound = 2.0 ** -8 * (parts.abs().sum(0) * 1.01 + parts.sum(0).abs()) + 100 * 2.0 ** -23 * mags.sum(0)
    assert ((dw.double() - parts.sum(0)).abs() <= bound * 1.01 + 1e-30).all()
    none = x.detach()[:0].requires_grad_()
    y = prime_moe.grouped_mm(none, w.expand(3, N, K), torch.zeros_like(off))
    dx, dw = torch.autograd.grad(y, (none, w), dy[:0])
    assert dx.shape == (0, K) and (dw == 0).all()
    with torch.no_grad():
        assert not prime_moe.grouped_mm(x, w.expand(3, N, K), off).requires_grad


def test_offsets_that_change_before_the_backward_pass_are_noticed(device):
    import prime_moe
    off = ends_tensor([3, 8], device)
    x, w = torch.ones((8, 16), dtype=torch.bfloat16, device=device, requires_grad=True), torch.ones((2, 8, 16), dtype=torch.bfloat16, device=device)
    y = prime_moe.grouped_mm(x, w, off)
    off[0] = 5
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_sums_are_held_in_32_bits(device, cus):
    """A long contraction of small terms onto a large one: sums in 16 bits would lose them."""
    import prime_moe
    K = 16384
    x = torch.full((3, K), 2.0 ** -7, dtype=torch.bfloat16, device=device)
    x[:, 0] = 256.0
    w = torch.ones((1, 8, K), dtype=torch.bfloat16, device=device)
    y = prime_moe.grouped_mm(x, w, ends_tensor([3], device))
    assert (y == 384.0).all()  # 256 + 16383 / 128 = 383.99
    dy = x[:1].t().contiguous().expand(K, 8).contiguous()
    dw = prime_moe.grouped_mm_wgrad(dy, torch.ones((K, 8), dtype=torch.bfloat16, device=device), ends_tensor([K], device))
    assert (dw == 384.0).all()


@pytest.mark.parametrize("what", ["x", "out", "dy"])
def test_beyond_32_bit_offsets(device, cus, what):
    """Operands and outputs above 4 GiB: rows near both ends."""
    import prime_moe
    gen = torch.Generator(device=device).manual_seed(8)
    M = (1 << 20) + 4133
    wide, narrow = 2304, 16
    K, N = (narrow, wide) if what == "out" else (wide, narrow)
    ends = [1, 700000, M - 3]
    off = ends_tensor(ends, device)
    big = torch.randn((M, wide), dtype=torch.bfloat16, device=device, generator=gen)
    assert big.numel() * 2 > 1 << 32
    small = torch.randn((M, narrow), dtype=torch.bfloat16, device=device, generator=gen)
    at = torch.tensor([0, 1, 2, 699999, 700000, 700001, M - 5, M - 4, M - 3, M - 1], device=device)
    if what == "dy":
        got = prime_moe.grouped_mm_wgrad(big, small, off)
        for g, (a, b) in enumerate(zip([0] + ends[:-1], ends)):
            ref = torch.zeros((wide, narrow), dtype=torch.float64, device=device)
            mags = torch.zeros_like(ref)
            for r in range(a, b, 1 << 16):
                p, q = big[r:min(b, r + (1 << 16))].double(), small[r:min(b, r + (1 << 16))].double()
                ref += p.t() @ q
                mags += p.abs().t() @ q.abs()
            # (partial sums of random signs: far below the sum of magnitudes that the plain bound would multiply by the depth)
            assert ((got[g].double() - ref).abs() <= 2.0 ** -8 * ref.abs() * 1.01 + 2.0 ** -23 * mags + 1e-6).all()
        return
    w = torch.randn((3, N, K), dtype=torch.bfloat16, device=device, generator=gen)
    x = small if what == "out" else big
    y = prime_moe.grouped_mm(x, w, off)
    group = torch.bucketize(at, torch.tensor(ends, device=device), right=True)
    for r, g in zip(at.tolist(), group.tolist()):
        ref, mags = R.mm(x[r:r + 1], w[min(g, 2)][None], [1 if g < 3 else 0])
        R.check(y[r:r + 1], ref, mags, K)


def test_offsets_out_of_order_do_no_harm(device, cus):
    """Offsets that are not ends of groups: every access stays inside the arguments (rows come out as something)."""
    import prime_moe
    gen = torch.Generator().manual_seed(9)
    x, w = make((100, 64), gen, torch.bfloat16, device), make((4, 40, 64), gen, torch.bfloat16, device)
    for bad in ([50, 20, 120, 90], [-7, -1, 1 << 30, 3], [200, 200, 200, 200], [2 ** 31 - 1, -(2 ** 31), 0, 60]):
        y = prime_moe.grouped_mm(x, w, ends_tensor(bad, device))
        dw = prime_moe.grouped_mm_wgrad(make((100, 40), gen, torch.bfloat16, device), x, ends_tensor(bad, device))
        torch.cuda.synchronize()
        assert y.shape == (100, 40) and dw.shape == (4, 40, 64)


def test_same_bits_again_and_on_poisoned_lds(device, cus):
    import prime_moe
    from prime_moe import _native
    gen = torch.Generator().manual_seed(10)
    ends = R.sized(1500, 9, gen)
    x, w = make((1511, 264), gen, torch.bfloat16, device), make((9, 328, 264), gen, torch.bfloat16, device)
    dy, off = make((1511, 328), gen, torch.bfloat16, device), ends_tensor(ends, device)
    word = torch.zeros((1,), dtype=torch.int32, device=device)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    calls = [lambda: prime_moe.grouped_mm(x, w, off), lambda: prime_moe.grouped_mm(x, wt, off), lambda: prime_moe.grouped_mm_wgrad(dy, x, off),
             lambda: prime_moe.grouped_mm(x[:29], w[:1], off[:1].clamp(max=20))]
    for call in calls:
        first = call()
        _native.check(_native.load().pmoe_poison_lds(word.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(call(), first)


def test_captured_training_step(device):
    """Forward and both gradients in one graph: replays on new inputs, between eager work on the same tensors."""
    import prime_moe
    gen = torch.Generator().manual_seed(11)
    E, N, K, M = 6, 200, 264, 600
    w = make((E, N, K), gen, torch.bfloat16, device, 0.1).requires_grad_()
    x = make((M, K), gen, torch.bfloat16, device).requires_grad_()
    dy, off = make((M, N), gen, torch.bfloat16, device), ends_tensor(R.sized(M - 10, E, gen), device)

    def step():
        y = prime_moe.grouped_mm(x, w, off)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(make((M, K), gen, torch.bfloat16, device))
            dy.copy_(make((M, N), gen, torch.bfloat16, device))
            off.copy_(ends_tensor(R.sized(M - 10 - i, E, gen), device))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_two_streams_at_once(device, cus):
    import prime_moe
    gen = torch.Generator().manual_seed(12)
    ends = R.sized(3000, 5, gen)
    off, w = ends_tensor(ends, device), make((5, 512, 512), gen, torch.bfloat16, device, 0.05)
    xs = [make((3000, 512), gen, torch.bfloat16, device) for _ in range(2)]
    want = [prime_moe.grouped_mm(x, w, off) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(prime_moe.grouped_mm(xs[i], w, off))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_backward_of_another_stream(device):
    import prime_moe
    gen = torch.Generator().manual_seed(21)
    ends = R.sized(900, 4, gen)
    off = ends_tensor(ends, device)
    x, w = make((900, 256), gen, torch.bfloat16, device), make((4, 128, 256), gen, torch.bfloat16, device, 0.05)
    g = make((900, 128), gen, torch.bfloat16, device)
    want = (prime_moe.grouped_mm(g, w.transpose(1, 2), off), prime_moe.grouped_mm_wgrad(g, x, off))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = prime_moe.grouped_mm(a, b, off)
    torch.cuda.current_stream().wait_stream(side)
    got = torch.autograd.grad(y, (a, b), g)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_traced_training_step(device):
    import prime_moe
    gen = torch.Generator().manual_seed(22)
    ends = R.sized(300, 4, gen)
    off = ends_tensor(ends, device)
    x = make((300, 256), gen, torch.bfloat16, device).requires_grad_()
    w = make((4, 128, 256), gen, torch.bfloat16, device, 0.05).requires_grad_()
    g = make((300, 128), gen, torch.bfloat16, device)

    def step(x, w, off):
        return prime_moe.grouped_mm(x, w, off)

    want = torch.autograd.grad(step(x, w, off), (x, w), g)
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(x, w, off), (x, w), g)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_registration(device):
    """Schemas, fake implementations and autograd registration as torch checks them, and one compiled call."""
    import prime_moe
    gen = torch.Generator().manual_seed(13)
    off = ends_tensor([3, 3, 17], device)
    x, w = make((20, 64), gen, torch.bfloat16, device).requires_grad_(), make((3, 40, 64), gen, torch.bfloat16, device).requires_grad_()
    dy = make((20, 40), gen, torch.bfloat16, device)
    q, s = prime_moe.quantize_int8(x.detach())
    qw, sw = prime_moe.quantize_int8(w.detach())
    ids, total = torch.zeros((20,), dtype=torch.int32, device=device), torch.tensor([18], dtype=torch.int32, device=device)
    ops = torch.ops.prime_moe
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.grouped_mm.default, (x, w, off), test_utils=tests + ("test_autograd_registration",))
    torch.library.opcheck(ops.grouped_mm_wgrad.default, (dy, x.detach(), off), test_utils=tests)
    torch.library.opcheck(ops.grouped_mm_int8.default, (q, qw, s, sw, off, torch.float16), test_utils=tests)
    torch.library.opcheck(ops.quantize_int8.default, (x.detach(),), test_utils=tests)
    torch.library.opcheck(ops.expert_offsets.default, (ids, total, 3), test_utils=tests)
    fn = torch.compile(lambda a, b: prime_moe.grouped_mm(a, b, off), backend="eager", fullgraph=True)
    assert torch.equal(fn(x.detach(), w.detach()), prime_moe.grouped_mm(x.detach(), w.detach(), off))


@pytest.mark.parametrize("E,n", [(1, 1), (8, 0), (8, 5), (8, 4096), (257, 65536), (1024, 3000)])
def test_expert_offsets(device, E, n):
    import prime_moe
    gen = torch.Generator().manual_seed(E + n)
    ids = torch.randint(-1, E + 1, (n,), generator=gen, dtype=torch.int32).to(device)  # some of no expert
    if n:
        order, experts, total = torch.ops.prime_moe.moe_align(ids, E, 1, 1)
        assert order.numel() == n
    else:  # (moe_align takes no empty list)
        experts, total = ids, torch.zeros((1,), dtype=torch.int32, device=device)
    got = prime_moe.expert_offsets(experts, total, E)
    want = torch.cumsum(torch.bincount(ids[(ids >= 0) & (ids < E)].long(), minlength=E), 0)
    assert got.dtype == torch.int32 and torch.equal(got.long(), want)
    # ids that are not sorted, or a count beyond the schedule: nothing outside the arguments is touched
    prime_moe.expert_offsets(ids, torch.tensor([n + 100], dtype=torch.int32, device=device), E)
    prime_moe.expert_offsets(ids, torch.tensor([-5], dtype=torch.int32, device=device), E)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------- a layer of them

def swiglu(h):
    gate, up = h.float().chunk(2, -1)
    return (torch.nn.functional.silu(gate) * up).to(h.dtype)


def layer(prime_moe, x, w1, w2, logits, top_k):
    """An MoE layer out of the ragged products, as a program that trains would write it."""
    E = w1.shape[0]
    ids, weights, order, experts, total = prime_moe.route(logits, top_k, block_m=1)
    offsets = prime_moe.expert_offsets(experts, total, E)
    order = order.long()
    token = order // top_k
    h = prime_moe.grouped_mm(x[token], w1, offsets)
    y = prime_moe.grouped_mm(swiglu(h), w2, offsets)
    return torch.zeros(x.shape, device=x.device).index_add(0, token, y.float() * weights.view(-1)[order][:, None])


def layer64(x, w1, w2, ids, weights):
    out = torch.zeros_like(x)
    for e in range(w1.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        gate, up = (x[t] @ w1[e].t()).chunk(2, -1)
        out = out.index_add(0, t, ((torch.nn.functional.silu(gate) * up) @ w2[e].t()) * weights[t, j][:, None])
    return out


def test_layer_and_its_gradients(device):
    import prime_moe
    gen = torch.Generator().manual_seed(14)
    T, K, E, N, top_k = 150, 256, 8, 512, 2
    x = make((T, K), gen, torch.bfloat16, device).requires_grad_()
    w1 = make((E, N, K), gen, torch.bfloat16, device, K ** -0.5).requires_grad_()
    w2 = make((E, K, N // 2), gen, torch.bfloat16, device, (N // 2) ** -0.5).requires_grad_()
    logits = torch.randn((T, E), generator=gen).to(device)
    out = layer(prime_moe, x, w1, w2, logits, top_k)
    g = torch.randn((T, K), generator=gen).to(device)
    grads = torch.autograd.grad(out, (x, w1, w2), g)
    ids, weights, *schedule = prime_moe.route(logits, top_k)
    args = [t.detach().double().requires_grad_() for t in (x, w1, w2)]
    ref = layer64(*args, ids.long(), weights.double())
    refs = torch.autograd.grad(ref, args, g.double())
    # a value passes at most five roundings to bf16 (2^-8 each) on its way to a gradient; their errors are independent, and
    # in the 2-norm they do not add up to more than their sum
    for got, want in zip((out.detach(), *grads), (ref.detach(), *refs)):
        assert float((got.double() - want).norm() / want.norm()) < 5 * 2.0 ** -8
    fused = torch.empty((T, K), dtype=torch.bfloat16, device=device)
    prime_moe.fused_moe_bf16(x.detach(), w1.detach(), w2.detach(), *schedule, weights, fused, top_k, 128, 64, 4, 2)
    assert float((out.detach().double() - fused.double()).norm() / fused.double().norm()) < 5 * 2.0 ** -8


def test_layer_in_int8(device):
    """quantise -> up -> SwiGLU -> quantise -> down, every step against 64 bits on the values that it was given."""
    import prime_moe
    gen = torch.Generator().manual_seed(15)
    T, K, E, N, top_k = 130, 512, 8, 768, 4
    x = make((T, K), gen, torch.bfloat16, device)
    q1, s1 = prime_moe.quantize_int8(make((E, N, K), gen, torch.bfloat16, device, K ** -0.5))
    q2, s2 = prime_moe.quantize_int8(make((E, K, N // 2), gen, torch.bfloat16, device, (N // 2) ** -0.5))
    ids, weights, order, experts, total = prime_moe.route(torch.randn((T, E), generator=gen).to(device), top_k, block_m=1)
    off = prime_moe.expert_offsets(experts, total, E)
    ends = off.tolist()
    xq, xs = prime_moe.quantize_int8(x)
    token = order.long() // top_k
    xq, xs = xq[token], xs[token]
    h = prime_moe.grouped_mm_int8(xq, q1, xs, s1, off)
    ref = R.mm_int8(xq, q1, xs, s1, ends)
    assert ((h.double() - ref).abs() <= 2.0 ** -8 * 1.001 * ref.abs()).all()
    a = swiglu(h)
    aq, as_ = prime_moe.quantize_int8(a)
    assert ((aq.double() * as_.double()[:, None] - a.double()).abs() <= 0.5001 * as_.double()[:, None]).all()
    y = prime_moe.grouped_mm_int8(aq, q2, as_, s2, off, torch.float32)
    ref = R.mm_int8(aq, q2, as_, s2, ends)
    assert ((y.double() - ref).abs() <= 2.0 ** -22 * ref.abs()).all()
