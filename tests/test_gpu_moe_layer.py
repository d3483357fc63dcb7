"""The whole layer for a few tokens on the GPU, with weights of 16 and of 4 bits, against its definition in 64 bits."""
import pytest
import torch

import int4_ref as R
from layer_ref import Layer, select

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def inputs(T, K, H, E, dtype, device, seed, bias=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((T, K), generator=gen).to(dtype).to(device)
    gate = (torch.randn((E, K), generator=gen) * K ** -0.5).to(dtype).to(device)
    b = (torch.randn((E,), generator=gen) * 0.5).to(device) if bias else None
    return gen, x, gate, b


def wide(gen, H, K, E, dtype, device):
    w1 = (torch.randn((E, 2 * H, K), generator=gen) * K ** -0.5).to(dtype).to(device)
    w2 = (torch.randn((E, K, H), generator=gen) * H ** -0.5).to(dtype).to(device)
    return w1, w2


def narrow(gen, H, K, E, dtype, group, device):
    out = []
    for n, k in ((2 * H, K), (K, H)):
        values = torch.randint(-8, 8, (E, n, k), generator=gen, dtype=torch.int8)
        scale = ((torch.rand((E, n, k // group), generator=gen) + 0.5) * 0.2 * k ** -0.5).to(dtype)
        out.append((values.to(device), scale.to(device)))
    return out


def layer_of_4_bits(x, gate, packed, top_k, bias, group, K, H):
    (v1, s1), (v2, s2) = packed
    ones = lambda v, s: 55 * R.weights(torch.ones_like(v), s).abs()
    return Layer(x, gate, R.weights(v1, s1), R.weights(v2, s2), top_k, bias, ones(v1, s1), ones(v2, s2), 2 * group + K / group + 30, 2 * group + H / group + 30)


SHAPES = [  # K, H, E, top_k
    (8, 8, 1, 1),
    (128, 128, 4, 2),
    (136, 72, 5, 3),      # contractions that end inside a step, columns inside a job
    (1000, 24, 3, 1),
    (2048, 768, 128, 8),
    (512, 40, 512, 32),   # every limit of the routing
    (4096, 256, 8, 4),
]


@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 9, 16])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("K,H,E,top_k", SHAPES)
def test_layer(device, K, H, E, top_k, dtype, T):
    import prime_moe
    gen, x, gate, bias = inputs(T, K, H, E, dtype, device, K + T, bias=T % 2 == 0)
    w1, w2 = wide(gen, H, K, E, dtype, device)
    out, ids, weights = prime_moe.moe_layer(x, gate, w1, w2, top_k, bias)
    assert out.shape == x.shape and out.dtype == dtype and ids.dtype == torch.int32 and weights.dtype == torch.float32
    Layer(x, gate, w1, w2, top_k, bias).check(out, ids, weights)


@pytest.mark.parametrize("T", [1, 2, 7, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("K,H,E,top_k", [(128, 128, 1, 1), (384, 256, 6, 3), (2048, 768, 32, 8), (4096, 128, 37, 9), (256, 128, 512, 32)])
def test_layer_int4(device, K, H, E, top_k, dtype, group, T):
    import prime_moe
    gen, x, gate, bias = inputs(T, K, H, E, dtype, device, K + T + group, bias=T % 2 == 1)
    packed = narrow(gen, H, K, E, dtype, group, device)
    q = [prime_moe.pack_int4(*p) for p in packed]
    out, ids, weights = prime_moe.moe_layer_int4(x, gate, *q[0], *q[1], top_k, bias)
    layer_of_4_bits(x, gate, packed, top_k, bias, group, K, H).check(out, ids, weights)


@pytest.mark.parametrize("K,H,group", [(32, 32, 32), (160, 96, 32), (192, 64, 64), (64, 320, 64)])
def test_layer_int4_with_tiles_that_end_early(device, K, H, group):
    import prime_moe
    for T in (1, 5, 16):
        gen, x, gate, bias = inputs(T, K, H, 3, BF16, device, K + T)
        packed = narrow(gen, H, K, 3, BF16, group, device)
        q = [prime_moe.pack_int4(*p) for p in packed]
        got = prime_moe.moe_layer_int4(x, gate, *q[0], *q[1], 2, bias)
        layer_of_4_bits(x, gate, packed, 2, bias, group, K, H).check(*got)


@pytest.mark.parametrize("kind", ["wide", "narrow"])
@pytest.mark.parametrize("T,E,top_k", [(16, 8, 1), (16, 4, 4), (13, 2, 1), (9, 300, 1), (16, 32, 32)])
def test_how_tokens_meet_experts(device, T, E, top_k, kind):
    """Everybody on one expert (up to 16 rows), on all of them, every token on its own."""
    import prime_moe
    K, H = 256, 128
    gen, x, gate, _ = inputs(T, K, H, E, BF16, device, T + E, bias=False)
    for bias in (None, torch.where(torch.arange(E) == E // 2, 50.0, 0.0).to(device)):
        if kind == "wide":
            w1, w2 = wide(gen, H, K, E, BF16, device)
            got = prime_moe.moe_layer(x, gate, w1, w2, top_k, bias)
            Layer(x, gate, w1, w2, top_k, bias).check(*got)
        else:
            packed = narrow(gen, H, K, E, BF16, 64, device)
            q = [prime_moe.pack_int4(*p) for p in packed]
            got = prime_moe.moe_layer_int4(x, gate, *q[0], *q[1], top_k, bias)
            layer_of_4_bits(x, gate, packed, top_k, bias, 64, K, H).check(*got)
        if bias is not None:
            assert (got[1][:, 0] == E // 2).all()


def test_ties_go_to_the_lower_expert(device):
    """Integers: every logit is exact, and most are equal."""
    import prime_moe
    gen = torch.Generator().manual_seed(1)
    T, K, H, E = 16, 64, 16, 64
    x = torch.randint(-1, 2, (T, K), generator=gen).to(BF16).to(device)
    gate = torch.randint(-1, 2, (E, K), generator=gen).to(BF16).to(device)
    w1, w2 = wide(gen, H, K, E, BF16, device)
    for top_k in (1, 7, 32):
        _, ids, weights = prime_moe.moe_layer(x, gate, w1, w2, top_k)
        scores = x.double() @ gate.double().t()
        assert torch.equal(ids.long(), select(scores, top_k))
        assert torch.allclose(weights.double(), torch.softmax(scores.gather(-1, ids.long()), -1), rtol=1e-5, atol=0)
    x.zero_()
    out, ids, weights = prime_moe.moe_layer(x, gate, w1, w2, 5)
    assert (ids == torch.arange(5, device=device)).all() and (weights == 0.2).all() and (out == 0).all()


def test_agrees_with_route_and_the_fused_layer(device):
    """The path that takes any number of tokens: the same experts, outputs as far apart as its two roundings (activation, pairs)."""
    import prime_moe
    T, K, H, E, top_k = 6, 1024, 256, 16, 4
    gen, x, gate, bias = inputs(T, K, H, E, BF16, device, 77)
    w1, w2 = wide(gen, H, K, E, BF16, device)
    out, ids, weights = prime_moe.moe_layer(x, gate, w1, w2, top_k, bias)
    rids, rweights, s, e, n = prime_moe.route(x.float() @ gate.float().t(), top_k, bias=bias)
    assert torch.equal(ids, rids) and torch.allclose(weights, rweights, rtol=1e-4, atol=1e-6)
    other = prime_moe.fused_moe_bf16(x, w1, w2, s, e, n, rweights, torch.empty_like(x), top_k, 128, 64, 4, 2)
    assert ((out.double() - other.double()).abs() <= 2e-2 * other.double().abs().clamp_min(1.0)).all()


@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_a_token_that_is_not_finite_stays_alone(device, kind):
    import prime_moe
    T, K, H, E, top_k = 7, 256, 128, 8, 2
    gen, x, gate, bias = inputs(T, K, H, E, BF16, device, 5)
    w = wide(gen, H, K, E, BF16, device) if kind == "wide" else [t for p in narrow(gen, H, K, E, BF16, 32, device) for t in prime_moe.pack_int4(*p)]
    run = lambda: (prime_moe.moe_layer if kind == "wide" else prime_moe.moe_layer_int4)(x, gate, *w, top_k, bias)
    want = run()
    x[2, 9], x[5, 200] = float("nan"), float("inf")
    got = run()
    rest = [0, 1, 3, 4, 6]
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, want))
    assert torch.isnan(got[0][2]).all() and not torch.isfinite(got[0][5]).any()


def test_an_expert_that_nobody_takes_is_not_read(device):
    import prime_moe
    T, K, H, E = 4, 128, 64, 8
    gen, x, gate, _ = inputs(T, K, H, E, BF16, device, 6)
    w1, w2 = wide(gen, H, K, E, BF16, device)
    bias = torch.tensor([0, 0, -1e9, 0, 0, -float("inf"), 0, 0], device=device)
    want = prime_moe.moe_layer(x, gate, w1, w2, 2, bias)
    w1[[2, 5]], w2[[2, 5]] = float("nan"), float("nan")
    got = prime_moe.moe_layer(x, gate, w1, w2, 2, bias)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.isfinite(got[0]).all()


def test_the_last_bit_of_the_activation_counts(device):
    """One rounding: outputs are within what the rounding of `out` and fp32 sums leave, 1.02 half steps, in all but a few of a million
    (an activation rounded to bfloat16 would leave as much again)."""
    import prime_moe
    T, K, H, E = 16, 2048, 512, 4
    gen, x, gate, _ = inputs(T, K, H, E, BF16, device, 7, bias=False)
    w1, w2 = wide(gen, H, K, E, BF16, device)
    out, ids, weights = prime_moe.moe_layer(x, gate, w1, w2, 2)
    ref = Layer(x, gate, w1, w2, 2, None).check(out, ids, weights)
    # half a step of every value's binade, and 2^-14 of the row's size for the sums
    step = 2.0 ** (torch.floor(torch.log2(ref.abs())) - 8)
    over = (out.double() - ref).abs() > step + 2.0 ** -14 * ref.abs().amax(-1, keepdim=True)
    assert int(over.sum()) == 0


@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_graphs_streams_and_the_same_bits(device, kind):
    import prime_moe
    T, K, H, E, top_k = 5, 1024, 384, 16, 4
    gen, x, gate, bias = inputs(T, K, H, E, BF16, device, 8)
    w = wide(gen, H, K, E, BF16, device) if kind == "wide" else [t for p in narrow(gen, H, K, E, BF16, 64, device) for t in prime_moe.pack_int4(*p)]
    y = torch.randn((T, K), generator=gen).to(BF16).to(device)
    run = lambda v: (prime_moe.moe_layer if kind == "wide" else prime_moe.moe_layer_int4)(v, gate, *w, top_k, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    pool = torch.cuda.graph_pool_handle()
    for g, v in zip(graphs, (x, y)):  # two graphs that share their memory: replayed one behind the other
        with torch.cuda.graph(g, pool=pool):
            got.append(run(v)[0].clone())
    for turn in range(3):
        x.copy_(torch.randn((T, K), generator=gen).to(BF16))
        for g, o, v in zip(graphs, got, (x, y)):
            want = run(v)[0]
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)
    # several calls in flight on several streams
    want = [run(v) for v in (x, y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    many = []
    for turn in range(12):
        with torch.cuda.stream(streams[turn % 3]):
            many.append((turn % 2, run((x, y)[turn % 2])))
    torch.cuda.synchronize()
    for i, r in many:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_decoding_as_it_is_used(device):
    """A layer quantised once, decoded with token by token and in a batch: the batch's rows are the tokens' own results."""
    import prime_moe
    T, K, H, E, top_k = 9, 512, 256, 16, 4
    gen, x, gate, bias = inputs(T, K, H, E, F16, device, 12)
    w1, w2 = wide(gen, H, K, E, F16, device)
    q1, q2 = prime_moe.quantize_int4(w1, 32), prime_moe.quantize_int4(w2, 32)
    packed = [R.quantize(w1, 32, F16), R.quantize(w2, 32, F16)]
    batch = prime_moe.moe_layer_int4(x, gate, *q1, *q2, top_k, bias)
    layer_of_4_bits(x, gate, packed, top_k, bias, 32, K, H).check(*batch)
    for t in range(T):
        one = prime_moe.moe_layer_int4(x[t:t + 1], gate, *q1, *q2, top_k, bias)
        assert torch.equal(one[1][0], batch[1][t])
        layer_of_4_bits(x[t:t + 1], gate, packed, top_k, bias, 32, K, H).check(*one)
    assert prime_moe.moe_layer(x[:0], gate, w1, w2, top_k)[0].shape == (0, K)


@pytest.fixture(params=[1, 7, 0])
def compute_units(request):
    """Grids of two workgroups, of 14, and of the whole card."""
    from prime_moe import _native
    _native.load().pmoe_set_compute_units(request.param)
    yield request.param
    _native.load().pmoe_set_compute_units(0)


@pytest.mark.parametrize("kind", ["wide", "narrow"])
@pytest.mark.parametrize("T", [1, 6, 16])
def test_workgroups_that_have_many_jobs(device, compute_units, kind, T):
    import prime_moe
    K, H, E, top_k = (264, 72, 6, 3) if kind == "wide" else (352, 160, 6, 3)
    gen, x, gate, bias = inputs(T, K, H, E, BF16, device, 40 + T)
    if kind == "wide":
        w1, w2 = wide(gen, H, K, E, BF16, device)
        Layer(x, gate, w1, w2, top_k, bias).check(*prime_moe.moe_layer(x, gate, w1, w2, top_k, bias))
    else:
        packed = narrow(gen, H, K, E, BF16, 32, device)
        q = [prime_moe.pack_int4(*p) for p in packed]
        layer_of_4_bits(x, gate, packed, top_k, bias, 32, K, H).check(*prime_moe.moe_layer_int4(x, gate, *q[0], *q[1], top_k, bias))


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_workgroups_that_share_columns_of_the_output(device, compute_units, kind, T):
    """More than 128 MB of touched weights, strips and experts in numbers that no grid divides; twice, for the same bits."""
    import prime_moe
    dtype = F16 if kind == "wide" else BF16
    K, H, E, top_k = (2056, 2728, 6, 6) if kind == "wide" else (4128, 2080, 11, 11)
    _, x, gate, bias = inputs(T, K, H, E, dtype, device, 50 + T)
    gen = torch.Generator(device=device).manual_seed(T)
    rand = lambda *s, **k: torch.randn(s, generator=gen, device=device, dtype=torch.float32)
    if kind == "wide":
        w1, w2 = (rand(E, 2 * H, K) * K ** -0.5).to(dtype), (rand(E, K, H) * H ** -0.5).to(dtype)
        assert E * 3 * K * H * 2 > 128 << 20
        run = lambda: prime_moe.moe_layer(x, gate, w1, w2, top_k, bias)
        ref = Layer(x, gate, w1, w2, top_k, bias)
    else:
        packed = [(torch.randint(-8, 8, (E, n, k), generator=gen, device=device, dtype=torch.int8), ((rand(E, n, k // 32).abs() + 0.5) * 0.1 * k ** -0.5).to(dtype))
                  for n, k in ((2 * H, K), (K, H))]
        assert E * 3 * K * H // 2 > 128 << 20
        q = [prime_moe.pack_int4(*p) for p in packed]
        run = lambda: prime_moe.moe_layer_int4(x, gate, *q[0], *q[1], top_k, bias)
        ref = layer_of_4_bits(x, gate, packed, top_k, bias, 32, K, H)
    first = run()
    ref.check(*first)
    for a, b in zip(first, run()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_experts_behind_4_gb(device, kind):
    import prime_moe
    T, top_k = 3, 2
    K, H, E = (4096, 2048, 140) if kind == "wide" else (4096, 4096, 260)
    gen, x, gate, bias = inputs(T, K, H, E, BF16, device, 70)
    bias[:-2] -= 1e4  # the last two experts are everybody's
    def all_experts(two):
        whole = torch.zeros((E, *two.shape[1:]), dtype=two.dtype, device=device)
        whole[-2:] = two
        return whole
    if kind == "wide":
        w1, w2 = wide(gen, H, K, 2, BF16, device)
        whole = [all_experts(t) for t in (w1, w2)]
        ref = Layer(x, gate[-2:], w1, w2, top_k, bias[-2:])
        out, ids, weights = prime_moe.moe_layer(x, gate, *whole, top_k, bias)
    else:
        packed = narrow(gen, H, K, 2, BF16, 128, device)
        whole = [all_experts(t) for p in packed for t in prime_moe.pack_int4(*p)]
        ref = layer_of_4_bits(x, gate[-2:], packed, top_k, bias[-2:], 128, K, H)
        out, ids, weights = prime_moe.moe_layer_int4(x, gate, *whole, top_k, bias)
    assert whole[0].numel() * whole[0].element_size() > 1 << 32
    ref.check(out, ids - (E - 2), weights)


@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_calls_of_several_threads(device, kind):
    """Calls of several host threads on streams of their own, each with rows of a longer batch."""
    import threading

    import prime_moe
    K, H, E, top_k = 512, 256, 16, 4
    gen, x, gate, bias = inputs(12, K, H, E, F16, device, 71)
    w = wide(gen, H, K, E, F16, device) if kind == "wide" else [t for p in narrow(gen, H, K, E, F16, 32, device) for t in prime_moe.pack_int4(*p)]
    run = lambda v: (prime_moe.moe_layer if kind == "wide" else prime_moe.moe_layer_int4)(v, gate, *w, top_k, bias)
    want = [run(x[4 * i:4 * i + 4]) for i in range(3)]
    torch.cuda.synchronize()
    got = [[] for _ in range(3)]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(run(x[4 * i:4 * i + 4]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(3):
        assert len(got[i]) == 20
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
