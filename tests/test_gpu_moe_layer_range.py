"""The whole layer for a few tokens where its activation leaves the sizes of a 16-bit type, against its definition in 64 bits."""
import pytest
import torch

import int4_ref as R
from layer_ref import ULP

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def check(got, x, w1, w2, bias, step, mag1=None, mag2=None, depth1=None, depth2=None):
    """A layer whose gate is zero and whose experts are everybody's.  `step`: what the activation is off by relative to itself: nothing as
    fp32; as the sum of two bf16 numbers, the second of which is below 2^-8 of the value's binade and rounded by half of its last
    place, 2^-17.  Everything else as in layer_ref.Layer: sums of `depth` additions in fp32 of magnitudes `mag`; |silu'| <= 1.1, |silu(g)| <= |g|;
    exponential, reciprocal and two products 2^-18 (1 + |g|) of the value; one rounding at the end."""
    out, ids, weights = got
    E, K, H = w2.shape
    order = torch.argsort(bias, descending=True)
    share = torch.softmax(bias.double()[order], 0)
    assert (ids == order).all() and ((weights.double() - share).abs() <= 2.0 ** -18).all()
    mag1, mag2 = w1.abs() if mag1 is None else mag1, w2.abs() if mag2 is None else mag2
    depth1, depth2 = depth1 or K / 16 + 30, depth2 or H / 8 + 30
    x = x.double()
    ref, bound = torch.zeros_like(x), torch.zeros_like(x)
    for e, a in zip(order.tolist(), share.tolist()):
        (g, u), (dg, du) = (t.chunk(2, -1) for t in (x @ w1[e].double().t(), depth1 * ULP * (x.abs() @ mag1[e].double().t())))
        act = g * torch.sigmoid(g) * u
        bent = 1.1 * u.abs() * dg + g.abs() * du + 1.1 * dg * du
        bent = bent + (2.0 ** -18 * (1 + g.abs()) + step) * (act.abs() + bent)
        y = act @ w2[e].double().t()
        dy = bent @ w2[e].double().abs().t() + depth2 * ULP * ((act.abs() + bent) @ mag2[e].double().t())
        ref += a * y
        bound += a * dy + 2.0 ** -18 * (y.abs() + dy) + 40 * ULP * a * y.abs()
    info = torch.finfo(out.dtype)
    bound = bound + info.eps / 2 * (ref.abs() + bound) + info.smallest_normal * info.eps / 2
    assert torch.isfinite(out).all()
    bad = (out.double() - ref).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((out.double() - ref).abs() / bound).max()))
    return act, ref


# of the gate rows, the up rows and the down projection: activations of a few 10^5, of 10^-6 and (bf16) of 10^36
SIZES = {"large": (1.0, 2.0 ** 16, 2.0 ** -10), "small": (2.0 ** -10, 2.0 ** -10, 2.0 ** 11), "largest": (1.0, 2.0 ** 119, 2.0 ** -119)}


@pytest.mark.parametrize("T", [1, 2, 3, 5, 9, 16])
@pytest.mark.parametrize("K,H", [(256, 128), (136, 72), (1000, 24), (2048, 768)])
@pytest.mark.parametrize("dtype,size", [(F16, "large"), (F16, "small"), (BF16, "large"), (BF16, "small"), (BF16, "largest")])
def test_activations_of_every_size(device, dtype, size, K, H, T):
    import prime_moe
    gate_size, up_size, down_size = SIZES[size]
    E = 3
    gen = torch.Generator().manual_seed(K + T)
    x = torch.randn((T, K), generator=gen).to(dtype).to(device)
    w1 = torch.randn((E, 2 * H, K), generator=gen) * K ** -0.5
    w1[:, :H] *= gate_size
    w1[:, H:] *= up_size
    w2 = torch.randn((E, K, H), generator=gen) * H ** -0.5 * down_size
    w1, w2 = w1.to(dtype).to(device), w2.to(dtype).to(device)
    bias = torch.tensor([0.25, 0.5, 0.0], device=device)
    got = prime_moe.moe_layer(x, torch.zeros((E, K), dtype=dtype, device=device), w1, w2, E, bias)
    act, ref = check(got, x, w1, w2, bias, 0.0 if dtype == F16 else 2.0 ** -17)
    most = act.abs().amax()
    assert {"large": most > 65504, "small": most < 2.0 ** -12, "largest": most > 1e35}[size] and ref.abs().amax() > 2.0 ** -12


@pytest.mark.parametrize("T", [1, 2, 5, 9, 16])
@pytest.mark.parametrize("K,H,group", [(256, 128, 128), (160, 96, 32), (192, 320, 64)])
@pytest.mark.parametrize("dtype,size", [(F16, "large"), (F16, "small"), (BF16, "large"), (BF16, "small")])
def test_activations_of_every_size_with_4_bits(device, dtype, size, K, H, group, T):
    import prime_moe
    gate_size, up_size, down_size = SIZES[size]
    E = 3
    gen = torch.Generator().manual_seed(K + T + group)
    x = torch.randn((T, K), generator=gen).to(dtype).to(device)
    weights = []
    for n, k, sizes in ((2 * H, K, (gate_size, up_size)), (K, H, (down_size, down_size))):
        values = torch.randint(-8, 8, (E, n, k), generator=gen, dtype=torch.int8)
        scale = (torch.rand((E, n, k // group), generator=gen) + 0.5) * 0.2 * k ** -0.5
        scale[:, :n // 2] *= sizes[0]
        scale[:, n // 2:] *= sizes[1]
        weights.append((values.to(device), scale.to(dtype).to(device)))
    bias = torch.tensor([0.25, 0.5, 0.0], device=device)
    packed = [t for w in weights for t in prime_moe.pack_int4(*w)]
    got = prime_moe.moe_layer_int4(x, torch.zeros((E, K), dtype=dtype, device=device), *packed, E, bias)
    ones = lambda v, s: 55 * R.weights(torch.ones_like(v), s).abs()  # (int4_ref.sums_bound)
    act, ref = check(got, x, R.weights(*weights[0]), R.weights(*weights[1]), bias, 2.0 ** -17, ones(*weights[0]), ones(*weights[1]),
                     2 * group + K / group + 30, 2 * group + H / group + 30)
    most = act.abs().amax()
    assert (most > 65504 if size == "large" else most < 2.0 ** -12) and ref.abs().amax() > 2.0 ** -12


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_small_activations_count_in_every_place(device, dtype):
    """One column of the activation at a time, at a size that has no second number in fp16: each reaches the outputs that its weights
    say, and by as much as they say."""
    import prime_moe
    K, H = 136, 40
    x = torch.zeros((1, K), dtype=dtype, device=device)
    x[0, 0] = 2.0 ** -9
    gate, bias = torch.zeros((1, K), dtype=dtype, device=device), torch.zeros(1, device=device)
    gen = torch.Generator().manual_seed(4)
    w2 = (torch.randn((1, K, H), generator=gen) * 1024).to(dtype).to(device)
    for column in range(H):
        w1 = torch.zeros((1, 2 * H, K), dtype=dtype, device=device)
        w1[0, column, 0], w1[0, H + column, 0] = 1.0, 1.3
        check(prime_moe.moe_layer(x, gate, w1, w2, 1, bias), x, w1, w2, bias, 2.0 ** -17)


def test_an_activation_between_the_largest_numbers_of_two_types(device):
    """Above the largest bf16 number and below that of fp32."""
    import prime_moe
    K, H = 64, 32
    x = torch.zeros((1, K), dtype=BF16, device=device)
    x[0, :2] = 1.0
    w1 = torch.zeros((1, 2 * H, K), dtype=BF16, device=device)
    w1[0, :H, 0] = 64.0
    w1[0, H:, 0], w1[0, H:, 1] = 1.9921875 * 2.0 ** 121, 0.005859375 * 2.0 ** 121  # 64 times their sum: 1.998 x 2^127
    w2 = torch.full((1, K, H), 2.0 ** -126, dtype=BF16, device=device)
    gate, bias = torch.zeros((1, K), dtype=BF16, device=device), torch.zeros(1, device=device)
    check(prime_moe.moe_layer(x, gate, w1, w2, 1, bias), x, w1, w2, bias, 2.0 ** -17)
    w1[0, H:, :2] *= -1
    check(prime_moe.moe_layer(x, gate, w1, w2, 1, bias), x, w1, w2, bias, 2.0 ** -17)


def test_gates_that_take_back_what_their_product_would_be(device):
    """gate * up beyond fp32, the activation far inside."""
    import prime_moe
    K, H = 64, 32
    x = torch.zeros((2, K), dtype=BF16, device=device)
    x[0, 0], x[1, 0] = 1.0, 1.125
    w1 = torch.zeros((1, 2 * H, K), dtype=BF16, device=device)
    w1[0, :H, 0] = torch.arange(-64, -32)
    w1[0, H:, 0] = 2.0 ** 125
    w2 = torch.full((1, K, H), 2.0 ** -60, dtype=BF16, device=device)
    bias = torch.zeros(1, device=device)
    check(prime_moe.moe_layer(x, torch.zeros((1, K), dtype=BF16, device=device), w1, w2, 1, bias), x, w1, w2, bias, 2.0 ** -17)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["wide", "narrow"])
def test_infinite_activations(device, dtype, kind):
    """An activation beyond fp32, or not a number, leaves outputs that are not finite, the other tokens theirs, and no wait open."""
    import prime_moe
    K, H, E, T, group = 256, 64, 2, 5, 32
    gen = torch.Generator().manual_seed(9)
    x = torch.randn((T, K), generator=gen).to(dtype).to(device)
    gate = torch.zeros((E, K), dtype=dtype, device=device)
    if kind == "wide":
        w = [torch.randn(s, generator=gen).to(dtype).to(device) * 0.1 for s in ((E, 2 * H, K), (E, K, H))]
        run = lambda v: prime_moe.moe_layer(v, gate, *w, E)
    else:
        w = [t for s in ((E, 2 * H, K), (E, K, H)) for t in prime_moe.pack_int4(
            torch.randint(-8, 8, s, generator=gen, dtype=torch.int8).to(device), torch.full((*s[:-1], s[-1] // group), 0.02, dtype=dtype, device=device))]
        run = lambda v: prime_moe.moe_layer_int4(v, gate, *w, E)
    want = run(x)[0]
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[3, 100] = bad
        got = run(y)[0]
        rest = [0, 1, 2, 4]
        assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[3]).any()
    if dtype == BF16:
        y = x.clone()
        y[3] = 2.0 ** 100
        got = run(y)[0]
        assert torch.equal(got[rest], want[rest]) and not torch.isfinite(got[3]).any()
