"""The choice of one token's experts, which a workgroup makes by ranks in four forms, by how many there are."""
import pytest
import torch

from layer_ref import Layer, select

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("E", [1, 2, 3, 5, 31, 33, 63, 64, 65, 100, 127, 128, 129, 160, 200, 255, 256, 257, 300, 511, 512])
def test_one_token_and_every_number_of_experts(device, E):
    import prime_moe
    K, H = 64, 16
    gen = torch.Generator().manual_seed(E)
    w1 = (torch.randn((E, 2 * H, K), generator=gen) * K ** -0.5).to(BF16).to(device)
    w2 = (torch.randn((E, K, H), generator=gen) * H ** -0.5).to(BF16).to(device)
    gate = (torch.randn((E, K), generator=gen) * K ** -0.5).to(BF16).to(device)
    x = torch.randn((1, K), generator=gen).to(BF16).to(device)
    for top_k in sorted({1, min(E, 8), min(E, 32)}):
        for bias in (None, torch.randn((E,), generator=gen).to(device), torch.linspace(-3, 3, E).to(device)):
            Layer(x, gate, w1, w2, top_k, bias).check(*prime_moe.moe_layer(x, gate, w1, w2, top_k, bias))
        # equal scores, the last expert alone above them, infinities
        bias = torch.zeros(E, device=device)
        bias[-1] = 1.0
        none = torch.zeros_like(gate)
        for last in (1.0, -float("inf")):
            bias[-1] = last
            ids = prime_moe.moe_layer(x, none, w1, w2, top_k, bias)[1]
            assert torch.equal(ids.long(), select(bias.double()[None], top_k))
