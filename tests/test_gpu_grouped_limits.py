"""The ragged products at the largest sizes that they accept."""
import pytest
import torch

import grouped_ref as R
from test_gpu_int8 import check

pytestmark = pytest.mark.gpu


def test_widest_rows_of_fp32(device):
    """int8 products whose rows of fp32 are 2^30 bytes: the store's row offsets pass 32 bits."""
    import prime_moe
    gen = torch.Generator(device=device).manual_seed(1)
    M, N, K = 24, 1 << 28, 16
    w = torch.randint(-128, 128, (N, K), dtype=torch.int8, device=device, generator=gen)
    x = torch.randint(-128, 128, (M, K), dtype=torch.int8, device=device, generator=gen)
    xs, ws = torch.rand((M,), device=device, generator=gen), torch.rand((N,), device=device, generator=gen)
    y = prime_moe.grouped_mm_int8(x, w, xs, ws, out_dtype=torch.float32)
    cols = torch.cat([torch.arange(0, 600), torch.arange(N - 600, N), torch.randint(0, N, (4096,))]).to(device)
    check(y[:, cols], R.mm_int8(x, w[cols][None], xs, ws[cols][None], [M]))
    del y, w, ws
    torch.cuda.empty_cache()
