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


def test_more_jobs_than_a_launch_has_threads(device):
    """A row for each of 1024 experts, whose weights are so wide that the kernel for few rows would need 2^32 threads."""
    import prime_moe
    gen = torch.Generator(device=device).manual_seed(2)
    E, N, K = 1024, 1 << 19, 8
    x = torch.randn((E, K), device=device, generator=gen).to(torch.bfloat16)
    w = torch.randn((N, K), device=device, generator=gen).to(torch.bfloat16)
    y = prime_moe.grouped_mm(x, w.expand(E, N, K), torch.arange(1, E + 1, dtype=torch.int32, device=device))
    for cols in (slice(0, 1 << 12), slice(N // 2 - 40, N // 2 + 40), slice(N - (1 << 12), N)):
        R.check(y[:, cols], *R.mm(x, w[cols][None], [E]), K)
    del y
    torch.cuda.empty_cache()
