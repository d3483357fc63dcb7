"""Gradients of the ragged products that lie in memory in other ways than the kernels take them."""
import pytest
import torch

import grouped_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("start", [0, 3, 8, 12])
def test_contiguous_gradients_that_begin_anywhere(device, start):
    """A piece of a flat gradient (of a cat, of a flattened tensor) is contiguous wherever it begins; the products take it from
    16-byte aligned addresses on."""
    import prime_moe
    gen = torch.Generator().manual_seed(start)
    ends, M, N, K = [5, 5, 40], 43, 24, 32
    off = torch.tensor(ends, dtype=torch.int32, device=device)
    x, w, dy = (torch.randn(s, generator=gen).to(torch.bfloat16).to(device).requires_grad_() for s in ((M, K), (3, N, K), (M, N)))
    extra = torch.zeros((start,), dtype=torch.bfloat16, device=device, requires_grad=True)

    def through_cat(y):
        flat = torch.cat([extra, y.flatten()])
        g = torch.randn(flat.shape, generator=gen).to(torch.bfloat16).to(device)
        return flat, g, g[start:].view(y.shape)

    flat, g, part = through_cat(prime_moe.grouped_mm(x, w, off))
    assert part.is_contiguous() and part.storage_offset() == start
    dx, dw = torch.autograd.grad(flat, (x, w), g)
    R.check(dx, *R.mm(part, w.detach().transpose(1, 2), ends), N)
    R.check(dw, *R.wgrad(part, x.detach(), ends), max(ends))
    flat, g, part = through_cat(prime_moe.grouped_mm_wgrad(dy, x, off))
    ddy, dx = torch.autograd.grad(flat, (dy, x), g)
    R.check(ddy, *R.mm(x.detach(), part, ends), K)
    R.check(dx, *R.mm(dy.detach(), part.transpose(1, 2), ends), N)
