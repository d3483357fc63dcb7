"""Offsets that are not ends of groups: what the products still promise, and that nothing next to their outputs is written."""
import pytest
import torch

import grouped_ref as R
from test_gpu_grouped import cus  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
BAD = [[50, 20, 120, 90], [-7, -1, 1 << 30, 3], [200, 200, 200, 200], [2 ** 31 - 1, -(2 ** 31), 0, 60], [10, 60, 40, 70], [0, 0, 0, -5]]
GUARD = 4096


def guarded(shape, dtype, device):
    """(all, the part in the middle): bytes of a known pattern on both sides."""
    n = torch.Size(shape).numel() * torch.empty((), dtype=dtype).element_size()
    everything = torch.full((n + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=device)
    return everything, everything[GUARD:GUARD + n].view(dtype).view(shape)


def check_guards(everything):
    assert (everything[:GUARD] == 0xA5).all() and (everything[-GUARD:] == 0xA5).all()


@pytest.mark.parametrize("M", [100, 40])  # tiles or blocks; the kernel for few rows
@pytest.mark.parametrize("offsets", BAD)
def test_outputs_stay_where_they_belong(device, cus, M, offsets):
    """Rows by their expert's weights: an end counts as the nearest inside, a group begins at the furthest end in front of it,
    so every row is one group's or none's.  Gradients of weights: unspecified, but inside."""
    from prime_moe import _native
    lib, stream = _native.load(), torch.cuda.current_stream().cuda_stream
    gen = torch.Generator().manual_seed(M)
    E, N, K = 4, 40, 64
    off = torch.tensor(offsets, dtype=torch.int32, device=device)
    x, w, dy = (torch.randn(s, generator=gen).to(torch.bfloat16).to(device) for s in ((M, K), (E, N, K), (M, N)))
    wt = w.transpose(1, 2).contiguous()
    far, ends = 0, []
    for o in offsets:
        far = max(far, min(max(o, 0), M))
        ends.append(far)
    ref, mags = R.mm(x, w, ends)
    for weights, across, stride in ((w, 0, K), (wt, 1, N)):
        everything, y = guarded((M, N), torch.bfloat16, device)
        _native.check(lib.pmoe_grouped_mm(x.data_ptr(), weights.data_ptr(), y.data_ptr(), off.data_ptr(), E, M, N, K, K, stride, N * K, across, 1, stream))
        R.check(y, ref, mags, K)
        assert (y[far:] == 0).all()
        check_guards(everything)
    q, qw = (torch.randint(-128, 128, s, generator=gen, dtype=torch.int8).to(device) for s in ((M, K), (E, N, K)))
    one = torch.ones((E * N + M,), device=device)
    everything, y = guarded((M, N), torch.float32, device)
    _native.check(lib.pmoe_grouped_mm_int8(q.data_ptr(), qw.data_ptr(), one.data_ptr(), one.data_ptr(), y.data_ptr(), off.data_ptr(), E, M, N, K, K, K,
                                           N * K, 0, stream))
    assert torch.equal(y.double(), R.mm_int8(q, qw, one[:M], one[:E * N].view(E, N), ends))
    check_guards(everything)
    everything, dw = guarded((E, N, K), torch.bfloat16, device)
    _native.check(lib.pmoe_grouped_mm_wgrad(dy.data_ptr(), x.data_ptr(), dw.data_ptr(), off.data_ptr(), E, M, N, K, N, K, 1, stream))
    check_guards(everything)
