"""Differentiation of the ragged products without a GPU: fake tensors that say they are on one."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16 = torch.bfloat16


def operands():
    dev = "cuda"
    x, w, dy = (torch.empty(s, dtype=BF16, device=dev) for s in ((10, 64), (3, 32, 64), (10, 32)))
    return x, w, dy, torch.empty((3,), dtype=torch.int32, device=dev)


def test_tangents_are_refused():
    """Forward mode: an output without a tangent would count as one that does not change."""
    import prime_moe
    import torch.autograd.forward_ad as fw
    with FakeTensorMode():
        x, w, dy, off = operands()
        for grads in (False, True):
            x.requires_grad_(grads)
            for call, dual in ((lambda t: prime_moe.grouped_mm(t, w, off), x), (lambda t: prime_moe.grouped_mm(x, t, off), w),
                               (lambda t: prime_moe.grouped_mm_wgrad(t, x, off), dy), (lambda t: prime_moe.grouped_mm_wgrad(dy, t, off), x)):
                with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode derivatives are not implemented"):
                    call(fw.make_dual(dual, torch.empty_like(dual)))
                with torch.no_grad(), fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode derivatives are not implemented"):
                    call(fw.make_dual(dual, torch.empty_like(dual)))
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not implemented"):
                torch.func.jvp(lambda t: prime_moe.grouped_mm(t, w, off), (x.detach(),), (torch.empty_like(x),))
        with fw.dual_level():  # level entered, no tangent
            assert prime_moe.grouped_mm(x, w, off).requires_grad
