"""Host side of the whole layer for a few tokens, without a GPU: what is refused, in the package and in the C ABI, and the fakes."""
import pytest
import torch

BF16, F16 = torch.bfloat16, torch.float16


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def packed(*shape, group=32, dtype=BF16):
    import prime_moe
    return prime_moe.pack_int4(torch.zeros(shape, dtype=torch.int8), torch.ones((*shape[:-1], shape[-1] // group), dtype=dtype))


def wide(x=None, gate=None, w1=None, w2=None, top_k=2, bias=None):
    return (t(3, 64) if x is None else x, t(4, 64) if gate is None else gate, t(4, 96, 64) if w1 is None else w1,
            t(4, 64, 48) if w2 is None else w2, top_k, bias)


def narrow(x=None, gate=None, w1=None, w2=None, top_k=2, bias=None):
    w1, w2 = w1 or packed(4, 128, 64), w2 or packed(4, 64, 64)
    return (t(3, 64) if x is None else x, t(4, 64) if gate is None else gate, *w1, *w2, top_k, bias)


REFUSED = [
    (wide, dict(x=t(64)), "2-D"),
    (wide, dict(x=t(3, 72)), "gate 2-D"),
    (wide, dict(gate=t(4, 72)), "gate 2-D"),
    (wide, dict(x=t(3, 64, dtype=torch.float32)), "bfloat16 or float16"),
    (wide, dict(gate=t(4, 64, dtype=F16)), "same dtype"),
    (wide, dict(w1=t(4, 96, 64, dtype=F16)), "same dtype"),
    (wide, dict(w2=t(4, 64, 48, dtype=F16)), "same dtype"),
    (wide, dict(x=t(17, 64)), "up to 16 tokens"),
    (wide, dict(gate=t(513, 64), w1=t(513, 16, 64), w2=t(513, 64, 8)), "1..512"),
    (wide, dict(gate=t(0, 64), w1=t(0, 16, 64), w2=t(0, 64, 8)), "1..512"),
    (wide, dict(top_k=0), "top_k"),
    (wide, dict(top_k=5), "top_k"),
    (wide, dict(gate=t(64, 64), w1=t(64, 16, 64), w2=t(64, 64, 8), top_k=33), "top_k"),
    (wide, dict(w1=t(4, 95, 64)), r"\(E, 2H, K\)"),
    (wide, dict(w1=t(3, 96, 64)), r"\(E, 2H, K\)"),
    (wide, dict(w1=t(4, 96, 56)), r"\(E, 2H, K\)"),
    (wide, dict(w2=t(4, 64, 40)), r"\(E, K, H\)"),
    (wide, dict(w2=t(4, 56, 48)), r"\(E, K, H\)"),
    (wide, dict(w1=t(4, 40, 64), w2=t(4, 64, 20)), "multiples of 8"),
    (wide, dict(x=t(3, 60), gate=t(4, 60), w1=t(4, 96, 60), w2=t(4, 60, 48)), "multiples of 8"),
    (wide, dict(x=t(3, 0), gate=t(4, 0), w1=t(4, 96, 0), w2=t(4, 0, 48)), "multiples of 8"),
    (wide, dict(w1=t(4, 0, 64), w2=t(4, 64, 0)), "multiples of 8"),
    (wide, dict(x=t(64, 3).t()), "contiguous"),
    (wide, dict(x=t(3, 128)[:, :64]), "contiguous"),
    (wide, dict(gate=t(64, 4).t()), "contiguous"),
    (wide, dict(w1=t(4, 64, 96).transpose(1, 2)), "contiguous"),
    (wide, dict(w2=t(4, 48, 64).transpose(1, 2)), "contiguous"),
    (wide, dict(bias=t(4)), "bias"),
    (wide, dict(bias=torch.zeros(5)), "bias"),
    (wide, dict(bias=torch.zeros(1, 4)), "bias"),
    (wide, dict(bias=torch.zeros(8)[::2]), "bias"),
    (narrow, dict(x=t(17, 64)), "up to 16 tokens"),
    (narrow, dict(w1=packed(3, 128, 64)), "experts of gate"),
    (narrow, dict(w2=packed(3, 64, 64)), "experts of gate"),
    (narrow, dict(w1=packed(4, 112, 64)), "multiple of 32"),
    (narrow, dict(w1=packed(4, 128, 256)), "does not fit"),
    (narrow, dict(w2=packed(4, 64, 256)), "does not fit"),
    (narrow, dict(w2=packed(4, 48, 64)), "rows"),
    (narrow, dict(w2=packed(4, 64, 64, group=64)), "same size"),
    (narrow, dict(w1=packed(4, 128, 64, dtype=F16)), "same dtype"),
    (narrow, dict(w2=packed(4, 64, 64, dtype=F16)), "same dtype"),
    (narrow, dict(w1=packed(128, 64)), "must be uint8 of shape"),
    (narrow, dict(x=t(3, 40), gate=t(4, 40)), "does not fit"),
]


@pytest.mark.parametrize("make,change,message", REFUSED)
def test_refused(make, change, message):
    from prime_moe import _torch_ops
    with pytest.raises(RuntimeError, match=message):
        getattr(_torch_ops, "validate_moe_layer" if make is wide else "validate_moe_layer_int4")(*make(**change))


def test_accepted():
    from prime_moe import _torch_ops
    _torch_ops.validate_moe_layer(*wide())
    _torch_ops.validate_moe_layer(*wide(x=t(0, 64), bias=torch.zeros(4)))
    _torch_ops.validate_moe_layer_int4(*narrow())
    _torch_ops.validate_moe_layer_int4(*narrow(x=t(16, 64, dtype=F16), gate=t(4, 64, dtype=F16), w1=packed(4, 192, 64, dtype=F16),
                                               w2=packed(4, 64, 96, dtype=F16)))


def test_cpu_tensors_are_refused():
    import prime_moe
    with pytest.raises((RuntimeError, NotImplementedError)):
        prime_moe.moe_layer(*wide())
    with pytest.raises((RuntimeError, NotImplementedError)):
        prime_moe.moe_layer_int4(*narrow())


def test_c_side_refuses():
    from prime_moe import _native
    lib, at = _native.load(), 1 << 20

    def layer(x=at, gate=at, bias=None, w1=at, s1=at, w2=at, s2=at, group=32, out=at, ids=at, weights=at, T=3, K=64, H=64, E=4, top_k=2, dtype=1,
              ws=at, ws_bytes=1 << 30):
        return lib.pmoe_moe_layer(x, gate, bias, w1, s1, w2, s2, group, out, ids, weights, T, K, H, E, top_k, dtype, ws, ws_bytes, None)

    need = lib.pmoe_moe_layer_workspace_bytes(3, 64, 4, 2)
    assert need > 0 and lib.pmoe_moe_layer_workspace_bytes(0, 64, 4, 2) == 0
    for bad in (dict(dtype=0), dict(dtype=3), dict(T=17), dict(T=-1), dict(E=0), dict(E=513), dict(top_k=0), dict(top_k=5), dict(E=64, top_k=33),
                dict(group=16), dict(K=72), dict(H=48), dict(K=0), dict(H=0), dict(K=1 << 21), dict(H=1 << 21), dict(group=0, K=60),
                dict(group=0, H=60), dict(group=64, H=96), dict(x=None), dict(gate=None), dict(w1=None), dict(w2=None), dict(s1=None), dict(s2=None), dict(out=None),
                dict(ids=None), dict(weights=None), dict(ws=None), dict(ws=at + 128), dict(ws_bytes=need - 1), dict(x=at + 8), dict(gate=at + 2),
                dict(w1=at + 8), dict(w2=at + 4), dict(s1=at + 8), dict(s2=at + 8), dict(out=at + 8)):
        assert layer(**bad) == 1, bad
    assert layer(T=0, x=None, ws=None) == 0


def test_fake_implementations():
    import prime_moe
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dtype=F16: torch.empty(s, dtype=dtype, device="cuda")
        for got in (prime_moe.moe_layer(e(3, 64), e(4, 64), e(4, 96, 64), e(4, 64, 48), 2, e(4, dtype=torch.float32)),
                    prime_moe.moe_layer_int4(e(3, 64), e(4, 64), *prime_moe.quantize_int4(e(4, 128, 64), 64), *prime_moe.quantize_int4(e(4, 64, 64), 64), 2)):
            assert got[0].shape == (3, 64) and got[0].dtype == F16
            assert got[1].shape == got[2].shape == (3, 2) and got[1].dtype == torch.int32 and got[2].dtype == torch.float32
