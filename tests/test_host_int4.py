"""Host side of the weights of 4 bits, without a GPU: their layout, what is refused, the fake implementations."""
import pytest
import torch

import int4_ref as R

BF16, F16 = torch.bfloat16, torch.float16


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def packed(*shape, group=64, dtype=BF16):
    import prime_moe
    return prime_moe.pack_int4(torch.zeros(shape, dtype=torch.int8), torch.ones((*shape[:-1], shape[-1] // group), dtype=dtype))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("lead,n,k", [((), 16, 128), ((3,), 48, 384), ((2, 2), 16, 640), ((), 32, None)])
def test_pack_is_the_described_layout(lead, n, k, group):
    import prime_moe
    k = k or group  # (one group: less than a tile)
    gen = torch.Generator().manual_seed(n + group)
    values = torch.randint(-8, 8, (*lead, n, k), generator=gen, dtype=torch.int8)
    scale = torch.rand((*lead, n, k // group), generator=gen).to(BF16)
    q, s = prime_moe.pack_int4(values, scale)
    assert q.shape == (*lead, n // 16, (k + 127) // 128, 1024) and s.shape == (*lead, n // 16, (k + 127) // 128, 16, 128 // group)
    back = R.unpack(q, s, k)
    assert torch.equal(back[0], values) and torch.equal(back[1], scale)
    # what a last tile has behind the columns stands for zero
    full = R.unpack(q, s, (k + 127) // 128 * 128)
    assert (full[0][..., k:] == 0).all() and (full[1][..., k // group:] == 0).all()


@pytest.mark.parametrize("make,message", [
    (lambda: (t(16, 128, dtype=torch.uint8), t(16, 1)), "int8"),
    (lambda: (t(128, dtype=torch.int8), t(1)), "int8"),
    (lambda: (t(16, 128, dtype=torch.int8), t(16, 1, dtype=torch.float32)), "bfloat16 or float16"),
    (lambda: (t(16, 128, dtype=torch.int8), t(16, 8)), "group of 32"),
    (lambda: (t(16, 128, dtype=torch.int8), t(15, 1)), "group of 32"),
    (lambda: (t(16, 96, dtype=torch.int8), t(16, 2)), "group of 32"),
    (lambda: (t(16, 128, dtype=torch.int8), t(16, 0)), "group of 32"),
    (lambda: (t(24, 128, dtype=torch.int8), t(24, 1)), "multiple of 16"),
    (lambda: (torch.full((16, 128), 8, dtype=torch.int8), t(16, 1)), "-8 .. 7"),
    (lambda: (torch.full((16, 128), -9, dtype=torch.int8), t(16, 1)), "-8 .. 7"),
])
def test_pack_refuses(make, message):
    import prime_moe
    with pytest.raises(RuntimeError, match=message):
        prime_moe.pack_int4(*make())


def off(*v):
    return torch.tensor(v, dtype=torch.int32)


REFUSED = [
    ("validate_grouped_mm_int4", lambda: (t(4, 64, dtype=torch.float32), *packed(32, 64), None), "bfloat16 or float16"),
    ("validate_grouped_mm_int4", lambda: (t(64), *packed(32, 64), None), "2-D"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), *packed(32, 64, dtype=F16), None), "same dtype"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), *packed(2, 32, 64), None), "must be uint8 of shape"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), *packed(32, 64), off(4)), "must be uint8 of shape"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(32, 64)[0].to(torch.int8), packed(32, 64)[1], None), "must be uint8"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(32, 64)[0], t(32, 1), None), "scales of w"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(32, 64)[0], t(2, 1, 16, 3), None), "scales of w"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(32, 64)[0], t(1, 1, 16, 2), None), "scales of w"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(32, 64)[0], t(2, 1, 16, 2, dtype=torch.float32), None), "bfloat16 or float16"),
    ("validate_grouped_mm_int4", lambda: (t(4, 256), *packed(32, 128), None), "does not fit"),
    ("validate_grouped_mm_int4", lambda: (t(4, 96), *packed(32, 128), None), "does not fit"),
    ("validate_grouped_mm_int4", lambda: (t(4, 0), *packed(32, 128), None), "positive multiple"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), *packed(2, 32, 64), off(4)), "one entry per matrix"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), *packed(2, 32, 64), off(1, 4).long()), "int32"),
    ("validate_grouped_mm_int4", lambda: (t(64, 4).t(), *packed(32, 64), None), "last dimension of x"),
    ("validate_grouped_mm_int4", lambda: (t(4, 68)[:, :64], *packed(32, 64), None), "rows of x"),
    ("validate_grouped_mm_int4", lambda: (t(4, 64), packed(64, 64)[0][::2], packed(32, 64)[1], None), "contiguous"),
    ("validate_quantize_int4", lambda: (t(16, 128, dtype=torch.int8), 32, BF16), "bfloat16, float16 or float32"),
    ("validate_quantize_int4", lambda: (t(16, 128), 32, torch.float32), "scale_dtype"),
    ("validate_quantize_int4", lambda: (t(16, 128), 16, BF16), "32, 64 or 128"),
    ("validate_quantize_int4", lambda: (t(128), 32, BF16), "two dimensions"),
    ("validate_quantize_int4", lambda: (t(24, 128), 32, BF16), "multiple of 16"),
    ("validate_quantize_int4", lambda: (t(16, 96), 64, BF16), "multiple of 64"),
    ("validate_quantize_int4", lambda: (t(16, 0), 64, BF16), "positive"),
    ("validate_quantize_int4", lambda: (t(128, 16).t(), 64, BF16), "contiguous"),
    ("validate_dequantize_int4", lambda: (t(16, 128, dtype=torch.uint8), t(16, 1), 128), "quantize_int4 makes it"),
    ("validate_dequantize_int4", lambda: (*packed(32, 256), 128), "does not fit"),
    ("validate_dequantize_int4", lambda: (*packed(32, 128), 32), "multiple of 64"),
    ("validate_dequantize_int4", lambda: (*packed(32, 128), 0), "positive"),
]


@pytest.mark.parametrize("name,make,message", REFUSED)
def test_refused(name, make, message):
    from prime_moe import _torch_ops
    with pytest.raises(RuntimeError, match=message):
        getattr(_torch_ops, name)(*make())


def test_accepted():
    from prime_moe import _torch_ops
    _torch_ops.validate_grouped_mm_int4(t(4, 72)[:, :64], *packed(32, 64), None)
    _torch_ops.validate_grouped_mm_int4(t(0, 64), *packed(2, 32, 64), off(0, 0))
    _torch_ops.validate_dequantize_int4(*packed(2, 3, 32, 192), 192)
    _torch_ops.validate_quantize_int4(t(0, 16, 64, dtype=torch.float32), 64, F16)


def test_cpu_tensors_are_refused():
    import prime_moe
    with pytest.raises((RuntimeError, NotImplementedError)):
        prime_moe.grouped_mm_int4(t(4, 64), *packed(32, 64))


def test_c_side_refuses():
    from prime_moe import _native
    lib, at = _native.load(), 1 << 20

    def mm(x=at, w=at, s=at, out=at, off=None, groups=1, m=4, n=32, k=128, group=64, stride=128, dtype=1):
        return lib.pmoe_grouped_mm_int4(x, w, s, out, off, groups, m, n, k, group, stride, dtype, None)

    for bad in (dict(dtype=0), dict(groups=0), dict(groups=2), dict(group=16), dict(n=24), dict(n=0), dict(k=96), dict(k=0), dict(stride=120),
                dict(stride=132), dict(m=-1), dict(x=None), dict(w=None), dict(s=None), dict(out=None), dict(x=at + 8), dict(w=at + 8),
                dict(s=at + 8), dict(out=at + 2), dict(off=at, groups=1025)):
        assert mm(**bad) == 1, bad
    assert mm(m=0, x=None) == 0
    for bad in ((at, 3, at, at, 1, 16, 128, 64), (at, 1, at, at, 0, 16, 128, 64), (at, 1, at, at, 1, 8, 128, 64), (at, 1, at, at, 1, 16, 96, 64),
                (at, 1, at, at, 1, 16, 128, 48), (None, 1, at, at, 1, 16, 128, 64), (at + 8, 1, at, at, 1, 16, 128, 64), (at, 1, at + 4, at, 1, 16, 128, 64),
                (at, 1, at, at + 2, 1, 16, 128, 64)):
        assert lib.pmoe_quantize_int4(*bad, None) == 1, bad
    for bad in ((at, at, at, 0, 16, 128, 64), (at, at, at, 1, 15, 128, 64), (at, at, None, 1, 16, 128, 64), (at, at + 8, at, 1, 16, 128, 64)):
        assert lib.pmoe_dequantize_int4(*bad, None) == 1, bad
    assert lib.pmoe_quantize_int4(None, 1, None, None, 1, 0, 128, 64, None) == 0
    assert lib.pmoe_dequantize_int4(None, None, None, 1, 0, 128, 64, None) == 0


def test_fake_implementations():
    import prime_moe
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        w = torch.empty((3, 32, 192), dtype=F16, device="cuda")
        q, s = prime_moe.quantize_int4(w, 64)
        assert q.shape == (3, 2, 2, 1024) and q.dtype == torch.uint8 and s.shape == (3, 2, 2, 16, 2) and s.dtype == F16
        assert prime_moe.dequantize_int4(q, s, 192).shape == w.shape and prime_moe.dequantize_int4(q, s).shape == (3, 32, 256)
        x, o = torch.empty((5, 192), dtype=F16, device="cuda"), torch.empty((3,), dtype=torch.int32, device="cuda")
        y = prime_moe.grouped_mm_int4(x, q, s, o)
        assert y.shape == (5, 32) and y.dtype == F16
        assert prime_moe.quantize_int4(torch.empty((16, 32), device="cuda"), 32)[1].dtype == BF16
