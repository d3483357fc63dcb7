"""Host side of the ragged expert products, without a GPU: what they refuse, in the package and in the C ABI, their schemas
and fake implementations, and that no kernel uses M0 behind the copies' back."""
import os
import re
import subprocess

import pytest
import torch

BF16, F16 = torch.bfloat16, torch.float16


def t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def off(*v):
    return torch.tensor(v, dtype=torch.int32)


REFUSED = [
    # grouped_mm
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 72), off(1, 4)), "must equal w.size"),
    ("validate_grouped_mm", lambda: (t(4, 64, dtype=torch.float32), t(2, 32, 64, dtype=torch.float32), off(1, 4)), "bfloat16 or float16"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 64, dtype=F16), off(1, 4)), "same dtype"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(32, 64), off(4)), "3-D"),
    ("validate_grouped_mm", lambda: (t(4, 60), t(2, 32, 60), off(1, 4)), "multiple of 8"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 33, 64), off(1, 4)), "multiple of 8"),
    ("validate_grouped_mm", lambda: (t(4, 0), t(2, 32, 0), off(1, 4)), "positive multiple"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 64), off(4)), "one entry per matrix"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 64), off(1, 4).long()), "int32"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 64), off(1, 2, 3, 4)[::2]), "contiguous int32"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(0, 32, 64), off()), "1..1024"),
    ("validate_grouped_mm", lambda: (t(4, 8), t(1, 8, 8).expand(1025, 8, 8), torch.zeros(1025, dtype=torch.int32)), "1..1024"),
    ("validate_grouped_mm", lambda: (t(64, 4).t(), t(2, 32, 64), off(1, 4)), "last dimension of x"),
    ("validate_grouped_mm", lambda: (t(4, 68)[:, :64], t(2, 32, 64), off(1, 4)), "rows of x"),
    ("validate_grouped_mm", lambda: (t(1, 64).expand(4, 64), t(2, 32, 64), off(1, 4)), "rows of x"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 128)[:, :, ::2], off(1, 4)), "must be contiguous"),
    ("validate_grouped_mm", lambda: (t(4, 64), t(2, 32, 68)[:, :, :64], off(1, 4)), "rows of w"),
    ("validate_grouped_mm", lambda: (t(4, 64), torch.empty_strided((2, 32, 64), (32 * 64 + 4, 64, 1), dtype=BF16), off(1, 4)), "matrices of w"),
    ("validate_grouped_mm", lambda: (torch.empty_strided((2, 8), (1 << 23, 1), dtype=BF16, device="meta"), t(2, 8, 8), off(1, 2)), "rows of x"),
    # grouped_mm_wgrad
    ("validate_grouped_mm_wgrad", lambda: (t(4, 32), t(5, 64), off(4)), "same number of rows"),
    ("validate_grouped_mm_wgrad", lambda: (t(4, 32), t(4, 64, dtype=F16), off(4)), "same dtype"),
    ("validate_grouped_mm_wgrad", lambda: (t(4, 36), t(4, 64), off(4)), "multiple of 8"),
    ("validate_grouped_mm_wgrad", lambda: (t(4, 32), t(4, 64), off(4).float()), "int32"),
    ("validate_grouped_mm_wgrad", lambda: (t(32, 4).t(), t(4, 64), off(4)), "last dimension of dy"),
    ("validate_grouped_mm_wgrad", lambda: (t(4, 32), t(4, 64), off()), "1..1024"),
]


def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def f32(*shape):
    return torch.zeros(shape)


REFUSED += [
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(32, 64), f32(4), f32(32), off(4), BF16), "3-D"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(2, 32, 64), f32(4), f32(2, 32), None, BF16), "2-D"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), t(32, 64), f32(4), f32(32), None, BF16), "int8"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 72), i8(32, 72), f32(4), f32(32), None, BF16), "multiple of 16"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(30, 64), f32(4), f32(30), None, BF16), "multiple of 8"),
    ("validate_grouped_mm_int8", lambda: (i8(1, 131072), i8(8, 131072), f32(1), f32(8), None, BF16), "below 131072"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(32, 64), f32(5), f32(32), None, BF16), "x_scale"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(32, 64), f32(4), f32(31), None, BF16), "w_scale"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(2, 32, 64), f32(4), f32(32), off(1, 4), BF16), "w_scale"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(32, 64), f32(4).double(), f32(32), None, BF16), "x_scale"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(32, 64), f32(4), f32(32), None, torch.int32), "out_dtype"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(64, 32).t(), f32(4), f32(32), None, BF16), "last dimension of w"),
    ("validate_grouped_mm_int8", lambda: (i8(4, 64), i8(2, 64, 32).transpose(1, 2), f32(4), f32(2, 32), off(1, 4), BF16), "last dimension of w"),
    ("validate_quantize_int8", lambda: (i8(4, 64),), "bfloat16, float16 or float32"),
    ("validate_quantize_int8", lambda: (t(4, 60),), "multiple of 8"),
    ("validate_quantize_int8", lambda: (t(4, 0),), "positive multiple"),
    ("validate_quantize_int8", lambda: (t(),), "dimension"),
    ("validate_quantize_int8", lambda: (t(64, 8).t(),), "contiguous"),
    ("validate_quantize_int8", lambda: (t(2, 4, 72)[..., :64],), "contiguous"),
    ("validate_quantize_int8", lambda: (t(4, 68)[:, :64],), "rows of x"),
    ("validate_expert_offsets", lambda: (off(0, 1).long(), off(2), 4), "int32"),
    ("validate_expert_offsets", lambda: (off(0, 1), off(), 4), "empty"),
    ("validate_expert_offsets", lambda: (off(0, 1), off(2), 0), "1..1024"),
    ("validate_expert_offsets", lambda: (off(0, 1), off(2), 1025), "1..1024"),
    ("validate_expert_offsets", lambda: (off(0, 0, 1, 1)[::2], off(2), 2), "contiguous"),
]


@pytest.mark.parametrize("check,args,match", REFUSED)
def test_refusals(check, args, match):
    from prime_moe import _torch_ops
    with pytest.raises(RuntimeError, match=re.escape(match)):
        getattr(_torch_ops, check)(*args())


def test_what_is_taken():
    from prime_moe import _torch_ops as ops
    ops.validate_grouped_mm(t(4, 64), t(2, 32, 64), off(1, 4))
    ops.validate_grouped_mm(t(4, 80)[:, 8:72], t(2, 64, 32).transpose(1, 2), off(1, 4))
    ops.validate_grouped_mm(t(1, 67)[:, :64], t(1, 32, 64).expand(5, 32, 64), off(0, 0, 0, 0, 1))  # a stride that no access uses
    ops.validate_grouped_mm(t(0, 64), t(2, 32, 64), off(0, 0))
    ops.validate_grouped_mm_wgrad(t(0, 32), t(0, 64), off(0))
    ops.validate_grouped_mm_int8(i8(0, 64), i8(32, 64), f32(0), f32(32), None, torch.float32)
    ops.validate_quantize_int8(t(3, 5, 64))
    ops.validate_quantize_int8(t(0, 64))
    ops.validate_expert_offsets(off(), off(0), 4)


def test_c_side_refuses_before_any_launch():
    from prime_moe import _native
    lib = _native.load()
    for rc in (
        lib.pmoe_grouped_mm(None, None, None, None, 2, 4, 32, 64, 64, 64, 2048, 0, 0, None),        # fp32
        lib.pmoe_grouped_mm(None, None, None, None, 1025, 4, 32, 64, 64, 64, 2048, 0, 1, None),     # groups
        lib.pmoe_grouped_mm(None, None, None, None, 2, 4, 33, 64, 64, 64, 2048, 0, 1, None),        # N
        lib.pmoe_grouped_mm(None, None, None, None, 2, 4, 32, 64, 60, 64, 2048, 0, 1, None),        # stride
        lib.pmoe_grouped_mm(None, None, None, None, 2, 4, 32, 64, 64, 1 << 23, 2048, 0, 1, None),   # stride
        lib.pmoe_grouped_mm(None, None, None, None, 2, 1 << 31, 32, 64, 64, 64, 2048, 0, 1, None),  # rows
        lib.pmoe_grouped_mm(None, None, None, None, 2, 4, 32, 64, 64, 64, 2048, 0, 1, None),        # null
        lib.pmoe_grouped_mm_wgrad(None, None, None, None, 2, 4, 32, 64, 32, 60, 1, None),
        lib.pmoe_grouped_mm_wgrad(None, None, None, None, 2, 4, 32, 64, 32, 64, 1, None),
        lib.pmoe_grouped_mm_int8(None, None, None, None, None, None, 2, 4, 32, 64, 64, 64, 2048, 1, None),      # groups without offsets
        lib.pmoe_grouped_mm_int8(None, None, None, None, None, None, 1, 4, 32, 131072, 131072, 131072, 0, 1, None),
        lib.pmoe_grouped_mm_int8(None, None, None, None, None, None, 1, 4, 32, 64, 64, 64, 0, 7, None),
        lib.pmoe_quantize_int8(None, 1, None, None, 4, 60, 60, None),
        lib.pmoe_quantize_int8(None, 1, None, None, 4, 64, 68, None),
        lib.pmoe_expert_offsets(None, None, None, 4, 0, None),
    ):
        assert rc == 1 and lib.pmoe_last_error()
    # no rows: nothing to do, nothing looked at
    assert lib.pmoe_grouped_mm(None, None, None, None, 2, 0, 32, 64, 64, 64, 2048, 0, 1, None) == 0
    assert lib.pmoe_grouped_mm_int8(None, None, None, None, None, None, 1, 0, 32, 64, 64, 64, 0, 1, None) == 0
    assert lib.pmoe_quantize_int8(None, 1, None, None, 0, 64, 64, None) == 0


def test_c_side_refuses_addresses_that_are_not_aligned():
    from prime_moe import _native
    lib, at = _native.load(), 1 << 20
    for off_by in ((8, 0, 0), (0, 8, 0), (0, 0, 2)):
        x, w, out = (at + o for o in off_by)
        assert lib.pmoe_grouped_mm(x, w, out, at, 2, 4, 32, 64, 64, 64, 2048, 0, 1, None) == 1
        assert b"aligned" in lib.pmoe_last_error()
        assert lib.pmoe_grouped_mm_wgrad(x, w, out, at, 2, 4, 32, 64, 32, 64, 1, None) == 1
        assert b"aligned" in lib.pmoe_last_error()
        assert lib.pmoe_grouped_mm_int8(x, w, at, at, out, None, 1, 4, 32, 64, 64, 64, 0, 1, None) == 1
        assert b"aligned" in lib.pmoe_last_error()


def test_cpu_tensors_are_refused():
    import prime_moe
    for call in (lambda: prime_moe.grouped_mm(t(4, 64), t(2, 32, 64), off(1, 4)), lambda: prime_moe.grouped_mm_wgrad(t(4, 32), t(4, 64), off(4)),
                 lambda: prime_moe.grouped_mm_int8(i8(4, 64), i8(32, 64), f32(4), f32(32)), lambda: prime_moe.quantize_int8(t(4, 64)),
                 lambda: prime_moe.expert_offsets(off(0), off(1), 2)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()


def test_fake_implementations():
    import prime_moe
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        dev = "cuda"
        x, w, o = (torch.empty(s, dtype=BF16, device=dev) for s in ((10, 64), (3, 32, 64), (3,)))
        assert prime_moe.grouped_mm(x, w, o).shape == (10, 32)
        assert prime_moe.grouped_mm_wgrad(prime_moe.grouped_mm(x, w, o), x, o).shape == (3, 32, 64)
        q, s = prime_moe.quantize_int8(w)
        assert q.shape == (3, 32, 64) and q.dtype == torch.int8 and s.shape == (3, 32) and s.dtype == torch.float32
        assert prime_moe.grouped_mm_int8(q[0], q, s[0], s, o, F16).dtype == F16


def test_no_compiler_use_of_m0(tmp_path):
    """The copies of csrc/moe_ring.h and grouped_tile.h set M0 inside inline assembly without telling the compiler: a kernel
    that contains one names M0 nowhere else, and no source uses a builtin that makes the compiler hold a value there."""
    from prime_moe import build
    names = ("grouped_mm.hip", "grouped_int8.hip")
    banned = re.compile(r"__builtin_amdgcn_(global_load_lds|raw_buffer_load_lds|struct_buffer_load_lds|ds_gws\w*|s_sendmsg\w*|s_movrel\w*|mov_dpp8)")
    for f in [n for n in os.listdir(build.CSRC) if n.startswith("grouped")]:
        assert not banned.search(open(os.path.join(build.CSRC, f)).read()), f
    for name in names:
        asm = tmp_path / (name + ".s")
        cmd = [build.hipcc(), f"--offload-arch={build.ARCH}", "-O3", "-std=c++17", "-munsafe-fp-atomics", *build.DEVICE_FLAGS,
               "-S", "--cuda-device-only", os.path.join(build.CSRC, name), "-o", str(asm)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        kernel, in_asm, copies, stray = None, False, set(), {}
        for line in open(asm):
            m = re.match(r"^(_Z\w+):", line)
            kernel = m.group(1) if m else kernel
            in_asm = ";;#ASMSTART" in line or (in_asm and ";;#ASMEND" not in line)
            code = line.split(";")[0]
            if kernel is None or not code.strip() or code.lstrip().startswith("."):
                continue
            if "global_load_lds" in code:
                assert in_asm, (kernel, line)
                copies.add(kernel)
            elif re.search(r"\bm0\b", code) and not in_asm:
                stray.setdefault(kernel, []).append(line.strip())
        assert copies
        for k in copies:
            assert k not in stray, (k, stray[k][:5])
