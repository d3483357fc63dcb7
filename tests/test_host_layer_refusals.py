"""What a refused batch of a whole layer is sent on to takes its types."""
import pytest
import torch

from test_host_moe_layer import F16, narrow, t, wide


@pytest.mark.parametrize("make,change,onward", [
    (wide, {}, {"fused_moe_bf16"}),
    (wide, dict(gate=t(4, 64, dtype=F16), w1=t(4, 96, 64, dtype=F16), w2=t(4, 64, 48, dtype=F16)), {"expert_offsets", "grouped_mm"}),
    (narrow, {}, {"expert_offsets", "grouped_mm_int4", "grouped_mm", "dequantize_int4"}),
    (narrow, dict(gate=t(4, 64, dtype=F16)), {"expert_offsets", "grouped_mm_int4", "grouped_mm", "dequantize_int4"}),
])
def test_more_tokens_are_sent_to_what_takes_them(make, change, onward):
    import prime_moe
    from prime_moe import _torch_ops
    x = t(17, 64, dtype=change["gate"].dtype if change else torch.bfloat16)
    with pytest.raises(RuntimeError, match="up to 16 tokens") as refused:
        getattr(_torch_ops, "validate_moe_layer" if make is wide else "validate_moe_layer_int4")(*make(x=x, **change))
    named = {w for w in str(refused.value).replace(",", " ").replace(")", " ").split() if hasattr(prime_moe, w) and not w.startswith("moe_layer")}
    assert named == onward | {"route"}


def test_the_c_side_too():
    from prime_moe import _native
    lib, at = _native.load(), 1 << 20
    for dtype, group, named in ((1, 0, b"fused_moe_bf16"), (2, 0, b"grouped_mm)"), (1, 32, b"grouped_mm_int4"), (2, 64, b"grouped_mm_int4")):
        assert lib.pmoe_moe_layer(at, at, None, at, at, at, at, group, at, at, at, 17, 64, 64, 4, 2, dtype, at, 1 << 30, None) == 1
        assert named in lib.pmoe_last_error()
