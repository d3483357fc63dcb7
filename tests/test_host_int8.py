"""Host side of the int8 quantiser, without a GPU."""


def test_c_side_refuses_addresses_that_are_not_aligned():
    """Rows are read 16 bytes at a time from where they begin; the address is looked at before any launch."""
    from prime_moe import _native
    lib, at = _native.load(), 1 << 20
    for dtype in (0, 1, 2):
        for off_by in ((8, 0), (2, 0), (0, 8), (0, 1)):
            assert lib.pmoe_quantize_int8(at + off_by[0], dtype, at + off_by[1], at, 4, 64, 64, None) == 1
            assert b"aligned" in lib.pmoe_last_error()
