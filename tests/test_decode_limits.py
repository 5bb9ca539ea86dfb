"""Host-only checks of the decode-step records at their limits (include/vecops_b200/decode_cuda.h); no pointer is ever read."""
from ctypes import byref, c_uint32, c_uint64

import pytest

from tests.test_decode_host import code_of, matmul_record, prefix_record
from vecops_b200 import capi


@pytest.mark.parametrize("name", ["m", "n", "k"])
def test_products_whose_tiles_pass_32_bits_are_left_to_the_simple_kernel(library, name):
    chosen = c_uint32(9)
    # operands on rows of their own, whatever the extent
    wide = dict(a_stride_m=1 << 31, b_stride_n=1 << 31, c_stride_m=1 << 31)
    for extent, kernel in (((1 << 31) - 256, None), ((1 << 31) - 255, capi.F8_GENERIC), ((1 << 31) - 1, capi.F8_GENERIC)):
        record = matmul_record(**{**wide, name: extent})
        if kernel is None:
            kernel = capi.F8_TILED if name == "m" else capi.F8_STREAM
        assert code_of("vecops_b200_matmul_f8_select", record, byref(chosen))[0] == capi.OK
        assert chosen.value == kernel, extent
        for forced in (capi.F8_STREAM, capi.F8_TILED):
            if kernel == capi.F8_GENERIC:
                assert code_of("vecops_b200_matmul_f8_select", matmul_record(**{**wide, name: extent, "kernel": forced}), byref(chosen))[0] == capi.NOT_APPLICABLE
    assert code_of("vecops_b200_matmul_f8_select", matmul_record(**{**wide, name: 1 << 31}), byref(chosen))[0] == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [dict(q=0x10002), dict(out=0x10008), dict(k_cache=0x10004), dict(v_cache=0x1000e), dict(q_stride_token=513), dict(out_stride_head=65),
                                     dict(k_stride_slot=132, k_stride_page=2112), dict(v_stride_page=2052), dict(table_stride=1 << 20)])
def test_scratch_of_the_attention_goes_by_its_extents(library, changes):
    def need(record):
        size = c_uint64(0)
        assert code_of("vecops_b200_prefix_sdpa_workspace", record, byref(size))[0] == capi.OK
        return size.value

    for extents in (dict(), dict(tokens=64, batch=64, prefix_len=8192)):
        assert need(prefix_record(**extents)) > 0
        assert need(prefix_record(**{**extents, **changes})) == need(prefix_record(**extents))
