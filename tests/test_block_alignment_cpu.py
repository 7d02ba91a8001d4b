"""Row ends that are no aligned int32 are refused by every entry that reads them, before any device work."""
import ctypes

import pytest

from nanochat_cpp_b200 import capi

lib = capi.lib
PTR = 1 << 20  # any aligned address: refused calls never follow it


@pytest.mark.parametrize("off", [1, 2, 3])
def test_quantizer(off):
    assert lib.mxb200_block_quantize(PTR, 4, 128, 128, PTR + off, 2, PTR, PTR, 0, PTR, PTR, None) == capi.ERR_ALIGNMENT


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("kind", range(5))
def test_product(off, kind):
    args = capi.BlockGemmArgs(PTR, PTR, PTR, PTR, PTR, PTR + off, 8, 128, 128, 2, kind, capi.OUT_BF16, 0)
    assert lib.mxb200_block_gemm(ctypes.byref(args), None) == capi.ERR_ALIGNMENT
