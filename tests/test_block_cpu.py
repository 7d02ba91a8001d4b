"""The block-of-128 entry points of the C ABI, as far as they go without a GPU: what they refuse before any device work, in the
order of their checks, and the sizes that they state."""
import ctypes

import pytest

from nanochat_cpp_b200 import capi

lib = capi.lib
PTR = 1 << 20  # any aligned address: refused calls never follow it


def gemm(**change):
    a = dict(a=PTR, a_scale=PTR, b=PTR, b_scale=PTR, d=PTR, ends=None, tokens=8, in_features=128, out_features=128, experts=1,
             kind=capi.BLOCK_FORWARD, out_kind=capi.OUT_BF16, b_ld=0)
    a.update(change)
    args = capi.BlockGemmArgs(*(a[f[0]] for f in capi.BlockGemmArgs._fields_))
    return lib.mxb200_block_gemm(ctypes.byref(args), None)


@pytest.mark.parametrize("change,status", [
    (dict(kind=5), capi.ERR_ARGUMENT), (dict(kind=-1), capi.ERR_ARGUMENT), (dict(out_kind=2), capi.ERR_ARGUMENT),
    (dict(out_kind=capi.OUT_F32), capi.ERR_ARGUMENT),
    (dict(tokens=-1), capi.ERR_SHAPE), (dict(tokens=1 << 31), capi.ERR_SHAPE), (dict(in_features=0), capi.ERR_SHAPE),
    (dict(in_features=24), capi.ERR_SHAPE), (dict(out_features=8), capi.ERR_SHAPE), (dict(experts=0), capi.ERR_SHAPE),
    (dict(experts=1025, ends=PTR), capi.ERR_SHAPE), (dict(experts=2), capi.ERR_NULL),
    (dict(b_ld=128, kind=capi.BLOCK_INPUT_GRAD), capi.ERR_ARGUMENT), (dict(b_ld=112), capi.ERR_SHAPE), (dict(b_ld=132), capi.ERR_SHAPE),
    (dict(b_ld=128, kind=capi.BLOCK_FORWARD_SCALED), capi.ERR_ARGUMENT),
    (dict(kind=capi.BLOCK_FORWARD_SCALED, out_kind=capi.OUT_F32), capi.ERR_ARGUMENT),
])
def test_gemm_refusals(change, status):
    assert gemm(**change) == status


@pytest.mark.parametrize("rows,cols,ld,ends,experts,status", [
    (-1, 128, 128, None, 1, capi.ERR_SHAPE), (4, 120, 128, None, 1, capi.ERR_SHAPE), (4, 128, 112, None, 1, capi.ERR_SHAPE),
    (4, 128, 132, None, 1, capi.ERR_SHAPE), (4, 0, 128, None, 1, capi.ERR_SHAPE), (4, 128, 128, PTR, 1025, capi.ERR_SHAPE),
    (4, 128, 128, None, 2, capi.ERR_NULL), (0, 128, 128, None, 1, capi.OK),
])
def test_quantizer_refusals(rows, cols, ld, ends, experts, status):
    assert lib.mxb200_block_quantize(PTR, rows, cols, ld, ends, experts, PTR, PTR, 0, None, None, None) == status


def test_quantizer_needs_an_output():
    assert lib.mxb200_block_quantize(PTR, 4, 128, 128, None, 1, None, None, 0, None, None, None) == capi.ERR_NULL
    assert lib.mxb200_block_quantize(PTR, 4, 128, 128, None, 1, PTR, PTR, 1, None, None, None) == capi.ERR_ARGUMENT


@pytest.mark.parametrize("experts,rows,cols", [(0, 128, 128), (1025, 128, 128), (1, 120, 128), (1, 128, 8), (1, 0, 128)])
def test_weight_quantizer_refusals(experts, rows, cols):
    assert lib.mxb200_block_quantize_weight(PTR, 1, experts, rows, cols, PTR, PTR, 0, None) == capi.ERR_SHAPE


@pytest.mark.parametrize("rows,cols,status", [(4, 24, capi.ERR_SHAPE), (4, 16400, capi.ERR_SHAPE), (-1, 128, capi.ERR_SHAPE),
                                              (0, 128, capi.OK)])
def test_norm_refusals(rows, cols, status):
    args = capi.BlockNormArgs(PTR, None, None, None, None, PTR, PTR, PTR, rows, cols, 0, 1e-5)
    assert lib.mxb200_block_norm_fwd(ctypes.byref(args), None) == status
    if status != capi.OK:
        back = capi.BlockNormBwdArgs(PTR, None, PTR, PTR, None, PTR, None, rows, cols, 0)
        assert lib.mxb200_block_norm_bwd(ctypes.byref(back), None, 0, None) == status


def test_null_arguments():
    assert lib.mxb200_block_gemm(None, None) == capi.ERR_NULL
    assert lib.mxb200_block_norm_fwd(None, None) == capi.ERR_NULL
    assert lib.mxb200_block_norm_bwd(None, None, 0, None) == capi.ERR_NULL


def test_token_blocks_bound_every_split_into_experts():
    import random
    rng = random.Random(0)
    for _ in range(300):
        experts, tokens = rng.randint(1, 40), rng.choice([0, 1, 5, 127, 128, 129, rng.randint(0, 5000)])
        cuts = sorted(rng.randint(0, tokens) for _ in range(experts))
        need = sum(-(-(b - a) // 128) for a, b in zip([0] + cuts[:-1], cuts))
        assert need <= lib.mxb200_block_token_blocks(tokens, experts)
    assert lib.mxb200_block_token_blocks(1000, 1) == 8 and lib.mxb200_block_token_blocks(0, 4) == 0
