"""Each kernel of the products in blocks of 128 against the 64-bit form, at sizes that are known to reach it: the test asks which
kernel a call takes before it looks at the result."""
import ctypes

import pytest
import torch

import block_ref as ref
from test_block_linear_gpu import activation, assert_product, ends_of, generator, given_weight, nc  # noqa: F401

pytestmark = pytest.mark.gpu

# last rows of an expert's tiles: 1, 31, 33, 129, 255 of 256, 1, 31, 33, 1, 127 of 128, whole tiles, none
RAGGED = [1, 31, 33, 129, 255, 0, 257, 512]

# (kernel, CTAs that share a tile's contraction), contraction, features, tokens or rows by expert, rows behind the last expert's
CASES = [
    (("32", 1), 2064, 1040, 70, 0),
    (("32", 1), 528, 2064, [1, 31, 33, 129, 255, 0, 64, 97, 32], 127),
    (("32", 8), 6144, 272, 40, 0),
    (("32", 3), 8192, 528, 200, 0),
    (("32", 8), 6144, 272, [31, 0, 33], 36),
    (("few", 1), 1040, 2064, 1001, 0),
    (("few", 1), 400, 4112, 2049, 0),
    (("few", 2), 6144, 1536, 700, 0),    # the last tile has 60 rows: one half of its columns
    (("few", 2), 6144, 1536, 741, 0),    # 101: both
    (("few", 2), 6144, 1536, 768, 0),
    (("few", 1), 528, 2064, [*RAGGED, 443], 77),
    (("few", 3), 6144, 528, [129, 0, 481, 255], 135),
    (("few", 3), 6144, 528, [33, 1, 31, 860], 75),
    (("many", 1), 1664, 6656, 3001, 0),
    (("many", 1), 272, 2064, 1111, 0),
    (("many", 1), 528, 2064, [*RAGGED, 700, 600], 82),
    (("many", 1), 528, 2064, [1, 31, 33, 129, 255, 0, 64, 97], 127),
    (("many", 1), 144, 4112, [255, 1, 31, 0, 129, 33, 1400, 256, 511], 384),
]


@pytest.mark.parametrize("kernel,contraction,features,counts,tail", CASES, ids=lambda v: f"{len(v)}x{sum(v)}" if isinstance(v, list) else str(v))
@pytest.mark.parametrize("kind", ["forward", "input_grad"])
def test_given_scales(nc, kernel, contraction, features, counts, tail, kind):  # noqa: F811
    g, capi, forward = generator(1), nc.capi, kind == "forward"
    dense = isinstance(counts, int)
    tokens, experts = (counts, 1) if dense else (sum(counts) + tail, len(counts))
    ends = None if dense else ends_of(counts)
    cin, cout = (contraction, features) if forward else (features, contraction)
    x, w = activation(g, tokens, contraction), given_weight(nc, g, experts, cout, cin)
    q = nc.quantize_block(x)
    y = torch.full((tokens, features), 7.0, device="cuda", dtype=torch.bfloat16)
    args = capi.BlockGemmArgs(w.data.data_ptr(), w.scale.data_ptr(), q.data.data_ptr(), q.scale.data_ptr(), y.data_ptr(),
                              None if dense else ends.data_ptr(), tokens, cin, cout, experts,
                              capi.BLOCK_FORWARD if forward else capi.BLOCK_INPUT_GRAD, capi.OUT_BF16, 0)
    splits = ctypes.c_int()
    name = capi.lib.mxb200_block_gemm_kernel(ctypes.byref(args), ctypes.byref(splits)).decode()
    assert (name, splits.value) == (f"{kind}_{kernel[0]}", kernel[1])
    capi.check(capi.lib.mxb200_block_gemm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "block_gemm")
    xv = ref.row_values(x)
    for e, (a, b) in enumerate([(0, tokens)] if dense else ref.spans(ends.tolist(), tokens)):
        wv = ref.weight_values(w.data[e], w.scale[e])
        if b > a:
            assert_product(y[a:b], xv[a:b], wv if forward else wv.t(), f"rows of expert {e}")
    if not dense:
        assert not y[sum(counts):].any()
    again = torch.empty_like(y)
    args.d = again.data_ptr()
    capi.check(capi.lib.mxb200_block_gemm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "block_gemm")
    assert torch.equal(again, y) and capi.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,kernel", [([4500, 0, 8300, 1, 4096, 4097], "weight_grad_long"), ([1300, 0, 129, 1, 2600], "weight_grad")],
                         ids=["long", "short"])
def test_weight_gradients_of_several_experts(nc, counts, kernel, dtype):  # noqa: F811
    """Sums of none, one, part of one and several segments side by side."""
    tokens, cin, cout, g, capi = sum(counts) + 50, 272, 400, generator(2), nc.capi
    args = capi.BlockGemmArgs(None, None, None, None, None, None, tokens, cin, cout, len(counts), capi.BLOCK_WEIGHT_GRAD, capi.OUT_F32, 0)
    assert capi.lib.mxb200_block_gemm_kernel(ctypes.byref(args), None).decode() == kernel
    x = activation(g, tokens, cin)
    w = torch.randn(len(counts), cout, cin, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = (0.01 * torch.randn(tokens, cout, device="cuda", generator=g)).bfloat16()
    ends = ends_of(counts)
    dw, = torch.autograd.grad(nc.fp8_block_experts(x, w, ends), w, dy)
    for e, (a, b) in enumerate(ref.spans(ends.tolist(), tokens)):
        if b > a:
            assert_product(dw[e], ref.tokens(dy[a:b])[0].t(), ref.tokens(x[a:b])[0].t(), f"dw of expert {e}")
        else:
            assert not dw[e].any()


def test_which_kernel_is_asked_for(nc):  # noqa: F811
    capi = nc.capi

    def name(tokens, kind, b_ld=0, out=capi.OUT_BF16, features=1536):
        args = capi.BlockGemmArgs(None, None, None, None, None, None, tokens, 1536, features, 1, kind, out, b_ld)
        got = capi.lib.mxb200_block_gemm_kernel(ctypes.byref(args), None)
        return got.decode() if got is not None else None
    assert name(1, capi.BLOCK_FORWARD, 1536) == "quantize_few" and name(1, capi.BLOCK_FORWARD) == "forward_32"
    assert name(16384, capi.BLOCK_FORWARD_SCALED) == "forward_scaled" and name(16384, capi.BLOCK_INPUT_GRAD_SCALED) == "input_grad_scaled"
    assert name(4096, capi.BLOCK_WEIGHT_GRAD, out=capi.OUT_F32) == "weight_grad"
    assert name(4097, capi.BLOCK_WEIGHT_GRAD) == "weight_grad_long"
    # what the product refuses
    assert name(0, capi.BLOCK_FORWARD) is None and name(1, 9) is None and name(1, capi.BLOCK_FORWARD, out=capi.OUT_F32) is None
    assert name(1, capi.BLOCK_FORWARD, features=24) is None and name(-1, capi.BLOCK_FORWARD) is None
