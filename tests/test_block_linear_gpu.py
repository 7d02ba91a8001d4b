"""The Linear and the experts' Linears in blocks of 128, and their quantizers, against plain 64-bit forms."""
import pytest
import torch

import block_ref as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16 = torch.finfo(torch.bfloat16).eps / 2


@pytest.fixture(scope="module")
def nc():
    import nanochat_cpp_b200 as nc
    return nc


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def activation(g, rows, cols):
    return (torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))).bfloat16()


def given_weight(nc, g, *shape):
    """A quantized checkpoint's weight: any scales."""
    n, k = shape[-2:]
    data = (100 * torch.randn(*shape, device="cuda", generator=g)).clamp(-448, 448).to(E4M3)
    scale = 1e-3 * (0.5 + torch.rand(*shape[:-2], -(-n // 128), -(-k // 128), device="cuda", generator=g))
    return nc.BlockTensor(data, scale)


def assert_close(got, want, slack, what):
    """Within `slack` and one rounding to got's type of the 64-bit value."""
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    bound = slack + half * (want.abs() + slack)
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound.clamp(min=1e-300)).max()):.3g} of its bound"


def assert_product(got, a, b, what):
    """got = a . b^T"""
    assert_close(got, a @ b.t(), ref.product_bound(a.size(1), a.abs() @ b.abs().t()), what)


# ------------------------------------------------------------------------------------------------ quantizers

@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 1536), (3, 128), (127, 144), (128, 256), (300, 1040), (513, 2000)])
def test_rows_are_exact(nc, rows, cols):
    x = activation(generator(1), rows, cols)
    if rows > 2:
        x[0] = 0
        x[1, 5], x[1, 6] = float("nan"), float("inf")
        x[2] = 1.75 * 2.0 ** -130  # the smallest scale
    q = nc.quantize_block(x)
    data, scale = ref.rows(x)
    assert q.data.dtype == E4M3 and q.scale.shape == (-(-cols // 128), rows)
    assert torch.equal(q.scale.double(), scale)
    assert torch.equal(torch.nan_to_num(q.data.double(), nan=1e9), torch.nan_to_num(data, nan=1e9))


@pytest.mark.parametrize("shape", [(16, 16), (128, 128), (144, 400), (3, 256, 272), (2, 1040, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_are_exact(nc, shape, dtype):
    w = torch.randn(*shape, device="cuda", generator=generator(2)).to(dtype)
    w[..., :3, :] *= 50
    q = nc.quantize_block_weight(w)
    for e in range(shape[0] if len(shape) == 3 else 1):
        data, scale = ref.weight(w[e] if len(shape) == 3 else w)
        assert torch.equal((q.data[e] if len(shape) == 3 else q.data).double(), data)
        assert torch.equal((q.scale[e] if len(shape) == 3 else q.scale).double(), scale)


def test_rows_of_a_strided_and_of_a_misaligned_view(nc):
    x = activation(generator(3), 40, 512)
    for v in (x[:, 64:320], x[::2, :256], x[1:, 3:259], x.t()[:16 * 8, :16].contiguous().t()[:, :128]):
        q, p = nc.quantize_block(v), nc.quantize_block(v.clone(memory_format=torch.contiguous_format))
        assert torch.equal(q.data.view(torch.uint8), p.data.view(torch.uint8)) and torch.equal(q.scale, p.scale)


# ------------------------------------------------------------------------------------------------ dense

TOKENS = [1, 2, 17, 64, 127, 128, 129, 200, 257, 700]
FEATURES = [(16, 16), (128, 128), (144, 272), (1536, 1536), (400, 2064), (2064, 400)]


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("cin,cout", FEATURES)
def test_forward(nc, tokens, cin, cout):
    g = generator(4)
    x, w = activation(g, tokens, cin), given_weight(nc, g, cout, cin)
    y = nc.fp8_block_matmul(x, w)
    assert y.shape == (tokens, cout) and y.dtype == torch.bfloat16
    assert_product(y, ref.row_values(x), ref.weight_values(w.data, w.scale), "y")
    again = nc.fp8_block_matmul(None, w, x_block=nc.quantize_block(x))
    assert torch.equal(y, again)


@pytest.mark.parametrize("tokens", [1, 2, 5, 8, 15, 16])
@pytest.mark.parametrize("cin,cout", [(16, 16), (144, 272), (1536, 1536), (2064, 400), (6144, 128)])
def test_quantized_by_the_product(nc, tokens, cin, cout):
    """The C entry that takes bf16 rows: the bits of quantizing first, dense and by expert."""
    import ctypes
    g, capi = generator(16), nc.capi
    x, w = activation(g, tokens, 2 * cin), given_weight(nc, g, 2, cout, cin)
    x[0, 0], x[-1, 3] = float("nan"), float("inf")
    for experts, ends in ((1, None), (2, ends_of([tokens // 3, tokens // 2]))):
        data, scale = w.data[:experts].contiguous(), w.scale[:experts].contiguous()
        got = torch.full((tokens, cout), 7.0, device="cuda", dtype=torch.bfloat16)
        args = capi.BlockGemmArgs(data.data_ptr(), scale.data_ptr(), x.data_ptr(), None, got.data_ptr(),
                                  ends.data_ptr() if ends is not None else None, tokens, cin, cout, experts, capi.BLOCK_FORWARD,
                                  capi.OUT_BF16, 2 * cin)
        capi.check(capi.lib.mxb200_block_gemm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "block_gemm")
        q, weight = nc.quantize_block(x[:, :cin]), nc.BlockTensor(data, scale)
        want = nc.fp8_block_experts(None, weight, ends, x_block=q) if experts > 1 else nc.fp8_block_matmul(
            None, nc.BlockTensor(data[0], scale[0]), x_block=q)
        assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))


@pytest.mark.parametrize("counts", [[0, 1, 2, 0] * 20, [40, 0, 70, 3], [33] * 3], ids=str)
def test_experts_quantized_by_the_product(nc, counts):
    """More rows than the small tile has, in the C entry that quantizes them; and what the experts' call takes by itself."""
    import ctypes
    g, capi, cin, cout = generator(19), nc.capi, 272, 400
    rows, ends = sum(counts) + 5, ends_of(counts)
    x, w = activation(g, rows, cin), given_weight(nc, g, len(counts), cout, cin)
    got = torch.full((rows, cout), 7.0, device="cuda", dtype=torch.bfloat16)
    args = capi.BlockGemmArgs(w.data.data_ptr(), w.scale.data_ptr(), x.data_ptr(), None, got.data_ptr(), ends.data_ptr(), rows, cin, cout,
                              len(counts), capi.BLOCK_FORWARD, capi.OUT_BF16, cin)
    capi.check(capi.lib.mxb200_block_gemm(ctypes.byref(args), torch.cuda.current_stream().cuda_stream), "block_gemm")
    called = nc.fp8_block_experts(x, w, ends)
    xr = ref.row_values(x)
    for y in (got, called):
        for e, (a, b) in enumerate(ref.spans(ends.tolist(), rows)):
            if b > a:
                assert_product(y[a:b], xr[a:b], ref.weight_values(w.data[e], w.scale[e]), f"y of expert {e}")
        assert not y[sum(counts):].any()


@pytest.mark.parametrize("tokens,cin,cout,experts", [
    (1, 1536, 1536, 1), (16, 1536, 400, 1), (100, 128, 144, 1), (40, 272, 640, 1), (32, 1536, 272, 16), (24, 272, 400, 80), (200, 128, 128, 40)])
def test_bits_do_not_depend_on_who_quantizes(nc, tokens, cin, cout, experts):
    g = generator(23)
    assert nc.capi.lib.mxb200_block_quantizes(tokens, cin, cout, experts)
    x, w = activation(g, tokens, cin), given_weight(nc, g, experts, cout, cin)
    if experts == 1:
        w = nc.BlockTensor(w.data[0], w.scale[0])
        assert torch.equal(nc.fp8_block_matmul(x, w), nc.fp8_block_matmul(None, w, x_block=nc.quantize_block(x)))
    else:
        ends = torch.sort(torch.randint(0, tokens + 1, (experts,), generator=g, device="cuda")).values.int()
        assert torch.equal(nc.fp8_block_experts(x, w, ends), nc.fp8_block_experts(None, w, ends, x_block=nc.quantize_block(x)))


@pytest.mark.parametrize("tokens", [1, 16, 129, 384, 1000])
@pytest.mark.parametrize("cin,cout", [(16, 16), (272, 144), (128, 640), (1040, 2000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(nc, tokens, cin, cout, dtype):
    g = generator(5)
    x = activation(g, tokens, cin).requires_grad_()
    w = torch.randn(cout, cin, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = (0.01 * torch.randn(tokens, cout, device="cuda", generator=g)).bfloat16()
    y = nc.fp8_block_matmul(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wv = ref.weight_values(*ref.weight(w.detach()))
    assert_product(y.detach(), ref.row_values(x.detach()), wv, "y")
    assert dx.dtype == torch.bfloat16 and dw.dtype == dtype
    assert_product(dx, ref.row_values(dy), wv.t(), "dx")
    assert_product(dw, ref.tokens(dy)[0].t(), ref.tokens(x.detach())[0].t(), "dw")


@pytest.mark.parametrize("cin,cout", [(640, 1552), (1040, 2000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_scaled_by_the_tensor_core(nc, cin, cout, dtype):
    tokens, g = 5001, generator(17)
    assert nc.capi.lib.mxb200_block_scaled(tokens, cin, cout, 1)
    x = activation(g, tokens, cin).requires_grad_()
    w = torch.randn(cout, cin, device="cuda", generator=g).to(dtype).requires_grad_()
    dy = (0.01 * torch.randn(tokens, cout, device="cuda", generator=g)).bfloat16()
    y = nc.fp8_block_matmul(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wv = ref.weight_values(*ref.weight(w.detach()))
    assert_product(y.detach(), ref.row_values(x.detach()), wv, "y")
    assert_product(dx, ref.row_values(dy), wv.t(), "dx")
    assert_product(dw, ref.tokens(dy)[0].t(), ref.tokens(x.detach())[0].t(), "dw")
    # only one of the gradients wanted
    one = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(nc.fp8_block_matmul(x.detach(), one), one, dy)[0], dw)
    one = x.detach().requires_grad_()
    assert_product(torch.autograd.grad(nc.fp8_block_matmul(one, w.detach()), one, dy)[0], ref.row_values(dy), wv.t(), "dx")


def test_long_sums_do_not_lose_precision(nc):
    """The tensor core cuts its running sums off, an error that grows with their length; beyond 4096 tokens they go on in
    registers, so that 16384 tokens' gradient is as good as 4096's (and 4500's last segment is short)."""
    def error(tokens):
        g = generator(tokens)
        x = torch.randn(tokens, 256, device="cuda", generator=g).bfloat16()
        w = torch.randn(256, 256, device="cuda", generator=g).requires_grad_()
        dy = torch.randn(tokens, 256, device="cuda", generator=g).bfloat16()
        dw, = torch.autograd.grad(nc.fp8_block_matmul(x, w), w, dy)
        want = ref.tokens(dy)[0].t() @ ref.tokens(x)[0]
        return float((dw.double() - want).norm() / want.norm())
    short = error(4096)
    assert error(4500) <= 1.5 * short and error(16384) <= 1.5 * short


def test_only_the_wanted_gradients(nc):
    g = generator(6)
    x, w = activation(g, 70, 256), torch.randn(128, 256, device="cuda", generator=g)
    dy = torch.randn(70, 128, device="cuda", generator=g).bfloat16()
    both_x, both_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(nc.fp8_block_matmul(both_x, both_w), (both_x, both_w), dy)
    one_x, one_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(nc.fp8_block_matmul(one_x, w), one_x, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(nc.fp8_block_matmul(x, one_w), one_w, dy)[0], dw)
    # blocks of the input and of the weight made beforehand: the same bits
    q, cache = nc.quantize_block(x), nc.Fp8WeightCache(True)
    for _ in range(2):
        one_x, one_w = x.clone().requires_grad_(), both_w.detach().requires_grad_()
        got = torch.autograd.grad(nc.fp8_block_matmul(one_x, one_w, x_block=q, cache=cache), (one_x, one_w), dy)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    frozen = nc.quantize_block_weight(w)
    one_x = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(nc.fp8_block_matmul(one_x, frozen), one_x, dy)[0], dx)


def test_an_expanded_gradient(nc):
    g = generator(7)
    x, w = activation(g, 33, 128).requires_grad_(), torch.randn(144, 128, device="cuda", generator=g).requires_grad_()
    nc.fp8_block_matmul(x, w).sum().backward()
    dx, dw = torch.autograd.grad(nc.fp8_block_matmul(x, w), (x, w), torch.ones(33, 144, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


def test_differences(nc):
    """On inputs whose blocks hold their values exactly, with steps that stay so, the product is linear: differences are exact."""
    g = generator(8)
    x = torch.randint(-4, 5, (40, 256), device="cuda", generator=g).bfloat16()
    x[:, ::128] = 256  # scale 1: small integers are E4M3 values
    w = torch.randint(-1, 2, (48, 256), device="cuda", generator=g).float()
    w[0, 0], w[0, 128] = 256, 256
    w[:, ::128] *= (w[:, ::128].abs() > 1)  # the 256s of x meet zeros, but for one feature: y stays small and exact
    dy = torch.zeros(40, 48, device="cuda", dtype=torch.bfloat16)
    xg = x.clone().requires_grad_()
    for f in (1, 17, 47):
        dy.zero_()
        dy[:, f] = 1.0
        dx, = torch.autograd.grad(nc.fp8_block_matmul(xg, w), xg, dy)
        for c in (1, 100, 129, 255):
            up, down = x.clone(), x.clone()
            up[:, c] += 1
            down[:, c] -= 1
            diff = (nc.fp8_block_matmul(up, w).float() - nc.fp8_block_matmul(down, w).float())[:, f] / 2
            assert torch.equal(diff, dx[:, c].float())


def test_nan_and_inf_stay_in_their_rows(nc):
    g = generator(9)
    x, w = activation(g, 130, 256), given_weight(nc, g, 256, 256)
    clean = nc.fp8_block_matmul(x, w)
    x[3, 7], x[129, 200] = float("nan"), float("inf")
    y = nc.fp8_block_matmul(x, w)
    assert torch.isnan(y[3]).all()
    keep = [r for r in range(130) if r not in (3, 129)]
    assert torch.equal(y[keep], clean[keep])


def test_no_tokens(nc):
    w = torch.randn(128, 64, device="cuda").requires_grad_()
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = nc.fp8_block_matmul(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 128) and dx.shape == (0, 64) and not dw.any()
    q = nc.quantize_block(x.detach())
    assert q.data.shape == (0, 64) and q.scale.shape == (1, 0)


def test_the_same_bits_again_and_on_another_stream(nc):
    g = generator(10)
    x, w = activation(g, 1000, 1040), torch.randn(2000, 1040, device="cuda", generator=g)
    dy = torch.randn(1000, 2000, device="cuda", generator=g).bfloat16()

    def step():
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = nc.fp8_block_matmul(a, b)
        return [y.detach(), *torch.autograd.grad(y, (a, b), dy)]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        third = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


# ------------------------------------------------------------------------------------------------ experts

COUNTS = [
    [5],
    [0, 0, 0],
    [1, 0, 128, 0, 129],
    [127, 1, 300, 0, 0, 64, 2, 511],
    [1] * 40,
    [0, 700, 0, 31],
    [3, 0] * 64,
]


def ends_of(counts):
    return torch.tensor(counts, device="cuda").cumsum(0).to(torch.int32)


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("tail", [0, 3, 200])
@pytest.mark.parametrize("cin,cout", [(16, 16), (272, 144), (640, 400)])
def test_experts(nc, counts, tail, cin, cout):
    g = generator(11)
    rows, ends = sum(counts) + tail, ends_of(counts)
    x = activation(g, rows, cin).requires_grad_()
    w = torch.randn(len(counts), cout, cin, device="cuda", generator=g).requires_grad_()
    dy = (0.01 * torch.randn(rows, cout, device="cuda", generator=g)).bfloat16()
    y = nc.fp8_block_experts(x, w, ends)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    given = given_weight(nc, g, len(counts), cout, cin)
    served = nc.fp8_block_experts(x.detach(), given, ends)
    xr, gr = ref.row_values(x.detach()), ref.row_values(dy)
    for e, (a, b) in enumerate(ref.spans(ends.tolist(), rows)):
        wv = ref.weight_values(*ref.weight(w[e].detach()))
        if b > a:
            assert_product(y[a:b].detach(), xr[a:b], wv, f"y of expert {e}")
            assert_product(dx[a:b], gr[a:b], wv.t(), f"dx of expert {e}")
            assert_product(dw[e], ref.tokens(dy[a:b])[0].t(), ref.tokens(x[a:b].detach())[0].t(), f"dw of expert {e}")
            assert_product(served[a:b], xr[a:b], ref.weight_values(given.data[e], given.scale[e]), f"served by expert {e}")
        else:
            assert not dw[e].any()
    last = sum(counts)
    assert not y[last:].any() and not dx[last:].any() and not served[last:].any()


@pytest.mark.parametrize("tail", [0, 77])
def test_experts_scaled_by_the_tensor_core(nc, tail):
    counts, cin, cout, g = [700, 0, 1, 129, 2000, 300, 256, 900, 1200, 0], 1040, 2000, generator(18)
    rows, ends = sum(counts) + tail, ends_of(counts)
    assert nc.capi.lib.mxb200_block_scaled(rows, cin, cout, len(counts))
    x = activation(g, rows, cin).requires_grad_()
    w = torch.randn(len(counts), cout, cin, device="cuda", generator=g).requires_grad_()
    dy = (0.01 * torch.randn(rows, cout, device="cuda", generator=g)).bfloat16()
    y = nc.fp8_block_experts(x, w, ends)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xr, gr = ref.row_values(x.detach()), ref.row_values(dy)
    for e, (a, b) in enumerate(ref.spans(ends.tolist(), rows)):
        wv = ref.weight_values(*ref.weight(w[e].detach()))
        if b > a:
            assert_product(y[a:b].detach(), xr[a:b], wv, f"y of expert {e}")
            assert_product(dx[a:b], gr[a:b], wv.t(), f"dx of expert {e}")
            assert_product(dw[e], ref.tokens(dy[a:b])[0].t(), ref.tokens(x[a:b].detach())[0].t(), f"dw of expert {e}")
        else:
            assert not dw[e].any()
    assert not y[sum(counts):].any() and not dx[sum(counts):].any()


def test_one_expert_is_the_dense_linear(nc):
    g = generator(12)
    x, w = activation(g, 333, 272), torch.randn(1, 400, 272, device="cuda", generator=g)
    dy = torch.randn(333, 400, device="cuda", generator=g).bfloat16()
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = nc.fp8_block_experts(a, b, ends_of([333]))
    got = torch.autograd.grad(y, (a, b), dy)
    c, d = x.clone().requires_grad_(), w[0].clone().requires_grad_()
    z = nc.fp8_block_matmul(c, d)
    want = torch.autograd.grad(z, (c, d), dy)
    assert torch.equal(y, z) and torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1])


@pytest.mark.parametrize("ends", [[50, 20, 70], [-5, 30, 1000], [0, 0, 2 ** 31 - 1], [90, 10, 10]])
def test_ends_out_of_order_or_range_count_as_their_bounds(nc, ends):
    g = generator(13)
    x, w = activation(g, 90, 128), given_weight(nc, g, 3, 256, 128)
    y = nc.fp8_block_experts(x, w, torch.tensor(ends, device="cuda", dtype=torch.int32))
    good = torch.tensor([b for _, b in ref.spans(ends, 90)], device="cuda", dtype=torch.int32)
    assert torch.equal(y, nc.fp8_block_experts(x, w, good))
    assert not y[int(good[-1]):].any()


def test_most_experts(nc):
    g = generator(14)
    counts = torch.randint(0, 3, (1024,), generator=torch.Generator().manual_seed(3)).tolist()
    rows = sum(counts)
    x = activation(g, rows, 128).requires_grad_()
    w = torch.randn(1024, 48, 128, device="cuda", generator=g).bfloat16().requires_grad_()
    dy = torch.randn(rows, 48, device="cuda", generator=g).bfloat16()
    y = nc.fp8_block_experts(x, w, ends_of(counts))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xr, gr = ref.row_values(x.detach()), ref.row_values(dy)
    for e, (a, b) in enumerate(ref.spans(ends_of(counts).tolist(), rows)):
        if b > a and (e < 40 or e > 1000):
            wv = ref.weight_values(*ref.weight(w[e].detach()))
            assert_product(y[a:b].detach(), xr[a:b], wv, f"y of expert {e}")
            assert_product(dx[a:b], gr[a:b], wv.t(), f"dx of expert {e}")
            assert_product(dw[e], ref.tokens(dy[a:b])[0].t(), ref.tokens(x[a:b].detach())[0].t(), f"dw of expert {e}")
        elif b == a:
            assert not dw[e].any()


# ------------------------------------------------------------------------------------------------ graphs

def test_captured_and_replayed_with_other_counts(nc):
    """A captured training pass over experts, replayed on new inputs and row counts. (No eager graph of the same leaves may live
    while a backward is captured: torch then ties the capture to that graph's stream and refuses it, whatever the operators.)"""
    g = generator(15)
    x = activation(g, 300, 256).requires_grad_()
    w = torch.randn(4, 144, 256, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(300, 144, device="cuda", generator=g).bfloat16()
    ends = ends_of([100, 0, 150, 50])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(nc.fp8_block_experts(x, w, ends), (x, w), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = nc.fp8_block_experts(x, w, ends)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    for counts in ([100, 0, 150, 50], [0, 299, 0, 1], [10, 20, 30, 40]):
        with torch.no_grad():
            ends.copy_(ends_of(counts))
            x.copy_(activation(g, 300, 256))
        graph.replay()
        a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        z = nc.fp8_block_experts(a, b, ends.clone())
        want = torch.autograd.grad(z, (a, b), dy)
        assert torch.equal(y, z) and torch.equal(dx, want[0]) and torch.equal(dw, want[1])

# ------------------------------------------------------------------------------------------------ refusals

def test_refusals(nc):
    x, w = torch.zeros(8, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(64, 128, device="cuda")
    ends, w3 = torch.tensor([4, 8], device="cuda", dtype=torch.int32), torch.zeros(2, 64, 128, device="cuda")
    bad = [
        lambda: nc.fp8_block_matmul(x.float(), w),
        lambda: nc.fp8_block_matmul(x.half(), w),
        lambda: nc.fp8_block_matmul(x, w.half()),
        lambda: nc.fp8_block_matmul(x[:, :120], w[:, :120]),
        lambda: nc.fp8_block_matmul(x, w[:24]),
        lambda: nc.fp8_block_matmul(x, w[:, :64]),
        lambda: nc.fp8_block_matmul(x[0], w),
        lambda: nc.fp8_block_matmul(x, w3),
        lambda: nc.fp8_block_matmul(x.cpu(), w),
        lambda: nc.fp8_block_matmul(x, w.cpu()),
        lambda: nc.fp8_block_matmul(None, w),
        lambda: nc.fp8_block_matmul(None, w.requires_grad_(), x_block=nc.quantize_block(x)),
        lambda: nc.fp8_block_matmul(x, nc.BlockTensor(w.detach().to(E4M3), torch.ones(1, 2, device="cuda"))),
        lambda: nc.fp8_block_matmul(x, nc.BlockTensor(w.detach().to(E4M3), torch.ones(1, 1, device="cuda", dtype=torch.bfloat16))),
        lambda: nc.fp8_block_matmul(x, w.detach(), x_block=nc.quantize_block(x[:4])),
        lambda: nc.fp8_block_experts(x, w.detach(), ends),
        lambda: nc.fp8_block_experts(x, w3, ends.long()),
        lambda: nc.fp8_block_experts(x, w3, ends[:1]),
        lambda: nc.fp8_block_experts(x, w3, ends.cpu()),
        lambda: nc.fp8_block_experts(x, w3, ends.repeat(2)[::2]),
        lambda: nc.quantize_block(x.float()),
        lambda: nc.quantize_block(x[:, :8]),
        lambda: nc.quantize_block_weight(w.detach()[0]),
        lambda: nc.quantize_block_weight(w.detach().half()),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was taken")
    torch.cuda.synchronize()


def test_a_second_derivative_is_refused(nc):
    x = torch.randn(16, 128, device="cuda").bfloat16().requires_grad_()
    y = nc.fp8_block_matmul(x, torch.randn(128, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
