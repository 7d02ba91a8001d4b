"""The residual RMS norm with its result in blocks of 128, its backward, and the path norm -> Linear / experts -> back."""
import pytest
import torch

import block_ref as ref
from test_block_linear_gpu import activation, assert_close, assert_product, ends_of, generator, given_weight, nc  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


def reference(x, r, gain, eps):
    res = (x.float() + r.float()).bfloat16() if r is not None else x
    v = res.double()
    rstd = 1 / torch.sqrt(v.square().mean(-1) + eps)
    hat = v * rstd[..., None]
    return res, rstd, hat, hat * gain.double() if gain is not None else hat


SHAPES = [(1, 16), (1, 1536), (3, 144), (7, 512), (33, 528), (64, 1024), (129, 1040), (50, 1552), (300, 2048), (5, 2064), (40, 5040),
          (9, 8192), (3, 16384), (1000, 128)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("add", [True, False])
@pytest.mark.parametrize("gain_type", [None, torch.float32, torch.bfloat16])
def test_forward_and_backward(nc, rows, cols, add, gain_type):  # noqa: F811
    g, eps = generator(1), 1e-5
    x = activation(g, rows, cols).requires_grad_()
    r = torch.randn(rows, cols, device="cuda", generator=g).bfloat16().requires_grad_() if add else None
    gain = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(gain_type).requires_grad_() if gain_type is not None else None
    dn = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    dres = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    res, n, q, rstd = nc.residual_norm_block(x, r, gain, eps=eps)
    want_res, want_rstd, hat, want_n = reference(x.detach(), r.detach() if add else None, gain.detach() if gain is not None else None, eps)
    assert torch.equal(res, want_res)
    # at most 64 squares in a thread and 13 sums of threads: each a rounding of a positive sum, halved by the root
    assert ((rstd.double() - want_rstd).abs() <= 43 * U * want_rstd).all()
    assert_close(n.detach(), want_n, 46 * U * want_n.abs(), "n")
    again = nc.quantize_block(n.detach())
    assert torch.equal(q.data.view(torch.uint8), again.data.view(torch.uint8)) and torch.equal(q.scale, again.scale)
    with torch.no_grad():
        bare = nc.residual_norm_block(x, r, gain, eps=eps, with_n=False)
    assert bare[1] is None and torch.equal(bare[0], res) and torch.equal(bare[2].data.view(torch.uint8), q.data.view(torch.uint8))

    inputs = [t for t in (x, r, gain) if t is not None]
    grads = torch.autograd.grad((res, n), inputs, (dres, dn))
    d = dn.double() * (gain.detach().double() if gain is not None else 1.0)
    mean, size = (d * hat).mean(-1, keepdim=True), (d * hat).abs().mean(-1, keepdim=True)
    scale = want_rstd[:, None]
    slack = U * (200 * scale * (d.abs() + hat.abs() * size) + 4 * dres.double().abs())
    assert_close(grads[0], scale * (d - hat * mean) + dres.double(), slack, "dx")
    if add:
        assert torch.equal(grads[1], grads[0])
    if gain is not None:
        terms = dn.double() * hat
        assert grads[-1].dtype == gain_type
        assert_close(grads[-1], terms.sum(0), (rows + 100) * U * terms.abs().sum(0), "dgain")


def test_gradients_by_differences(nc):  # noqa: F811
    """Directional differences of the 64-bit form against the kernel's gradients."""
    g, eps = generator(2), 1e-5
    x = activation(g, 20, 272).requires_grad_()
    r = torch.randn(20, 272, device="cuda", generator=g).bfloat16()
    gain = (1 + 0.2 * torch.randn(272, device="cuda", generator=g)).requires_grad_()
    dn, dres = (torch.randn(20, 272, device="cuda", generator=g).bfloat16() for _ in range(2))
    res, n, _, _ = nc.residual_norm_block(x, r, gain, eps=eps)
    dx, dgain = torch.autograd.grad((res, n), (x, gain), (dres, dn))

    def f(v, k):
        return ((v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * k * dn.double()).sum() + (v * dres.double()).sum())
    v, k, h = res.detach().double(), gain.detach().double(), 1e-5
    for _ in range(4):
        a = torch.randn(20, 272, device="cuda", generator=g).double()
        b = torch.randn(272, device="cuda", generator=g).double()
        by_x, by_k = (f(v + h * a, k) - f(v - h * a, k)) / (2 * h), (f(v, k + h * b) - f(v, k - h * b)) / (2 * h)
        # dx is rounded to bf16 (2^-8 of each term); differences are good to about 1e-7 of the sums
        assert abs(float((dx.double() * a).sum() - by_x)) <= float((dx.double() * a).abs().sum()) * (2.0 ** -8 + 1e-5)
        assert abs(float((dgain.double() * b).sum() - by_k)) <= float((dgain.double() * b).abs().sum()) * 1e-4


def test_only_one_of_the_outputs_is_used(nc):  # noqa: F811
    g = generator(3)
    x = activation(g, 10, 256).requires_grad_()
    gain = torch.ones(256, device="cuda").requires_grad_()
    dy = torch.randn(10, 256, device="cuda", generator=g).bfloat16()
    res, n, _, _ = nc.residual_norm_block(x, x.detach(), gain)
    dx, dgain = torch.autograd.grad(res, (x, gain), dy)
    assert torch.equal(dx, dy) and not dgain.any()
    res, n, _, _ = nc.residual_norm_block(x, x.detach(), gain)
    zero = torch.zeros_like(dy)
    a = torch.autograd.grad(n, x, dy)[0]
    res, n, _, _ = nc.residual_norm_block(x, x.detach(), gain)
    assert torch.equal(a, torch.autograd.grad((res, n), x, (zero, dy))[0])


def test_rows_of_zeros_and_leading_dimensions(nc):  # noqa: F811
    x = torch.zeros(2, 3, 144, device="cuda", dtype=torch.bfloat16)
    res, n, q, rstd = nc.residual_norm_block(x, eps=1e-6)
    assert n.shape == x.shape and q.data.shape == (6, 144) and rstd.shape == (6,)
    assert not n.any() and torch.allclose(rstd, torch.full_like(rstd, 1e3))
    empty = nc.residual_norm_block(x[:0].reshape(0, 144), x[:0].reshape(0, 144))
    assert empty[0].shape == (0, 144) and empty[2].scale.shape == (2, 0)


def test_refusals(nc):  # noqa: F811
    x = torch.zeros(4, 128, device="cuda", dtype=torch.bfloat16)
    wide = torch.zeros(1, 16400, device="cuda", dtype=torch.bfloat16)
    needs = x.clone().requires_grad_()
    bad = [
        lambda: nc.residual_norm_block(x.float()),
        lambda: nc.residual_norm_block(x[:, :24]),
        lambda: nc.residual_norm_block(wide),
        lambda: nc.residual_norm_block(x.cpu()),
        lambda: nc.residual_norm_block(x, x[:2]),
        lambda: nc.residual_norm_block(x, x.float()),
        lambda: nc.residual_norm_block(x, None, torch.ones(64, device="cuda")),
        lambda: nc.residual_norm_block(x, None, torch.ones(128, device="cuda", dtype=torch.float16)),
        lambda: nc.residual_norm_block(x, None, torch.ones(128)),
        lambda: nc.residual_norm_block(x, eps=-1.0),
        lambda: nc.residual_norm_block(needs, with_n=False),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {k} was taken")


@pytest.mark.parametrize("rows", [1, 70, 400])
def test_a_block_of_a_model(nc, rows):  # noqa: F811
    """norm -> projection -> add and norm -> experts, forward and backward, against the composition of the 64-bit forms on the
    tensors in between."""
    g, eps, c, hidden = generator(4), 1e-5, 272, 400
    x = activation(g, rows, c).requires_grad_()
    gain = (1 + 0.1 * torch.randn(c, device="cuda", generator=g)).requires_grad_()
    w = (torch.randn(c, c, device="cuda", generator=g) / c ** 0.5).requires_grad_()
    we = (torch.randn(3, hidden, c, device="cuda", generator=g) / c ** 0.5).requires_grad_()
    ends = ends_of([rows // 3, 0, rows - rows // 3 - rows // 8])
    dy = torch.randn(rows, hidden, device="cuda", generator=g).bfloat16()
    res, n, q, _ = nc.residual_norm_block(x, None, gain, eps=eps)
    h = nc.fp8_block_matmul(n, w, x_block=q)
    res2, n2, q2, _ = nc.residual_norm_block(h, res, None, eps=eps)
    y = nc.fp8_block_experts(n2, we, ends, x_block=q2)
    for t in (n, h, n2, res2):
        t.retain_grad()
    y.backward(dy)
    wv = ref.weight_values(*ref.weight(w.detach()))
    assert_product(h.detach(), ref.row_values(n.detach()), wv, "h")
    assert_product(n.grad, ref.row_values(h.grad), wv.t(), "dn")
    assert_product(w.grad, ref.tokens(h.grad)[0].t(), ref.tokens(n.detach())[0].t(), "dw")
    for e, (a, b) in enumerate(ref.spans(ends.tolist(), rows)):
        v = ref.weight_values(*ref.weight(we[e].detach()))
        if b > a:
            assert_product(y[a:b].detach(), ref.row_values(n2.detach())[a:b], v, "y")
            assert_product(n2.grad[a:b], ref.row_values(dy)[a:b], v.t(), "dn2")
            assert_product(we.grad[e], ref.tokens(dy[a:b])[0].t(), ref.tokens(n2.detach()[a:b])[0].t(), "dwe")
    assert torch.isfinite(x.grad).all() and torch.isfinite(gain.grad).all()
