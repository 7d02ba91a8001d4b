"""A backward pass in blocks of 128 computes what it is asked for: the gradients that autograd wants at that time, not those that
the inputs could have had."""
import pytest
import torch

from test_block_linear_gpu import activation, ends_of, generator, given_weight, nc  # noqa: F401

pytestmark = pytest.mark.gpu


def launches_of(nc, call):  # noqa: F811
    before = nc.capi.launch_count()
    out = call()
    return out, nc.capi.launch_count() - before


@pytest.mark.parametrize("tokens,scaled", [(70, False), (5001, True)])
@pytest.mark.parametrize("experts", [0, 3])
def test_linears(nc, tokens, scaled, experts):  # noqa: F811
    cin, cout, g = 640, 1552, generator(1)
    x = activation(g, tokens, cin).requires_grad_()
    w = torch.randn(*([experts] if experts else []), cout, cin, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(tokens, cout, device="cuda", generator=g).bfloat16()
    ends = ends_of([tokens // 2, 0, tokens // 3]) if experts else None
    assert bool(nc.capi.lib.mxb200_block_scaled(tokens, cin, cout, max(1, experts))) == scaled

    def forward(a=x, b=w, **given):
        return nc.fp8_block_experts(a, b, ends, **given) if experts else nc.fp8_block_matmul(a, b, **given)

    # one quantizer for the incoming gradient, one product for each gradient that is wanted
    y = forward()
    (dx, dw), both = launches_of(nc, lambda: torch.autograd.grad(y, (x, w), dy, retain_graph=True))
    (only_x,), for_x = launches_of(nc, lambda: torch.autograd.grad(y, x, dy, retain_graph=True))
    (only_w,), for_w = launches_of(nc, lambda: torch.autograd.grad(y, w, dy))
    assert (both, for_x, for_w) == (3, 2, 2)
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    # the input in blocks beforehand: the weight gradient quantizes it along its tokens too
    y = forward(x_block=nc.quantize_block(x))
    (dx, dw), both = launches_of(nc, lambda: torch.autograd.grad(y, (x, w), dy, retain_graph=True))
    (only_x,), for_x = launches_of(nc, lambda: torch.autograd.grad(y, x, dy, retain_graph=True))
    (only_w,), for_w = launches_of(nc, lambda: torch.autograd.grad(y, w, dy))
    assert (both, for_x, for_w) == (4, 2, 3)
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    # a weight without a gradient of its own
    frozen = given_weight(nc, g, *w.shape)
    (dx,), for_x = launches_of(nc, lambda: torch.autograd.grad(forward(x, frozen), x, dy))
    assert dx.shape == x.shape and for_x <= 4  # the forward's one or two among them


def test_a_gradient_that_is_not_asked_for_takes_no_memory(nc):  # noqa: F811
    tokens, cin, cout, experts, g = 64, 1024, 2048, 64, generator(2)
    x = activation(g, tokens, cin).requires_grad_()
    w = torch.randn(experts, cout, cin, device="cuda", generator=g).requires_grad_()  # its gradient: 512 MB
    y = nc.fp8_block_experts(x, w, ends_of([1] * experts))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.cuda.max_memory_allocated() - before < 16 << 20


def test_accumulated_into_the_leaves_that_want_it(nc):  # noqa: F811
    g = generator(3)
    x, w = activation(g, 33, 128).requires_grad_(), torch.randn(144, 128, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(33, 144, device="cuda", generator=g).bfloat16()
    y = nc.fp8_block_matmul(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    y.backward(dy, inputs=[w], retain_graph=True)
    assert x.grad is None and torch.equal(w.grad, dw)
    y.backward(dy, inputs=[x])
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


@pytest.mark.parametrize("add", [True, False])
@pytest.mark.parametrize("gain_type", [torch.float32, torch.bfloat16])
def test_norm(nc, add, gain_type):  # noqa: F811
    g = generator(4)
    x = activation(g, 300, 528).requires_grad_()
    r = torch.randn(300, 528, device="cuda", generator=g).bfloat16().requires_grad_() if add else None
    gain = (1 + 0.2 * torch.randn(528, device="cuda", generator=g)).to(gain_type).requires_grad_()
    dn = torch.randn(300, 528, device="cuda", generator=g).bfloat16()
    res, n, _, _ = nc.residual_norm_block(x, r, gain)
    (dx, dgain), both = launches_of(nc, lambda: torch.autograd.grad(n, (x, gain), dn, retain_graph=True))
    (only_x,), for_x = launches_of(nc, lambda: torch.autograd.grad(n, x, dn, retain_graph=True))
    (only_gain,), for_gain = launches_of(nc, lambda: torch.autograd.grad(n, gain, dn, retain_graph=True))
    assert (both, for_x, for_gain) == (2, 1, 2)
    assert torch.equal(only_x, dx) and torch.equal(only_gain, dgain)
    if add:
        (only_r,), for_r = launches_of(nc, lambda: torch.autograd.grad(n, r, dn, retain_graph=True))
        assert for_r == 1 and torch.equal(only_r, dx)
    # through the residual alone: the norm's gain has no part in it
    (through,), none = launches_of(nc, lambda: torch.autograd.grad(res, x, dn))
    assert none == 0 and torch.equal(through, dn)
