"""The autograd nodes of the operators in blocks of 128 beside what else a program does with autograd: forward-mode and function
transforms, saved-tensor hooks, recomputation, batched and accumulated gradients, captured backward passes."""
import pytest
import torch

from test_block_linear_gpu import activation, ends_of, generator, given_weight, nc  # noqa: F401

pytestmark = pytest.mark.gpu


def calls(nc):  # noqa: F811
    """(name, f of one differentiable bf16 activation, its shape)"""
    g = generator(1)
    w, we = torch.randn(144, 256, device="cuda", generator=g), torch.randn(2, 144, 256, device="cuda", generator=g)
    gain, given = torch.ones(256, device="cuda"), given_weight(nc, g, 144, 256)
    ends = ends_of([30, 20])
    return [
        ("matmul", lambda x: nc.fp8_block_matmul(x, w)),
        ("given", lambda x: nc.fp8_block_matmul(x, given)),
        ("experts", lambda x: nc.fp8_block_experts(x, we, ends)),
        ("norm", lambda x: nc.residual_norm_block(x, None, gain)[1]),
        ("residual", lambda x: nc.residual_norm_block(x.detach(), x, gain)[1]),
    ]


NAMES = ["matmul", "given", "experts", "norm", "residual"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_and_function_transforms_are_refused(nc, name):  # noqa: F811
    f, x = dict(calls(nc))[name], activation(generator(2), 60, 256)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            f(dual)
        with torch.no_grad(), pytest.raises(RuntimeError):
            f(dual)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: f(v).float().sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    f(x)  # and afterwards everything is as before
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", [60, 5001])
def test_saved_tensors_through_hooks(nc, tokens):  # noqa: F811
    """What the nodes keep may be packed and unpacked, on the CPU too; 5001 tokens take the scaled products."""
    cin, cout, g = 640, 1552, generator(3)
    x = activation(g, tokens, cin).requires_grad_()
    w = torch.randn(cout, cin, device="cuda", generator=g).requires_grad_()
    we = torch.randn(3, cout, cin, device="cuda", generator=g).requires_grad_()
    gain = torch.randn(cin, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(tokens, cout, device="cuda", generator=g).bfloat16()
    ends = ends_of([tokens // 2, 0, tokens // 3])

    def step():
        res, n, q, _ = nc.residual_norm_block(x, None, gain)
        y = nc.fp8_block_matmul(n, w, x_block=q) + nc.fp8_block_matmul(n, w) + nc.fp8_block_experts(res, we, ends)
        return y, (x, w, we, gain)
    y, leaves = step()
    want = torch.autograd.grad(y, leaves, dy)
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t)):
        with hooks:
            y, _ = step()
        for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(a, b)


def test_recomputed_in_backward(nc):  # noqa: F811
    from torch.utils.checkpoint import checkpoint
    g = generator(4)
    x = activation(g, 70, 256).requires_grad_()
    w = torch.randn(256, 256, device="cuda", generator=g).requires_grad_()

    def layer(h):
        _, n, q, _ = nc.residual_norm_block(h)
        return nc.fp8_block_matmul(n, w, x_block=q)
    dy = torch.randn(70, 256, device="cuda", generator=g).bfloat16()
    want = torch.autograd.grad(layer(layer(x)), (x, w), dy)
    got = torch.autograd.grad(checkpoint(layer, checkpoint(layer, x, use_reentrant=False), use_reentrant=False), (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_changes_between_forward_and_backward_is_noticed(nc):  # noqa: F811
    g = generator(5)
    x = activation(g, 70, 256)
    w = torch.randn(2, 144, 256, device="cuda", generator=g).requires_grad_()
    ends = ends_of([30, 40])
    y = nc.fp8_block_experts(x, w, ends)
    ends.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    given = given_weight(nc, g, 144, 256)
    xg = x.clone().requires_grad_()
    y = nc.fp8_block_matmul(xg, given)
    given.scale.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    h = x.clone().requires_grad_()
    res, n, _, _ = nc.residual_norm_block(h * 1, x)
    with torch.no_grad():
        res.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.sum().backward()


def test_the_same_tensor_twice(nc):  # noqa: F811
    g = generator(6)
    x = activation(g, 40, 256).requires_grad_()
    dn = torch.randn(40, 256, device="cuda", generator=g).bfloat16()
    res, n, _, _ = nc.residual_norm_block(x, x)
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    res2, n2, _, _ = nc.residual_norm_block(a, b)
    assert torch.equal(res, res2) and torch.equal(n, n2)
    da, db = torch.autograd.grad(n2, (a, b), dn)
    assert torch.equal(torch.autograd.grad(n, x, dn)[0], da + db)
    # two leaves do not end up with one gradient buffer
    res2, n2, _, _ = nc.residual_norm_block(a, b)
    n2.backward(dn)
    assert a.grad.data_ptr() != b.grad.data_ptr() and torch.equal(a.grad, b.grad)
    n3 = nc.residual_norm_block(a, b)[1]
    n3.backward(dn)
    assert torch.equal(a.grad, da + da) and torch.equal(b.grad, da + da)


def test_backward_into_grad_captured(nc):  # noqa: F811
    """A training step with .backward(), captured once and replayed on other values; gradients are accumulated in place."""
    g = generator(7)
    x = activation(g, 200, 256)
    gain = torch.ones(256, device="cuda").requires_grad_()
    w = torch.randn(144, 256, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(200, 144, device="cuda", generator=g).bfloat16()

    def step():
        _, n, q, _ = nc.residual_norm_block(x, None, gain)
        nc.fp8_block_matmul(n, w, x_block=q).backward(dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for t in (w, gain):
        t.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        x.copy_(activation(g, 200, 256))
        for t in (w, gain):
            t.grad.zero_()
        graph.replay()
        got = [t.grad.clone() for t in (w, gain)]
        b, c = w.detach().clone().requires_grad_(), gain.detach().clone().requires_grad_()
        _, n, q, _ = nc.residual_norm_block(x.clone(), None, c)
        nc.fp8_block_matmul(n, b, x_block=q).backward(dy)
        assert torch.equal(got[0], b.grad) and torch.equal(got[1], c.grad)


def test_two_threads_at_once(nc):  # noqa: F811
    import threading
    g = generator(8)
    x = activation(g, 300, 1040)
    w = torch.randn(528, 1040, device="cuda", generator=g)
    dy = torch.randn(300, 528, device="cuda", generator=g).bfloat16()

    def step():
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        _, n, q, _ = nc.residual_norm_block(a)
        return torch.autograd.grad(nc.fp8_block_matmul(n, b, x_block=q), (a, b), dy)
    want, bad = step(), []
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and nc.capi.device_status() == 0
