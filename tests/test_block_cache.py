"""Weight caches of the Linears in blocks of 128."""
import pytest
import torch

import nanochat_cpp_b200 as nc
from nanochat_cpp_b200 import engine


class Counting:
    """Any object with a get() is a cache."""

    def __init__(self):
        self.asked = []

    def get(self, kind, weights, make):
        self.asked.append((kind, weights))
        return ["data", "scale"]


class Sub(nc.Fp8WeightCache):
    def get(self, kind, weights, make):
        return ["data", "scale"]


def test_a_cache_that_is_off_is_none():
    w = torch.zeros(128, 128)  # on the CPU: quantizing it would raise
    for cache in (None, nc.Fp8WeightCache(), nc.Fp8WeightCache(False)):
        assert engine._block_operands(w, None, cache) == (w, None, None, None, None)


def test_a_subclass_and_another_class_are_asked():
    w, other = torch.zeros(128, 128), Counting()
    assert engine._block_operands(w, None, other) == (w, None, None, "data", "scale")
    assert other.asked == [(2, [w])]
    assert engine._block_operands(w, None, Sub(False)) == (w, None, None, "data", "scale")


@pytest.mark.gpu
def test_a_cache_that_is_off_takes_the_same_products():
    """At a size where a training pass lets the tensor core scale: no cache and one that is off give the same bits."""
    tokens, cin, cout, g = 5001, 640, 1552, torch.Generator(device="cuda").manual_seed(1)
    assert nc.capi.lib.mxb200_block_scaled(tokens, cin, cout, 1)
    x = torch.randn(tokens, cin, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.randn(cout, cin, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(tokens, cout, device="cuda", generator=g).bfloat16()

    def step(**given):
        launches = nc.capi.launch_count()
        y = nc.fp8_block_matmul(x, w, **given)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)], nc.capi.launch_count() - launches
    want, launches = step()
    got, same = step(cache=nc.Fp8WeightCache(False))
    assert same == launches and all(torch.equal(a, b) for a, b in zip(got, want))
    w3, ends = w.detach()[None].clone().requires_grad_(), torch.tensor([tokens], device="cuda", dtype=torch.int32)
    for cache in (None, nc.Fp8WeightCache()):
        y = nc.fp8_block_experts(x, w3, ends, cache=cache)
        dx, dw = torch.autograd.grad(y, (x, w3), dy)
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1]) and torch.equal(dw[0], want[2])


@pytest.mark.gpu
def test_a_weight_changed_in_place_is_quantized_again():
    """Between two calls, and between a forward pass and its backward, which goes by the weight of the forward."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(70, 256, device="cuda", generator=g).bfloat16().requires_grad_()
    w = torch.randn(144, 256, device="cuda", generator=g).requires_grad_()
    dy = torch.randn(70, 144, device="cuda", generator=g).bfloat16()
    cache = nc.Fp8WeightCache(True)
    before = nc.fp8_block_matmul(x, w)
    want_dx, = torch.autograd.grad(before, x, dy)
    y = nc.fp8_block_matmul(x, w, cache=cache)
    assert torch.equal(y, before)
    with torch.no_grad():
        w.mul_(-3)
    after = nc.fp8_block_matmul(x, w, cache=cache)
    assert torch.equal(after, nc.fp8_block_matmul(x, w)) and not torch.equal(after, before)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want_dx)
    with torch.no_grad():
        again = nc.fp8_block_matmul(x, w, cache=cache)
    assert torch.equal(again, after)
