"""The operators in blocks of 128 where offsets pass 32 bits, on two streams at once, and replayed from graphs that share their
inputs."""
import pytest
import torch

import block_ref as ref
from test_block_linear_gpu import activation, assert_product, ends_of, generator, given_weight, nc  # noqa: F401

pytestmark = pytest.mark.gpu


def test_rows_beyond_32_bits(nc):  # noqa: F811
    rows, cols = 270000, 16384  # 4.4e9 values
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    g = generator(1)
    x[-300:] = activation(g, 300, cols)
    w = given_weight(nc, g, 32, cols)
    q = nc.quantize_block(x)
    data, scale = ref.rows(x[-300:])
    assert torch.equal(q.data[-300:].double(), data) and torch.equal(q.scale[:, -300:].double(), scale)
    assert not q.data[: rows - 300].view(torch.uint8).any()
    y = nc.fp8_block_matmul(None, w, x_block=q)
    assert_product(y[-300:], ref.row_values(x[-300:]), ref.weight_values(w.data, w.scale), "y")
    assert not y[:-300].any()
    del q, y
    res, n, q, rstd = nc.residual_norm_block(x, eps=1e-3)
    again = nc.quantize_block(n[-300:])
    assert torch.equal(q.data[-300:].view(torch.uint8), again.data.view(torch.uint8)) and torch.equal(q.scale[:, -300:], again.scale)
    want = x[-300:].double() / torch.sqrt(x[-300:].double().square().mean(1, keepdim=True) + 1e-3)
    assert ((n[-300:].double() - want).abs() <= 2.0 ** -8 * want.abs()).all()


def test_gradients_beyond_32_bits(nc):  # noqa: F811
    tokens, cin, cout = 270000, 16384, 16
    g = generator(2)
    x = torch.zeros(tokens, cin, device="cuda", dtype=torch.bfloat16)
    x[-300:] = activation(g, 300, cin)
    dy = torch.zeros(tokens, cout, device="cuda", dtype=torch.bfloat16)
    dy[-300:] = torch.randn(300, cout, device="cuda", generator=g).bfloat16()
    w = torch.randn(cout, cin, device="cuda", generator=g).requires_grad_()
    x.requires_grad_()
    dx, dw = torch.autograd.grad(nc.fp8_block_matmul(x, w), (x, w), dy)
    wv = ref.weight_values(*ref.weight(w.detach()))
    assert_product(dx[-300:], ref.row_values(dy[-300:]), wv.t(), "dx")
    assert not dx[:-300].any()
    first = tokens - tokens % 128 - 384  # whole blocks: the rows before are zeros
    assert_product(dw, ref.tokens(dy[first:])[0].t(), ref.tokens(x.detach()[first:])[0].t(), "dw")


def test_weights_beyond_32_bits(nc):  # noqa: F811
    experts, cout, cin = 1024, 2048, 2304  # 4.8e9 values
    w = torch.zeros(experts, cout, cin, device="cuda", dtype=torch.bfloat16)
    g = generator(3)
    w[-1] = torch.randn(cout, cin, device="cuda", generator=g).bfloat16()
    q = nc.quantize_block_weight(w)
    data, scale = ref.weight(w[-1])
    assert torch.equal(q.data[-1].double(), data) and torch.equal(q.scale[-1].double(), scale)
    for rows in (40, 700):
        x = activation(g, rows, cin)
        ends = torch.zeros(experts, device="cuda", dtype=torch.int32)
        ends[-1] = rows
        assert_product(nc.fp8_block_experts(x, q, ends), ref.row_values(x), ref.weight_values(data, scale), "y")


def test_two_streams_at_once(nc):  # noqa: F811
    g = generator(4)
    shapes = [(1, 1536, 1536), (40, 1536, 2048), (700, 640, 1552), (3000, 1536, 1536)]
    work = [(activation(g, t, k), given_weight(nc, g, n, k)) for t, k, n in shapes]
    want = [nc.fp8_block_matmul(x, w) for x, w in work]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for j in range(len(work)):
                    x, w = work[(i + j) % len(work)]
                    got.append(((i + j) % len(work), nc.fp8_block_matmul(x, w)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for k, y in got:
        assert torch.equal(y, want[k])
    assert nc.capi.device_status() == 0


def test_graphs_of_one_decoding_step(nc):  # noqa: F811
    """Two graphs over the same inputs, replayed in turn on new values: a token's norm, projection and experts."""
    g = generator(5)
    x, r = activation(g, 4, 1536), activation(g, 4, 1536)
    gain = 1 + 0.1 * torch.randn(1536, device="cuda", generator=g)
    w, we = given_weight(nc, g, 2048, 1536), given_weight(nc, g, 8, 400, 2048)
    ends = ends_of([0, 1, 0, 2, 0, 0, 1, 0])

    def step():
        res, _, q, _ = nc.residual_norm_block(x, r, gain, with_n=False)
        h = nc.fp8_block_matmul(None, w, x_block=q)
        return res, h, nc.fp8_block_experts(h, we, ends)
    graphs, outs = [], []
    step()
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for k in range(6):
        x.copy_(activation(g, 4, 1536))
        ends.copy_(ends_of([k % 3, 0, 0, 1, 0, 0, 0, 3 - k % 3]))
        want = step()
        graphs[k % 2].replay()
        for a, b in zip(outs[k % 2], want):
            assert torch.equal(a, b)
