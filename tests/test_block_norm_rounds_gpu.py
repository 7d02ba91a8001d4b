"""The norm's backward over more rows than its CTAs have at a time, at every width's kernel, and the size of its grid."""
import pytest
import torch

from test_block_linear_gpu import activation, assert_close, generator, nc  # noqa: F401
from test_block_norm_gpu import U, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [4112, 5040, 8192, 8208, 16384])
def test_wide_rows_take_one_round(nc, cols):  # noqa: F811
    """Beyond 4096 columns an SM has room for one CTA, each of which leaves one row of partial sums."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert nc.capi.lib.mxb200_block_norm_workspace_bytes(100000, cols) == sms * cols * 4
    assert nc.capi.lib.mxb200_block_norm_workspace_bytes(3, cols) == 3 * cols * 4


@pytest.mark.parametrize("rows,cols", [(9001, 16), (5001, 528), (2501, 2048), (1201, 2064), (701, 4096), (593, 4112), (450, 8192), (447, 8208),
                                       (300, 16384), (148, 16384), (149, 8192)])
@pytest.mark.parametrize("gain_type", [torch.float32, torch.bfloat16])
def test_many_rows(nc, rows, cols, gain_type):  # noqa: F811
    g, eps = generator(1), 1e-5
    x = activation(g, rows, cols).requires_grad_()
    r = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    gain = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(gain_type).requires_grad_()
    dn = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    dres = torch.randn(rows, cols, device="cuda", generator=g).bfloat16()
    res, n, _, _ = nc.residual_norm_block(x, r, gain, eps=eps)
    dx, dgain = torch.autograd.grad((res, n), (x, gain), (dres, dn))
    _, rstd, hat, want_n = reference(x.detach(), r, gain.detach(), eps)
    assert_close(n.detach(), want_n, 46 * U * want_n.abs(), "n")
    d = dn.double() * gain.detach().double()
    mean, size = (d * hat).mean(-1, keepdim=True), (d * hat).abs().mean(-1, keepdim=True)
    scale = rstd[:, None]
    slack = U * (200 * scale * (d.abs() + hat.abs() * size) + 4 * dres.double().abs())
    assert_close(dx, scale * (d - hat * mean) + dres.double(), slack, "dx")
    # every sum has at most `rows` terms in some order, each a product of three roundings at most, and 46 of n's
    terms = dn.double() * hat
    assert_close(dgain, terms.sum(0), (rows + 100) * U * terms.abs().sum(0), "dgain")
