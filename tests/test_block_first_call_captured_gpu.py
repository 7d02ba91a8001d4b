"""A process whose first call of each operator in blocks of 128 is captured into a graph: what the operators ask the device once
for is asked under capture then."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
import torch
import nanochat_cpp_b200 as nc
def blocks_up(n): return -(-n // 128)
def given(out, cin): return nc.BlockTensor(torch.ones(out, cin, device="cuda").to(torch.float8_e4m3fn), torch.full((blocks_up(out), blocks_up(cin)), 0.5, device="cuda"))
x = torch.full((5001, 640), 2.0, device="cuda", dtype=torch.bfloat16).requires_grad_()
wide = torch.full((300, 5040), 2.0, device="cuda", dtype=torch.bfloat16).requires_grad_()
w = torch.ones(1552, 640, device="cuda").requires_grad_()
gain = torch.ones(5040, device="cuda").requires_grad_()
dy, dn = torch.ones(5001, 1552, device="cuda", dtype=torch.bfloat16), torch.ones(300, 5040, device="cuda", dtype=torch.bfloat16)
w1, w2 = given(1536, 640), given(2064, 640)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = nc.fp8_block_matmul(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    n = nc.residual_norm_block(wide, None, gain)[1]
    dwide, dgain = torch.autograd.grad(n, (wide, gain), dn)
    with torch.no_grad():
        one, some, many = (nc.fp8_block_matmul(x[:k], v) for k, v in ((1, w1), (1001, w2), (5001, w2)))
graph.replay()
torch.cuda.synchronize()
assert (y == 1280).all() and (dx == 1552).all() and (dw == 10002).all()
assert (one == 640).all() and (some == 640).all() and (many == 640).all()
assert (n == 1).all() and (dgain - 300).abs().max() < 0.01 and dwide.abs().max() < 1e-2
assert nc.capi.device_status() == 0
print("captured")
"""


@pytest.mark.gpu
def test_first_calls_captured():
    out = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]
