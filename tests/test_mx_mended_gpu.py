"""The 4-bit layer's operators on the GPU: calls beside those of test_mx_gpu.py.  Oracle, inputs and the derivation of the tolerances are the same."""
import pytest
import torch

import _mx_oracle as mo
from dist_amd import lib as L
from dist_amd import ops
from test_mx_gpu import BF, F32, U, act, close, gen, half, operand, rows8, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(5, 64, 96), (70, 128, 288), (300, 256, 256), (2600, 1024, 96)])
@pytest.mark.parametrize("out", [BF, F32])
def test_product_beside_its_residual(M, N, K, out, gpu_lib):
    # out and res are the columns of one buffer, either way round
    B, A = operand(N, K, 1)[0], operand(M, K, 2)[0]
    res = torch.randn(M, N, generator=gen(4)).to(out).cuda()
    want = ops.gemm_mxfp4(A, B, res=res, out_dtype=out)
    for left in (0, N):
        buf = torch.empty(M, 2 * N, dtype=out, device="cuda")
        o, r = buf[:, left:left + N], buf[:, N - left:2 * N - left]
        r.copy_(res)
        ops.gemm_mxfp4(A, B, res=r, out=o)
        same_bits(o, want)
        same_bits(r, res)


@pytest.mark.parametrize("C", [768, 1411, 8200])
def test_norm_beside_its_input(C, gpu_lib):
    rows = 70
    x, r, w = act(rows, C, BF, 1), act(rows, C, BF, 2), torch.rand(C, generator=gen(3)).cuda()
    buf = torch.empty(rows, 2 * C, dtype=BF, device="cuda")
    a, b = buf[:, :C], buf[:, C:]
    a.copy_(x)
    n = ops.rmsnorm(a, w, res=r, h=b)
    assert n["h"] is b
    same_bits(a, x)
    same_bits(b, (x.float() + r.float()).to(BF))
    rstd = mo.rms(x, w)[1].float().cuda()
    want = ops.rmsnorm_bwd(a, rstd, r, w)
    got = ops.rmsnorm_bwd(a, rstd, r, w, dh=b)
    same_bits(a, x)
    for u, v in zip(got, want):
        same_bits(u, v)
