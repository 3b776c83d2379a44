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


@pytest.mark.parametrize("rows,C", [((1 << 20) + 5, 2), ((1 << 24) + 3, 3), ((1 << 20) + 1, 7)])
def test_norm_gradient_of_more_short_rows_than_workgroups(rows, C, gpu_lib):
    h = torch.randn(rows, C, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(BF)
    d = torch.randn(rows, C, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF)
    w = torch.rand(C, generator=gen(3)).cuda()
    rstd = 1 / torch.sqrt(h.float().square().mean(1) + 1e-6)
    dh, dw = ops.rmsnorm_bwd(h, rstd, d, w)
    n, g = h.double() * rstd.double()[:, None], d.double() * w.double()
    want = rstd.double()[:, None] * (g - n * (g * n).mean(1, keepdim=True))
    # as test_norm_gradient's: every addition and product around the sum of C terms
    inner = rstd.double()[:, None] * (4 * g.abs() + n.abs() * ((C + 8 + 4) * (g * n).abs().mean(1, keepdim=True) + 6 * (g * n).mean(1, keepdim=True).abs()))
    assert bool(((dh.double() - want).abs() <= half(BF) * want.abs() + 1.01 * U * inner).all())
    # a slice's chain of rows, 64 slices, and the products
    assert bool(((dw.double() - (d.double() * n).sum(0)).abs() <= (rows // 64 + 64 + 4) * U * (d.double() * n).abs().sum(0)).all())
    c = h.clone()
    same_bits(ops.rmsnorm_bwd(c, rstd, d, w, dh=c)[0], dh)
