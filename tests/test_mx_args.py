"""CPU: argument checks of the norm / MXFP4 entry points, in the library (bad arguments return before any launch) and in the Python wrappers; the oracle's format against
torch's own e2m1 arithmetic; the formula of the norm's gradient against differences."""
import ctypes as C

import pytest
import torch

import _mx_oracle as mo
from dist_amd import lib as L
from dist_amd import ops

P = 1 << 20                   # an address that is never read: every call below is refused first


def _rms(**kw):
    a = L.RmsArgs()
    base = dict(x=P, w=P, y=P, scale=P, rows=4, ldx=64, ldy=64, ldres=64, ldh=64, C=64, fmt=L.RMS_SAME, dtype=L.BF16, eps=1e-6)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return L.load().dist_op_rmsnorm(C.byref(a), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(w=None), dict(y=None), dict(fmt=3), dict(fmt=L.RMS_E4M3, scale=None), dict(dtype=7), dict(rows=-1), dict(C=0), dict(C=-8),
                                dict(ldx=63), dict(ldy=63), dict(res=P, ldres=63), dict(h=P, ldh=63), dict(x=P + 1), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(fmt=L.RMS_MXFP4, y=P + 4)])
def test_rmsnorm_refuses(kw):
    assert _rms(**kw) == -1


def test_zero_rows_are_nothing_to_do():
    assert _rms(rows=0) == 0 and _rms(rows=0, x=None, y=None) == 0
    l = L.load()
    assert l.dist_op_quant_mxfp4(None, L.BF16, 0, 64, 64, 0, None, None, None) == 0
    assert l.dist_op_dequant_mxfp4(None, None, 0, 64, None, L.F32, None) == 0
    a = L.GemmMxArgs()
    a.M, a.N, a.K = 0, 5, 64
    assert l.dist_op_gemm_mxfp4(C.byref(a), None) == 0
    assert l.dist_op_rmsnorm(None, None) == -1 and l.dist_op_rmsnorm_bwd(None, None) == -1 and l.dist_op_gemm_mxfp4(None, None) == -1


def _bwd(**kw):
    a = L.RmsBwdArgs()
    base = dict(h=P, rstd=P, dy=P, w=P, dh=P, dw=P, scratch=P, scratch_elems=1 << 30, rows=4, ldh=64, lddy=64, lddres=64, lddh=64, C=64, dtype=L.BF16, dy_dtype=L.F32)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return L.load().dist_op_rmsnorm_bwd(C.byref(a), None)


@pytest.mark.parametrize("kw", [dict(h=None), dict(rstd=None), dict(dy=None), dict(w=None), dict(dw=None), dict(scratch=None), dict(C=0), dict(rows=-1), dict(ldh=1), dict(lddy=1),
                                dict(dres=P, lddres=1), dict(lddh=1), dict(dtype=9), dict(dy_dtype=9), dict(dy=P + 2)])
def test_rmsnorm_bwd_refuses(kw):
    assert _bwd(**kw) == -1


def test_rmsnorm_bwd_scratch_is_checked():
    n = L.load().dist_op_rmsnorm_bwd_scratch(4, 64)
    assert n > 0 and _bwd(scratch_elems=n - 1) == -3
    assert L.load().dist_op_rmsnorm_bwd_scratch(-1, 64) == -1 and L.load().dist_op_rmsnorm_bwd_scratch(4, 0) == -1


@pytest.mark.parametrize("args", [(None, 1, 4, 64, 64, 0, P, P), (P, 1, 4, 64, 64, 0, None, P), (P, 1, 4, 64, 64, 0, P, None), (P, 5, 4, 64, 64, 0, P, P), (P, 1, 4, 64, 63, 0, P, P),
                                  (P, 1, -1, 64, 64, 0, P, P), (P, 1, 4, 0, 0, 0, P, P), (P, 1, 0, 64, 64, 1, P, P), (P, 1, 4, 64, 64, 0, P + 8, P), (P + 1, 1, 4, 64, 64, 0, P, P),
                                  (P, 1, 4, 64, 64, 0, P, P + 4)])
def test_quant_refuses(args):
    assert L.load().dist_op_quant_mxfp4(*args, None) == -1


@pytest.mark.parametrize("args", [(None, P, 4, 64, P, 1), (P, None, 4, 64, P, 1), (P, P, 4, 64, None, 1), (P, P, 4, 48, P, 1), (P, P, -4, 64, P, 1), (P, P, 4, 64, P, 2), (P, P, 4, 64, P + 2, 1)])
def test_dequant_refuses(args):
    assert L.load().dist_op_dequant_mxfp4(*args, None) == -1


def _gemm(**kw):
    a = L.GemmMxArgs()
    base = dict(A=P, a_scale=P, B=P, b_scale=P, C=P, M=4, N=8, K=64, lda=64, ldc=8, ldres=8, a_fmt=L.MX_A_MXFP4, dtype=L.BF16)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return L.load().dist_op_gemm_mxfp4(C.byref(a), None)


@pytest.mark.parametrize("kw", [dict(A=None), dict(a_scale=None), dict(B=None), dict(b_scale=None), dict(C=None), dict(M=-1), dict(N=0), dict(K=0), dict(K=48), dict(ldc=7),
                                dict(res=P, ldres=7), dict(a_fmt=2), dict(dtype=2), dict(a_fmt=L.MX_A_E4M3, dtype=L.F32), dict(a_fmt=L.MX_A_E4M3, lda=63), dict(a_fmt=L.MX_A_E4M3, lda=72), dict(K=(1 << 22) + 32), dict(a_fmt=L.MX_A_E4M3, lda=(1 << 22) + 16),
                                dict(A=P + 8), dict(B=P + 8), dict(b_scale=P + 4), dict(a_scale=P + 4), dict(C=P + 1), dict(bias=P + 2)])
def test_gemm_refuses(kw):
    assert _gemm(**kw) == -1


def test_gemm_scratch_is_checked():
    """a long axis over few tiles is cut into slices, whose partial results need a place"""
    l = L.load()
    n = l.dist_op_gemm_mxfp4_scratch(128, 128, 16384, L.MX_A_MXFP4)
    assert n > 0 and n % (128 * 128) == 0 and l.dist_op_gemm_mxfp4_scratch(64, 128, 16384, L.MX_A_MXFP4) == 0 and l.dist_op_gemm_mxfp4_scratch(50432, 2304, 768, L.MX_A_E4M3) == 0
    big = dict(M=128, N=128, K=16384, ldc=128)
    assert _gemm(**big) == -3 and _gemm(**big, scratch=P, scratch_elems=n - 1) == -3 and _gemm(**big, scratch=P + 4, scratch_elems=n) == -3


def test_wrappers_refuse_before_they_reach_the_library():
    x, w = torch.randn(4, 64), torch.ones(64)
    op = (torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 8, 8, dtype=torch.uint8))
    for call, what in ((lambda: ops.rmsnorm(x, w), "GPU"), (lambda: ops.rmsnorm(x, w, fmt="e5m2"), "fmt"), (lambda: ops.rmsnorm(x, w[:5]), "w"), (lambda: ops.rmsnorm(x[None], w), "x"),
                       (lambda: ops.rmsnorm(x.t(), torch.ones(4)), "rows must be contiguous"), (lambda: ops.rmsnorm(x[:1].expand(4, 64), w), "overlap"),
                       (lambda: ops.rmsnorm(x, w, res=x[:2]), "res"), (lambda: ops.rmsnorm(x, w, res=x.bfloat16()), "res"), (lambda: ops.rmsnorm(x, w, rstd=torch.empty(3)), "rstd"),
                       (lambda: ops.rmsnorm_bwd(x, torch.ones(3), x, w), "rstd"), (lambda: ops.rmsnorm_bwd(x, torch.ones(4), x[:3], w), "dy"), (lambda: ops.rmsnorm_bwd(x, torch.ones(4), x, w), "GPU"),
                       (lambda: ops.quant_mxfp4(x[0]), "matrix"), (lambda: ops.quant_mxfp4(x), "GPU"), (lambda: ops.quant_mxfp4(x[:, :0]), "empty"), (lambda: ops.quant_mxfp4(x[:0], transpose=True), "empty"),
                       (lambda: ops.dequant_mxfp4(op[0], op[1][:, :7]), "scales"), (lambda: ops.dequant_mxfp4(op[0][:, :24], op[1]), "codes"),
                       (lambda: ops.gemm_mxfp4(op, op), "GPU"), (lambda: ops.gemm_mxfp4(op[0], op), "A"), (lambda: ops.gemm_mxfp4((torch.zeros(8, 48, dtype=torch.uint8), torch.zeros(1, 8, 8, dtype=torch.uint8)), op), "A has 96"),
                       (lambda: ops.gemm_mxfp4((torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8)), op), "A")):
        with pytest.raises(L.DistError, match=what):
            call()
    with pytest.raises(TypeError):
        ops.rmsnorm(x.half(), w)
    with pytest.raises(TypeError):
        ops.quant_mxfp4(x.double())


def test_struct_mirrors_and_sizes():
    l = L.load()
    for name, mirror in (("dist_rms_args", L.RmsArgs), ("dist_rms_bwd_args", L.RmsBwdArgs), ("dist_gemm_mx_args", L.GemmMxArgs)):
        assert l.dist_abi_sizeof(name.encode()) == C.sizeof(mirror)
    assert l.dist_op_mxfp4_scale_bytes(5, 300) == 2 * 5 * 8 and l.dist_op_mxfp4_scale_bytes(0, 32) == 0 and l.dist_op_mxfp4_scale_bytes(5, 0) == -1
    assert l.dist_op_gemm_mxfp4_scratch(4, 4, 48, 0) == -1 and l.dist_op_gemm_mxfp4_scratch(4, 4, 64, 0) >= 0


def test_oracle_format():
    """the oracle's rounding against arithmetic rounding on the grid's three steps, its layout against itself, and its special blocks"""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 96, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (7, 1), generator=g).double())
    x[0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, -0.25, -0.75, -5.0, -7.9, 0.0, -0.0, 4.0] * 2)
    x[1, 32:64] = 0
    code, byte = mo.codes_of(x)
    v = x.view(7, 3, 32) * torch.exp2(-(byte - 127).double())[..., None]
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    want = torch.copysign((torch.round(a / step) * step).clamp(max=6), v) * torch.exp2((byte - 127).double())[..., None]
    assert torch.equal(mo.values_of(code, byte), want.view(7, 96))
    assert torch.equal(torch.stack(mo.unpack(*mo.pack(code, byte))[0:1])[0], code) and torch.equal(mo.unpack(*mo.pack(code, byte))[1], byte)
    assert int(byte[1, 1]) == 0
    x[2, 5], x[3, 40] = float("inf"), float("nan")
    byte = mo.codes_of(x)[1]
    assert int(byte[2, 0]) == int(byte[3, 1]) == 255 and int((byte == 255).sum()) == 2


def test_gradient_formula_against_differences():
    g = torch.Generator().manual_seed(1)
    x, w, d, r = (torch.randn(3, 10, generator=g, dtype=torch.float64) for _ in range(4))
    w = w[0] + 1.5
    loss = lambda x, w: float((mo.rms(x, w)[2] * d).sum() + (x * r).sum())  # noqa: E731
    h, rstd, _ = mo.rms(x, w)
    dh, dw = mo.rms_bwd(h, rstd, d, w, r)
    e = 1e-5                                     # central differences: error e^2 f''' + 2^-53 f / e, both under 1e-9 here
    for i in range(3):
        for j in range(10):
            step = torch.zeros_like(x)
            step[i, j] = e
            assert abs((loss(x + step, w) - loss(x - step, w)) / (2 * e) - float(dh[i, j])) < 1e-8
    for j in range(10):
        step = torch.zeros_like(w)
        step[j] = e
        assert abs((loss(x, w + step) - loss(x, w - step)) / (2 * e) - float(dw[j])) < 1e-8
