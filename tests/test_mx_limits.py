"""CPU: calls of the 4-bit layer's entry points that no launch can hold (2^32 work items along an axis) are refused before anything runs."""
import ctypes as C

import pytest

from dist_amd import lib as L
from test_mx_args import P, _bwd, _gemm, _rms


@pytest.mark.parametrize("kw", [dict(rows=(1 << 28) + 16), dict(rows=(1 << 26) + 4, C=1024, ldx=1024, ldy=1024), dict(rows=1 << 24, C=16384, ldx=16384, ldy=16384),
                                dict(rows=1 << 24, C=20000, ldx=20000, ldy=20000), dict(rows=1 << 24, C=20000, ldx=20000, fmt=L.RMS_E4M3, ldy=20000), dict(rows=(1 << 28) + 16, fmt=L.RMS_MXFP4)])
def test_norm_of_too_many_rows(kw):
    assert _rms(**kw) == -1


@pytest.mark.parametrize("C", [1 << 26, 1 << 30])
def test_gradient_of_too_wide_rows(C):
    for rows in (1, 100):
        assert _bwd(rows=rows, C=C, ldh=C, lddy=C, lddh=C, scratch_elems=1 << 40) == -1


@pytest.mark.parametrize("dtype", [L.BF16, L.F32])
def test_quantisation_of_too_many_blocks(dtype):
    l = L.load()
    for rows, cols, transpose in (((1 << 27) + 8, 32, 0), (1 << 20, 1 << 16, 0), (1 << 30, 1 << 10, 1), ((1 << 23) * 256, 64, 1)):
        assert l.dist_op_quant_mxfp4(P, dtype, rows, cols, cols, transpose, P, P, None) == -1
    assert l.dist_op_dequant_mxfp4(P, P, 1 << 30, 64, P, dtype, None) == -1


def test_products_of_too_many_tiles():
    for N in (1 << 28, (1 << 30) + 1, (1 << 31) - 1):
        assert _gemm(N=N, ldc=N) == -1
    assert _gemm(M=1 << 20, N=1 << 30, ldc=1 << 30) == -1
    assert L.load().dist_op_gemm_mxfp4_scratch(100, (1 << 31) - 1, 64, L.MX_A_MXFP4) == -1
