"""CPU: which buffers of the 4-bit layer's operators count as overlapping."""
import pytest
import torch

from dist_amd import lib as L
from dist_amd import ops


def _bytes(t):
    """the set of byte numbers that a view covers"""
    es = t.element_size()
    first = t.data_ptr()
    at = torch.zeros(t.shape, dtype=torch.int64)
    for n, (size, step) in enumerate(zip(t.shape, t.stride())):
        shape = [1] * t.dim()
        shape[n] = size
        at = at + (torch.arange(size) * step).view(shape)
    return {first + int(e) * es + k for e in at.flatten() for k in range(es)}


def test_columns_of_one_buffer_lie_apart():
    b = torch.zeros(16, 128, dtype=torch.bfloat16)
    for out, t in ((b[:, :64], b[:, 64:]), (b[:, 64:], b[:, :64]), (b[:8, 96:], b[8:, :32]), (b[:, 8:16], b[:, :8]), (b[3:4, :64], b[:, 64:]), (b[:, 64:], b[3:4, :64]),
                   (b[:, :1], b[:, 1:2]), (b[4:, :32], b[:, 32:64])):
        ops._apart(out, "out", t)
    for out, t in ((b[:, :65], b[:, 64:]), (b[:, 63:], b[:, :64]), (b[1:], b[:-1]), (b[:8], b[7:]), (b[3:4], b[:, 64:]), (b[:, 64:], b[3:4])):
        with pytest.raises(L.DistError, match="overlaps"):
            ops._apart(out, "out", t)


def test_meeting_is_exact_for_one_pitch_and_never_missed():
    g = torch.Generator().manual_seed(0)

    def n(low, high):
        return int(torch.randint(low, high + 1, (1,), generator=g))

    base = torch.zeros(400, dtype=torch.float32)

    def view(pitch):
        rows, at = n(1, 6), n(0, 120)
        cols = n(1, pitch)
        if n(0, 4) == 0:
            return base[at:at + cols]                                        # a vector
        if n(0, 1):
            return base[at:].as_strided((rows, cols), (pitch, 1), at)
        return base.view(torch.bfloat16).as_strided((rows, 2 * cols), (2 * pitch, 1), 2 * at)

    both = [0, 0]
    for _ in range(4000):
        pa = n(1, 40)
        pb = pa if n(0, 3) else n(1, 40)
        a, b = view(pa), view(pb)
        real, said = bool(_bytes(a) & _bytes(b)), ops._meet(ops._runs(a), ops._runs(b))
        assert said or not real
        runs = ops._runs(a)[2], ops._runs(b)[2]
        if 0 in runs or runs[0] == runs[1]:
            assert said == real
            both[real] += 1
    assert min(both) > 500


def _share(shape, dtype, other, at=0):
    """a tensor of this shape and type in `other`'s memory, `at` bytes behind its start"""
    n = torch.empty(shape, dtype=dtype).numel() * dtype.itemsize
    return other.view(-1).view(torch.uint8)[at:at + n].view(dtype).view(shape)


def test_every_buffer_is_checked_against_every_operand():
    """(CPU tensors: the refusal comes before the one of their place, which a call without an overlap ends with)"""
    F = torch.float32
    C, rows, N = 64, 16, 64
    x, r, w, rs = torch.zeros(rows, C), torch.zeros(rows, C), torch.zeros(C), torch.zeros(rows)
    d, dw, dh = torch.zeros(rows, C), torch.zeros(C), torch.zeros(rows, C)
    q, sa = torch.zeros(N, 32, dtype=torch.uint8), torch.zeros(1, N, 8, dtype=torch.uint8)
    B, sb = torch.zeros(N, 32, dtype=torch.uint8), torch.zeros(1, N, 8, dtype=torch.uint8)
    q8, s8 = torch.zeros(4, C, dtype=torch.uint8), torch.zeros(256)[:4]
    big = torch.zeros(4096)                                          # (longer than any operand, which lie in it)
    bf = torch.bfloat16
    h = torch.zeros(rows, C)

    def wide(t):
        """the operand moved into `big`, behind the place of the output"""
        return _share(t.shape, t.dtype, big)

    calls = [
        lambda: ops.rmsnorm(x, w, rstd=_share((rows,), F, x)), lambda: ops.rmsnorm(x, w, res=r, rstd=_share((rows,), F, r, 128)), lambda: ops.rmsnorm(x, w, rstd=w[:rows]),
        lambda: ops.rmsnorm(x, w, h=h, rstd=_share((rows,), F, h, 64)), lambda: ops.rmsnorm(x, wide(w), h=_share((rows, C), F, big)), lambda: ops.rmsnorm(x, w, h=h[:], res=_share((rows, C), F, big), rstd=_share((rows,), F, big)),
        lambda: ops.rmsnorm_bwd(h, rs, d, wide(w), dh=_share((rows, C), F, big)), lambda: ops.rmsnorm_bwd(h, wide(rs), d, w, dh=_share((rows, C), F, big)),
        lambda: ops.rmsnorm_bwd(h, rs, d, w, dh=dh, dw=_share((C,), F, dh)), lambda: ops.rmsnorm_bwd(h, rs, d, w, dw=w), lambda: ops.rmsnorm_bwd(h, rs, d, w, dw=_share((C,), F, h, 256)),
        lambda: ops.rmsnorm_bwd(h, rs, d, w, dw=_share((C,), F, d)), lambda: ops.rmsnorm_bwd(h, rs, d, w, dres=r, dw=_share((C,), F, r)),
        lambda: ops.rmsnorm_bwd(h[:, :16], _share((rows,), F, big), d[:, :16], w[:16], dw=_share((16,), F, big)),
        lambda: ops.gemm_mxfp4((q, sa), (B, sb), bias=wide(torch.zeros(N)), out=_share((N, N), bf, big)),
        lambda: ops.gemm_mxfp4((q, wide(sa)), (B, sb), out=_share((N, N), bf, big)), lambda: ops.gemm_mxfp4((q, sa), (B, wide(sb)), out=_share((N, N), bf, big)),
        lambda: ops.gemm_mxfp4((wide(q), sa), (B, sb), out=_share((N, N), bf, big)), lambda: ops.gemm_mxfp4((q, sa), (wide(B), sb), out=_share((N, N), bf, big)),
        lambda: ops.gemm_mxfp4((q8, wide(s8)), (B, sb), out=_share((4, N), bf, big)),
    ]
    for n, call in enumerate(calls):
        with pytest.raises(L.DistError) as e:
            call()
        assert "overlaps" in str(e.value), f"call {n}: {e.value}"
    for call in (lambda: ops.rmsnorm(x, w, res=r, h=x, rstd=rs), lambda: ops.rmsnorm(x, w, res=r, h=r, rstd=rs), lambda: ops.rmsnorm(x, w, res=x, h=x), lambda: ops.rmsnorm_bwd(h, rs, d, w, dres=r, dh=h, dw=dw),
                 lambda: ops.rmsnorm_bwd(h, rs, d, w, dres=r, dh=d, dw=dw), lambda: ops.rmsnorm_bwd(h, rs, d, w, dres=r, dh=r, dw=dw), lambda: ops.rmsnorm_bwd(h, rs, h, w, dh=h),
                 lambda: ops.gemm_mxfp4((q, sa), (B, sb), res=x.new_zeros(N, N, dtype=bf), out=x.new_zeros(N, N, dtype=bf)), lambda: ops.gemm_mxfp4((B, sb), (B, sb))):
        with pytest.raises(L.DistError, match="GPU"):
            call()
