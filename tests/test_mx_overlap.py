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
        real, said = bool(_bytes(a) & _bytes(b)), ops._meet(a, b)
        assert said or not real
        runs = ops._runs(a)[2], ops._runs(b)[2]
        if 0 in runs or runs[0] == runs[1]:
            assert said == real
            both[real] += 1
    assert min(both) > 500
