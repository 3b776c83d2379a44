"""Definitions in 64 bits of the norm, the MXFP4 format and its product, for the tests of rmsnorm / quant_mxfp4 / gemm_mxfp4."""
import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half(dtype):
    """half a step, relative to the value"""
    return torch.finfo(dtype).eps / 2


def codes_of(x):
    """x [rows, K] -> (codes 0..15 [rows, Kp], scale bytes [rows, Kp / 32]) as int64"""
    rows, K = x.shape
    Kp = -(-K // 32) * 32
    b = torch.zeros(rows, Kp, dtype=torch.float64)
    b[:, :K] = x.double().cpu()
    b = b.view(rows, -1, 32)
    a = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    fl = torch.frexp(torch.where((a > 0) & ~bad, a, torch.ones_like(a)))[1] - 1
    byte = (fl - 2 + 127).clamp(0, 254)
    byte = torch.where(a == 0, torch.zeros_like(byte), byte)
    byte = torch.where(bad, torch.full_like(byte, 255), byte).long()
    v = torch.where(bad[..., None], torch.zeros_like(b), b) * torch.exp2(-(byte.clamp(max=254) - 127).double())[..., None]
    m = v.abs()
    code = torch.zeros_like(m, dtype=torch.int64)
    for k in range(1, 8):
        border = float(LEVELS[k - 1] + LEVELS[k]) / 2
        code = torch.where((m > border) | ((m == border) & (k % 2 == 0)), k, code)          # a tie goes to the even code
    sign = torch.signbit(b) & ~bad[..., None]
    code = code + 8 * sign.long()
    return code.view(rows, Kp), byte


def values_of(code, byte):
    rows = code.shape[0]
    v = LEVELS[(code % 8)] * (1 - 2 * (code // 8)).double()
    v = v.view(rows, -1, 32) * torch.exp2((byte - 127).double())[..., None]
    v = torch.where((byte == 255)[..., None], torch.full_like(v, float("nan")), v)
    return v.reshape(rows, -1)


def pack(code, byte):
    """-> the stored layout (codes uint8 [rows, Kp / 2], scales uint8 [chunks, rows, 8])"""
    rows, Kp = code.shape
    q = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    nb = Kp // 32
    sc = torch.zeros(-(-nb // 8), rows, 8, dtype=torch.uint8)
    for b in range(nb):
        sc[b // 8, :, 2 * (b % 4) + (b // 4) % 2] = byte[:, b].to(torch.uint8)
    return q, sc


def unpack(codes, scales):
    codes, scales = codes.cpu().long(), scales.cpu().long()
    rows, n = codes.shape
    code = torch.empty(rows, 2 * n, dtype=torch.int64)
    code[:, 0::2], code[:, 1::2] = codes % 16, codes // 16
    byte = torch.stack([scales[b // 8, :, 2 * (b % 4) + (b // 4) % 2] for b in range(2 * n // 32)], 1)
    return code, byte


def read(op):
    return values_of(*unpack(*op))


def rms(x, w, res=None, eps=1e-6):
    h = x.double().cpu() + (res.double().cpu() if res is not None else 0.0)
    rstd = 1 / torch.sqrt(h.square().mean(1) + eps)
    return h, rstd, h * rstd[:, None] * w.double().cpu()


def rms_bwd(h, rstd, dy, w, dres=None):
    h, rstd, dy, w = (t.double().cpu() for t in (h, rstd, dy, w))
    n, g = h * rstd[:, None], dy * w
    dh = rstd[:, None] * (g - n * (g * n).mean(1, keepdim=True)) + (dres.double().cpu() if dres is not None else 0.0)
    return dh, (dy * n).sum(0)
