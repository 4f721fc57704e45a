"""MXFP4 in 64 bits for the tests: levels, scales and codes from their definitions (torch tensors of any device)."""
import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pitch(cols):
    return 4 * -(-cols // 128)


def nearest(q):
    """Codes of f64 values of magnitude below 7: the nearest level, of two the one with the even code; bit 3 the sign."""
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=q.device)
    d = (q.abs()[..., None] - lv).abs()
    best = d == d.amin(-1, keepdim=True)
    even = best & (torch.arange(8, device=q.device) % 2 == 0)
    code = torch.where(even.any(-1), even.byte().argmax(-1), best.byte().argmax(-1))
    return (code + 8 * torch.signbit(q)).to(torch.uint8)


def level(code):
    lv = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=code.device)
    return lv[code.long()]


def quantize(x):
    """f64 x [rows, cols] -> (codes [rows, cols], one a byte, scale bytes [rows, ceil(cols / 32)])."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % 32)).view(rows, -1, 32)
    odd = ~torch.isfinite(b).all(-1)
    b = torch.where(odd[..., None], torch.zeros_like(b), b)
    m = b.abs().amax(-1)
    # Tried one by one: the smallest exponent from -127 on under which m is below 7.
    f, e = torch.frexp(m)
    byte = torch.full_like(m, 127)
    for k in (0, -1, -2, -3, -4):
        s = torch.clamp(e + k, min=-127)
        fits = (m > 0) & (m * torch.exp2(-s.double()) < 7)   # exact, unlike ldexp on the GPU
        byte = torch.where(fits, (s + 127).double(), byte)
    byte = torch.where(odd, torch.full_like(byte, 255), byte)
    s = torch.where(odd, torch.ones_like(byte), torch.exp2(byte - 127))
    code = nearest(b / s[..., None])
    code = torch.where(odd[..., None], torch.zeros_like(code), code)
    return code.view(rows, -1)[:, :cols], byte.to(torch.uint8)


def values(code, byte):
    """f64 values of codes [rows, cols] under scale bytes [rows, >= ceil(cols / 32)]; NaN under 255."""
    cols = code.shape[1]
    s = torch.where(byte == 255, torch.full_like(byte, 127).double() * float("nan"), torch.exp2(byte.double() - 127))
    return level(code) * s.repeat_interleave(32, 1)[:, :cols]


def pack(code, byte):
    """Codes two a byte [rows, ceil(cols / 2)] and scales [rows, pitch]."""
    rows, cols = code.shape
    code = torch.nn.functional.pad(code, (0, cols % 2))
    scales = torch.full((rows, pitch(cols)), 127, dtype=torch.uint8, device=code.device)
    scales[:, :byte.shape[1]] = byte
    return (code[:, ::2] | (code[:, 1::2] << 4)).contiguous(), scales


def unpack(codes, cols):
    return torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1)[:, :cols]
