"""Rows in four bits from their definition, in plain torch: codes, scales, tiles, and what they stand for."""
import torch

#: values of the codes 0 to 7; 8 to 15 are their negatives
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def up(n, to):
    return (n + to - 1) // to * to


def nearest(t):
    """Codes of the nearest values, ties to the even code, saturating; t in 64 bits, NaN as the largest."""
    grid = torch.tensor(VALUES, dtype=torch.float64, device=t.device)
    size = torch.nan_to_num(t.abs(), nan=6.0).clamp(max=6.0)
    off = (size.unsqueeze(-1) - grid).abs()
    best = off.min(-1, keepdim=True).values
    ties = off == best
    even = torch.arange(8, device=t.device) % 2 == 0
    # the even one of two equally near codes
    code = torch.where(ties.sum(-1, keepdim=True) > 1, ties & even, ties).float().argmax(-1)
    return code + 8 * (torch.signbit(t) & ~torch.isnan(t))


def rounded_32(t):
    return t.float().double()


def quantised(t, block, scale=None):
    """(codes, scale bytes) of rows t, in whole blocks of 32 channels; t: values that are exact in 64 bits.  Product and quotient of scales are rounded to
    32 bits each, as defined."""
    rows, c = t.shape
    t = torch.nn.functional.pad(t.double(), (0, up(c, 32) - c)).reshape(rows, -1, block)
    most = t.abs().amax(-1)
    finite = torch.isfinite(t).all(-1)
    if block == 16:
        g = 1.0 if scale is None else float(scale)
        six = rounded_32(torch.tensor(6 * g, dtype=torch.float64)).item()
        s = rounded_32(torch.where(finite, most, 1.0) / six).clamp(2.0 ** -9, 448.0).float().to(torch.float8_e4m3fn)
        step = rounded_32(s.double() * g)
        byte = torch.where(finite, s.view(torch.uint8), 0x7F)
    else:
        exponent = torch.frexp(torch.where(finite & (most > 0), most, 2.0 ** -127))[1].double() - 3
        exponent = exponent.clamp(min=-127)
        step = torch.exp2(exponent)
        byte = torch.where(finite, exponent + 127, 255.0).to(torch.uint8)
    codes = nearest(rounded_32(t / step.unsqueeze(-1)))
    return codes.reshape(rows, -1).to(torch.uint8), byte


def packed(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpacked(codes):
    """Codes, one a byte, of rows of float4_e2m1fn_x2."""
    b = codes.view(torch.uint8).reshape(-1, codes.shape[-1])
    return torch.stack([b & 15, b >> 4], -1).flatten(1)


def tiled(scale_bytes):
    """Scale bytes in tiles, place by place."""
    rows, blocks = scale_bytes.shape
    tall, wide = up(rows, 128), up(blocks, 4)
    out = torch.zeros(tall * wide, dtype=torch.uint8, device=scale_bytes.device)
    r = torch.arange(rows, device=out.device).unsqueeze(1)
    b = torch.arange(blocks, device=out.device).unsqueeze(0)
    out[(r // 128 * (wide // 4) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = scale_bytes
    return out.reshape(tall, wide)


def untiled(scales, rows, blocks):
    """The inverse: scale bytes by row and block."""
    flat, wide = scales.view(torch.uint8).reshape(-1), scales.shape[1]
    r = torch.arange(rows, device=flat.device).unsqueeze(1)
    b = torch.arange(blocks, device=flat.device).unsqueeze(0)
    return flat[(r // 128 * (wide // 4) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4]


def scale_values(byte, block):
    return byte.contiguous().view(torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu).float().double()


def values(codes, scales, scale=None):
    """What the kernels' codes and scales stand for, in 64 bits, rows flattened: (rows, whole blocks of channels)."""
    block = 16 if scales.dtype == torch.float8_e4m3fn else 32
    one = unpacked(codes)
    rows, wide = one.shape
    v = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=one.device)[one.long()]
    s = scale_values(untiled(scales, rows, wide // block), block) * (1.0 if scale is None else scale.double())
    return (v.reshape(rows, -1, block) * s.unsqueeze(-1)).reshape(rows, wide)
