"""Plain 64-bit forms of the operators on token rows, and the error bounds of the kernels' arithmetic.

Bounds, with u the unit roundoff of a type (half the distance of 1 from the next number: fp32 2^-24, fp16 2^-11, bf16 2^-8): a result in type T is rounded once, which
costs u(T) of its magnitude (or half the smallest subnormal step), and the fp32 arithmetic in front of it costs a number of
u(fp32) that is counted beside each bound, relative to the magnitudes that enter the sum.
"""
import torch

U32 = 2.0 ** -24
U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
STEP = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rms(x, weight, residual, eps, offset):
    """(y, s, rstd) in 64 bits"""
    s = x.double() if residual is None else x.double() + residual.double()
    rstd = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    w = 1.0 if weight is None else offset + weight.double()
    return s * rstd * w, s, rstd


def rms_grads(dy, ds, s, rstd, weight, offset):
    """(d, dweight, magnitudes of the terms of d, magnitudes of the terms of dweight) in 64 bits"""
    c = s.shape[-1]
    n = s * rstd
    g = dy.double() * (1.0 if weight is None else offset + weight.double())
    d = rstd * (g - n * (g * n).sum(-1, keepdim=True) / c)
    size = rstd * (g.abs() + n.abs() * (g * n).abs().sum(-1, keepdim=True) / c)
    if ds is not None:
        d = d + ds.double()
        size = size + ds.double().abs()
    flat = (dy.double() * n).reshape(-1, c)
    return d, flat.sum(0), size, flat.abs().sum(0)


def within(got, want, bound):
    """All finite, and nowhere further off than `bound` (a tensor or a number)."""
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all()
    off = (got - want).abs() - bound
    assert off.numel() == 0 or off.max() <= 0, "off by %.3e more than the bound, at %s" % (off.max(), (off == off.max()).nonzero()[0].tolist())


def rounded(want, dtype):
    """What one rounding to `dtype` may cost"""
    return U[dtype] * want.abs() + STEP[dtype]


def turned(t, cos, sin, interleaved):
    """t: (..., tokens, heads, D); cos, sin: (..., tokens, 1, pairs)"""
    pairs = cos.shape[-1]
    out = t.clone()
    if interleaved:
        a, b = t[..., 0:2 * pairs:2], t[..., 1:2 * pairs:2]
        out[..., 0:2 * pairs:2], out[..., 1:2 * pairs:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = t[..., :pairs], t[..., pairs:2 * pairs]
        out[..., :pairs], out[..., pairs:2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return out


def angles(positions, inv_freq, sections):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[..., axis] * inv_freq.double()).unsqueeze(-2)
    return angle.cos(), angle.sin()


def rotary(t, weight, positions, inv_freq, sections, eps, interleaved, offset):
    """(output, normed without the weight, rstd) in 64 bits"""
    cos, sin = angles(positions, inv_freq, sections)
    t = t.double()
    n, rstd, w = t, None, 1.0
    if weight is not None:
        rstd = 1.0 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
        n, w = t * rstd, offset + weight.double()
    return turned(n * w, cos, sin, interleaved), n, rstd


def rotary_grads(dout, weight, n, rstd, positions, inv_freq, sections, interleaved, offset):
    """(dx, dweight, magnitudes of the terms of dx, of dweight) in 64 bits"""
    cos, sin = angles(positions, inv_freq, sections)
    g = turned(dout.double(), cos, -sin, interleaved)
    big = turned(dout.double().abs(), cos.abs(), -sin.abs(), interleaved).abs() + turned(dout.double().abs(), cos.abs(), sin.abs(), interleaved).abs()
    if weight is None:
        return g, None, big, None
    w = offset + weight.double()
    gw, bw = g * w, big * w.abs()
    d = rstd * (gw - n * (gw * n).mean(-1, keepdim=True))
    size = rstd * (bw + n.abs() * (bw * n.abs()).mean(-1, keepdim=True))
    c = n.shape[-1]
    return d, (g * n).reshape(-1, c).sum(0), size, (big * n.abs()).reshape(-1, c).sum(0)
