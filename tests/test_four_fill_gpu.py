"""What lies behind a row's channels, up to a whole unit of 32, where the row has infinities or NaN: zeros, by every route."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import four_reference as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _check_fill(codes, scales, c, block, bad):
    """bad: rows whose channels are all NaN.  Codes behind the channels are zeros, of either sign, their blocks' scales the smallest; blocks of channels have the NaN."""
    rows, wide = bad.shape[0], codes.shape[-1] * 2
    assert (R.unpacked(codes)[:, c:] & 7 == 0).all()
    byte = R.untiled(scales, rows, wide // block)
    held = R.up(c, block) // block  # blocks that have a channel
    nan = 0x7F if block == 16 else 0xFF
    assert ((byte[:, :held] == nan) == bad.unsqueeze(1)).all()
    assert (byte[:, held:] == 1).all()  # 2^-9 in e4m3 (in blocks of 32 the last one has a channel)


# groups of lanes of a warp, CTAs, rows beyond what a CTA holds; the last unit with one block of channels and with two, aligned and odd
@pytest.mark.parametrize("c", [3, 16, 24, 40, 48, 67, 72, 520, 1064, 1111, 1125, 4112, 8200, 8213, 16400, 20001, 33000, 40003])
@pytest.mark.parametrize("dtype,residual", [(BF16, None), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("block", [16, 32])
def test_norm(c, dtype, residual, block):
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn((7, c), device="cuda", generator=g).to(dtype)
    r = None if residual is None else torch.randn((7, c), device="cuda", generator=g).to(residual)
    w = torch.rand(c + 1, device="cuda", generator=g).to(dtype)
    x[1, c // 2], x[4, 0], x[6, c - 1] = float("nan"), float("nan"), float("nan")
    bad = torch.tensor([0, 1, 0, 0, 1, 0, 1], device="cuda", dtype=torch.bool)
    routes = [pkg.rms_norm_quant_4bit(x, weight, r, block=block) for weight in (w[:c].clone(), w[1:])]  # (a weight off 16 bytes takes another route)
    for out in routes:
        _check_fill(out[0], out[1], c, block, bad)
    same = pkg.rms_norm_quant_4bit(x, w[1:].clone(), r, block=block)
    assert all(torch.equal(a.view(torch.uint8)[bad], b.view(torch.uint8)[bad]) for a, b in zip(routes[1][:1], same[:1]))
    assert torch.equal(routes[1][1].view(torch.uint8), same[1].view(torch.uint8))


@pytest.mark.parametrize("c", [16, 24, 48, 72, 1111])
def test_norm_of_zeros_without_eps(c):
    """An infinite root: the row is NaN, what lies behind it is not."""
    x = torch.zeros(3, c, device="cuda")
    x[1] = 1.0
    codes, scales = pkg.rms_norm_quant_4bit(x, eps=0.0)
    _check_fill(codes, scales, c, 16, torch.tensor([1, 0, 1], device="cuda", dtype=torch.bool))


@pytest.mark.parametrize("c", [3, 24, 40, 67, 1111])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block,scale", [(16, None), (16, 0.25), (32, None)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_quantize(c, dtype, block, scale, what):
    """The last block has the NaN for its scale and zeros for the codes behind the channels."""
    x = torch.randn(5, c, device="cuda").to(dtype)
    x[3, c - 1] = what
    codes, scales = pkg.quantize_4bit(x, block, None if scale is None else torch.full((1,), scale, device="cuda"))
    assert (R.unpacked(codes)[:, c:] & 7 == 0).all()
    byte = R.untiled(scales, 5, codes.shape[-1] * 2 // block)
    nan = 0x7F if block == 16 else 0xFF
    assert byte[3, (c - 1) // block] == nan and (byte == nan).sum() == 1
