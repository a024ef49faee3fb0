"""Rows in four bits at the ends of their range: the largest numbers over small scales of the tensor, and the smallest."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import four_reference as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _check(x, scale):
    """Codes and scale bytes are those of the definition: IEEE quotients, saturating."""
    codes, scales = pkg.quantize_4bit(x, 16, scale)
    want, byte = R.quantised(x, 16, scale)
    assert torch.equal(scales.view(torch.uint8), R.tiled(byte))
    assert torch.equal(codes.view(torch.uint8), R.packed(want))
    return codes, scales


@pytest.mark.parametrize("c", [160, 163])  # aligned rows, and odd ones
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -14, 1e-4, 1 / 449, 1.0, 2.0 ** 100, 2.0 ** 117])
def test_largest_numbers(c, dtype, scale):
    """A quotient beyond the largest float saturates with its own sign, and leaves the other codes of its block as they are."""
    g = torch.tensor([scale], device="cuda")
    x = torch.zeros(6, c, device="cuda", dtype=dtype)
    big = torch.finfo(dtype).max
    d = 448 * scale
    ordinary = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.5, -1.5, -2.5, -5.0, 7.0], device="cuda").mul(d).clamp(-big, big).to(dtype)
    for row, most in enumerate((big, -big, 1e38, -1e38, 1e37, -1e36)):
        x[row, :14], x[row, 14], x[row, 15] = ordinary, most, -most / 2
        x[row, 16:32] = most
        x[row, 32:48], x[row, 40] = 0.0, most
        x[row, c - 1] = most
    codes, scales = _check(x, g)
    if d < 1e35:  # all of these saturate
        code = R.unpacked(codes)
        for row, sign in enumerate((0, 8, 0, 8, 0, 8)):
            assert code[row, 14] == 7 + sign and code[row, 15] == 15 - sign and (code[row, 16:32] == 7 + sign).all() and code[row, c - 1] == 7 + sign


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -99 * 1.37, 2.0 ** -60, 2.0 ** 110, 2.0 ** 117])
def test_ends_of_the_scale(dtype, scale):
    """Numbers of a block's own size where products and quotients are near the ends of fp32; those midway between two codes among them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((200, 320), device="cuda", generator=g, dtype=torch.float64)
    # scales of blocks from the smallest to the largest, no number beyond the type
    x *= torch.exp2(torch.randint(-12, 12, (200, 20), device="cuda", generator=g).double()).repeat_interleave(16, -1)
    x = (x * scale).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    codes, scales = _check(x, torch.tensor([scale], device="cuda"))
    # midway, over the scales just found: those of blocks whose largest number stays in place
    step = (R.scale_values(R.untiled(scales, 200, 20), 16) * float(torch.tensor(scale))).repeat_interleave(16, -1)
    places = torch.arange(320, device="cuda") % 16
    halves = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda", dtype=torch.float64)[places % 7]
    _check(torch.where((places < 14) & (x.reshape(200, 20, 16).abs().argmax(-1).repeat_interleave(16, -1) != places), halves * step, x.double()).to(dtype),
           torch.tensor([scale], device="cuda"))


@pytest.mark.parametrize("c,weight_at", [(64, 0), (67, 0), (64, 1)])  # aligned, odd, and without a common frame
def test_largest_numbers_of_the_norm(c, weight_at):
    """The norm's output over its scales saturates with its own sign too."""
    g = torch.tensor([2.0 ** -100], device="cuda")
    x = torch.randn(40, c, device="cuda").sign()
    weight = torch.full((c + 1,), 2.0 ** 100, device="cuda")[weight_at : c + weight_at]
    codes, scales = pkg.rms_norm_quant_4bit(x, weight, scale=g)
    assert torch.equal(R.unpacked(codes)[:, :c].to(torch.int32), torch.where(x > 0, 7, 15).int())
    assert (scales.float()[:1, :1] == 448).all()
