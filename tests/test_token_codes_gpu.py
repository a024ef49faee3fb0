"""The 8-bit codes of rms_norm_quant: those of y / scale, as a division rounds it, and what infinities and NaN leave."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
LARGEST = {E4M3: 448.0, torch.int8: 127.0}


def _codes(quotients, dtype):
    quotients = quotients.clamp(-LARGEST[dtype], LARGEST[dtype])
    return quotients.to(E4M3).float() if dtype == E4M3 else quotients.round()


# groups of lanes, a CTA with few and with many vectors, the same for odd rows, rows beyond what a CTA holds
@pytest.mark.parametrize("c", [64, 640, 4096, 8192, 1111, 9957, 33001])
@pytest.mark.parametrize("block", [0, 32, 128])
@pytest.mark.parametrize("dtype", [E4M3, torch.int8])
def test_codes_are_the_rounded_quotients(c, block, dtype):
    # fp32, whose y is stored as the kernel has it: the codes follow from y and the scales.  Values of eight bits put many quotients
    # midway between two codes or close to it.
    rows = max(64, min(4096, (1 << 21) // c))
    g = torch.Generator(device="cuda").manual_seed(c + block)
    x = torch.randn(rows, c, device="cuda", generator=g).bfloat16().float()
    x[0] = 0.0
    w = (torch.rand(c, device="cuda", generator=g) + 0.5).bfloat16().float()
    y = pkg.rms_norm(x, w)
    q, scale = pkg.rms_norm_quant(x, w, block=block, dtype=dtype)
    per = scale.repeat_interleave(block or c, -1)[:, :c]
    assert torch.equal(q.float(), _codes(y / per, dtype))


@pytest.mark.parametrize("c", [640, 1111, 4096, 33001])
@pytest.mark.parametrize("block", [0, 64])
def test_infinite_scale(c, block):
    x = torch.randn(3, c, device="cuda")
    w = torch.ones(c, device="cuda")
    w[5] = float("inf")
    q, scale = pkg.rms_norm_quant(x, w, block=block)
    assert torch.isinf(scale[:, 0]).all()
    last = c if block == 0 else block
    got = q.float()
    assert torch.isnan(got[:, 5]).all()  # infinity over itself
    got[:, 5] = 0
    assert (got[:, :last] == 0).all()  # what is finite over infinity
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("c", [640, 1111, 4096, 33001])
def test_nan_in_a_row_of_int8_codes(c):
    x = torch.randn(4, c, device="cuda")
    clean = pkg.rms_norm_quant(x, block=32, dtype=torch.int8)
    x[2, c // 3] = float("nan")
    for block in (0, 32):
        q, scale = pkg.rms_norm_quant(x, block=block, dtype=torch.int8)
        assert torch.isnan(scale[2]).all() and torch.isfinite(scale[[0, 1, 3]]).all()  # (the codes of such a row mean nothing)
        if block:
            assert torch.equal(q[[0, 1, 3]], clean[0][[0, 1, 3]]) and torch.equal(scale[[0, 1, 3]], clean[1][[0, 1, 3]])
