"""Gradients of fp32 norm weights beside 16-bit queries and keys: the angles and the reciprocal root mean square behind them are fp32's."""
import math

import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _weight_gradient(x, dout, position, inv_freq, interleaved=False):
    """that of one token's one head"""
    w = torch.ones(x.numel(), device="cuda", requires_grad=True)
    at = torch.full((1, 1), position, device="cuda", dtype=torch.int64)
    q, _ = pkg.rotary(x.view(1, 1, -1), None, at, inv_freq, (inv_freq.numel(),), w, None, 0.0, interleaved)
    return torch.autograd.grad(q, w, dout.view(1, 1, -1))[0]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [128, 40, 14])
def test_sines_and_cosines(dtype, interleaved, d):
    # a head of ones has a root mean square of exactly one (the sum of ones is exact; the mean is one but for inv_d's rounding, which
    # makes it at most u off and the root half of that); against a gradient of one in each pair's first channel the weight's gradient is the cosine there,
    # less the sine in the second.  Each is off by the angle's last rounding (2^-26 turns, pi / 2 u) and one unit of sincospi (u).
    pairs = d // 2
    inv_freq = (10000.0 ** -(torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)).float()
    x = torch.ones(d, device="cuda", dtype=dtype)
    dout = torch.zeros(d, device="cuda", dtype=dtype)
    first = torch.arange(pairs, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    dout[first] = 1
    bound = (math.pi / 2 + 1) * ref.U32 + (0 if d == 128 else 1.5 * ref.U32)  # (half of u for the mean, one for the product by the root)
    for position in [1, 2, 3, 100, 997] + list(range(1500, 4500, 61)):
        got = _weight_gradient(x, dout, position, inv_freq, interleaved).double()
        angle = position * inv_freq.double()
        assert (got[first] - angle.cos()).abs().max() <= bound
        assert (got[second] + angle.sin()).abs().max() <= bound


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_root_mean_square(dtype):
    # a head of 128 equal values: their squares' sum has at most 22 + 7 bits in fp16 and 16 + 7 in bf16, so with values of eight bits it is exact;
    # one rounding of the root, one of the product
    inv_freq = torch.ones(64, device="cuda")
    for k in range(128, 256):
        x = torch.full((128,), k / 64.0, device="cuda", dtype=dtype)
        got = _weight_gradient(x, torch.ones_like(x), 0, inv_freq).double()
        assert (got - 1).abs().max() <= 2 * ref.U32 * (1 + ref.U32)
