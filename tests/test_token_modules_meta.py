"""Modules that are built on the meta device, given memory and loaded afterwards."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg


def _emptied(m, device="cpu"):
    """`to_empty`, with memory that holds something else"""
    m.to_empty(device=device)
    with torch.no_grad():
        for p in m.parameters():
            p.fill_(float("nan"))
    return m


@pytest.mark.parametrize("shared", [False, True])
def test_rotary_frequencies_come_back(shared):
    args = dict(base=500.0, shared=shared, qk_norm=True)
    want = pkg.AxialRotary(16, (2, 3, 3), **args)
    with torch.no_grad():
        want.q_weight.normal_()
    m = _emptied(pkg.AxialRotary(16, (2, 3, 3), device="meta", **args))
    assert not any(m.load_state_dict(want.state_dict()))
    assert torch.equal(m.inv_freq, want.inv_freq) and torch.equal(m.q_weight, want.q_weight)
    with torch.device("meta"):
        m = pkg.AxialRotary(16, (2, 3, 3), **args)
    m = _emptied(m.half())
    m.reset_parameters()
    assert torch.equal(m.inv_freq, want.inv_freq) and m.inv_freq.dtype == torch.float32
    assert (m.q_weight == 1).all() and (m.k_weight == 1).all() and m.q_weight.dtype == torch.float16


def test_rotary_frequencies_are_not_emptied_and_ones_of_the_user_are_kept():
    m = pkg.AxialRotary(16, (8,))
    before = m.inv_freq.clone()
    assert torch.equal(_emptied(m).inv_freq, before)
    m.inv_freq = torch.arange(8.0) * 0.1
    assert torch.equal(m.half().inv_freq, torch.arange(8.0) * 0.1)
    assert torch.equal(_emptied(m).inv_freq, torch.arange(8.0) * 0.1)
    m.reset_parameters()
    assert torch.equal(m.inv_freq, before)
    assert m.to("meta").inv_freq.is_meta


def test_norm_weight_comes_back():
    m = _emptied(pkg.RMSNorm(8, offset=1.0, device="meta", dtype=torch.bfloat16))
    m.reset_parameters()
    assert (m.weight == 0).all() and m.weight.dtype == torch.bfloat16
    assert pkg.RMSNorm(8, offset=0.25).weight.tolist() == [0.75] * 8
    pkg.RMSNorm(8, affine=False).reset_parameters()
