"""Host side of the operators on token rows, without a GPU: refusals of the Python functions and of the C ABI, shapes of the
traced ops, modules."""
import ctypes

import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from channels_last_groupnorm_b200 import _native as nt

from .test_host import _buffer


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.rms_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.rms_norm_quant(x)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.RMSNorm(64)(x)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.rotary(x.view(4, 1, 64), None, torch.zeros(4, 1), torch.ones(32), (32,))
    with pytest.raises(RuntimeError, match="CUDA"):
        torch.ops.gnb200.rms_fwd(x, None, None, 1e-6, 0.0)


def test_modules():
    m = pkg.RMSNorm(8, offset=1.0)
    assert (m.weight == 0).all() and list(m.state_dict()) == ["weight"]
    assert pkg.RMSNorm(8, affine=False).weight is None
    with pytest.raises(ValueError, match="expected input"):
        m(torch.zeros(2, 9))
    r = pkg.AxialRotary(16, (2, 3, 3), base=100.0, qk_norm=True)
    assert sorted(r.state_dict()) == ["k_weight", "q_weight"]
    want = [100.0 ** -(i / n) for n in (2, 3, 3) for i in range(n)]
    assert torch.allclose(r.inv_freq, torch.tensor(want))
    assert r.half().inv_freq.dtype == torch.float32 and r.q_weight.dtype == torch.float16
    for bad in ((5, 4), (), (-1, 4), (0,)):
        with pytest.raises(ValueError):
            pkg.AxialRotary(16, bad)


def test_traced_shapes():
    x = torch.empty(2, 5, 300, device="meta", dtype=torch.bfloat16)
    r = torch.empty(2, 5, 300, device="meta")
    y, s, rstd = torch.ops.gnb200.rms_fwd(x, r, None, 1e-6, 0.0)
    assert y.shape == x.shape and y.dtype == x.dtype and s.dtype == torch.float32 and rstd.shape == (2, 5)
    assert torch.ops.gnb200.rms_fwd(x, None, None, 1e-6, 0.0)[1].numel() == 0
    q, scale, s = torch.ops.gnb200.rms_quant(x, r, None, 1e-6, 0.0, 128, 0)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (2, 5, 3) and s.shape == r.shape
    assert torch.ops.gnb200.rms_quant(x, None, None, 1e-6, 0.0, 0, 1)[1].shape == (2, 5, 1)
    heads = torch.empty(2, 5, 4, 64, device="meta")
    out = torch.ops.gnb200.rotary(heads, heads[:, :, :2], torch.empty(2, 5, 1, device="meta"), torch.empty(32, device="meta"), [32], None, None,
                                  1e-6, 0.0, False)
    assert out[0].shape == heads.shape and out[1].shape == (2, 5, 2, 64) and out[1].is_contiguous()


def test_rms_refusals_of_the_c_abi():
    one = _buffer(1 << 16)
    fwd = nt.lib.gnb200_rms_fwd

    def call(rows=2, c=8, dtype=0, rdtype=0, wdtype=0, x=one, r=None, w=None, y=one, s=None):
        return fwd(x, c, r, c, w, rows, c, 1e-6, 0.0, dtype, rdtype, wdtype, y, s, None, None)

    assert call(dtype=7) == -1 and "dtype" in nt.lib.gnb200_last_error().decode()
    assert call(c=0) == -1 and call(rows=-1) == -1
    assert call(x=None) == -1 and call(y=None) == -1
    assert call(r=one) == -1  # a residual without a place for the sum
    assert call(dtype=1, rdtype=2, r=one, s=one) == -1 and call(dtype=1, wdtype=2, w=one) == -1
    assert call(c=(1 << 30) + 8) == -4
    assert call(rows=0) == 0
    q = nt.lib.gnb200_rms_fwd_8bit

    def codes(block=0, form=0, scale=one):
        return q(one, 8, None, 8, None, 2, 8, 1e-6, 0.0, 0, 0, 0, block, form, one, scale, None, None)

    assert codes(block=16) == -1 and codes(form=2) == -1 and codes(scale=None) == -1
    bwd = nt.lib.gnb200_rms_bwd

    def back(dy=one, rstd=one, dw=None, w=None, ds_out=None, rows=2):
        return bwd(dy, 8, None, 8, one, 8, None, 8, w, rstd, rows, 8, 0.0, 0, 0, 0, one, ds_out, dw, None, 0, None)

    assert back(dy=None) == -1 and back(rstd=None) == -1
    assert back(dw=one) == -1  # a gradient of no weight
    assert back(ds_out=one) == -1  # the sum has dy's type: one gradient
    assert back(rows=0) == 0


def test_rotary_refusals_of_the_c_abi():
    one = _buffer(1 << 16)
    strides = (ctypes.c_int64 * 3)(64, 64, 64)

    def args(**kw):
        a = nt.RotaryArgs(batch=1, tokens=1, q_heads=1, k_heads=0, head_dim=64, positions=one, pos_type=1, axes=1, inv_freq=one, eps=1e-6)
        a.sections[0] = 32
        for name, v in kw.items():
            if name == "sections":
                for i, s in enumerate(v):
                    a.sections[i] = s
            else:
                setattr(a, name, v)
        return a

    def call(q=one, out=one, **kw):
        a = args(**kw)
        return nt.lib.gnb200_rotary_fwd(ctypes.byref(a), q, strides, None, None, out, None, None)

    for kw in ({"dtype": 5}, {"pos_type": 3}, {"head_dim": 1}, {"q_heads": 0}, {"q_heads": -1, "k_heads": 3}, {"axes": 0}, {"axes": 9}, {"sections": (33,)},
               {"sections": (-1,)}, {"sections": (0,)}, {"positions": None}, {"inv_freq": None}, {"q": None}, {"out": None}, {"batch": -1},
               {"dtype": 1, "q_weight": one, "q_weight_dtype": 2}, {"k_heads": 1}):
        assert call(**kw) == -1, kw
    assert call(head_dim=514) == -4 and call(q_heads=(1 << 20) + 1) == -4
    assert call(tokens=0) == 0
    assert nt.lib.gnb200_rotary_fwd(None, one, strides, None, None, one, None, None) == -1
    a = args(q_weight=one)
    assert nt.lib.gnb200_rotary_bwd(ctypes.byref(a), one, strides, None, None, None, None, None, None, one, None, one, None, None, 0, None) == -1  # no q
    assert nt.lib.gnb200_rotary_bwd(ctypes.byref(a), one, strides, None, None, one, strides, None, None, one, None, None, None, None, 0, None) == -1
