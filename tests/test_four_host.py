"""Rows in four bits and dropout without a GPU: the definition's own checks, refusals, traced shapes, modules."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from channels_last_groupnorm_b200 import _native as nt
from tests import dropout_reference as D
from tests import four_reference as R

from .test_host import _buffer


def test_definition_of_codes():
    t = torch.tensor([0.0, 0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 6.0, 100.0, -0.3, float("nan")], dtype=torch.float64)
    assert R.nearest(t).tolist() == [0, 0, 1, 2, 2, 4, 4, 6, 6, 7, 7, 7, 9, 7]


def test_tiles_are_read_back():
    scales = torch.arange(300 * 7, dtype=torch.int64).remainder(251).to(torch.uint8).view(300, 7)
    tiles = R.tiled(scales)
    assert tiles.shape == (384, 8)
    assert torch.equal(R.untiled(tiles, 300, 7), scales)
    # row 33 of block 5: second tile along the row, lane 1, word 1, byte 1
    assert tiles.reshape(-1)[512 + 16 + 4 + 1] == scales[33, 5]


def test_sizes():
    assert nt.lib.gnb200_4bit_code_bytes(3, 33) == 3 * 32
    assert nt.lib.gnb200_4bit_scale_bytes(3, 33, 16) == 128 * 4 and nt.lib.gnb200_4bit_scale_bytes(129, 129, 32) == 2 * 2 * 512
    assert nt.lib.gnb200_4bit_scale_bytes(3, 33, 8) == 0


def test_traced_shapes():
    x = torch.empty(2, 70, 100, device="meta", dtype=torch.bfloat16)
    codes, scales = torch.ops.gnb200.quantize_4bit(x, 16, None)
    assert codes.shape == (2, 70, 64) and codes.dtype == torch.float4_e2m1fn_x2
    assert scales.shape == (256, 8) and scales.dtype == torch.float8_e4m3fn
    codes, scales, s = torch.ops.gnb200.rms_quant_4bit(x, x.float(), None, 1e-6, 0.0, 32, None)
    assert scales.shape == (256, 4) and scales.dtype == torch.float8_e8m0fnu and s.dtype == torch.float32
    assert torch.ops.gnb200.dequantize_4bit(codes, scales, 100, None, torch.float16).shape == x.shape
    w, ws = torch.ops.gnb200.quantize_4bit(torch.empty(9, 100, device="meta"), 32, None)
    y = torch.ops.gnb200.linear_4bit(codes, scales, w, ws, None, None, None, torch.float16)
    assert y.shape == (2, 70, 9) and y.dtype == torch.float16
    s = torch.ops.gnb200.dropout_add(x, x.float(), 0.1, None, 0, 0)
    assert s.shape == x.shape and s.dtype == torch.float32


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    for call in (pkg.quantize_4bit, pkg.rms_norm_quant_4bit, pkg.dropout_add, pkg.RMSNorm(64).quantize_4bit, pkg.DropoutAdd(), pkg.Linear4bit):
        with pytest.raises(ValueError, match="CUDA"):
            call(x)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8).view(torch.float4_e2m1fn_x2), torch.zeros(128, 4).to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.dequantize_4bit(codes, scales)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.linear_4bit(codes, scales, codes, scales)
    for call in (lambda: torch.ops.gnb200.quantize_4bit(x, 16, None), lambda: torch.ops.gnb200.dropout_add(x, None, 0.1, None, 0, 0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_refusals_of_the_c_abi():
    one = _buffer(1 << 16)
    lib = nt.lib

    def said(rc, words):
        return rc < 0 and words in lib.gnb200_last_error().decode()

    def quantize(rows=2, c=64, dtype=0, block=16, g=None, x=one, codes=one, scales=one):
        return lib.gnb200_quantize_4bit(x, c, rows, c, dtype, block, g, codes, scales, None)

    assert said(quantize(dtype=3), "dtype") and said(quantize(block=8), "block") and said(quantize(block=32, g=one), "whole tensor")
    assert said(quantize(rows=-1), "rows") and said(quantize(c=0), "rows") and said(quantize(x=None), "null") and said(quantize(scales=None), "null")
    assert quantize(rows=2 ** 31) == -4 and quantize(c=2 ** 30 + 1) == -4
    assert said(quantize(codes=one.value + 8 if hasattr(one, "value") else int(one) + 8), "16 bytes")
    assert quantize(rows=0, x=None) == 0

    def back(rows=2, c=64, block=16, g=None, dtype=0, codes=one):
        return lib.gnb200_dequantize_4bit(codes, one, rows, c, block, g, dtype, one, None)

    assert said(back(dtype=3), "dtype") and said(back(block=64), "block") and said(back(codes=None), "null") and back(rows=0) == 0

    def norm(rows=2, c=64, dtype=1, rdtype=1, wdtype=1, r=None, s=None, block=16):
        return lib.gnb200_rms_fwd_4bit(one, c, r, c, None, rows, c, 1e-6, 0.0, dtype, rdtype, wdtype, block, None, one, one, s, None)

    assert said(norm(r=one), "null") and said(norm(r=one, s=one, rdtype=2), "residual") and said(norm(block=0), "block") and norm(rows=0) == 0

    def linear(tokens=2, features=8, c=64, block=16, g=None, bias_dtype=0, dtype=0, w=one):
        return lib.gnb200_linear_4bit(one, one, g, w, one, None, None, tokens, features, c, block, bias_dtype, dtype, one, None)

    assert said(linear(dtype=5), "dtype") and said(linear(bias_dtype=-1), "dtype") and said(linear(block=0), "block")
    assert said(linear(block=32, g=one), "whole tensor") and said(linear(tokens=-1), "negative") and said(linear(c=0), "positive") and said(linear(w=None), "null")
    assert linear(tokens=2 ** 31) == -4 and linear(features=2 ** 30 + 1) == -4 and linear(tokens=0) == 0 and linear(features=0) == 0

    def dropout(n=8, p=0.1, x=one, r=None, dtype=1, out_dtype=1, out=one):
        return lib.gnb200_dropout_add(x, r, n, p, None, 1, 2, dtype, out_dtype, out, None)

    assert said(dropout(dtype=4), "dtype") and said(dropout(out_dtype=2), "types") and said(dropout(dtype=0, r=one), "residual")
    assert said(dropout(n=-1), "negative") and said(dropout(p=1.0), "p is") and said(dropout(p=-0.1), "p is") and said(dropout(p=float("nan")), "p is")
    assert said(dropout(x=None), "null") and said(dropout(out=None), "null") and dropout(n=0) == 0


def test_words_of_the_generator():
    # the published answers of Philox 4x32-10 to counters and keys of zeros and of ones
    assert D.philox(0, 0, 0).tolist() == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert D.philox(2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1).tolist() == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_modules():
    assert pkg.DropoutAdd(0.25, layer=3).extra_repr() == "p=0.25, layer=3"
    for p in (1.0, -0.1, float("nan")):
        with pytest.raises(ValueError, match="less than 1"):
            pkg.DropoutAdd(p)
