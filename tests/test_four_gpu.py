"""Rows to four bits, back, and through the norm, against the definition in 64 bits."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import four_reference as R
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# one channel; parts of a vector, a block, a unit; a tile of scales and one more block; odd; rows of a CTA and beyond
WIDTHS = [1, 3, 16, 31, 32, 33, 48, 64, 72, 130, 264, 1000, 1111, 1352, 4096, 5120]
ROWS = [1, 2, 31, 33, 127, 128, 129, 700]


def _rows(rows, c, dtype, seed=0, spread=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, c), device="cuda", generator=g)
    if spread:  # blocks of very different sizes, some of zeros, some that saturate
        x *= torch.exp2(torch.randint(-14, 9, (rows, c // 16 + 1), device="cuda", generator=g).float()).repeat_interleave(16, -1)[:, :c]
        x *= (torch.rand((rows, c // 16 + 1), device="cuda", generator=g) > 0.1).float().repeat_interleave(16, -1)[:, :c]
    return x.to(dtype)


def _scale(value):
    return None if value is None else torch.full((1,), value, device="cuda")


def _check_codes(x, codes, scales, block, scale):
    c = x.shape[-1]
    want, byte = R.quantised(x.reshape(-1, c), block, scale)
    assert codes.dtype == torch.float4_e2m1fn_x2 and codes.shape == x.shape[:-1] + (R.up(c, 32) // 2,)
    assert scales.dtype == (torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu)
    tiles = R.tiled(byte)
    assert scales.shape == tiles.shape and torch.equal(scales.view(torch.uint8), tiles)
    assert torch.equal(codes.view(torch.uint8).reshape(-1, codes.shape[-1]), R.packed(want))


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block,scale", [(16, None), (16, 2.0 ** -7), (16, 0.0371), (32, None)])
def test_quantize(c, dtype, block, scale):
    x, s = _rows(7, c, dtype, c), _scale(scale)
    _check_codes(x, *pkg.quantize_4bit(x, block, s), block, s)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("c", [40, 512, 1111])
@pytest.mark.parametrize("block", [16, 32])
def test_quantize_rows(rows, c, block):
    x = _rows(rows, c, BF16, rows)
    _check_codes(x, *pkg.quantize_4bit(x, block), block, None)


@pytest.mark.parametrize("rows,c", [(40000, 64), (20000, 200), (9001, 1111)])
def test_quantize_many_rows(rows, c):
    """More rows than lanes, and rows whose lanes are a part of a warp."""
    x = _rows(rows, c, BF16, 1, spread=False)
    _check_codes(x, *pkg.quantize_4bit(x, 16), 16, None)


def test_halfway_values():
    """Quotients midway between two codes go to the even one, whatever the scale."""
    q = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device="cuda")
    q = torch.cat([q, -q])
    for scale in (1.0, 1.125, 1.75, 0.013671875, 2.0 ** -9, 448.0):  # e4m3 values
        x = (q * scale).reshape(1, 16)
        codes, scales = pkg.quantize_4bit(x, 16)
        assert R.unpacked(codes)[0, :16].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 8, 10, 10, 12, 12, 14, 14, 15]
        assert scales.float().reshape(-1)[0].item() == scale


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_unusual_values(block, dtype):
    """Infinities and NaN make their block NaN and no other; blocks of zeros, of the largest and of the smallest numbers."""
    x = torch.ones(5, 160, device="cuda", dtype=dtype)
    x[0, 5], x[1, 37], x[2, 64], x[3, 159] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[4, :32], x[4, 32:64], x[4, 64:96], x[4, 96:128] = 0.0, torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal, -torch.finfo(dtype).smallest_normal / 2
    codes, scales = pkg.quantize_4bit(x, block)
    _, byte = R.quantised(x, block)
    assert torch.equal(scales.view(torch.uint8), R.tiled(byte))
    y = pkg.dequantize_4bit(codes, scales, 160, dtype=F32)
    bad = ~torch.isfinite(x.reshape(5, -1, block)).all(-1, keepdim=True)
    assert torch.equal(torch.isnan(y).reshape(5, -1, block), bad.expand(5, 160 // block, block))
    assert (y[4, :32] == 0).all() and not torch.isnan(y[4]).any()
    # 1 / 6 is 0.171875 in e4m3, 1 / 0.171875 the code of 6; or 2^-2 and the code of 4
    assert (y[0, 32:] == (6 * 0.171875 if block == 16 else 1.0)).all()


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block,scale", [(16, None), (16, 0.0371), (32, None)])
def test_dequantize(c, dtype, block, scale):
    x, s = _rows(131, c, F32, c, spread=False), _scale(scale)
    codes, scales = pkg.quantize_4bit(x, block, s)
    y = pkg.dequantize_4bit(codes, scales, c, s, dtype)
    want = R.values(codes, scales, s)[:, :c]
    assert y.dtype == dtype and y.is_contiguous()
    assert torch.equal(y, want.float().to(dtype))  # (code times block scale is exact in 32 bits)
    # no further from x than half a step of the codes and the scale's rounding: 1 of 6 between the largest codes, 2^-4 of the scale
    step = x.abs().reshape(131, -1).amax() * (1 / 6 + 2.0 ** -4)
    assert (want - x.double()).abs().max() <= (step if block == 16 else step * 1.5)


def test_layouts_and_batches():
    """Slices of wider rows, rows that begin off a vector, transposed rows, three dimensions: the same codes as of a copy."""
    wide = _rows(64, 1000, BF16, 5)
    for x in (wide[:, 8:520], wide[:, 3:515], wide[::2, :96], wide.t()[:, :40], wide[:, :960].view(8, 8, 960), wide[:60, :96].view(4, 15, 96)[:, 2:9]):
        for block in (16, 32):
            a, b = pkg.quantize_4bit(x, block), pkg.quantize_4bit(x.contiguous().clone(), block)
            assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))
            _check_codes(x, *a, block, None)
    flat = _rows(1, 64 * 96 + 1, F16, 6).reshape(-1)[1:].view(64, 96)  # contiguous, off every vector
    _check_codes(flat, *pkg.quantize_4bit(flat, 16), 16, None)


def test_nothing():
    for shape in ((0, 64), (3, 0, 64)):
        codes, scales = pkg.quantize_4bit(torch.empty(shape, device="cuda"))
        assert codes.shape == shape[:-1] + (32,) and scales.shape == (0, 4)
        assert pkg.dequantize_4bit(codes, scales).shape == shape
        w = pkg.quantize_4bit(torch.ones(8, 64, device="cuda"))
        assert pkg.linear_4bit(codes, scales, *w).shape == shape[:-1] + (8,)


# ---------------------------------------------------------------------------------------------- norm

# the arithmetic of the norm before its codes, relative: as in the tests of rms_norm
NORM = 48 * ref.U32


def _check_norm(x, w, r, block, scale, eps=1e-6, offset=0.0):
    c = x.shape[-1]
    out = pkg.rms_norm_quant_4bit(x, w, r, eps, offset, block, scale)
    codes, scales = out[:2]
    want, sums, _ = ref.rms(x, w, r, eps, offset)
    if r is not None:
        assert torch.equal(out[2], (x.float() + r.float()).to(r.dtype))
    rows, wide = want.reshape(-1, c).shape[0], codes.shape[-1] * 2
    y = torch.nn.functional.pad(want.reshape(rows, c), (0, wide - c)).reshape(rows, -1, block)
    g = 1.0 if scale is None else float(scale)
    step = R.scale_values(R.untiled(scales, rows, wide // block), block).unsqueeze(-1)
    most = y.abs().amax(-1, keepdim=True)
    if block == 16:  # the scale is off by half a step of e4m3, or cut off
        exact = (most / (6 * g)).clamp(2.0 ** -9, 448.0)
        assert ((step - exact).abs() <= exact * (2.0 ** -4 + NORM) + 2.0 ** -10).all()
    else:  # a power of two, of the largest magnitude
        low, high = torch.exp2(torch.floor(torch.log2(most * (1 - NORM))) - 2), torch.exp2(torch.floor(torch.log2(most * (1 + NORM))) - 2)
        assert ((step >= low.clamp(min=2.0 ** -127)) & (step <= high.clamp(min=2.0 ** -127))).all()
    q = y / (step * g)
    half = torch.where(q.abs() <= 2, 0.25, torch.where(q.abs() <= 4, 0.5, 1.0))
    value = R.values(codes, scales).reshape(rows, -1, block) / step
    assert ((value - q.clamp(-6, 6)).abs() <= half + 2 * NORM * q.abs() + 1e-9).all()
    assert torch.equal(scales.view(torch.uint8), R.tiled(R.untiled(scales, rows, wide // block)))  # zeros where there is nothing
    flat = R.unpacked(codes)
    assert (flat[:, c:] % 8 == 0).all()
    return out


def _norm_inputs(rows, c, dtype, residual, weight, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, c), device="cuda", generator=g).to(dtype)
    r = None if residual is None else (torch.randn((rows, c), device="cuda", generator=g) * 3).to(residual)
    w = None if weight is None else (torch.rand(c, device="cuda", generator=g) + 0.5).to(weight)
    return x, w, r


@pytest.mark.parametrize("c", WIDTHS + [8200, 16384, 16400, 20001, 33000])
@pytest.mark.parametrize("dtype,residual,weight", [(F32, F32, F32), (BF16, BF16, BF16), (F16, F32, F16), (BF16, None, F32), (F16, F16, None)])
def test_norm(c, dtype, residual, weight):
    for block, scale in ((16, None), (16, 0.004), (32, None)):
        _check_norm(*_norm_inputs(5, c, dtype, residual, weight, c), block, _scale(scale), 1e-5, 0.25)


@pytest.mark.parametrize("rows", [1, 2, 129, 1183, 1184, 3001])
@pytest.mark.parametrize("c", [24, 264, 640, 1000, 1111])
def test_norm_rows(rows, c):
    _check_norm(*_norm_inputs(rows, c, BF16, F32, BF16, rows), 16, _scale(2.0 ** -8))


def test_norm_is_the_norm_then_the_codes():
    """In 32 bits, where nothing is rounded between: but for sums in another order, quantize_4bit of rms_norm."""
    x, w, r = _norm_inputs(300, 2048, F32, F32, F32)
    codes, scales, s = pkg.rms_norm_quant_4bit(x, w, r, block=32)
    y, t = pkg.rms_norm(x, w, r)
    want, tiles = pkg.quantize_4bit(y, 32)
    assert torch.equal(s, t) and torch.equal(scales.view(torch.uint8), tiles.view(torch.uint8))
    # a code changes where a border lies in the last places of y: 48 u of them, in steps of an eighth at least
    assert (codes.view(torch.uint8) != want.view(torch.uint8)).float().mean() <= 16 * 48 * ref.U32 * 8


def test_norm_layouts():
    wide = _rows(64, 1000, BF16, 5, spread=False)
    w = torch.rand(1001, device="cuda").bfloat16()
    for x in (wide[:, 8:520], wide[:, 3:515], wide[::2, :96], wide.t()[:, :40]):
        for weight in (w[: x.shape[1]], w[1 : x.shape[1] + 1], w[::2][:40] if x.shape[1] == 40 else None):
            a = _check_norm(x, weight, x.flip(0), 16, None)
            b = pkg.rms_norm_quant_4bit(x.contiguous(), None if weight is None else weight.clone(), x.flip(0).contiguous())
            assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a[:2], b[:2]))


def test_norm_keeps_nan_in_its_row():
    x = torch.randn(6, 1111, device="cuda").bfloat16()
    x[2, 700], x[4, 3] = float("nan"), float("inf")
    codes, scales = pkg.rms_norm_quant_4bit(x)
    y = pkg.dequantize_4bit(codes, scales, 1111, dtype=F32)
    assert torch.isnan(y[[2]]).all() and torch.isnan(y[4, :16]).any()
    assert torch.isfinite(y[[0, 1, 3, 5]]).all()


def test_norm_sum_in_the_residual_buffer():
    """Through the C ABI the stream may be written where it was read."""
    from channels_last_groupnorm_b200 import _native as nt

    for c in (512, 1111, 40000):
        x, w, r = _norm_inputs(9, c, BF16, F32, BF16)
        want = pkg.rms_norm_quant_4bit(x, w, r)
        codes, scales, s = torch.zeros_like(want[0].view(torch.uint8)), torch.zeros_like(want[1].view(torch.uint8)), r.clone()
        rc = nt.lib.gnb200_rms_fwd_4bit(x.data_ptr(), c, s.data_ptr(), c, w.data_ptr(), 9, c, 1e-6, 0.0, 2, 0, 2, 16, None, codes.data_ptr(), scales.data_ptr(),
                                        s.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(codes, want[0].view(torch.uint8)) and torch.equal(scales, want[1].view(torch.uint8)) and torch.equal(s, want[2])


# ---------------------------------------------------------------------------------------------- use


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    one = torch.ones(1, device="cuda")
    codes, scales = pkg.quantize_4bit(x)
    for call, words in ((lambda: pkg.quantize_4bit(x.int()), "float32"), (lambda: pkg.quantize_4bit(x, 8), "block"), (lambda: pkg.quantize_4bit(x, 32, one), "whole tensor"),
                        (lambda: pkg.quantize_4bit(x, 16, one.double()), "scale"), (lambda: pkg.quantize_4bit(x, 16, one.cpu()), "scale"),
                        (lambda: pkg.quantize_4bit(x, 16, torch.ones(2, device="cuda")), "scale"), (lambda: pkg.quantize_4bit(x[:, :0]), "channels"),
                        (lambda: pkg.quantize_4bit(x.clone().requires_grad_(True)), "gradient"),
                        (lambda: pkg.rms_norm_quant_4bit(x, torch.ones(64, device="cuda").requires_grad_(True)), "gradient"),
                        (lambda: pkg.rms_norm_quant_4bit(x, torch.ones(65, device="cuda")), "weight"), (lambda: pkg.rms_norm_quant_4bit(x, None, x[:3]), "residual"),
                        (lambda: pkg.rms_norm_quant_4bit(x, None, x.half()), "residual"), (lambda: pkg.rms_norm_quant_4bit(x, block=0), "block"),
                        (lambda: pkg.dequantize_4bit(codes, scales, 65), "channels"), (lambda: pkg.dequantize_4bit(codes, scales, 32), "channels"),
                        (lambda: pkg.dequantize_4bit(codes.view(torch.uint8), scales), "codes"), (lambda: pkg.dequantize_4bit(codes, scales.float()), "scales"),
                        (lambda: pkg.dequantize_4bit(codes, scales[:64]), "scales"), (lambda: pkg.dequantize_4bit(codes, scales, dtype=torch.float64), "dtype"),
                        (lambda: pkg.RMSNorm(65).cuda().quantize_4bit(x), "expected input")):
        with pytest.raises(ValueError, match=words):
            call()
    with torch.no_grad():
        pkg.quantize_4bit(x.clone().requires_grad_(True))


def test_other_stream_and_graph():
    x, w, r = _norm_inputs(40, 512, BF16, BF16, BF16)
    scale = _scale(0.01)
    want = [pkg.rms_norm_quant_4bit(t, w, r, scale=scale) for t in (x, x * 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.rms_norm_quant_4bit(x, w, r, scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want[0]))
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.rms_norm_quant_4bit(held, w, r, scale=scale)
    for i in (1, 0):
        held.copy_((x, x * 2)[i])
        graph.replay()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want[i]))


@pytest.mark.parametrize("block", [16, 32])
def test_compiled(block):
    x, w, r = _norm_inputs(9, 200, BF16, F32, BF16)

    def call(x, w, r):
        a = pkg.quantize_4bit(x, block)
        b = pkg.rms_norm_quant_4bit(x, w, r, block=block)
        return a + b + (pkg.dequantize_4bit(a[0], a[1], 200),)

    torch._dynamo.reset()
    got, want = torch.compile(call, backend="aot_eager", fullgraph=True)(x, w, r), call(x, w, r)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


def test_far_rows():
    """Rows whose elements and bytes are counted in more than 32 bits."""
    rows, c = 36000, 131072  # 4.7e9 elements, 2.4e9 bytes of codes
    x = torch.empty(rows, c, device="cuda", dtype=BF16)
    x[-130:] = _rows(130, c, BF16, 3, spread=False)
    codes, scales = pkg.quantize_4bit(x, 32)
    want, tiles = pkg.quantize_4bit(x[-160:].clone(), 32)  # (whole tiles of scales end the call: 36000 = 281 * 128 + 32)
    assert torch.equal(codes[-130:].view(torch.uint8), want[-130:].view(torch.uint8))
    byte = R.untiled(scales[-128:], 32, c // 32)
    assert torch.equal(byte, R.untiled(tiles, 160, c // 32)[-32:])
    y = pkg.dequantize_4bit(codes, scales, c)
    assert torch.equal(y[-32:], pkg.dequantize_4bit(want, tiles, c)[-32:])


def test_codes_of_another_maker():
    """Codes and tiles laid out as documented, without the kernels, are read back and normed rows agree with them after a round trip."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for block in (16, 32):
        codes = torch.randint(0, 16, (77, 96), device="cuda", generator=g, dtype=torch.uint8)
        byte = torch.randint(0x30, 0x50, (77, 96 // block), device="cuda", generator=g).to(torch.uint8)
        kind = torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu
        rows, tiles = R.packed(codes).view(torch.float4_e2m1fn_x2), R.tiled(byte).view(kind)
        y = pkg.dequantize_4bit(rows, tiles, 96, dtype=F32)
        assert torch.equal(y.double(), R.values(rows, tiles))


def test_rows_behind_the_last_are_left():
    """Through the C ABI: codes and tiles of a call, and nothing behind them."""
    from channels_last_groupnorm_b200 import _native as nt

    for rows, c in ((5, 100), (130, 64), (33, 1111)):
        x = _rows(rows, c, BF16, 1)
        want = pkg.quantize_4bit(x)
        norm = pkg.rms_norm_quant_4bit(x)
        n, m = nt.lib.gnb200_4bit_code_bytes(rows, c), nt.lib.gnb200_4bit_scale_bytes(rows, c, 16)
        stream = torch.cuda.current_stream().cuda_stream
        for expect, call in ((want, lambda a, b: nt.lib.gnb200_quantize_4bit(x.data_ptr(), c, rows, c, 2, 16, None, a, b, stream)),
                             (norm, lambda a, b: nt.lib.gnb200_rms_fwd_4bit(x.data_ptr(), c, None, c, None, rows, c, 1e-6, 0.0, 2, 2, 2, 16, None, a, b, None, stream))):
            codes, tiles = (torch.full((k + 1024,), 0xA5, dtype=torch.uint8, device="cuda") for k in (n, m))
            assert call(codes.data_ptr(), tiles.data_ptr()) == 0
            assert torch.equal(codes[:n], expect[0].view(torch.uint8).reshape(-1)) and torch.equal(tiles[:m], expect[1].view(torch.uint8).reshape(-1))
            assert (codes[n:] == 0xA5).all() and (tiles[m:] == 0xA5).all()
