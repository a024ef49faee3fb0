"""The C entry points of the norm on rows that all begin between vector boundaries, as far behind one as each other: the vector kernels take
them in a shifted frame.  Everything around the inputs is NaN, around the outputs a pattern that has to stay."""
import ctypes

import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from channels_last_groupnorm_b200 import _native as nt
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODES = {F32: 0, F16: 1, BF16: 2}
GUARD = 64
# as in test_token_norm_gpu.py: at most 64 terms a thread and 14 levels of additions, halved by the root, and the norm's own operations
FORWARD = 48 * ref.U32
EPS = 1e-6


class Framed:
    """(rows, c) values `skew` elements behind a vector boundary, in a buffer of NaN or, as an output, of a pattern"""

    def __init__(self, skew, rows, c, dtype, values=None, gap=0):
        self.out = values is None
        stride = c + gap
        size = (rows - 1) * stride + c
        self.flat = torch.empty(2 * GUARD + skew + size, device="cuda", dtype=dtype)
        raw = self.flat.view(torch.uint8)
        raw.fill_(0x5A)
        if not self.out:
            self.flat.fill_(float("nan"))
        self.view = self.flat[GUARD + skew:].as_strided((rows, c), (stride, 1))
        if not self.out:
            self.view.copy_(values)
        self.at = ctypes.c_void_p(self.view.data_ptr())
        self.ends = (GUARD + skew, GUARD + skew + size)

    def untouched(self):
        one = torch.tensor([0x5A], device="cuda", dtype=torch.uint8)
        return bool((self.flat[:self.ends[0]].view(torch.uint8) == one).all() and (self.flat[self.ends[1]:].view(torch.uint8) == one).all())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _at(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


TYPES = [(BF16, BF16), (F16, F32), (F32, F32), (BF16, None)]
# narrower than the overhang of a vector; lanes of a warp, with one and with several vectors; a CTA with few and with many; rows of one, two
# and several turns; even rows that begin at odd places
SHAPES = [(1, 4), (2, 9), (3, 1), (3, 4), (5, 3), (6, 700), (7, 2), (9, 5000), (31, 17), (150, 3), (640, 65), (999, 2000), (1111, 2), (1111, 3000), (2050, 300),
          (4096, 5), (9957, 301), (12345, 2), (16385, 1)]


def _values(c, rows, dtype, wide):
    g = torch.Generator(device="cuda").manual_seed(c)

    def normal(dt):
        return torch.randn(rows, c, device="cuda", generator=g).to(dt)

    x, dy, w = normal(dtype), normal(dtype), (torch.rand(c, device="cuda", generator=g) + 0.5).to(dtype)
    return (x, dy, w) + ((None, None) if wide is None else (normal(wide), normal(wide)))


@pytest.mark.parametrize("c,rows", SHAPES)
@pytest.mark.parametrize("dtype,wide", TYPES)
def test_forward_and_backward(c, rows, dtype, wide):
    x, dy, w, r, ds = _values(c, rows, dtype, wide)
    ve = 4 if dtype == F32 else 8
    want, sums, rstd = ref.rms(x, w, r, EPS, 0.0)
    stored = None if wide is None else (x.float() + r.float()).to(wide)
    again = wide not in (None, F32)  # (the residual and x instead of the stored sum)
    d, dw, size, wsize = ref.rms_grads(dy, ds, sums, rstd, w, 0.0)
    plain = pkg.rms_norm(x, w, r, EPS)
    plain = plain if wide is None else plain[0]
    s_code, wide_or = CODES[wide or dtype], wide or dtype
    need = nt.lib.gnb200_rms_bwd_workspace_bytes(rows, c, CODES[dtype], s_code)
    ws = torch.empty(max(1, need), device="cuda", dtype=torch.uint8)
    for skew in range(1, ve):
        gap = 0 if skew % 2 else 2 * ve  # rows at another distance that keeps the frame
        X, Y, rs = Framed(skew, rows, c, dtype, x, gap), Framed(skew, rows, c, dtype), torch.empty(rows, device="cuda")
        R = S = None
        if wide is not None:
            R, S = Framed(skew, rows, c, wide, r, gap), Framed(skew, rows, c, wide)
        nt.check(nt.lib.gnb200_rms_fwd(X.at, c + gap, R and R.at, c + gap, _at(w), rows, c, EPS, 0.0, CODES[dtype], s_code, CODES[dtype], Y.at, S and S.at,
                                       _at(rs), _stream()))
        ref.within(Y.view, want, ref.rounded(want, dtype) + FORWARD * want.abs())
        ref.within(rs, rstd.squeeze(-1), FORWARD * rstd.squeeze(-1))
        assert Y.untouched()
        if c % ve:
            assert torch.equal(Y.view, plain)  # wherever the row stands
        if S:
            assert torch.equal(S.view, stored) and S.untouched()
        # backward: from x alone, from the sum, or from x and the residual
        DY, DX = Framed(skew, rows, c, dtype, dy, gap), Framed(skew, rows, c, dtype)
        SUM = X if wide is None else R if again else Framed(skew, rows, c, wide, stored, gap)
        DS = None if ds is None else Framed(skew, rows, c, wide_or, ds, gap)
        DO = Framed(skew, rows, c, wide) if wide is not None and wide != dtype else None
        got = torch.empty_like(w)
        nt.check(nt.lib.gnb200_rms_bwd(DY.at, c + gap, DS and DS.at, c + gap, SUM.at, c + gap, X.at if again else None, c + gap, _at(w), _at(rs), rows, c, 0.0,
                                       CODES[dtype], s_code, CODES[dtype], DX.at, DO and DO.at, _at(got), _at(ws), need, _stream()))
        ref.within(DX.view, d, ref.rounded(d, dtype) + 2 * FORWARD * size)
        assert DX.untouched()
        if DO:
            ref.within(DO.view, d, ref.rounded(d, wide) + 2 * FORWARD * size)
            assert DO.untouched()
        ref.within(got, dw, ref.rounded(dw, dtype) + (FORWARD + (rows + 64) * ref.U32) * wsize)


@pytest.mark.parametrize("c,rows", SHAPES)
@pytest.mark.parametrize("dtype,wide", TYPES)
@pytest.mark.parametrize("block,form", [(0, 0), (32, 0), (128, 0), (64, 1)])
def test_codes(c, rows, dtype, wide, block, form):
    x, _, w, r, _ = _values(c, rows, dtype, wide)
    ve = 4 if dtype == F32 else 8
    blocks = -(-c // block) if block else 1
    want = None
    plain = pkg.rms_norm_quant(x, w, r, EPS, block=block, dtype=torch.int8 if form else torch.float8_e4m3fn)
    for skew in range(1, ve):
        X, Q = Framed(skew, rows, c, dtype, x), Framed(skew, rows, c, torch.uint8)
        R = S = None
        if wide is not None:
            R, S = Framed(skew, rows, c, wide, r), Framed(skew, rows, c, wide)
        SC = Framed(0, rows, blocks, F32)
        nt.check(nt.lib.gnb200_rms_fwd_8bit(X.at, c, R and R.at, c, _at(w), rows, c, EPS, 0.0, CODES[dtype], CODES[wide or dtype], CODES[dtype], block, form, Q.at,
                                            SC.at, S and S.at, _stream()))
        assert Q.untouched() and SC.untouched() and (S is None or S.untouched())
        if want is None:
            want = (Q.view.clone(), SC.view.clone())
            y = ref.rms(x, w, r, EPS, 0.0)[0]
            most = torch.stack([p.abs().amax(-1) for p in y.split(block or c, -1)], -1) / (127.0 if form else 448.0)
            ref.within(SC.view, most.clamp_min(2.0 ** -126), (FORWARD + 2 * ref.U32) * most + 2.0 ** -140)
        if c % ve:  # wherever the row stands
            assert torch.equal(Q.view, plain[0].view(torch.uint8)) and torch.equal(SC.view, plain[1])
        assert torch.equal(Q.view, want[0]) and torch.equal(SC.view, want[1])


@pytest.mark.parametrize("c,rows", [(640, 300), (4096, 40), (16384, 3)])
@pytest.mark.parametrize("dtype,wide", TYPES)
def test_weights_off_vector_boundaries(c, rows, dtype, wide):
    # a weight that is a piece of a flat buffer of parameters: every result as with one of its own
    x, dy, w, r, ds = _values(c, rows, dtype, wide)
    flat = torch.full((c + 9,), float("nan"), device="cuda", dtype=dtype)
    odd = flat[3:3 + c]
    odd.copy_(w)
    want, sums, rstd = ref.rms(x, w, r, EPS, 0.0)
    leaves = [t.requires_grad_(True) for t in (x, odd.detach(), r) if t is not None]
    out = pkg.rms_norm(leaves[0], leaves[1], None if wide is None else leaves[2], EPS)
    outs, cots = ((out,), (dy,)) if wide is None else (out, (dy, ds))
    ref.within(outs[0].detach(), want, ref.rounded(want, dtype) + FORWARD * want.abs())
    grads = torch.autograd.grad(outs, leaves, cots)
    d, dw, size, wsize = ref.rms_grads(dy, ds, sums, rstd, w, 0.0)
    ref.within(grads[0], d, ref.rounded(d, dtype) + 2 * FORWARD * size)
    ref.within(grads[1], dw, ref.rounded(dw, dtype) + (FORWARD + (rows + 64) * ref.U32) * wsize)
    with torch.no_grad():
        q, scale = pkg.rms_norm_quant(x, odd, r, EPS, block=128)[:2]
    per = scale.double().repeat_interleave(128, -1)
    half = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * per)
    ref.within(q.double() * per, want, half * (1 + 2.0 ** -8) + 2 * FORWARD * want.abs())
