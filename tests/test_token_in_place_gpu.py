"""The C entry points with outputs in their inputs' own buffers: the bits of a call with buffers of its own, whichever kernel takes it."""
import ctypes

import pytest
import torch

from channels_last_groupnorm_b200 import _native as nt

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODES = {F32: 0, F16: 1, BF16: 2}


def _at(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _inputs(rows, c, dtype, wide):
    g = torch.Generator(device="cuda").manual_seed(c)
    x, dy = (torch.randn(rows, c, device="cuda", generator=g).to(dtype) for _ in range(2))
    r, ds = (torch.randn(rows, c, device="cuda", generator=g).to(wide) for _ in range(2))
    return x, r, (torch.rand(c, device="cuda", generator=g) + 0.5).to(dtype), dy, ds


# a group of lanes, a CTA, odd rows of both, rows beyond what a CTA holds (even and odd)
CASES = [(65, 640, BF16, BF16), (9, 4096, F16, F32), (700, 1111, BF16, BF16), (9, 12345, F16, F32), (5, 33000, BF16, BF16), (5, 33001, F32, F32),
         (5, 20000, BF16, F32)]


@pytest.mark.parametrize("rows,c,dtype,wide", CASES)
def test_forward(rows, c, dtype, wide):
    x, r, w, _, _ = _inputs(rows, c, dtype, wide)

    def call(x, r, y, s):
        rstd = torch.empty(rows, device="cuda")
        nt.check(nt.lib.gnb200_rms_fwd(_at(x), c, _at(r), c, _at(w), rows, c, 1e-6, 0.0, CODES[dtype], CODES[wide], CODES[dtype], _at(y), _at(s),
                                       _at(rstd), _stream()))
        return y, s, rstd

    want = call(x, r, torch.empty_like(x), torch.empty_like(r))
    x1, r1 = x.clone(), r.clone()
    for got in (call(x, r1, torch.empty_like(x), r1), call(x1, r.clone(), x1, torch.empty_like(r))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x2, r2 = x.clone(), r.clone()
    assert all(torch.equal(a, b) for a, b in zip(call(x2, r2, x2, r2), want))
    if dtype == wide:  # crosswise
        x3, r3 = x.clone(), r.clone()
        assert all(torch.equal(a, b) for a, b in zip(call(x3, r3, r3, x3), want))


@pytest.mark.parametrize("rows,c,dtype,wide", CASES)
@pytest.mark.parametrize("block", [0, 64])
def test_codes(rows, c, dtype, wide, block):
    x, r, w, _, _ = _inputs(rows, c, dtype, wide)

    def call(r, s):
        q = torch.empty(rows, c, device="cuda", dtype=torch.uint8)
        scale = torch.empty(rows, (c + block - 1) // block if block else 1, device="cuda")
        nt.check(nt.lib.gnb200_rms_fwd_8bit(_at(x), c, _at(r), c, _at(w), rows, c, 1e-6, 0.0, CODES[dtype], CODES[wide], CODES[dtype], block, 0, _at(q),
                                            _at(scale), _at(s), _stream()))
        return q, scale, s

    want = call(r, torch.empty_like(r))
    r1 = r.clone()
    assert all(torch.equal(a, b) for a, b in zip(call(r1, r1), want))


@pytest.mark.parametrize("rows,c,dtype,wide", CASES)
def test_backward(rows, c, dtype, wide):
    x, r, w, dy, ds = _inputs(rows, c, dtype, wide)
    again = wide != F32  # (the residual and x instead of the stored sum)
    s = r if again else x.float() + r
    rstd = torch.rsqrt((x.float() + r.float()).square().mean(-1) + 1e-6)
    ws = torch.empty(max(1, nt.lib.gnb200_rms_bwd_workspace_bytes(rows, c, CODES[dtype], CODES[wide])), device="cuda", dtype=torch.uint8)

    def call(dy, ds, dx, ds_out):
        dw = torch.empty_like(w)
        nt.check(nt.lib.gnb200_rms_bwd(_at(dy), c, _at(ds), c, _at(s), c, _at(x) if again else None, c, _at(w), _at(rstd), rows, c, 0.0, CODES[dtype],
                                       CODES[wide], CODES[dtype], _at(dx), _at(ds_out), _at(dw), _at(ws), ws.numel(), _stream()))
        return [t for t in (dx, ds_out, dw) if t is not None]

    out = None if dtype == wide else torch.empty_like(ds)
    want = call(dy, ds, torch.empty_like(dy), out)
    dy1, ds1 = dy.clone(), ds.clone()
    got = call(dy1, ds1, dy1, None if out is None else ds1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if dtype == wide:
        ds2 = ds.clone()
        assert all(torch.equal(a, b) for a, b in zip(call(dy, ds2, ds2, None), want))
