"""rms_norm and rms_norm_quant on the GPU against the definition in 64 bits."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# channels: one; fewer than a vector; one lane; odd; a group of lanes with a ragged end; one warp with several vectors a lane; one CTA with
# two and four vectors a thread; odd rows in a CTA with 4, 16 and 32 elements a thread; rows beyond what a CTA holds, aligned and odd
WIDTHS = [1, 3, 8, 31, 72, 256, 640, 1000, 1111, 1280, 4096, 5120, 8200, 12345, 16384, 16400, 20001, 33000]
# the sum of squares: at most 64 terms a thread or 5 + 9 levels of additions, each worth one u, halved by the square root; the
# square root, the division, two products and the addition of the residual: below 48 u
FORWARD = 48 * ref.U32


def _inputs(rows, c, dtype, residual=None, weight=None, seed=0, grads=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dt, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(dt)

    x = normal((rows, c), dtype)
    r = None if residual is None else normal((rows, c), residual, 3.0)
    w = None if weight is None else (torch.rand(c, device="cuda", generator=g) + 0.5).to(weight)
    if not grads:
        return x, w, r
    return x, w, r, normal((rows, c), dtype), None if residual is None else normal((rows, c), residual)


def _check_forward(x, w, r, eps=1e-6, offset=0.0):
    with torch.no_grad():
        out = pkg.rms_norm(x, w, r, eps, offset)
    y, s = (out, None) if r is None else out
    want, sums, _ = ref.rms(x, w, r, eps, offset)
    assert y.dtype == x.dtype and y.is_contiguous()
    ref.within(y, want, ref.rounded(want, x.dtype) + FORWARD * want.abs())
    if r is not None:
        assert s.dtype == r.dtype and s.is_contiguous()
        exact = (x.float() + r.float()).to(r.dtype)  # one addition in 32 bits, one rounding
        assert torch.equal(s, exact)


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype,residual,weight", [(F32, F32, F32), (BF16, BF16, BF16), (F16, F32, F16), (BF16, None, F32), (F16, F16, None)])
def test_forward(c, dtype, residual, weight):
    _check_forward(*_inputs(5, c, dtype, residual, weight))


@pytest.mark.parametrize("rows", [1, 2, 3, 33, 700, 9001])
@pytest.mark.parametrize("c", [24, 320, 1111, 2048])
def test_forward_rows(rows, c):
    _check_forward(*_inputs(rows, c, BF16, F32, F32))


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype,residual,weight", [(F32, F32, F32), (BF16, BF16, F32), (F16, F32, F16), (BF16, None, BF16), (F32, None, None),
                                                   (F16, F16, None)])
def test_backward(c, dtype, residual, weight, rows=7):
    x, w, r, dy, ds = _inputs(rows, c, dtype, residual, weight, grads=True)
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    out = pkg.rms_norm(x, w, r, 1e-5, 0.25)
    outs, cots = ((out,), (dy,)) if r is None else (out, (dy, ds))
    grads = list(torch.autograd.grad(outs, leaves, cots))
    # a 16-bit sum whose weight needs no gradient is taken as it was stored
    as_stored = r is not None and w is None and residual != F32
    stored = x.detach().double() if r is None else out[1].detach().double() if as_stored else x.detach().double() + r.detach().double()
    _, _, rstd = ref.rms(x.detach(), None, None if r is None else r.detach(), 1e-5, 0.0)
    d, dw, size, wsize = ref.rms_grads(dy, ds, stored, rstd, None if w is None else w.detach(), 0.25)
    # the dot product as the sum of squares above, and the terms' own operations
    fp32 = 2 * FORWARD
    dx = grads.pop(0)
    assert dx.dtype == dtype
    ref.within(dx, d, ref.rounded(d, dtype) + fp32 * size)
    if r is not None:
        dr = grads.pop(0)
        assert dr.dtype == residual
        ref.within(dr, d, ref.rounded(d, residual) + fp32 * size)
    if w is not None:
        got = grads.pop(0)
        assert got.dtype == weight
        ref.within(got, dw, ref.rounded(dw, weight) + (FORWARD + (rows + 64) * ref.U32) * wsize)


@pytest.mark.parametrize("rows,c", [(1, 64), (3, 48), (1000, 320), (5000, 136), (3000, 2056), (900, 999)])
def test_backward_many_rows(rows, c):
    test_backward(c, BF16, F32, BF16, rows)


def test_gradients_of_one_output_only():
    x, w, r, dy, ds = _inputs(9, 192, F32, F32, F32, grads=True)
    for t in (x, w, r):
        t.requires_grad_(True)
    y, s = pkg.rms_norm(x, w, r)
    gx, gr = torch.autograd.grad(s, (x, r), ds)  # the norm not used: the sum's gradient passes
    assert torch.equal(gx, ds) and torch.equal(gr, ds)
    y, s = pkg.rms_norm(x, w, r)
    gx, gr, gw = torch.autograd.grad(y, (x, r, w), dy)
    d, dw, size, wsize = ref.rms_grads(dy, None, (x + r).detach().double(), ref.rms(x.detach(), None, r.detach(), 1e-6, 0.0)[2], w.detach(), 0.0)
    ref.within(gx, d, 2 * FORWARD * size)
    assert torch.equal(gx, gr)
    ref.within(gw, dw, 2 * FORWARD * wsize)


def test_gradients_against_differences():
    x, w, r, dy, ds = _inputs(4, 96, F32, F32, F32, grads=True)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dirs = [torch.randn(t.shape, device="cuda", generator=gen) for t in (x, w, r)]

    def loss(h):
        with torch.no_grad():
            y, s = pkg.rms_norm(x + h * dirs[0], w + h * dirs[1], r + h * dirs[2], 1e-3)
        return (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()

    h = 2.0 ** -6
    slope = (loss(h) - loss(-h)) / (2 * h)
    for t in (x, w, r):
        t.requires_grad_(True)
    y, s = pkg.rms_norm(x, w, r, 1e-3)
    grads = torch.autograd.grad((y, s), (x, w, r), (dy, ds))
    along = sum((g.double() * v.double()).sum() for g, v in zip(grads, dirs))
    # 384 outputs of magnitude 4, each 48 u off: below 384 * 4 * 48 u / h in the difference; the third derivative's h^2 term: the function
    # bends on the scale of the rows' root mean square (3), so h^2 of the terms' magnitude, some 400
    assert (slope - along).abs() <= 384 * 4 * FORWARD / h + 400 * h * h


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows_and_views(dtype):
    wide = torch.randn(3, 7, 5 * 64, device="cuda").to(dtype)
    w = torch.rand(64, device="cuda") + 0.5
    part = wide[:, :, 64:128]           # rows at one distance: read in place
    _check_forward(part, w, wide[:, :, 192:256])
    _check_forward(wide[:, ::2, 3:67], w, None)  # not one distance, not aligned: copied
    _check_forward(wide[:, :, :64].transpose(1, 2).contiguous().transpose(1, 2), w, None)  # channels not contiguous
    _check_forward(wide[0, 0, 1:65], w, wide[0, 1, 2:66])  # one row, no vector boundary
    _check_forward(wide[:1, :1, :64].expand(4, 3, 64), w, None)  # one row many times


def test_empty_and_single():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y, s = pkg.rms_norm(x, w, x.detach())
    assert y.shape == s.shape == (0, 16)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert gx.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device="cuda"))
    q, scale = pkg.rms_norm_quant(torch.empty(2, 0, 16, device="cuda"))
    assert q.shape == (2, 0, 16) and scale.shape == (2, 0, 1)
    one = pkg.rms_norm(torch.full((1, 1), -3.0, device="cuda"), eps=0.0)
    assert one.item() == -1.0


@pytest.mark.parametrize("c", [40, 640, 1111, 2048, 33000])
def test_nan_and_infinity_stay_in_their_row(c):
    x, w, r = _inputs(6, c, F32, F32, F32)
    x[1, c // 2] = float("nan")
    x[3, c - 1] = float("inf")
    y, s = pkg.rms_norm(x, w, r)
    assert torch.isnan(y[1]).all()
    assert torch.isnan(y[3, c - 1]) and (y[3, : c - 1] == 0).all()  # infinity over itself; the others over infinity
    keep = [0, 2, 4, 5]
    _check_forward(x[keep], w, r[keep])
    assert torch.equal(y[keep], pkg.rms_norm(x[keep], w, r[keep])[0])
    for block in (0, 32, 128):
        q, scale, _ = pkg.rms_norm_quant(x, w, r, block=block)
        assert torch.isnan(scale[1]).all() and torch.isnan(q[1].float()).all()
        at = 0 if block == 0 else (c - 1) // block
        assert torch.isnan(scale[3, at]) and torch.isnan(q[3, c - 1].float())
        assert torch.isfinite(scale[keep]).all() and torch.isfinite(q[keep].float()).all()


def test_rows_of_zeros():
    x = torch.zeros(3, 512, device="cuda", dtype=BF16)
    assert (pkg.rms_norm(x) == 0).all()
    for dtype in (torch.float8_e4m3fn, torch.int8):
        for block in (0, 64):
            q, scale = pkg.rms_norm_quant(x, block=block, dtype=dtype)
            assert (q.float() == 0).all() and (scale == 2.0 ** -126).all()


def _check_quant(x, w, r, block, dtype, eps=1e-6, offset=0.0):
    with torch.no_grad():
        out = pkg.rms_norm_quant(x, w, r, eps, offset, block, dtype)
    q, scale = out[:2]
    want, _, _ = ref.rms(x, w, r, eps, offset)
    c = x.shape[-1]
    width = block or c
    largest = 448.0 if dtype == torch.float8_e4m3fn else 127.0
    most = torch.stack([p.abs().amax(-1) for p in want.split(width, -1)], -1) / largest
    assert q.dtype == dtype and scale.dtype == F32 and scale.shape == most.shape
    want_scale = most.clamp_min(2.0 ** -126)
    ref.within(scale, want_scale, (FORWARD + 2 * ref.U32) * want_scale)
    per = scale.double().repeat_interleave(width, -1)[..., :c]
    # half a step of the codes: e4m3 keeps three bits behind the first (2^-4 of the value), steps of 2^-9 below 2^-6; int8 half of one.  The value
    # that is rounded is as far off as y and the reciprocal of the scale are.
    half = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * per) if dtype == torch.float8_e4m3fn else 0.5 * per
    ref.within(q.double() * per, want, half * (1 + 2.0 ** -8) + 2 * FORWARD * want.abs())
    assert (q.double().abs() <= largest).all()
    if r is not None:
        assert torch.equal(out[2], (x.float() + r.float()).to(r.dtype))


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("block", [0, 32, 64, 128])
@pytest.mark.parametrize("dtype,residual,codes", [(BF16, BF16, torch.float8_e4m3fn), (F16, None, torch.int8), (F32, F32, torch.float8_e4m3fn),
                                                  (BF16, F32, torch.int8)])
def test_quant(c, block, dtype, residual, codes):
    x, w, r = _inputs(5, c, dtype, residual, dtype)
    _check_quant(x, w, r, block, codes)


def test_quant_many_rows_and_offset():
    x, w, r = _inputs(3001, 520, BF16, BF16, F32)
    _check_quant(x, w, r, 128, torch.float8_e4m3fn, offset=1.0)
    _check_quant(x, w, r, 0, torch.int8, eps=0.5)


def test_same_bits_every_time_and_on_another_stream():
    x, w, r, dy, ds = _inputs(4000, 768, BF16, BF16, F32, grads=True)
    for t in (x, w, r):
        t.requires_grad_(True)

    def step():
        y, s = pkg.rms_norm(x, w, r)
        return (y, s) + torch.autograd.grad((y, s), (x, r, w), (dy, ds))

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_in_a_graph():
    x, w, r = _inputs(300, 1280, F16, F16, F16)
    want = pkg.rms_norm(x, w, r)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, s = pkg.rms_norm(x, w, r)
        q, scale, _ = pkg.rms_norm_quant(x, w, r, block=128)
    x.copy_(torch.randn_like(x))
    graph.replay()
    again = pkg.rms_norm(x, w, r)
    assert torch.equal(y, again[0]) and torch.equal(s, again[1]) and not torch.equal(want[0], y)
    assert torch.equal(scale, pkg.rms_norm_quant(x, w, r, block=128)[1])


def test_offsets_beyond_32_bits():
    c, rows = 4096, 540000  # 2.2e9 elements
    x = torch.empty(rows, c, device="cuda", dtype=BF16)
    x[:-2].fill_(1.0)
    x[-2:].normal_()
    y = pkg.rms_norm(x)
    assert torch.equal(y[-2:], pkg.rms_norm(x[-2:].clone()))
    assert (y[:: 7919] - 1.0).abs()[:-1].max() == 0
    q, scale = pkg.rms_norm_quant(x[-540000:, :], block=128)
    assert torch.equal(scale[-2:], pkg.rms_norm_quant(x[-2:].clone(), block=128)[1])
    del y, q
    far = x.view(-1).as_strided((2, 64), (2 ** 31 + 64, 1))  # one row from the other's distance
    assert torch.equal(pkg.rms_norm(far), pkg.rms_norm(far.clone()))


def test_module_and_compiled_call():
    m = pkg.RMSNorm(256, eps=1e-5, offset=1.0, device="cuda", dtype=F32)
    assert (m.weight == 0).all()
    with torch.no_grad():
        m.weight.normal_()
    x, _, r = _inputs(12, 256, F16, F32)
    x.requires_grad_(True)
    y, s = m(x, r)
    with torch.no_grad():
        assert torch.equal(m.quantize(x, r, block=64)[2], s)
    gy = torch.randn_like(y)
    grads = torch.autograd.grad(y, (x, m.weight), gy)
    compiled = torch.compile(lambda a, b: m(a, b), backend="aot_eager", fullgraph=True)
    yc, sc = compiled(x, r)
    gc = torch.autograd.grad(yc, (x, m.weight), gy)
    for a, b in zip((y, s) + grads, (yc, sc) + gc):
        assert torch.equal(a, b)


def test_refusals():
    x, w, r = _inputs(4, 64, BF16, BF16, BF16)
    for bad in (lambda: pkg.rms_norm(x, w, r[:3]), lambda: pkg.rms_norm(x, w[:32], r), lambda: pkg.rms_norm(x, w, r.half()),
                lambda: pkg.rms_norm(x, w.half(), r), lambda: pkg.rms_norm(x.double(), None), lambda: pkg.rms_norm(x, w.cpu(), r),
                lambda: pkg.rms_norm(x, w, r.cpu()), lambda: pkg.rms_norm(x.int(), None), lambda: pkg.rms_norm(x[:, :0], None),
                lambda: pkg.rms_norm_quant(x, w, r, block=16), lambda: pkg.rms_norm_quant(x, w, r, dtype=torch.uint8),
                lambda: pkg.rms_norm_quant(x.clone().requires_grad_(True), w), lambda: pkg.RMSNorm(32, device="cuda")(x)):
        with pytest.raises(ValueError):
            bad()
    assert torch.isfinite(pkg.rms_norm(x, w, r)[0]).all()  # nothing was left broken


def test_rows_without_a_common_frame_through_the_c_abi():
    # the Python functions copy such tensors; the C entry points take them as they are
    import ctypes

    from channels_last_groupnorm_b200 import _native as nt

    rows, c = 9, 150
    base = torch.randn(rows, 157, device="cuda").to(BF16)
    x, r = base[:, 3:153], torch.randn(rows, 160, device="cuda").to(BF16)[:, 1:151]
    w = torch.rand(c, device="cuda").to(BF16)
    y, s = torch.full((rows * c + 5,), 7.0, device="cuda", dtype=BF16), torch.full((rows * c + 5,), 7.0, device="cuda", dtype=BF16)
    rstd = torch.empty(rows, device="cuda")
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    out = lambda t: ctypes.c_void_p(t.data_ptr() + 4)  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    nt.check(nt.lib.gnb200_rms_fwd(at(x), 157, at(r), 160, at(w), rows, c, 1e-6, 0.0, 2, 2, 2, out(y), out(s), at(rstd), stream))
    want, sums, root = ref.rms(x, w, r, 1e-6, 0.0)
    ref.within(y[2:-3].view(rows, c), want, ref.rounded(want, BF16) + FORWARD * want.abs())
    ref.within(rstd, root.squeeze(-1), FORWARD * root.squeeze(-1))
    for t in (y, s):
        assert (t[:2] == 7).all() and (t[-3:] == 7).all()
    dy = torch.randn(rows, 151, device="cuda").to(BF16)[:, :c]
    dx = torch.full((rows * c + 5,), 7.0, device="cuda", dtype=BF16)
    dw = torch.empty(c, device="cuda", dtype=BF16)
    need = nt.lib.gnb200_rms_bwd_workspace_bytes(rows, c, 2, 2)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    nt.check(nt.lib.gnb200_rms_bwd(at(dy), 151, None, 0, at(r), 160, at(x), 157, at(w), at(rstd), rows, c, 0.0, 2, 2, 2, out(dx), None, at(dw), at(ws),
                                   need, stream))
    d, dweight, size, wsize = ref.rms_grads(dy, None, x.double() + r.double(), root, w, 0.0)
    ref.within(dx[2:-3].view(rows, c), d, ref.rounded(d, BF16) + 2 * FORWARD * size)
    ref.within(dw, dweight, ref.rounded(dweight, BF16) + (FORWARD + (rows + 64) * ref.U32) * wsize)
    assert (dx[:2] == 7).all() and (dx[-3:] == 7).all()
    # a workspace that is too small is refused before anything is launched
    assert nt.lib.gnb200_rms_bwd(at(dy), 151, None, 0, at(r), 160, at(x), 157, at(w), at(rstd), rows, c, 0.0, 2, 2, 2, out(dx), None, at(dw), at(ws),
                                 16, stream) == -2


@pytest.mark.parametrize("c", [31, 150, 1111, 2050, 12345])
@pytest.mark.parametrize("rows", [1, 2, 17, 3000])
def test_odd_rows_write_nothing_beside_them(c, rows):
    # outputs in the middle of larger buffers, rows of every skew; all parts of a row beside rows of other values
    if rows * c > 2e7:
        rows = 301
    x, w, r, dy, ds = _inputs(rows, c, BF16, BF16, BF16, seed=3, grads=True)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = pkg.rms_norm(x, w, r)
    grads = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    pick = sorted({0, 1, rows // 2, rows - 1} & set(range(rows)))
    one, two = pkg.rms_norm(x.detach()[pick], w.detach(), r.detach()[pick])
    assert torch.equal(y[pick], one) and torch.equal(s[pick], two)
    _, _, rstd = ref.rms(x.detach(), None, r.detach(), 1e-6, 0.0)
    d, dw, size, wsize = ref.rms_grads(dy, ds, x.detach().double() + r.detach().double(), rstd, w.detach(), 0.0)
    ref.within(grads[0], d, ref.rounded(d, BF16) + 2 * FORWARD * size)
    ref.within(grads[2], dw, ref.rounded(dw, BF16) + (FORWARD + (rows + 64) * ref.U32) * wsize)
    _check_quant(x.detach(), w.detach(), r.detach(), 64, torch.float8_e4m3fn)


def test_gradients_with_a_graph_of_their_own():
    x, w, r, dy, ds = _inputs(5, 72, BF16, BF16, F32, grads=True)
    for t in (x, w, r):
        t.requires_grad_(True)
    plain = torch.autograd.grad(pkg.rms_norm(x, w, r), (x, r, w), (dy, ds))
    graphed = torch.autograd.grad(pkg.rms_norm(x, w, r), (x, r, w), (dy, ds), create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b)
