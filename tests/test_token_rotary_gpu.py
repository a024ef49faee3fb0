"""rotary on the GPU against the definition in 64 bits."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# a pair's output: the angle is rounded once to fp32 in half turns (at most pi u off), sine and cosine 2 u, a product and a sum 2 u; the norm
# in front: at most 16 terms a lane and 5 levels, halved, and four more operations
TURN = 8 * ref.U32
NORM = 20 * ref.U32


def _inputs(lead, hq, hk, d, sections, dtype, norm=None, seed=0, pos=torch.int64, most=5000, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).mul_(1.5).to(dtype)

    if packed:
        both = normal(*lead, hq + 2 * hk, d)
        q, k = both[..., :hq, :], both[..., hq:hq + hk, :]
    else:
        q, k = normal(*lead, hq, d), normal(*lead, hk, d)
    positions = torch.randint(0, most, (*lead, len(sections)), device="cuda", generator=g)
    positions = positions.to(pos) if pos != F32 else positions.float() * 0.25 + 0.125
    n = sum(sections)
    inv_freq = (10000.0 ** -(torch.arange(n, device="cuda", dtype=torch.float64) / n)).float()
    ws = [None, None] if norm is None else [(torch.rand(d, device="cuda", generator=g) + 0.5).to(norm) for _ in range(2)]
    return q, k, positions, inv_freq, tuple(sections), ws[0], ws[1]


def _check(q, k, positions, inv_freq, sections, qw, kw, interleaved=False, offset=0.0, eps=1e-6, backward=True):
    q, k = q.detach(), k.detach()
    q.requires_grad_(backward)
    k.requires_grad_(backward)
    for w in (qw, kw):
        if w is not None:
            w.requires_grad_(backward)
    out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw, eps, interleaved, offset)
    g = torch.Generator(device="cuda").manual_seed(9)
    cots = [torch.randn(o.shape, device="cuda", generator=g).to(o.dtype) for o in out]
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(out, leaves, cots))) if backward else {}
    for t, w, o, c in ((q, qw, out[0], cots[0]), (k, kw, out[1], cots[1])):
        weight = None if w is None else w.detach()
        want, n, rstd = ref.rotary(t.detach(), weight, positions, inv_freq, sections, eps, interleaved, offset)
        big = n.abs() if weight is None else (n * (offset + weight.double())).abs()
        cos, sin = ref.angles(positions, inv_freq, sections)
        ones = torch.ones_like(cos)
        reach = ref.turned(big, ones, -ones, interleaved).abs() + ref.turned(big, ones, ones, interleaved).abs()  # at least |a| + |b|, twice at most
        assert o.dtype == t.dtype and o.is_contiguous()
        ref.within(o, want, ref.rounded(want, t.dtype) + (TURN + (0 if w is None else NORM)) * reach)
        if not backward:
            continue
        d, dw, size, wsize = ref.rotary_grads(c, weight, n, rstd, positions, inv_freq, sections, interleaved, offset)
        spread = c.double().abs()
        spread = ref.turned(spread, ones, -ones, interleaved).abs() + ref.turned(spread, ones, ones, interleaved).abs()
        if weight is not None:
            gw = spread * (offset + weight.double()).abs()
            spread_w = (spread * n.abs()).reshape(-1, n.shape[-1]).sum(0)
            spread = rstd * (gw + n.abs() * (gw * n.abs()).mean(-1, keepdim=True))
        ref.within(grads[id(t)], d, ref.rounded(d, t.dtype) + (TURN + 2 * NORM) * (size + spread))
        assert grads[id(t)].dtype == t.dtype
        if w is not None:
            rows = t.numel() // t.shape[-1]
            # a sum over all rows: at most as many additions in a row as there are rows
            ref.within(grads[id(w)], dw, ref.rounded(dw, w.dtype) + (TURN + NORM + (rows + 64) * ref.U32) * (wsize + spread_w))
            assert grads[id(w)].dtype == w.dtype


# head sizes: smallest; odd with a tail; each vector width; several slots a lane; the largest
HEADS = [(2, (1,)), (3, (1,)), (6, (1, 1)), (7, (2, 1)), (33, (5, 4, 3)), (40, (20,)), (64, (16, 16)), (72, (12, 12, 12)), (80, (12, 12, 12)),
         (96, (16, 16, 16)), (100, (10, 20, 20)), (128, (16, 24, 24)), (128, (8, 8)), (130, (65,)), (256, (64, 32, 32)), (264, (100, 0, 32)), (510, (255,)),
         (512, (64, 64, 64, 64)), (512, (200,))]


@pytest.mark.parametrize("d,sections", HEADS)
@pytest.mark.parametrize("dtype,norm", [(F32, None), (BF16, BF16), (F16, F32), (F32, F32), (BF16, None)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_sizes(d, sections, dtype, norm, interleaved):
    _check(*_inputs((2, 5), 6, 2, d, sections, dtype, norm), interleaved=interleaved, offset=0.25)


@pytest.mark.parametrize("lead,hq,hk", [((1,), 1, 1), ((1, 1), 32, 8), ((1, 1), 5, 1), ((3, 1), 7, 7), ((517,), 3, 1), ((2, 901), 4, 2), ((40, 50), 20, 20)])
@pytest.mark.parametrize("norm", [None, BF16])
def test_tokens_and_heads(lead, hq, hk, norm):
    _check(*_inputs(lead, hq, hk, 64, (8, 12, 12), BF16, norm))


@pytest.mark.parametrize("pos,most", [(torch.int32, 100000), (torch.int64, 2 ** 31), (F32, 3000)])
def test_positions(pos, most):
    # exact angles: the bound is the same for positions of a thousand million
    _check(*_inputs((2, 37), 4, 4, 64, (10, 11, 11), F32, None, pos=pos, most=most))


def test_negative_positions_turn_back():
    q, k, positions, inv_freq, sections, _, _ = _inputs((50,), 4, 4, 128, (22, 21, 21), F32)
    there = pkg.rotary(q, k, positions, inv_freq, sections)
    back = pkg.rotary(there[0], there[1], -positions, inv_freq, sections)
    ref.within(back[0], q.double(), 2 * TURN * 2 * q.double().abs().max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", [None, F32])
def test_strides(dtype, norm):
    _check(*_inputs((2, 31), 6, 2, 64, (32,), dtype, norm, packed=True))  # slices of one projection
    q, k, positions, *rest = _inputs((2, 6), 31, 31, 64, (16, 16), dtype, norm)
    q, k = q.transpose(1, 2), k.transpose(1, 2)  # (batch, heads, tokens, head_dim) memory
    positions = torch.randint(0, 50, (2, 2, 31), device="cuda").permute(0, 2, 1)  # axes in front
    _check(q, k, positions, *rest)
    one = torch.randint(0, 50, (1, 31, 2), device="cuda").expand(2, 31, 2)  # the same tokens in every sample
    _check(q, k, one, *rest)
    odd = torch.randn(2, 31, 6, 67, device="cuda").to(dtype)[..., 3:]  # heads that start on no vector boundary
    _check(odd, odd[:, :, :2].clone(), one, *rest)
    _check(odd[..., ::1].transpose(2, 3).contiguous().transpose(2, 3), odd[:, :, :2], one, *rest)  # channels not contiguous: copied
    narrow = torch.randn(2, 31, 1, 64, device="cuda").to(dtype).expand(2, 31, 6, 64)  # one head many times
    _check(narrow, narrow[:, :, :3], one, *rest)


def test_expanded_gradient():
    q, k, positions, inv_freq, sections, _, _ = _inputs((3, 5), 2, 1, 64, (32,), F32)
    q.requires_grad_(True)
    out, _ = pkg.rotary(q, k, positions, inv_freq, sections)
    (g,) = torch.autograd.grad(out.sum(), q)
    cos, sin = ref.angles(positions, inv_freq, sections)
    want = ref.turned(torch.ones_like(q, dtype=torch.float64), cos, -sin, False)
    ref.within(g, want, 2 * TURN * 2)


def test_queries_only_and_one_norm_only():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((4, 9), 6, 3, 64, (16, 16), BF16, BF16)
    full = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    alone, none = pkg.rotary(q, None, positions, inv_freq, sections, qw)
    assert none is None and torch.equal(alone, full[0])
    _check(q, k, positions, inv_freq, sections, qw, None)
    _check(q, k, positions, inv_freq, sections, None, kw.detach())
    for t in (q, k, qw, kw):
        t.detach_().requires_grad_(True)
    out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    dk = torch.randn_like(out[1])
    gk, gkw = torch.autograd.grad(out[1], (k, kw), dk)  # the queries' output not used
    both = torch.autograd.grad(pkg.rotary(q, k, positions, inv_freq, sections, qw, kw), (k, kw), (torch.zeros_like(out[0]), dk))
    assert torch.equal(gk, both[0])
    ref.within(gkw, both[1].double(), 2 ** -7 * both[1].double().abs() + 1e-4)  # (dealt out to other CTAs: another order of the sum)


def test_mixed_weight_types():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 33), 4, 4, 128, (64,), F16, F16)
    _check(q, k, positions, inv_freq, sections, qw, kw.float())


def test_gradients_against_differences():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 3), 2, 2, 32, (8, 8), F32, F32)
    gen = torch.Generator(device="cuda").manual_seed(3)
    dirs = [torch.randn(t.shape, device="cuda", generator=gen) for t in (q, k, qw, kw)]
    cots = [torch.randn(t.shape, device="cuda", generator=gen) for t in (q, k)]

    def loss(h):
        moved = [t.detach() + h * v for t, v in zip((q, k, qw, kw), dirs)]
        with torch.no_grad():
            out = pkg.rotary(moved[0], moved[1], positions, inv_freq, sections, moved[2], moved[3], 1e-3)
        return sum((o.double() * c.double()).sum() for o, c in zip(out, cots))

    h = 2.0 ** -7
    slope = (loss(h) - loss(-h)) / (2 * h)
    for t in (q, k, qw, kw):
        t.requires_grad_(True)
    grads = torch.autograd.grad(pkg.rotary(q, k, positions, inv_freq, sections, qw, kw, 1e-3), (q, k, qw, kw), cots)
    along = sum((g.double() * v.double()).sum() for g, v in zip(grads, dirs))
    # 768 outputs of magnitude up to 4 and (TURN + NORM) off; the third derivative's h^2 on sums of magnitude 800
    assert (slope - along).abs() <= 768 * 4 * 2 * (TURN + NORM) / h + 800 * h * h


def test_infinities_and_nan_in_channels_that_pass():
    q, k, positions, inv_freq, sections, _, _ = _inputs((6,), 2, 2, 64, (16,), BF16)
    q[..., 32:] = float("inf")
    q[..., 40] = float("nan")
    out, _ = pkg.rotary(q, k, positions, inv_freq, sections)
    assert torch.isfinite(out[..., :32]).all()
    assert (out[..., 32:40] == float("inf")).all() and torch.isnan(out[..., 40]).all()
    q[0, 0, 0] = float("nan")
    out, ok = pkg.rotary(q, k, positions, inv_freq, sections, torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))
    assert torch.isnan(out[0, 0]).all() and torch.isfinite(ok).all()


def test_empty():
    for lead in ((0,), (2, 0), (0, 3)):
        q, k, positions, inv_freq, sections, qw, kw = _inputs(lead, 2, 2, 64, (32,), BF16, BF16)
        for t in (q, qw, kw):
            t.requires_grad_(True)
        out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
        assert out[0].shape == q.shape and out[1].shape == k.shape
        grads = torch.autograd.grad(out, (q, qw, kw), [torch.empty_like(o) for o in out])
        assert grads[0].shape == q.shape and (grads[1] == 0).all() and (grads[2] == 0).all()


def test_same_bits_every_time_and_on_another_stream():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 3000), 8, 4, 128, (20, 22, 22), BF16, BF16)
    for t in (q, k, qw, kw):
        t.requires_grad_(True)

    def step():
        out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
        return tuple(out) + torch.autograd.grad(out, (q, k, qw, kw), [o.detach() for o in out])

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    s, h, d = 150000, 120, 128  # 2.3e9 elements
    q = torch.empty(s, h, d, device="cuda", dtype=BF16)
    q[:-3].fill_(1.0)
    q[-3:].normal_()
    positions = torch.arange(s, device="cuda").unsqueeze(-1)
    inv_freq = (10000.0 ** -(torch.arange(64, device="cuda") / 64.0)).float()
    out, _ = pkg.rotary(q, None, positions, inv_freq, (64,))
    tail, _ = pkg.rotary(q[-3:].clone(), None, positions[-3:], inv_freq, (64,))
    assert torch.equal(out[-3:], tail)


def test_module_and_compiled_call():
    m = pkg.AxialRotary(64, (8, 12, 12), qk_norm=True, interleaved=True, device="cuda").to(BF16)
    assert m.inv_freq.dtype == F32 and m.q_weight.dtype == BF16
    q, k, positions, *_ = _inputs((2, 40), 4, 2, 64, (8, 12, 12), BF16)
    q.requires_grad_(True)
    k.requires_grad_(True)
    out = m(q, k, positions)
    cots = [torch.randn_like(o) for o in out]
    grads = torch.autograd.grad(out, (q, k, m.q_weight, m.k_weight), cots)
    compiled = torch.compile(lambda a, b: m(a, b, positions), backend="aot_eager", fullgraph=True)
    outc = compiled(q, k)
    gradc = torch.autograd.grad(outc, (q, k, m.q_weight, m.k_weight), cots)
    for a, b in zip(tuple(out) + grads, tuple(outc) + gradc):
        assert torch.equal(a, b)
    shared = pkg.AxialRotary(64, (8, 12, 12), shared=True)
    assert torch.allclose(shared.inv_freq, 10000.0 ** -(torch.arange(32) / 32.0))


def test_refusals():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 5), 4, 2, 64, (16, 16), BF16, BF16)
    call = pkg.rotary
    for bad in (lambda: call(q[0, 0], None, positions, inv_freq, sections), lambda: call(q.double(), None, positions, inv_freq, sections),
                lambda: call(q, k[:1], positions, inv_freq, sections), lambda: call(q, k.float(), positions, inv_freq, sections),
                lambda: call(q, k[..., :32], positions, inv_freq, sections), lambda: call(q, k, positions[:, :3], inv_freq, sections),
                lambda: call(q, k, positions, inv_freq, (16, 20)), lambda: call(q, k, positions, inv_freq, (32,)),
                lambda: call(q, k, positions, inv_freq, (33, -1)), lambda: call(q, k, positions, inv_freq, ()),
                lambda: call(q, k, positions.cpu(), inv_freq, sections), lambda: call(q, k, positions.half(), inv_freq, sections),
                lambda: call(q, k, positions, inv_freq.half(), sections), lambda: call(q, k, positions, inv_freq[:20], sections),
                lambda: call(q, k, positions, inv_freq, sections, qw[:8], kw), lambda: call(q, k, positions, inv_freq, sections, qw.half(), kw),
                lambda: call(q, None, positions, inv_freq, sections, qw, kw),
                lambda: call(q, k, positions, inv_freq.clone().requires_grad_(True), sections),
                lambda: call(torch.empty(2, 5, 1, 514, device="cuda"), None, positions, inv_freq, sections),
                lambda: pkg.AxialRotary(64, (20, 20)), lambda: pkg.AxialRotary(64, ())):
        with pytest.raises(ValueError):
            bad()
    assert torch.isfinite(call(q, k, positions, inv_freq, sections, qw, kw)[0]).all()


def test_gradients_with_a_graph_of_their_own():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 7), 4, 2, 64, (16, 16), BF16, BF16)
    for t in (q, k, qw, kw):
        t.requires_grad_(True)
    out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    cots = [torch.randn_like(o) for o in out]
    plain = torch.autograd.grad(out, (q, k, qw, kw), cots)
    graphed = torch.autograd.grad(pkg.rotary(q, k, positions, inv_freq, sections, qw, kw), (q, k, qw, kw), cots, create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b)


def test_captured_in_a_graph():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((3, 50), 4, 2, 128, (20, 22, 22), F16, F16)
    pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    q.copy_(torch.randn_like(q))
    positions.add_(3)
    graph.replay()
    again = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_integer_and_list_arguments_take_the_other_path():
    q, k, positions, inv_freq, sections, qw, kw = _inputs((2, 5), 4, 2, 64, (16, 16), F32, F32)
    want = pkg.rotary(q, k, positions, inv_freq, sections, qw, kw, 1.0)
    got = pkg.rotary(q, k, positions, inv_freq, list(sections), qw, kw, 1, 0, 0)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for t in (q, k, qw, kw):
        t.requires_grad_(True)
    cots = [torch.randn_like(o) for o in want]
    a = torch.autograd.grad(pkg.rotary(q, k, positions, inv_freq, sections, qw, kw, 1.0), (q, k, qw, kw), cots)
    b = torch.autograd.grad(pkg.rotary(q, k, positions, inv_freq, list(sections), qw, kw, 1, 0, 0), (q, k, qw, kw), cots)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
