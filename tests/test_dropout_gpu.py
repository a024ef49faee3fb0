"""Dropout with the residual's addition against its definition: masks word by word, values and gradients in 64 bits."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import dropout_reference as D
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32), (F32, None), (F16, None), (BF16, None)]


def _inputs(shape, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(shape, device="cuda", generator=g) + 3).to(dtype)
    r = None if residual is None else (torch.randn(shape, device="cuda", generator=g) * 3).to(residual)
    ds = torch.randn(shape, device="cuda", generator=g).to(dtype if residual is None else residual)
    return x, r, ds


def _want(x, r, kept, p):
    d = torch.where(kept, x.double() / (1 - p), 0.0)
    return d if r is None else d + r.double()


def _check(x, r, ds, p, seed, layer):
    leaves = [t.requires_grad_(True) for t in (x, r) if t is not None]
    s = pkg.dropout_add(x, r, p, seed, layer)
    grads = torch.autograd.grad(s, leaves, ds)
    number = seed if isinstance(seed, int) else seed.item()
    kept = D.kept(x.numel(), p, number, layer, device="cuda").view(x.shape)
    want = _want(x.detach(), None if r is None else r.detach(), kept, p)
    assert s.dtype == (x.dtype if r is None else r.dtype) and s.is_contiguous()
    # 1 / (1 - p) rounded, one fma or product, one rounding to the type
    size = x.detach().double().abs() / (1 - p) + (0.0 if r is None else r.detach().double().abs())
    ref.within(s.detach(), want, ref.rounded(want, s.dtype) + 3 * ref.U32 * size)
    if r is not None:
        assert torch.equal(s.detach()[~kept], r.detach()[~kept])
        assert torch.equal(grads[1], ds)
    else:
        assert (s.detach()[~kept] == 0).all()
    dx = _want(ds, None, kept, p)
    assert grads[0].dtype == x.dtype
    ref.within(grads[0], dx, ref.rounded(dx, x.dtype) + 3 * ref.U32 * dx.abs())
    assert (grads[0][~kept] == 0).all()


# one element; parts of a counter, a vector; vectors and a rest; more than a CTA, more than the grid's CTAs
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 64, 1111, 4099, 640 * 64, 3000001])
@pytest.mark.parametrize("dtype,residual", TYPES)
def test_sizes(n, dtype, residual):
    _check(*_inputs((n,), dtype, residual, n), 0.25, 1234567890123456789, 3)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -32, 0.05, 0.1, 0.5, 0.999, 1 - 2.0 ** -30])
@pytest.mark.parametrize("dtype,residual", [(F32, F32), (BF16, None)])
def test_probabilities(p, dtype, residual):
    _check(*_inputs((33, 97), dtype, residual), p, 5, 0)


@pytest.mark.parametrize("seed", [0, 1, -1, 2 ** 63 - 1, -2 ** 63, 2 ** 32, 2 ** 64 - 1])
@pytest.mark.parametrize("layer", [0, 1, 2 ** 40 + 7, 2 ** 64 - 1])
def test_seeds_and_layers(seed, layer):
    _check(*_inputs((5, 72), F16, F16), 0.3, seed, layer)
    if seed < 2 ** 63:
        _check(*_inputs((5, 72), F16, F16), 0.3, torch.tensor([seed], device="cuda"), layer)


def test_masks_differ_and_are_fair():
    x = torch.ones(1 << 20, device="cuda")
    masks = [pkg.dropout_add(x, p=0.25, seed=s, layer=l) > 0 for s, l in ((0, 0), (1, 0), (0, 1), (1, 1))]
    for i, m in enumerate(masks):
        # six standard deviations of a million draws
        assert abs(m.float().mean().item() - 0.75) <= 6 * (0.25 * 0.75 / 2 ** 20) ** 0.5
        for other in masks[:i]:
            agree = (m == other).float().mean().item()
            assert abs(agree - (0.75 ** 2 + 0.25 ** 2)) <= 6 * 0.5 / 2 ** 10


def test_layouts():
    """The mask goes by the order of the elements: slices, transposes, views off a vector, expanded gradients."""
    wide, other = torch.randn(48, 200, device="cuda").bfloat16(), torch.randn(48, 200, device="cuda").bfloat16()
    for cut in (lambda t: t[:, 8:136], lambda t: t[:, 3:110], lambda t: t.t(), lambda t: t.reshape(-1)[1:4001].view(40, 100), lambda t: t.view(4, 12, 200)[:, ::3]):
        x, r = cut(wide), cut(other)
        got = pkg.dropout_add(x, r, 0.4, 9, 1)
        assert torch.equal(got, pkg.dropout_add(x.contiguous().clone(), r.contiguous().clone(), 0.4, 9, 1))
    x = wide.clone().requires_grad_(True)
    pkg.dropout_add(x, None, 0.4, 9).sum().backward()  # (a gradient of one element, expanded)
    kept = D.kept(x.numel(), 0.4, 9, device="cuda").view(x.shape)
    assert torch.equal(x.grad, torch.where(kept, 1 / 0.6, 0.0).bfloat16())


def test_dropped_elements_are_zero_whatever_they_were():
    x, r, _ = _inputs((64, 64), F32, F32)
    kept = D.kept(x.numel(), 0.5, 11, device="cuda").view(x.shape)
    x[~kept] = float("nan")
    x.view(-1)[int((~kept).view(-1).nonzero()[0])] = float("inf")
    assert torch.equal(pkg.dropout_add(x, r, 0.5, 11)[~kept], r[~kept])
    assert torch.isfinite(pkg.dropout_add(x, r, 0.5, 11)).all()


@pytest.mark.parametrize("dtype,residual", [(F32, F32), (BF16, F32), (F16, None)])
def test_second_derivatives(dtype, residual):
    """The gradient is linear: its own gradient is the mask again."""
    x, r, ds = _inputs((9, 40), dtype, residual)
    leaves = [t.requires_grad_(True) for t in (x, r, ds) if t is not None]
    s = pkg.dropout_add(x, r, 0.3, 21, 2)
    dx, = torch.autograd.grad(s, x, ds, create_graph=True)
    assert torch.equal(dx, torch.autograd.grad(pkg.dropout_add(x, r, 0.3, 21, 2), x, ds.detach())[0])
    v = torch.randn_like(dx)
    dds, = torch.autograd.grad(dx, ds, v)
    kept = D.kept(x.numel(), 0.3, 21, 2, device="cuda").view(x.shape)
    want = _want(v, None, kept, 0.3)
    assert dds.dtype == ds.dtype
    ref.within(dds, want, ref.rounded(want, ds.dtype) + 3 * ref.U32 * want.abs())
    assert len(leaves)


def test_gradients_against_differences():
    x, r, _ = (t if t is None else t.double() for t in _inputs((6, 10), F32, F32))
    v = torch.randn(6, 10, device="cuda", dtype=torch.float64)

    def call(a, b):
        return pkg.dropout_add(a.float(), b.float(), 0.25, 3).double()

    xs, rs = x.float().requires_grad_(True), r.float().requires_grad_(True)
    gx, gr = torch.autograd.grad(pkg.dropout_add(xs, rs, 0.25, 3), (xs, rs), v.float())
    h = 2.0 ** -4
    for which, got in ((0, gx), (1, gr)):
        for i in range(60):
            e = torch.zeros(60, device="cuda", dtype=torch.float64)
            e[i] = h
            e = e.view(6, 10)
            up, down = (call(x + s * e, r) if which == 0 else call(x, r + s * e) for s in (1, -1))
            slope = ((up - down) * v).sum() / (2 * h)
            # linear: the difference has the roundings of two values of up to 16 alone
            assert abs(slope - got.view(-1)[i]) <= 16 * 2 * ref.U32 / h * v.abs().max() + 1e-6


def test_only_what_is_asked_for():
    x, r, ds = _inputs((9, 40), BF16, F32)
    s = pkg.dropout_add(x, r.requires_grad_(True), 0.3, 21)
    g, = torch.autograd.grad(s, r, ds)
    assert torch.equal(g, ds)
    with torch.no_grad():
        assert not pkg.dropout_add(x, r, 0.3, 21).requires_grad
    assert torch.equal(s.detach(), pkg.dropout_add(x, r.detach(), 0.3, 21))


def test_seed_that_changed_before_the_backward():
    x, r, ds = _inputs((9, 40), BF16, BF16)
    seed = torch.tensor([4], device="cuda")
    s = pkg.dropout_add(x.requires_grad_(True), r, 0.3, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(s, x, ds)


def test_captured_step_follows_its_seed():
    x, r, ds = _inputs((33, 72), BF16, BF16)
    seed = torch.tensor([100], device="cuda")

    def step():
        leaf = x.detach().requires_grad_(True)
        s = pkg.dropout_add(leaf, r, 0.3, seed, 5)
        dx, = torch.autograd.grad(s, leaf, ds)
        return s.detach(), dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        seed.add_(1)
    for i in range(3):
        seed.fill_(200 + i)
        graph.replay()
        assert seed.item() == 201 + i
        for a, b in zip(out, ref_step(x, r, ds, 200 + i)):
            assert torch.equal(a, b)


def ref_step(x, r, ds, seed):
    leaf = x.detach().requires_grad_(True)
    s = pkg.dropout_add(leaf, r, 0.3, seed, 5)
    return s.detach(), torch.autograd.grad(s, leaf, ds)[0]


def test_other_stream():
    x, r, _ = _inputs((33, 72), BF16, BF16)
    want = pkg.dropout_add(x, r, 0.3, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.dropout_add(x, r, 0.3, 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("on_device", [False, True])
def test_compiled(on_device):
    x, r, ds = _inputs((9, 40), BF16, F32)
    seed = torch.tensor([7], device="cuda") if on_device else 7
    leaves = [x.requires_grad_(True), r.requires_grad_(True)]

    def call(x, r):
        return pkg.dropout_add(x, r, 0.3, seed, 2)

    torch._dynamo.reset()
    got, want = torch.compile(call, backend="aot_eager", fullgraph=True)(x, r), call(x, r)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, ds), torch.autograd.grad(want, leaves, ds)):
        assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    for kw, words in (({"p": 1.0}, "less than 1"), ({"p": -0.5}, "less than 1"), ({"p": float("nan")}, "less than 1"), ({"residual": x[:3]}, "residual"),
                      ({"residual": x.half()}, "residual"), ({"residual": x.cpu()}, "residual"), ({"seed": torch.ones(1, device="cuda")}, "seed"),
                      ({"seed": torch.tensor([1])}, "seed"), ({"seed": torch.ones(2, device="cuda", dtype=torch.int64)}, "seed"), ({"seed": 2 ** 64}, "64 bits"),
                      ({"layer": -2 ** 63 - 1}, "64 bits")):
        with pytest.raises(ValueError, match=words):
            pkg.dropout_add(x, **kw)
    with pytest.raises(ValueError, match="float32"):
        pkg.dropout_add(x.double())


def test_module_and_nothing():
    x, r, _ = _inputs((9, 40), BF16, F32)
    m = pkg.DropoutAdd(0.3, layer=4)
    assert torch.equal(m(x, r, 12), pkg.dropout_add(x, r, 0.3, 12, 4))
    m.eval()
    assert torch.equal(m(x, r, 12), x.float() + r)
    assert pkg.dropout_add(x[:0], r[:0], 0.3).shape == (0, 40)
    assert pkg.dropout_add(x[0, 0], p=0.0).shape == ()


def test_one_tensor_in_both_places():
    x, _, ds = _inputs((9, 40), F32, F32)
    x.requires_grad_(True)
    g, = torch.autograd.grad(pkg.dropout_add(x, x, 0.25, 3), x, ds)
    kept = D.kept(x.numel(), 0.25, 3, device="cuda").view(x.shape)
    want = ds.double() + torch.where(kept, ds.double() / 0.75, 0.0)
    ref.within(g, want, 6 * ref.U32 * want.abs() + 6 * ref.U32 * ds.double().abs())


def test_graphs_that_are_kept_and_dropped():
    """Twice through a graph that is kept; an error the second time where the seed, which it holds, is gone; hooks on what is saved; a checkpoint."""
    from torch.utils.checkpoint import checkpoint

    x, r, ds = _inputs((9, 40), BF16, BF16)
    x.requires_grad_(True)
    seed = torch.tensor([6], device="cuda")
    want, = torch.autograd.grad(pkg.dropout_add(x, r, 0.25, 6, 1), x, ds)
    s = pkg.dropout_add(x, r, 0.25, seed, 1)
    for keep in (True, False):
        assert torch.equal(torch.autograd.grad(s, x, ds, retain_graph=keep)[0], want)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(s, x, ds)
    with torch.autograd.graph.save_on_cpu():
        s = pkg.dropout_add(x, r, 0.25, seed, 1)
    assert torch.equal(torch.autograd.grad(s, x, ds)[0], want)
    s = checkpoint(lambda t: pkg.dropout_add(t, r, 0.25, seed, 1), x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(s, x, ds)[0], want)


@pytest.mark.parametrize("n", [2 ** 32 + 4096, 2 ** 34 + 4104])
def test_far_elements(n):
    """Elements, and counters, of more than 32 bits."""
    x = torch.empty(n, device="cuda", dtype=BF16)
    x[-8192:] = 1.0
    s = pkg.dropout_add(x, None, 0.5, 77)
    kept = D.kept(8192, 0.5, 77, begin=n - 8192, device="cuda")
    assert torch.equal(s[-8192:], kept.bfloat16() * 2)
