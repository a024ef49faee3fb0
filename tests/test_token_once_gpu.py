"""The operators on token rows are differentiable once: a second derivative is an error, whichever outputs were used."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu


def _leaves(*shapes):
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(s, device="cuda", generator=g).requires_grad_(True) for s in shapes]


def _refuses(outs, leaves, cots):
    """First derivatives as without a graph; a derivative of any of them is refused."""
    plain = torch.autograd.grad(outs, leaves, cots, retain_graph=True)
    graphed = torch.autograd.grad(outs, leaves, cots, create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b)
        assert b.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(b.square().sum(), leaves, retain_graph=True, allow_unused=True)


def test_norm():
    x, r, w, dy, ds = _leaves((5, 72), (5, 72), (72,), (5, 72), (5, 72))
    _refuses(pkg.rms_norm(x, w, r), (x, r, w), (dy.detach(), ds.detach()))
    _refuses(pkg.rms_norm(x, w), (x, w), dy.detach())
    _refuses(pkg.rms_norm(x, w, r)[:1], (x, r, w), (dy.detach(),))
    # through the gradient of the output too
    gx, = torch.autograd.grad(pkg.rms_norm(x, w), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gx.sum(), dy)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("used", ["both", "queries", "keys"])
def test_rotary(norm, used):
    q, k, qw, kw, dq, dk = _leaves((2, 7, 4, 64), (2, 7, 2, 64), (64,), (64,), (2, 7, 4, 64), (2, 7, 2, 64))
    if not norm:
        qw = kw = None
    positions = torch.arange(28, device="cuda").view(2, 7, 2)
    inv_freq = torch.linspace(1.0, 0.01, 32, device="cuda")
    out = pkg.rotary(q, k, positions, inv_freq, (16, 16), qw, kw)
    pick = {"both": slice(None), "queries": slice(0, 1), "keys": slice(1, 2)}[used]
    leaves = [t for pair in ((q, qw), (k, kw))[pick] for t in pair if t is not None]
    cots = [dq, dk][pick]
    if norm:
        _refuses(out[pick], leaves, [c.detach() for c in cots])
    grads = torch.autograd.grad(out[pick], leaves, cots, create_graph=True)
    assert all(g.requires_grad for g in grads)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(sum(g.square().sum() for g in grads), cots)


def test_functional_ops():
    x, w, dy = _leaves((5, 72), (72,), (5, 72))
    y, _, _ = torch.ops.gnb200.rms_fwd(x, None, w, 1e-6, 0.0)
    gx, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gx.sum(), dy)
