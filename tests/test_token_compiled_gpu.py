"""The operators on token rows under torch.compile: what the traced formulas keep for the backward, and that they compute what eager calls do."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _compiled(fn):
    torch._dynamo.reset()
    return torch.compile(fn, backend="aot_eager", fullgraph=True)


def _kept(call):
    """sizes of the tensors that `call` keeps for its backward"""
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(tuple(t.shape)) or t, lambda t: t):
        out = call()
    return out, sizes


@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("weights", ["none", "queries", "both"])
def test_rotary_keeps_what_its_backward_reads(compiled, weights):
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(2, 9, h, 64, device="cuda", generator=g).bfloat16().requires_grad_(True) for h in (4, 3))
    qw = torch.rand(64, device="cuda", generator=g).requires_grad_(True) if weights != "none" else None
    kw = torch.rand(64, device="cuda", generator=g).requires_grad_(True) if weights == "both" else None
    positions = torch.arange(18, device="cuda").view(2, 9, 1)
    inv_freq = torch.linspace(1.0, 0.01, 32, device="cuda")

    def eager(q, k):
        return pkg.rotary(q, k, positions, inv_freq, (32,), qw, kw)

    def op(q, k):  # what compiled code calls
        return torch.ops.gnb200.rotary(q, k, positions, inv_freq, [32], qw, kw, 1e-6, 0.0, False)

    out, sizes = _kept(lambda: (_compiled(eager) if compiled else op)(q, k))
    assert ((2, 9, 4, 64) in sizes) == (qw is not None)
    assert ((2, 9, 3, 64) in sizes) == (kw is not None)
    cots = [torch.randn(o.shape, device="cuda", generator=g).bfloat16() for o in out]
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    want = eager(q, k)
    for a, b in zip(list(out) + list(torch.autograd.grad(out, leaves, cots)), list(want) + list(torch.autograd.grad(want, leaves, cots))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("c", [256, 1111, 12345])
@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (F16, F32), (F32, None)])
def test_norm_as_in_eager_calls(c, dtype, residual):
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.randn(7, c, device="cuda", generator=g).to(dtype) for _ in range(2))
    r, ds = (None, None) if residual is None else (torch.randn(7, c, device="cuda", generator=g).to(residual) for _ in range(2))
    w = torch.rand(c, device="cuda", generator=g)
    leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]

    def call(x, w, r):
        return pkg.rms_norm(x, w, r, 1e-5, 0.5)

    def both(fn):
        out = fn(x, w, r)
        outs, cots = ((out,), (dy,)) if r is None else (out, (dy, ds))
        return tuple(outs) + torch.autograd.grad(outs, leaves, cots)

    for a, b in zip(both(call), both(_compiled(call))):
        assert torch.equal(a, b)
    if residual == BF16:  # the sum again from its terms: a weight's gradient as exact as fp32 has it
        _, sizes = _kept(lambda: _compiled(call)(x, w, r))
        assert sizes.count((7, c)) == 2


@pytest.mark.parametrize("c", [256, 1111, 12345])
@pytest.mark.parametrize("dtype,block", [(torch.float8_e4m3fn, 128), (torch.int8, 0)])
def test_codes_as_in_eager_calls(c, dtype, block):
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r = (torch.randn(7, c, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.rand(c, device="cuda", generator=g)

    def call(x, w, r):
        return pkg.rms_norm_quant(x, w, r, block=block, dtype=dtype)

    with torch.no_grad():
        for a, b in zip(call(x, w, r), _compiled(call)(x, w, r)):
            assert a.dtype == b.dtype and torch.equal(a.float(), b.float())
