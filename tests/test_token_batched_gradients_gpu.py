"""Backward of the norm and of rotary positions where others look at the gradients: batches of them, a dispatch mode."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _norm(residual):
    torch.manual_seed(1)
    x = torch.randn(9, 40, device="cuda").bfloat16().requires_grad_(True)
    w = torch.rand(40, device="cuda").requires_grad_(True)
    if residual is None:
        return [x, w], [pkg.rms_norm(x, w)]
    r = torch.randn(9, 40, device="cuda").to(residual).requires_grad_(True)
    return [x, w, r], list(pkg.rms_norm(x, w, r))


def _rotary(normed):
    torch.manual_seed(1)
    q, k = (torch.randn(2, 7, h, 48, device="cuda").bfloat16().requires_grad_(True) for h in (4, 2))
    positions, freq = torch.arange(14, device="cuda").view(2, 7, 1), torch.rand(20, device="cuda")
    weights = [torch.rand(48, device="cuda").requires_grad_(True) for _ in range(2)] if normed else [None, None]
    return [q, k] + [w for w in weights if normed], list(pkg.rotary(q, k, positions, freq, (20,), *weights))


CASES = {"norm": lambda: _norm(None), "norm over 16 bits": lambda: _norm(BF16), "norm over fp32": lambda: _norm(F32), "rotary": lambda: _rotary(False),
         "rotary with norm": lambda: _rotary(True)}


@pytest.mark.parametrize("case", list(CASES))
def test_batches(case):
    """As many gradients of each output at once: those of one after the other."""
    leaves, outs = CASES[case]()
    ds = [torch.randn((3,) + o.shape, device="cuda").to(o.dtype) for o in outs]
    got = torch.autograd.grad(outs, leaves, ds, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(outs, leaves, [d[i] for d in ds], retain_graph=True)):
            assert a.dtype == b.dtype and torch.equal(a[i], b)


@pytest.mark.parametrize("case", list(CASES))
def test_a_mode_in_the_backward_alone(case):
    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves, outs = CASES[case]()
    ds = [torch.randn_like(o) for o in outs]
    want = torch.autograd.grad(outs, leaves, ds, retain_graph=True)
    with Seen() as seen:
        got = torch.autograd.grad(outs, leaves, ds)
    assert any("gnb200" in name for name in seen.names)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
