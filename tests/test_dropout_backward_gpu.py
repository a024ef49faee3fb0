"""The backward of dropout where others look at its gradient: batches of gradients, dispatch modes."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import channels_last_groupnorm_b200 as pkg
from tests import dropout_reference as D

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _case(residual, on_device):
    torch.manual_seed(1)
    x = torch.randn(9, 40, device="cuda").bfloat16().requires_grad_(True)
    r = torch.randn(9, 40, device="cuda").to(residual).requires_grad_(True) if residual is not None else None
    seed = torch.tensor([6], device="cuda") if on_device else 6
    kept = D.kept(x.numel(), 0.25, 6, 2, device="cuda").view(9, 40)
    return x, r, seed, kept


@pytest.mark.parametrize("residual", [None, BF16, F32])
@pytest.mark.parametrize("on_device", [False, True])
def test_batched_gradients(residual, on_device):
    """Each gradient of a batch has the mask of the call."""
    x, r, seed, kept = _case(residual, on_device)
    leaves = [t for t in (x, r) if t is not None]
    s = pkg.dropout_add(x, r, 0.25, seed, 2)
    ds = torch.randn(3, 9, 40, device="cuda").to(s.dtype)
    got = torch.autograd.grad(s, leaves, ds, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(s, leaves, ds[i], retain_graph=True)):
            assert a[i].dtype == b.dtype and torch.equal(a[i], b)
    assert (got[0][:, ~kept] == 0).all()


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def test_a_mode_in_the_backward_alone():
    x, r, seed, _ = _case(F32, True)
    s = pkg.dropout_add(x, r, 0.25, seed, 2)
    ds = torch.randn_like(s)
    want = torch.autograd.grad(s, (x, r), ds, retain_graph=True)
    with Seen() as seen:
        got = torch.autograd.grad(s, (x, r), ds)
    assert any("dropout_mask" in name for name in seen.names)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
