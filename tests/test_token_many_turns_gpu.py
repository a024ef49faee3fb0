"""Odd rows that share a warp, over many turns of each group of lanes: a row's line in shared memory is written again and again."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

# as in test_token_norm_gpu.py: at most 64 terms a thread and 14 levels of additions, halved by the root, and the norm's own operations
FORWARD = 48 * ref.U32


@pytest.mark.parametrize("c", [3, 9, 31, 150, 301, 999])
def test_every_turn_has_its_own_row(c):
    rows = 60001
    g = torch.Generator(device="cuda").manual_seed(c)
    x, r, dy, ds = (torch.randn(rows, c, device="cuda", generator=g).bfloat16() for _ in range(4))
    w = torch.rand(c, device="cuda", generator=g) + 0.5
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = pkg.rms_norm(x, w, r)
    gx, gr, gw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    x, r, w = x.detach(), r.detach(), w.detach()
    want, sums, rstd = ref.rms(x, w, r, 1e-6, 0.0)
    ref.within(y.detach(), want, ref.rounded(want, y.dtype) + FORWARD * want.abs())
    d, _, size, _ = ref.rms_grads(dy, ds, sums, rstd, w, 0.0)
    ref.within(gx, d, ref.rounded(d, gx.dtype) + 2 * FORWARD * size)
    assert torch.equal(gx, gr)
    # the same bits where the rows come in calls of one turn
    for at in (0, 20000, rows - 64):
        assert torch.equal(y[at:at + 64], pkg.rms_norm(x[at:at + 64].clone(), w, r[at:at + 64].clone())[0])
    q, scale, _ = pkg.rms_norm_quant(x, w, r, block=32)
    most = torch.stack([p.abs().amax(-1) for p in want.split(32, -1)], -1) / 448.0
    ref.within(scale, most.clamp_min(2.0 ** -126), (FORWARD + 2 * ref.U32) * most + 2.0 ** -140)
