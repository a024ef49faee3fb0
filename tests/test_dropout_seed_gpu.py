"""Dropout without a seed: refused where it would repeat a mask without a word, taken where nothing is dropped."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu


def test_training_needs_a_seed():
    x, r = (torch.randn(9, 40, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
    m = pkg.DropoutAdd(0.3, layer=4)
    for call in (lambda: m(x, r), lambda: m(x), lambda: m(x, r, None), lambda: pkg.dropout_add(x, r, 0.3), lambda: pkg.dropout_add(x), lambda: pkg.dropout_add(x, r, 0.3, layer=7)):
        with pytest.raises(ValueError, match="seed is needed"):
            call()
    with torch.no_grad(), pytest.raises(ValueError, match="seed is needed"):
        m(x, r)
    assert torch.equal(m(x, r, 0), pkg.dropout_add(x, r, 0.3, 0, 4))
    with pytest.raises(ValueError, match="64 bits"):
        pkg.dropout_add(x, r, 0.3, layer=2 ** 64)


def test_nothing_to_drop_needs_none():
    x, r = (torch.randn(9, 40, device="cuda").requires_grad_(True) for _ in range(2))
    assert torch.equal(pkg.dropout_add(x, r, 0.0), x + r) and torch.equal(pkg.DropoutAdd(0.0)(x, r), x + r)
    m = pkg.DropoutAdd(0.3).eval()
    for seed in (None, 5):
        s = m(x, r, seed)
        assert torch.equal(s, x + r)
        ds = torch.randn_like(s)
        assert all(torch.equal(g, ds) for g in torch.autograd.grad(s, (x, r), ds))
    assert pkg.dropout_add(x[:0], r[:0], 0.3).shape == (0, 40)


def test_compiled_without_a_seed():
    x, r = torch.randn(9, 40, device="cuda"), torch.randn(9, 40, device="cuda")
    m = pkg.DropoutAdd(0.3).eval()
    torch._dynamo.reset()
    assert torch.equal(torch.compile(m, backend="aot_eager", fullgraph=True)(x, r), x + r)
    with pytest.raises(Exception, match="seed is needed"):
        torch.compile(m.train(), backend="aot_eager", fullgraph=True)(x, r)


def test_slices_need_seeds_of_their_own():
    """What the documentation says of ranks: the same seed drops the same elements of every slice."""
    x = torch.ones(4, 1 << 16, device="cuda")
    masks = [pkg.dropout_add(part, None, 0.25, 11) > 0 for part in x]
    assert all(torch.equal(m, masks[0]) for m in masks)
    masks = [pkg.dropout_add(part, None, 0.25, 11 * 4 + rank) > 0 for rank, part in enumerate(x)]
    for i, m in enumerate(masks):
        for other in masks[:i]:
            # six standard deviations of independent masks
            assert abs((m == other).float().mean().item() - (0.75 ** 2 + 0.25 ** 2)) <= 6 * 0.5 / 2 ** 8
