"""The operators together, as a transformer block uses them: trained with dropout into its residual stream, served in four bits."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import channels_last_groupnorm_b200 as pkg
from tests import dropout_reference as D
from tests import four_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(repo_root):
    spec = importlib.util.spec_from_file_location("video_block", os.path.join(repo_root, "examples", "video_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits,dropout", [(4, 0.1), (8, 0.1), (4, 0.0)])
def test_example_runs(example, bits, dropout):
    first, last, off = example.main(frames=2, size=8, channels=128, heads=2, steps=3, bits=bits, dropout=dropout)
    assert all(torch.isfinite(torch.tensor(v)) for v in (first, last, off))


def test_block_gradients_with_dropout(example):
    """The block's output and gradients against torch's own operations in 64 bits under the same masks."""
    torch.manual_seed(1)
    block = example.VideoBlock(96, 2, device="cuda", dtype=torch.float32, dropout=0.25)
    maps = torch.randn(2, 96, 5, 7, device="cuda").to(memory_format=torch.channels_last).requires_grad_(True)
    tokens = 2 * 5 * 7
    kept = [D.kept(tokens * 96, 0.25, 9, layer, device="cuda").view(tokens, 96) / 0.75 for layer in (0, 1)]
    weights = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}

    def plain_norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    def plain(m):
        b = weights
        stream = F.silu(F.group_norm(m, 32, b["norm_in.weight"], b["norm_in.bias"])).permute(0, 2, 3, 1).reshape(-1, 96)
        qkv = (plain_norm(stream, b["norm1.weight"]) @ b["qkv.weight"].t()).view(-1, 3, 2, 48)
        angle = block.positions(2, 5, 7, m.device).double()[:, [0] * 8 + [1] * 8 + [2] * 8] * block.rotary.inv_freq.double()
        cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)

        def turned(t, w):
            a, c = plain_norm(t, w).split(24, dim=-1)
            return torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)

        q, k = turned(qkv[:, 0], b["rotary.q_weight"]), turned(qkv[:, 1], b["rotary.k_weight"])
        o = torch.einsum("hqk,khd->qhd", (torch.einsum("qhd,khd->hqk", q, k) / 48 ** 0.5).softmax(-1), qkv[:, 2]).reshape(-1, 96)
        stream = stream + (o @ b["out.weight"].t()) * kept[0]
        out = stream + (F.gelu(plain_norm(stream, b["norm2.weight"]) @ b["up.weight"].t()) @ b["down.weight"].t()) * kept[1]
        return out.view(2, 5, 7, 96).permute(0, 3, 1, 2)

    torch.backends.cuda.matmul.allow_tf32 = False
    got, want = block(maps, seed=9), plain(maps.detach().double().requires_grad_(True))
    # as in the test of the block without dropout: sums of some hundreds of terms in 32 bits
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    direction = torch.randn_like(want)
    names = [n for n, _ in block.named_parameters()]
    leaf = maps.detach().double().requires_grad_(True)
    wanted = torch.autograd.grad(plain(leaf), [leaf] + [weights[n] for n in names], direction)
    found = torch.autograd.grad(got, [maps] + [p for _, p in block.named_parameters()], direction.float())
    for name, a, b in zip(["maps"] + names, found, wanted):
        assert (a - b).abs().max() <= 2e-4 * b.abs().max(), name
    # without dropout, in evaluation and with another seed it is another function
    assert not torch.equal(block(maps, seed=10), got)
    block.eval()
    assert torch.equal(block(maps, seed=10), block(maps, seed=9))


@pytest.mark.parametrize("block", [16, 32])
def test_serving_in_a_graph(block):
    """Norm, product, activation and product again, captured once and replayed on new tokens: the bits of the eager calls."""
    torch.manual_seed(2)
    norm = pkg.RMSNorm(320, device="cuda", dtype=torch.bfloat16)
    up, down = (pkg.Linear4bit(torch.randn(o, i, device="cuda").bfloat16() / i ** 0.5, block=block) for o, i in ((1280, 320), (320, 1280)))

    @torch.no_grad()
    def step(branch, stream):
        codes, scales, stream = norm.quantize_4bit(branch, stream, block=block)
        return down(F.gelu(up((codes, scales)))), stream

    branch, stream = (torch.randn(24, 320, device="cuda").bfloat16() for _ in range(2))
    for _ in range(2):
        step(branch, stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(branch, stream)
    for _ in range(3):
        branch.normal_()
        stream.normal_()
        graph.replay()
        for a, b in zip(out, step(branch, stream)):
            assert torch.equal(a, b)
    # and the first product against what its operands stand for
    with torch.no_grad():
        codes, scales, _ = norm.quantize_4bit(branch, stream, block=block)
    kind = pkg.token_four.SCALE_TYPES[block]
    want = R.values(codes, scales) @ R.values(up.weight_codes.view(torch.float4_e2m1fn_x2), up.weight_scales.view(kind), up.weight_scale).t()
    y = up((codes, scales)).double()
    assert (y - want).abs().max() <= 2.0 ** -8 * want.abs().max()  # one rounding to bf16, of the largest at most
