"""The example that runs group norm, token norms, rotary positions and 8-bit outputs together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(repo_root):
    spec = importlib.util.spec_from_file_location("video_block", os.path.join(repo_root, "examples", "video_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_block_learns_and_serves(example):
    first, last, off = example.main(frames=2, size=8, channels=128, heads=2, steps=12)
    assert last < 0.8 * first
    assert off < 0.06  # codes of three bits behind the first in two of the products: 2^-4 at most, a fraction of it on average


def test_block_against_plain_torch(example):
    torch.manual_seed(1)
    block = example.VideoBlock(96, 2, device="cuda", dtype=torch.float32)
    maps = torch.randn(2, 96, 5, 7, device="cuda").to(memory_format=torch.channels_last).requires_grad_(True)

    def plain_norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    def plain(m):
        m = m.double()
        b = {k: v.double() for k, v in block.state_dict().items()}
        stream = torch.nn.functional.silu(torch.nn.functional.group_norm(m, 32, b["norm_in.weight"], b["norm_in.bias"])).permute(0, 2, 3, 1).reshape(-1, 96)
        qkv = (plain_norm(stream, b["norm1.weight"]) @ b["qkv.weight"].t()).view(-1, 3, 2, 48)
        angle = block.positions(2, 5, 7, m.device).double()[:, [0] * 8 + [1] * 8 + [2] * 8] * block.rotary.inv_freq.double()
        cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)

        def turned(t, w):
            a, c = plain_norm(t, w).split(24, dim=-1)
            return torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)

        q, k = turned(qkv[:, 0], b["rotary.q_weight"]), turned(qkv[:, 1], b["rotary.k_weight"])
        scores = torch.einsum("qhd,khd->hqk", q, k) / 48 ** 0.5
        o = torch.einsum("hqk,khd->qhd", scores.softmax(-1), qkv[:, 2]).reshape(-1, 96)
        stream = stream + o @ b["out.weight"].t()
        y = plain_norm(stream, b["norm2.weight"])
        out = stream + torch.nn.functional.gelu(y @ b["up.weight"].t()) @ b["down.weight"].t()
        return out.view(2, 5, 7, 96).permute(0, 3, 1, 2)

    got = block(maps)
    want = plain(maps)
    torch.backends.cuda.matmul.allow_tf32 = False
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    direction = torch.randn_like(want)
    (g,) = torch.autograd.grad(got, maps, direction.float())
    (w,) = torch.autograd.grad(want, maps, direction)
    assert (g - w).abs().max() <= 2e-4 * w.abs().max()
