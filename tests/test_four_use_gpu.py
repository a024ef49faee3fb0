"""Rows in four bits and their products as programs use them: compiled modules, replays on other streams, tokens alone and in company, a served block."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import channels_last_groupnorm_b200 as pkg
from tests import four_reference as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("bias", [False, True])
def test_compiled_module(block, bias):
    """`Linear4bit`, whose forward views bytes as packed codes, on rows and on codes of the norm."""
    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 72, bias=bias).cuda().bfloat16()
    four, norm = pkg.Linear4bit.from_linear(linear, block), pkg.RMSNorm(200, device="cuda", dtype=BF16)

    def normed(x, r):
        codes, scales, s = norm.quantize_4bit(x, r, block=block)
        return four((codes, scales)), s

    x, r = (torch.randn(3, 5, 200, device="cuda").bfloat16() for _ in range(2))
    with torch.no_grad():
        torch._dynamo.reset()
        assert torch.equal(torch.compile(four, backend="aot_eager", fullgraph=True)(x), four(x))
        for a, b in zip(torch.compile(normed, backend="aot_eager", fullgraph=True)(x, r), normed(x, r)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_module_of_a_broken_weight(block, what):
    """A NaN or an infinity among the weights makes its feature NaN and leaves the others as they are."""
    torch.manual_seed(0)
    weight = torch.randn(72, 200, device="cuda").bfloat16()
    weight[9, :4] = 0.01
    x = torch.randn(5, 200, device="cuda").bfloat16()
    broken = weight.clone()
    broken[9, 3] = what
    with torch.no_grad():
        want, got = pkg.Linear4bit(weight, block=block)(x), pkg.Linear4bit(broken, block=block)(x)
    assert torch.isnan(got[:, 9]).all()
    rest = torch.arange(72, device="cuda") != 9
    assert torch.equal(got[:, rest], want[:, rest])


@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -60, 2.0 ** 100])
def test_module_of_far_weights(size):
    """Weights far from one, down to where the weight's own scale is cut off: as near as weights of one."""
    torch.manual_seed(0)
    weight, x = torch.randn(72, 200, device="cuda"), torch.randn(5, 200, device="cuda")
    with torch.no_grad():
        near, far = pkg.Linear4bit(weight)(x).double(), pkg.Linear4bit(weight * size)(x).double() / size
    if size < 2.0 ** -100:  # block scales have fewer bits there, but no sum is lost
        want = x.double() @ weight.double().t()
        assert (far - want).norm() <= 0.3 * want.norm()
    else:
        assert torch.equal(far, near)


def test_module_without_features():
    four = pkg.Linear4bit(torch.zeros(0, 200, device="cuda").bfloat16())
    assert four(torch.ones(3, 200, device="cuda").bfloat16()).shape == (3, 0)


def test_replay_on_another_stream():
    """A captured product follows its inputs on the stream of the replay."""
    rows, weights = torch.randn(40, 1024, device="cuda"), torch.randn(300, 1024, device="cuda")

    def call():
        return pkg.linear_4bit(*pkg.quantize_4bit(rows), *pkg.quantize_4bit(weights))

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    side = torch.cuda.Stream()
    for _ in range(3):
        rows.normal_()
        weights.normal_()
        want = call()
        out.fill_(7.0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, want) and not (out == 7.0).all()


@pytest.mark.parametrize("features,k", [(512, 4096), (4096, 1024), (20480, 512), (130, 96)])
@pytest.mark.parametrize("block", [16, 32])
def test_a_token_alone_and_in_company(features, k, block):
    """Up to 16 tokens take the same tile and share K out alike: a token's bits do not go by the others."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(n, k, device="cuda", generator=g) for n in (16, features))
    w = pkg.quantize_4bit(w, block)
    whole = pkg.linear_4bit(*pkg.quantize_4bit(x, block), *w, dtype=F32)
    for i in (0, 7, 15):
        assert torch.equal(pkg.linear_4bit(*pkg.quantize_4bit(x[i : i + 1], block), *w, dtype=F32), whole[i : i + 1])
    assert torch.equal(pkg.linear_4bit(*pkg.quantize_4bit(x[:9], block), *w, dtype=F32), whole[:9])


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("c", [96, 1111])
def test_codes_of_codes(block, c):
    """What codes of the norm stand for has the same codes again: the largest of a block is 6 times its scale, or 4 times where that is a power of two."""
    x, r = (torch.randn(77, c, device="cuda") * s for s in (1.0, 3.0))
    codes, scales, _ = pkg.rms_norm_quant_4bit(x, None, r, block=block)
    again = pkg.quantize_4bit(pkg.dequantize_4bit(codes, scales, c, dtype=F32), block)
    assert torch.equal(again[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[1].view(torch.uint8), scales.view(torch.uint8))


@pytest.fixture(scope="module")
def example(repo_root):
    spec = importlib.util.spec_from_file_location("video_block", os.path.join(repo_root, "examples", "video_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [16, 32])
def test_served_block(example, bits):
    """The example's block in four bits against the same steps with products, in 64 bits, of what codes and scales stand for."""
    torch.manual_seed(2)
    block = example.VideoBlock(128, 2, device="cuda", dtype=F32).eval()
    maps = torch.randn(2, 128, 6, 6, device="cuda").to(memory_format=torch.channels_last)
    weights = {n: pkg.Linear4bit.from_linear(getattr(block, n), bits) for n in ("qkv", "out", "up", "down")}

    def plain(name, x):
        m = weights[name]
        codes, scales = x if isinstance(x, tuple) else pkg.quantize_4bit(x, bits)
        w = R.values(m.weight_codes.view(torch.float4_e2m1fn_x2), m.weight_scales.view(pkg.token_four.SCALE_TYPES[bits]), m.weight_scale)
        return (R.values(codes, scales) @ w.t()).float()

    with torch.no_grad():
        stream = block.tokens_of(maps)
        rows = lambda x, norm: pkg.quantize_4bit(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm.weight, bits)  # noqa: E731
        attended = plain("out", block.attention(plain("qkv", rows(stream, block.norm1)), block.positions(2, 6, 6, maps.device)))
        stream = stream + attended
        want = block.maps_of(stream + plain("down", F.gelu(plain("up", rows(stream, block.norm2)))), maps)
        got = block.serve_4bit(maps, weights)
    # Sums in 32 bits move what is quantised next by some 1e-6, and with it single codes that lie at a border, of some 1e5 by a few: each a sixth of its
    # block's largest number at most, in one token's 128 channels or more.  Their part of the block's 72 tokens is below 1e-2; another weight, scale or residual
    # is of the order of one.
    assert (got - want).norm() <= 1e-2 * want.norm()
