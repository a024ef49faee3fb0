"""Products of rows in four bits against the definition in 64 bits."""
import pytest
import torch

import channels_last_groupnorm_b200 as pkg
from channels_last_groupnorm_b200 import _native as nt
from tests import four_reference as R
from tests import token_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U32 = ref.U32


def _exact(rows, k, block, seed):
    """Codes and scales of powers of two: with K up to some thousands every sum, in whatever order, has fewer than 24 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 16, (rows, k), device="cuda", generator=g, dtype=torch.uint8)
    if block == 16:
        byte = torch.tensor([0x30, 0x38, 0x40, 0x48], device="cuda", dtype=torch.uint8)[torch.randint(0, 4, (rows, k // 16), device="cuda", generator=g)]
    else:
        byte = torch.randint(125, 129, (rows, k // 32), device="cuda", generator=g).to(torch.uint8)
    return R.packed(codes).view(torch.float4_e2m1fn_x2), R.tiled(byte).view(torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu)


def _same(tokens, features, k, block):
    x, w = _exact(tokens, k, block, tokens), _exact(features, k, block, features + 1)
    # products are multiples of 2^-4 (codes of halves, scales of halves or quarters) up to 36 * 16 each: below 2^24 of these up to K = 1800, and the sums of
    # random signs far beyond
    got = pkg.linear_4bit(*x, *w, dtype=F32)
    assert torch.equal(got.double(), R.values(*x) @ R.values(*w).t())
    assert nt.wait_timeouts() == 0


# tokens: one; in and beyond tiles of 16, 32, 64 and 128, and several tiles
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 100, 128, 129, 200, 256, 257, 300, 511, 513, 777])
@pytest.mark.parametrize("block", [16, 32])
def test_tokens(tokens, block):
    _same(tokens, 384, 512, block)


# one K step and less; parts of a tile of scales; one K tile and less, more; K in clusters
@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 224, 256, 288, 352, 512, 544, 768, 1056, 1344, 2080])
@pytest.mark.parametrize("tokens", [5, 140, 300])
@pytest.mark.parametrize("block", [16, 32])
def test_channels(k, tokens, block):
    _same(tokens, 200, k, block)


@pytest.mark.parametrize("features", [1, 2, 7, 8, 127, 128, 129, 250, 256, 258, 1111, 4100])
@pytest.mark.parametrize("tokens", [3, 70, 260])
def test_features(features, tokens):
    _same(tokens, features, 320, 16)


@pytest.mark.parametrize("tokens,features,k", [(1000, 2000, 1024), (2048, 1536, 512), (4100, 1000, 256), (600, 20000, 288)])
@pytest.mark.parametrize("block", [16, 32])
def test_many_tiles(tokens, features, k, block):
    _same(tokens, features, k, block)


def _random(rows, c, block, seed, scale):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, c), device="cuda", generator=g)
    return pkg.quantize_4bit(x, block, scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("block,scaled", [(16, True), (16, False), (32, False)])
@pytest.mark.parametrize("bias", [None, F32, F16, BF16])
@pytest.mark.parametrize("tokens,features,c", [(1, 250, 1352), (77, 130, 1111), (300, 512, 640)])
def test_values(dtype, block, scaled, bias, tokens, features, c):
    sx, sw = (torch.full((1,), v, device="cuda") if scaled else None for v in (0.0123, 0.0045))
    x, w = _random(tokens, c, block, 1, sx), _random(features, c, block, 2, sw)
    b = None if bias is None else torch.randn(features, device="cuda").to(bias)
    got = pkg.linear_4bit(*x, *w, sx, sw, b, dtype)
    assert got.dtype == dtype and got.is_contiguous()
    vx, vw = R.values(*x, sx), R.values(*w, sw)
    want, size = vx @ vw.t(), vx.abs() @ vw.abs().t()
    if b is not None:
        want, size = want + b.double(), size + b.double().abs()
    # 64 products and the sum so far are added at a time; each may lose its last place in 32 bits, cut off (2 u), of what is added at the most; then a product
    # of scales, one with the sum, the bias
    steps = (c + 63) // 64
    ref.within(got, want, ref.rounded(want, dtype) + (65 * steps * 2 + 4) * U32 * size)


def test_nan_stays_in_its_row():
    x = torch.randn(300, 256, device="cuda")
    x[7, 200], x[130, 3] = float("nan"), float("inf")
    wx = torch.randn(260, 256, device="cuda")
    wx[255, 0] = float("nan")
    for rows in (300, 20):
        y = pkg.linear_4bit(*pkg.quantize_4bit(x[:rows].contiguous()), *pkg.quantize_4bit(wx), dtype=F32)
        bad = torch.zeros(300, 260, dtype=torch.bool, device="cuda")
        bad[7], bad[130], bad[:, 255] = True, True, True
        assert torch.equal(torch.isnan(y), bad[:rows])


def test_shapes_and_layouts():
    x, w = _exact(60, 128, 16, 1), _exact(40, 128, 16, 2)
    want = pkg.linear_4bit(*x, *w)
    assert torch.equal(pkg.linear_4bit(x[0].view(3, 20, 64), x[1], *w).view(60, 40), want)
    # codes with gaps between the rows are copied
    gaps = torch.zeros(60, 80, dtype=torch.uint8, device="cuda")
    gaps[:, :64] = x[0].view(torch.uint8)
    assert torch.equal(pkg.linear_4bit(gaps[:, :64].view(torch.float4_e2m1fn_x2), x[1], *w), want)
    bias = torch.randn(80, device="cuda")[::2]
    assert torch.equal(pkg.linear_4bit(*x, *w, bias=bias), pkg.linear_4bit(*x, *w, bias=bias.contiguous()))
    one = pkg.quantize_4bit(torch.ones(128, device="cuda"))
    assert one[0].shape == (64,) and pkg.linear_4bit(*one, *w).shape == (40,)


def test_same_bits_every_time():
    """Also of one token among others in its tile, and of a K that a cluster shares."""
    x, w = _random(16, 4096, 16, 1, None), _random(512, 4096, 16, 2, None)
    first = pkg.linear_4bit(*x, *w, dtype=F32)
    for _ in range(5):
        assert torch.equal(pkg.linear_4bit(*x, *w, dtype=F32), first)


def test_refusals():
    x, w = _exact(4, 64, 16, 1), _exact(8, 64, 16, 2)
    other, wide = _exact(8, 64, 32, 3), _exact(8, 96, 16, 4)
    one = torch.ones(1, device="cuda")
    for args, kw, words in (((x[0], x[1], w[0][0], w[1]), {}, "weight_codes"), ((*x, *other), {}, "blocks"), ((*x, *wide), {}, "channels"),
                            ((*x, w[0], w[1][:64]), {}, "scales"), ((x[0], x[1].t(), *w), {}, "scales"), ((*x, *w), {"scale": one.half()}, "scale"),
                            ((*other, *other), {"weight_scale": one}, "whole tensor"), ((*x, *w), {"bias": torch.ones(7, device="cuda")}, "bias"),
                            ((*x, *w), {"bias": torch.ones(8, device="cuda").double()}, "bias"), ((*x, *w), {"dtype": torch.int32}, "dtype"),
                            ((*x, *w), {"bias": torch.ones(8, device="cuda").requires_grad_(True)}, "gradient"),
                            ((x[0].view(torch.uint8), x[1], *w), {}, "codes"), ((*x, w[0].cpu(), w[1].cpu()), {}, "weight_codes")):
        with pytest.raises(ValueError, match=words):
            pkg.linear_4bit(*args, **kw)


def test_streams_and_graphs():
    """On another stream; two captured calls; a weight quantised right in front of its product."""
    x, w = _random(40, 1024, 16, 1, None), _random(300, 1024, 16, 2, None)
    want = pkg.linear_4bit(*x, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.linear_4bit(*x, *w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    rows, weights = torch.randn(40, 1024, device="cuda"), torch.randn(300, 1024, device="cuda")
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            a = pkg.quantize_4bit(rows)
            outs.append(pkg.linear_4bit(*a, *pkg.quantize_4bit(weights)))
    for step in range(3):
        rows.normal_()
        weights.normal_()
        want = pkg.linear_4bit(*pkg.quantize_4bit(rows), *pkg.quantize_4bit(weights))
        graphs[step % 2].replay()
        assert torch.equal(outs[step % 2], want)
    with torch.cuda.stream(side):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_compiled():
    x, w = torch.randn(20, 200, device="cuda").bfloat16(), pkg.quantize_4bit(torch.randn(72, 200, device="cuda"))
    bias = torch.randn(72, device="cuda")

    def call(x, bias):
        return pkg.linear_4bit(*pkg.quantize_4bit(x), *w, bias=bias, dtype=x.dtype)

    torch._dynamo.reset()
    assert torch.equal(torch.compile(call, backend="aot_eager", fullgraph=True)(x, bias), call(x, bias))


def test_far_outputs():
    """An output of more than 2^31 elements."""
    tokens, features = 70001, 32003
    x, w = _exact(tokens, 32, 32, 1), _exact(features, 32, 32, 2)
    y = pkg.linear_4bit(*x, *w, dtype=BF16)
    vx, vw = R.values(*x)[-300:], R.values(*w)
    assert torch.equal(y[-300:], (vx @ vw.t()).to(BF16))


@pytest.mark.parametrize("block", [16, 32])
def test_module(block):
    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 72).cuda().bfloat16()
    four = pkg.Linear4bit.from_linear(linear, block)
    x = torch.randn(3, 5, 200, device="cuda").bfloat16()
    norm = pkg.RMSNorm(200, device="cuda", dtype=BF16)
    with torch.no_grad():
        y = four(x)
        codes, scales = pkg.quantize_4bit(x, block)
        want = R.values(codes, scales) @ R.values(four.weight_codes.view(torch.float4_e2m1fn_x2), four.weight_scales.view(pkg.token_four.SCALE_TYPES[block]),
                                                  four.weight_scale).t() + linear.bias.double()
        assert y.shape == (3, 5, 72) and y.dtype == BF16
        ref.within(y.view(15, 72), want, ref.rounded(want, BF16) + 1e-3)
        # each operand is off by a tenth or so, so the product by a sixth at most
        plain = linear(x).float()
        assert (y.float() - plain).norm() <= 0.2 * plain.norm()
        assert torch.equal(four(norm.quantize_4bit(x, block=block)), four(pkg.rms_norm_quant_4bit(x, norm.weight, block=block)))
        # checkpoints, and casts that leave the weight's scale in 32 bits
        again = pkg.Linear4bit(torch.randn(72, 200, device="cuda").bfloat16(), torch.zeros(72, device="cuda").bfloat16(), block)
        again.load_state_dict(four.state_dict())
        assert torch.equal(again(x), y)
        if block == 16:
            kept = four.weight_scale.clone()
            assert four.half().weight_scale.dtype == F32 and torch.equal(four.weight_scale, kept)
    with pytest.raises(ValueError, match="expected input"):
        four(x[..., :199])


# pairs with tiles of 256 and of 128 features, clusters, single CTAs; outputs whose rows begin anywhere
@pytest.mark.parametrize("tokens,features,k", [(3000, 1111, 1344), (2100, 1536, 512), (777, 1111, 320), (300, 1110, 2080), (70, 1113, 1056), (9, 2500, 96)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_sixteen_bits(tokens, features, k, dtype, bias):
    x, w = _exact(tokens, k, 16, tokens), _exact(features, k, 16, features + 1)
    b = torch.randint(-64, 64, (features,), device="cuda").to(dtype) if bias else None
    got = pkg.linear_4bit(*x, *w, bias=b, dtype=dtype)
    want = R.values(*x) @ R.values(*w).t() + (b.double() if bias else 0.0)
    assert torch.equal(got, want.to(dtype))  # exact in 32 bits, rounded once


def test_outputs_of_any_address():
    """Through the C ABI: an output that begins off a vector, and what lies around it as it was."""
    for tokens, features in ((300, 512), (20, 512), (2100, 1536)):
        x, w = _exact(tokens, 512, 16, 1), _exact(features, 512, 16, 2)
        want = pkg.linear_4bit(*x, *w)
        room = torch.full((tokens * features + 64,), 7.0, device="cuda", dtype=BF16)
        rc = nt.lib.gnb200_linear_4bit(x[0].data_ptr(), x[1].data_ptr(), None, w[0].data_ptr(), w[1].data_ptr(), None, None, tokens, features, 512, 16, 0, 2,
                                       room.data_ptr() + 2, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(room[1:1 + tokens * features].view(tokens, features), want)
        assert (room[0] == 7).all() and (room[1 + tokens * features:] == 7).all()


def test_nothing_is_written_behind():
    """Rows and features that fill up a tile leave what lies behind the output as it was."""
    for tokens, features, k in ((130, 131, 256), (1, 1, 32), (17, 129, 544), (2000, 1111, 256)):
        x, w = _exact(tokens, k, 32, 1), _exact(features, k, 32, 2)
        room = torch.full((tokens * features + 4096,), 7.0, device="cuda")
        rc = nt.lib.gnb200_linear_4bit(x[0].data_ptr(), x[1].data_ptr(), None, w[0].data_ptr(), w[1].data_ptr(), None, None, tokens, features, k, 32, 0, 0,
                                       room.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert torch.equal(room[:tokens * features].view(tokens, features).double(), R.values(*x) @ R.values(*w).t())
        assert (room[tokens * features:] == 7).all()


def test_several_streams_at_once():
    """Calls of all kernels side by side on four streams: the bits of calls one by one."""
    shapes = [(300, 512, 512), (8, 4096, 2048), (2100, 1536, 512), (64, 1000, 4096)]
    calls = [(_exact(t, k, 16, t), _exact(n, k, 16, n)) for t, n, k in shapes]
    want = [pkg.linear_4bit(*x, *w) for x, w in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, ((x, w), s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(pkg.linear_4bit(*x, *w))
    torch.cuda.synchronize()
    for one, outs in zip(want, got):
        assert all(torch.equal(one, o) for o in outs)
    assert nt.wait_timeouts() == 0
