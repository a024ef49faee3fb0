"""What the token rows of a transformer block meet around its norms, as measurable cases: in training the dropout of a
branch with the residual's addition, whose mask is made from a counter wherever it is needed; in serving rows in four bits
with block scales - quantised, read back, normed straight into them - and the product of two such matrices.

`run` computes them in their plain form, elementary torch operations in 32 bits, rounded once at the end, or, where `own`
is true, by the package's operators.  `exact` gives the same from the definition in 64 bits.

Four bits: a block of 16 channels shares an e4m3 scale, below a scale of the whole tensor in 32 bits; a block of 32 shares
a power of two and has no scale above it.  Codes are e2m1, two a byte, the first one low; a row has whole blocks of 32 of them, zeros behind
its channels.  Scales lie in tiles of 128 rows and 4 blocks: row r, block b at ((r / 128) * (columns / 4) + b / 4) * 512 +
(r % 32) * 16 + (r % 128 / 32) * 4 + b % 4, zeros behind the rows and blocks there are.
"""
import math

import numpy
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

_package = None


def _ops():
    global _package
    if _package is None:
        import channels_last_groupnorm_b200 as _package
    return _package


def _pack(rows, c, dtype, block):
    return {"op": "pack", "rows": rows, "c": c, "dtype": dtype, "block": block}


def _linear(rows, c, out, dtype, block, bias=False):
    return {"op": "linear", "rows": rows, "c": c, "out": out, "dtype": dtype, "block": block, "bias": bias}


def _norm(rows, c, out, dtype, block, residual="same"):
    """residual: "none", "same" (the type of x) or "float32" """
    return {"op": "norm", "rows": rows, "c": c, "out": out, "dtype": dtype, "block": block, "residual": residual}


def _dropout(rows, c, dtype, p, residual="same", held="host"):
    """held: where the seed is, "host" (a number) or "device" (a tensor, as a captured step wants it)"""
    return {"op": "dropout", "rows": rows, "c": c, "dtype": dtype, "p": p, "residual": residual, "held": held}


def listed():
    return [
        # Half-precision image tokens kept in four bits and read back, a last block that is not whole.
        dict(_pack(777, 1352, "float16", 16), name="pack_ragged_777x1352_b16"),
        # A large projection's weight, or a long prompt's activations, stored and read back.
        dict(_pack(16384, 8192, "bfloat16", 32), name="pack_16384x8192_b32"),
        # One token being answered: the weights are what is read, launches are what is waited for.
        dict(_linear(1, 4096, 4096, "bfloat16", 16), name="linear_decode_1x4096x4096"),
        # Eight sequences answered at once, a wider feed-forward layer.
        dict(_linear(8, 5120, 20480, "bfloat16", 16), name="linear_decode_8x5120x20480"),
        # A prompt's tokens.
        dict(_linear(2048, 4096, 4096, "bfloat16", 16), name="linear_prompt_2048x4096x4096"),
        # Many prompts at a wide model: the product's own rate.
        dict(_linear(8192, 8192, 8192, "bfloat16", 16), name="linear_prompts_8192x8192x8192"),
        # Half precision, odd sizes everywhere, powers of two as scales, a bias.
        dict(_linear(777, 1352, 1111, "float16", 32, bias=True), name="linear_ragged_777x1352x1111_b32"),
        # Eight answered sequences through the norm with the residual's addition into the queries, keys and values.
        dict(_norm(8, 4096, 6144, "bfloat16", 16), name="norm_decode_8x4096x6144"),
        # A prompt through the norm into the feed-forward layer, residual stream in fp32.
        dict(_norm(2048, 4096, 16384, "bfloat16", 16, residual="float32"), name="norm_prompt_2048x4096x16384"),
        # A small training step: an image's tokens at a U-Net's second width; the seed is on the device, as in a captured step.
        dict(_dropout(64, 640, "float16", 0.1, held="device"), name="dropout_image_64x640"),
        # fp32 training at odd sizes, no residual.
        dict(_dropout(2077, 1111, "float32", 0.25, residual="none"), name="dropout_odd_2077x1111"),
        # A training step's batch of tokens in bf16.
        dict(_dropout(16384, 4096, "bfloat16", 0.1), name="dropout_16384x4096"),
    ]


#: most that a drawn case moves and computes, half of what the largest listed ones do
MOST_BYTES, MOST_FLOPS = 3e8, 5e11


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    n = rng.choice([320, 640, 1280, 2048, 2560, 4096, 5120, 8192, 10240]) if rng.random() < 0.4 else _between(rng, lo, hi)
    return n + 8 - n % 8 if rng.random() < 0.4 else n


def _drawn(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    op = rng.choice(["pack", "linear", "linear", "norm", "dropout"])
    rows = rng.choice([1, 2, 4, 8, 16, 32]) if rng.random() < 0.25 else _between(rng, 1, 16384)
    c, block = _width(rng, 64, 12288), rng.choice([16, 16, 32])
    if op == "pack":
        return _pack(rows, c, dtype, block)
    if op == "dropout":
        return _dropout(rows, c, dtype, rng.choice([0.05, 0.1, 0.1, 0.25, 0.5]), rng.choice(["none", "same", "same", "float32"]), rng.choice(["host", "device"]))
    if dtype == "float32":  # products answer in 16 bits
        dtype = "bfloat16"
    if op == "linear":
        return _linear(rows, c, _width(rng, 64, 16384), dtype, block, rng.random() < 0.3)
    return _norm(rows, c, _width(rng, 64, 16384), dtype, block, rng.choice(["none", "same", "same", "float32"]))


def draw(rng):
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= MOST_BYTES and work(case)["flops"] <= MOST_FLOPS:
            return case


# ---------------------------------------------------------------------------------------------- inputs


def _up(n, to):
    return -(-n // to) * to


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, op, rows, c = DTYPES[case["dtype"]], case["op"], case["rows"], case["c"]

    def normal(shape, scale, dt=dtype):
        return torch.randn(shape, device=dev, generator=gen, dtype=dt).mul_(scale)

    # some channels are much larger than the others
    state = {"case": case, "x": normal((rows, c), 1.0), "residual": None}
    state["x"][:, :: max(1, c // 5)] *= 8
    if op in ("norm", "dropout") and case["residual"] != "none":
        state["residual"] = normal((rows, c), 2.0, torch.float32 if case["residual"] == "float32" else dtype)
    if op == "dropout":
        state["ds"] = normal((rows, c), 0.1, dtype if state["residual"] is None else state["residual"].dtype)
        state["seed"] = torch.randint(-2 ** 62, 2 ** 62, (1,), device=dev, generator=gen)
        if case["held"] == "host":
            state["seed"] = int(state["seed"].item())
        state["layer"] = seed % 61
        for name in ("x", "residual"):
            if state[name] is not None:
                state[name].requires_grad_(True)
        return state
    # scales of whole tensors, as a calibration leaves them that keeps to powers of two: no rounding of their own
    state["scale"] = None if case["block"] == 32 else torch.full((1,), 2.0 ** -6, device=dev)
    if op == "pack":
        return state
    if op == "norm":
        state["norm_weight"] = torch.rand(c, device=dev, generator=gen).add_(0.5).to(dtype)
    state["weight_scale"] = None if case["block"] == 32 else torch.full((1,), 2.0 ** -14, device=dev)
    codes, scales = _quantised(normal((case["out"], c), 0.02, torch.float32), case["block"], state["weight_scale"])
    state["weight"] = (_packed(codes), _tiled(scales))
    state["bias"] = normal((case["out"],), 0.5) if case.get("bias") else None
    return state


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"pack": _plain_pack, "linear": _plain_linear, "norm": _plain_norm, "dropout": _plain_dropout}[state["case"]["op"]](state)


def _run_own(state):
    ops, case = _ops(), state["case"]
    x, r = state["x"], state["residual"]
    if case["op"] == "dropout":
        s = ops.dropout_add(x, r, case["p"], state["seed"], state["layer"])
        return (s.detach(),) + torch.autograd.grad(s, (x,) if r is None else (x, r), state["ds"])
    block, scale = case["block"], state["scale"]
    with torch.no_grad():
        if case["op"] == "pack":
            codes, scales = ops.quantize_4bit(x, block, scale)
            return ops.dequantize_4bit(codes, scales, case["c"], scale, x.dtype)
        stream = ()
        if case["op"] == "linear":
            codes, scales = ops.quantize_4bit(x, block, scale)
        else:
            codes, scales, *stream = ops.rms_norm_quant_4bit(x, state["norm_weight"], r, EPS, 0.0, block, scale)
        y = ops.linear_4bit(codes, scales, *state["weight"], scale, state["weight_scale"], state["bias"], x.dtype)
        return (y, *stream)


def _quantised(t, block, scale):
    """Codes (0 to 15) and scales of the rows of t (float32), whole blocks of 32 channels."""
    rows, c = t.shape
    wide = _up(c, 32)
    blocks = torch.nn.functional.pad(t, (0, wide - c)).reshape(rows, wide // block, block)
    most = blocks.abs().amax(dim=-1)
    if block == 16:
        one = torch.ones(1, device=t.device) if scale is None else scale
        scales = (most / (6.0 * one)).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
        over = blocks / (scales.float() * one).unsqueeze(-1)
    else:
        exponent = torch.clamp(torch.bitwise_right_shift(most.view(torch.int32), 23) - 2, 0, 254)
        scales = exponent.to(torch.uint8).view(torch.float8_e8m0fnu)
        over = blocks / scales.float().unsqueeze(-1)
    size = over.abs().clamp(max=6.0)
    # steps of a half up to 2, of one up to 4, of two up to 6; torch.round takes ties to the even one
    code = torch.where(size <= 2.0, torch.round(size * 2), torch.where(size <= 4.0, torch.round(size) + 2, torch.round(size / 2) + 4))
    return (code.to(torch.uint8) | (torch.signbit(over).to(torch.uint8) << 3)).reshape(rows, wide), scales


def _packed(codes):
    """Two codes a byte."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).view(torch.float4_e2m1fn_x2)


def _tiled(scales):
    rows, blocks = scales.shape
    tall, wide = _up(rows, 128), _up(blocks, 4)
    whole = torch.nn.functional.pad(scales.view(torch.uint8), (0, wide - blocks, 0, tall - rows))
    tiles = whole.reshape(tall // 128, 4, 32, wide // 4, 4).permute(0, 3, 2, 1, 4)
    return tiles.reshape(tall, wide).view(scales.dtype)


def _values(codes, scales, block):
    """What codes and scales stand for, in 32 bits, before the tensor's own scale."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    rows, wide = codes.shape
    return (table[codes.int()].reshape(rows, wide // block, block) * scales.float().unsqueeze(-1)).reshape(rows, wide)


def _plain_pack(state):
    case, one = state["case"], 1.0 if state["scale"] is None else state["scale"]
    codes, scales = _quantised(state["x"].float(), case["block"], state["scale"])
    return (_values(codes, scales, case["block"]) * one)[:, :case["c"]].to(state["x"].dtype)


def _plain_product(state, rows):
    case = state["case"]
    packed, tiles = state["weight"][0].view(torch.uint8), state["weight"][1]
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(1)
    tall, wide = tiles.shape
    scales = tiles.view(torch.uint8).reshape(tall // 128, wide // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tall, wide)
    scales = scales[:case["out"], :codes.shape[1] // case["block"]].contiguous().view(tiles.dtype)
    y = _values(*_quantised(rows, case["block"], state["scale"]), case["block"]) @ _values(codes, scales, case["block"]).t()
    if state["scale"] is not None:
        y = y * (state["scale"] * state["weight_scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _plain_linear(state):
    return (_plain_product(state, state["x"].float()),)


def _plain_norm(state):
    x, r = state["x"], state["residual"]
    s = x.float() if r is None else x.float() + r.float()
    y = s * (s.square().mean(dim=-1, keepdim=True) + EPS).rsqrt() * state["norm_weight"].float()
    return (_plain_product(state, y),) + (() if r is None else (s.to(r.dtype),))


LOW = 0xFFFFFFFF


def _kept(shape, p, seed, layer, dev):
    """Which elements a dropout leaves: element i by word i % 4 of Philox 4x32 with ten rounds (Salmon and others, 2011), counter (i / 4, layer), key
    the seed; dropped where the word is below p * 2^32.  64-bit products wrap, which leaves their low and high words."""
    n = math.prod(shape)
    at = torch.arange(-(-n // 4), device=dev)
    key = [seed & LOW, (seed >> 32) & LOW]
    words = [at & LOW, at >> 32, torch.full_like(at, layer & LOW), torch.full_like(at, (layer >> 32) & LOW)]
    for _ in range(10):
        first, second = words[0] * 0xD2511F53, words[2] * 0xCD9E8D57
        words = [((second >> 32) & LOW) ^ words[1] ^ key[0], second & LOW, ((first >> 32) & LOW) ^ words[3] ^ key[1], first & LOW]
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    return torch.stack(words, dim=-1).reshape(-1)[:n].reshape(shape) >= round(p * 2 ** 32)


def _plain_dropout(state):
    case, x, r, ds = state["case"], state["x"], state["residual"], state["ds"]
    kept = _kept(x.shape, case["p"], state["seed"], state["layer"], x.device)
    scale = 1.0 / (1.0 - case["p"])
    s = torch.where(kept, x.float() * scale, 0.0)
    dx = torch.where(kept, ds.float() * scale, 0.0).to(x.dtype)
    if r is None:
        return s.to(x.dtype), dx
    return (s + r.float()).to(r.dtype), dx, ds


# ---------------------------------------------------------------------------------------------- what it takes


def _four(rows, c, block):
    """Bytes of rows in four bits."""
    return rows * (_up(c, 32) // 2 + _up(c, 32) // block)


def work(case):
    size, rows, c = BYTES[case["dtype"]], case["rows"], case["c"]
    if case["op"] == "dropout":  # x and the residual in, their sum out; its gradient in, that of x out
        wide = 4 if case["residual"] == "float32" else size
        stream = 0 if case["residual"] == "none" else wide
        return {"bytes": rows * c * (2 * size + wide + wide + stream), "flops": rows * c * 4}
    if case["op"] == "pack":  # rows in, codes and scales out and in, rows out
        return {"bytes": 2 * rows * c * size + 2 * _four(rows, c, case["block"]), "flops": rows * c * 4}
    wide = 4 if case.get("residual") == "float32" else size
    stream = 2 * wide if case.get("residual", "none") != "none" else 0
    # rows in, codes out and in, weights in, answers out
    moved = rows * c * (size + stream) + 2 * _four(rows, c, case["block"]) + _four(case["out"], c, case["block"]) + rows * case["out"] * size
    return {"bytes": moved, "flops": 2 * rows * c * case["out"]}


# ---------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_dropout(case, state) if case["op"] == "dropout" else _exact_four(case, state)


def _nearest(t):
    """The nearest e2m1 value of each element, ties to the even code."""
    grid = torch.tensor(E2M1, device=t.device, dtype=torch.float64)
    size = torch.minimum(t.abs(), grid[-1])
    above = torch.bucketize(size, grid).clamp_(1, 7)  # grid[above - 1] < size <= grid[above]
    low, high = grid[above - 1], grid[above]
    middle = (low + high) / 2
    up = (size > middle) | ((size == middle) & (above % 2 == 0))
    return torch.copysign(torch.where(up, high, low), t)


def _exact_rows(t, block, scale):
    """What the quantised rows of t stand for."""
    pieces = []
    for part in t.split(block, dim=-1):
        most = part.abs().amax(dim=-1, keepdim=True)
        if block == 16:
            step = (most / (6 * scale)).clamp(2.0 ** -9, 448.0).to(torch.float32).to(torch.float8_e4m3fn).double() * scale
        else:
            step = torch.ldexp(torch.ones_like(most), torch.frexp(most)[1] - 3)
            step = torch.where(most < 2.0 ** -125, 2.0 ** -127, step)
        pieces.append(_nearest(part / step) * step)
    return torch.cat(pieces, dim=-1)


def _exact_four(case, state):
    block, t, out = case["block"], state["x"].double(), []
    scale = 1.0 if state["scale"] is None else float(state["scale"])
    if case["op"] == "norm":
        if state["residual"] is not None:
            t = t + state["residual"].double()
            out.append(t)
        size = torch.linalg.vector_norm(t, dim=-1, keepdim=True) / math.sqrt(case["c"])
        t = t / torch.sqrt(size * size + EPS) * state["norm_weight"].double()
    t = _exact_rows(t, block, scale)
    if case["op"] == "pack":
        return t
    # the weight, value by value from its bytes
    packed, tiles = state["weight"][0].view(torch.uint8), state["weight"][1].view(torch.uint8).reshape(-1)
    row = torch.arange(case["out"], device="cuda").unsqueeze(1)
    at = torch.arange(case["c"], device="cuda").unsqueeze(0)
    code = torch.bitwise_right_shift(packed[:, at[0] // 2], (at % 2 * 4).to(torch.uint8)) & 15
    grid = torch.tensor(E2M1, device="cuda", dtype=torch.float64)
    weight = grid[(code & 7).int()] * (1.0 - 2.0 * (code >> 3).double())
    del code
    unit = at // block
    columns = state["weight"][1].shape[1]
    place = (torch.div(row, 128, rounding_mode="floor") * (columns // 4) + unit // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + unit % 4
    byte = tiles[place]
    del place
    if block == 16:
        weight *= byte.view(torch.float8_e4m3fn).double() * float(state["weight_scale"])
    else:
        weight *= byte.view(torch.float8_e8m0fnu).double()
    y = torch.einsum("rc,oc->ro", t, weight)
    if state["bias"] is not None:
        y = y + state["bias"].double()
    return (y, *out)


def _exact_dropout(case, state):
    x, r, ds = state["x"], state["residual"], state["ds"]
    seed = numpy.uint64((state["seed"] if isinstance(state["seed"], int) else int(state["seed"].item())) % 2 ** 64)
    n, u32 = x.numel(), numpy.uint32
    drawn = numpy.empty((-(-n // 4), 4), dtype=u32)
    for begin in range(0, len(drawn), 1 << 20):  # (pieces that stay in a cache)
        at = numpy.arange(begin, min(begin + (1 << 20), len(drawn)), dtype=numpy.uint64)
        a, b = at.astype(u32), (at >> numpy.uint64(32)).astype(u32)
        c, d = numpy.full_like(a, state["layer"] % 2 ** 32), numpy.full_like(a, state["layer"] >> 32)
        for step in range(10):
            k0 = u32((int(seed) + step * 0x9E3779B9) % 2 ** 32)
            k1 = u32(((int(seed) >> 32) + step * 0xBB67AE85) % 2 ** 32)
            left, right = a.astype(numpy.uint64) * numpy.uint64(0xD2511F53), c.astype(numpy.uint64) * numpy.uint64(0xCD9E8D57)
            a, b, c, d = ((right >> numpy.uint64(32)).astype(u32) ^ b ^ k0, right.astype(u32),
                          (left >> numpy.uint64(32)).astype(u32) ^ d ^ k1, left.astype(u32))
        drawn[begin:begin + len(at)] = numpy.stack([a, b, c, d], axis=1)
    # a word below p 2^32 drops its element
    factor = torch.from_numpy(drawn.reshape(-1)[:n] >= u32(int(case["p"] * 2 ** 32 + 0.5))).to(x.device).reshape(x.shape).double() / (1.0 - case["p"])
    s = x.detach().double() * factor
    dx = ds.double() * factor
    return (s, dx) if r is None else (s + r.detach().double(), dx, ds.double())
