"""The operators around the attention and feed-forward blocks of transformers over image, video and text tokens, as
measurable cases: the root-mean-square norm with the residual's addition (inference and training), the same with its
output in 8 bits and scales, and rotary positions with several axes on queries and keys, with or without the norm of
each head in front.

`run` computes them in their plain form, elementary torch operations in 32 bits, rounded once at the end, or, where `own`
is true, by the package's operators.  `exact` gives the same from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
E4M3_MOST = 448.0
TINY = 2.0 ** -126  # the smallest scale
EPS = 1e-6

_package = None


def _ops():
    global _package
    if _package is None:
        import channels_last_groupnorm_b200 as _package
    return _package


def _norm(op, mode, rows, c, dtype, residual="same", weight="same", block=0):
    """residual: "none", "same" (the type of x) or "float32"; weight: "same" or "float32"; block: columns that share a
    scale, 0 for one scale a row."""
    return {"op": op, "mode": mode, "rows": rows, "c": c, "dtype": dtype, "residual": residual, "weight": weight, "block": block}


def _rotary(mode, b, s, hq, hk, d, sections, dtype, scheme="axial", base=10000.0, interleaved=False, norm=False, packed=False, grid=""):
    """sections: rotary pairs of each axis; scheme: "axial" (every axis has the whole range of frequencies) or "shared"
    (the axes divide one range); packed: q and k are slices of one projection's output; grid: frames x height x width
    of the tokens, "" for a stream of tokens that begins at some position."""
    return {"op": "rotary", "mode": mode, "b": b, "s": s, "hq": hq, "hk": hk, "d": d, "sections": sections, "dtype": dtype, "scheme": scheme,
            "base": base, "interleaved": interleaved, "norm": norm, "packed": packed, "grid": grid}


def listed():
    return [
        # One token being answered: the smallest call there is, latency and launches.
        dict(_norm("norm", "infer", 1, 4096, "bfloat16"), name="norm_decode_1x4096"),
        # Two images' 64 x 64 tokens at a U-Net's second width, half precision.
        dict(_norm("norm", "infer", 8192, 640, "float16"), name="norm_image_8192x640"),
        # A training step's batch of tokens in bf16 with fp32 master weights: forward, then the gradients of x,
        # residual and weight.
        dict(_norm("norm", "train", 16384, 4096, "bfloat16", weight="float32"), name="norm_train_16384x4096"),
        # fp32 training at odd sizes, no residual: rows that do not start on vector boundaries.
        dict(_norm("norm", "train", 2077, 1111, "float32", residual="none"), name="norm_train_odd_2077x1111"),
        # Eight sequences answered at once, in front of an 8-bit projection with one scale a token.
        dict(_norm("quant", "infer", 8, 5120, "bfloat16"), name="quant_decode_8x5120"),
        # A prompt in front of an 8-bit projection with a scale for every 128 columns.
        dict(_norm("quant", "infer", 2048, 4096, "bfloat16", block=128), name="quant_prompt_2048x4096_b128"),
        # Many prompts at a wide model, residual stream in fp32.
        dict(_norm("quant", "infer", 8192, 8192, "bfloat16", residual="float32"), name="quant_prompts_8192x8192"),
        # Half precision, no residual, a last block of columns that is not whole.
        dict(_norm("quant", "infer", 777, 1352, "float16", residual="none", block=128), name="quant_ragged_777x1352_b128"),
        # One token of text in a model that divides its frequencies over time, height and width; shared key heads.
        dict(_rotary("infer", 1, 1, 32, 8, 128, "16,24,24", "bfloat16", scheme="shared", base=1e6, packed=True), name="rotary_decode_1x32x8x128"),
        # Two images' tokens, queries and keys sliced out of one projection, the norm of each head in front.
        dict(_rotary("infer", 2, 4096, 20, 20, 64, "16,16", "float16", norm=True, packed=True, grid="1x64x64"), name="rotary_image_2x4096x20x64"),
        # A video's tokens in training: forward, then the gradients of q, k and both norm weights.
        dict(_rotary("train", 1, 16384, 32, 32, 128, "16,24,24", "bfloat16", interleaved=True, norm=True, grid="16x32x32"), name="rotary_video_train_16384x32x128"),
        # fp32 training with shared key heads, a length of no particular kind and a head that is rotated in part.
        dict(_rotary("train", 3, 631, 16, 4, 80, "12,12,12", "float32"), name="rotary_odd_train_3x631x16x80"),
    ]


#: bytes of the largest drawn case, a third of the largest listed one's
MOST_BYTES = 4.5e8


def _between(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]; 3071 in the place of the one after it."""
    n = min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))
    return 3071 if n == 3072 else n


def _drawn(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    op = rng.choice(["norm", "norm", "quant", "rotary", "rotary"])
    if op != "rotary":
        c = rng.choice([320, 640, 1280, 2048, 2560, 4096, 5120, 8192]) if rng.random() < 0.5 else _between(rng, 64, 16384)
        if rng.random() < 0.5 and c > 64:
            c += 8 - c % 8
        if c == 3072:
            c = 3080
        rows = 1 if rng.random() < 0.1 else _between(rng, 1, 32768)
        residual = rng.choice(["none", "same", "same", "float32"])
        if op == "quant":
            return _norm(op, "infer", rows, c, dtype, residual, rng.choice(["same", "float32"]), rng.choice([0, 0, 32, 64, 128, 128]))
        return _norm(op, rng.choice(["infer", "train"]), rows, c, dtype, residual, rng.choice(["same", "float32"]))
    d = rng.choice([40, 64, 64, 72, 80, 96, 128, 128, 128, 256])
    axes = rng.choice([1, 2, 3, 3])
    half = d // 2 if rng.random() < 0.75 else d // 2 - 4
    parts = [half // axes] * axes
    parts[0] += half - sum(parts)
    hk = rng.choice([1, 2, 4, 8, 12, 16, 20, 32])
    hq = hk * rng.choice([1, 1, 2, 4])
    if hq * d == 3072 or hk * d == 3072:
        hq, hk = 16, 4
    b, grid = rng.choice([1, 1, 2, 3, 16]), ""
    if axes > 1 and rng.random() < 0.6:
        t = 1 if axes == 2 else _between(rng, 1, 16)
        h, w = _between(rng, 4, 64), _between(rng, 4, 64)
        s, grid = t * h * w, "%dx%dx%d" % (t, h, w)
        if s == 3072:
            return _drawn(rng)
    else:
        s = 1 if rng.random() < 0.25 else _between(rng, 1, 16384)
    norm = rng.random() < 0.5
    return _rotary(rng.choice(["infer", "train"]), b, s, hq, hk, d, ",".join(str(p) for p in parts), dtype, rng.choice(["axial", "shared"]),
                   rng.choice([1e4, 1e6]), rng.random() < 0.5, norm, rng.random() < 0.5, grid)


def draw(rng):
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= MOST_BYTES:
            return case


# ---------------------------------------------------------------------------------------------- inputs


def _sections(case):
    return tuple(int(p) for p in case["sections"].split(","))


def _inv_freq(case, dev):
    """Inverse frequencies of the rotary pairs, in 32 bits."""
    parts = _sections(case)
    if case["scheme"] == "axial":
        exponents = torch.cat([torch.arange(p, device=dev, dtype=torch.float64) / p for p in parts])
    else:
        exponents = torch.arange(sum(parts), device=dev, dtype=torch.float64) / sum(parts)
    return torch.pow(torch.tensor(case["base"], device=dev, dtype=torch.float64), -exponents).float()


def _positions(case, gen, dev):
    b, s, axes = case["b"], case["s"], len(_sections(case))
    if case["grid"]:
        t, h, w = (int(n) for n in case["grid"].split("x"))
        at = torch.arange(s, device=dev)
        place = torch.stack([at // (h * w), at // w % h, at % w], dim=-1)[:, 3 - axes:]
        return place.expand(b, s, axes).contiguous()
    # A stream of tokens: all axes alike.  Short in fp32, where the angles of a long one are off by more than the type's
    # rounding already in the product of position and frequency.
    start = torch.randint(0, 40 if case["dtype"] == "float32" else 4096, (b, 1, 1), device=dev, generator=gen)
    at = torch.arange(s, device=dev)
    if case["dtype"] == "float32":
        at = at % 64
    return (start + at.reshape(1, s, 1)).expand(b, s, axes).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, scale, dt=dtype):
        return torch.randn(shape, device=dev, generator=gen, dtype=dt).mul_(scale)

    state = {"case": case}
    train = case["mode"] == "train"
    if case["op"] != "rotary":
        shape, r = (case["rows"], case["c"]), case["residual"]
        state["x"] = normal(shape, 1.0)
        # the residual stream carries some channels that are much larger than the others
        state["residual"] = None
        if r != "none":
            state["residual"] = normal(shape, 2.0, torch.float32 if r == "float32" else dtype)
            state["residual"][:, :: max(1, case["c"] // 5)] *= 8
        wt = torch.float32 if case["weight"] == "float32" else dtype
        state["weight"] = torch.rand(case["c"], device=dev, generator=gen).add_(0.5).to(wt)
        if train:
            state["dy"] = normal(shape, 0.1)
            state["ds"] = None if r == "none" else normal(shape, 0.1, state["residual"].dtype)
            for name in ("x", "residual", "weight"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    b, s, hq, hk, d = (case[n] for n in ("b", "s", "hq", "hk", "d"))
    if case["packed"]:
        both = normal((b, s, hq + 2 * hk, d), 1.5)
        state["q"], state["k"] = both[:, :, :hq].detach(), both[:, :, hq:hq + hk].detach()
    else:
        state["q"], state["k"] = normal((b, s, hq, d), 1.5), normal((b, s, hk, d), 1.5)
    state["q_weight"] = state["k_weight"] = None
    if case["norm"]:
        state["q_weight"] = torch.rand(d, device=dev, generator=gen).add_(0.5).to(dtype)
        state["k_weight"] = torch.rand(d, device=dev, generator=gen).add_(0.5).to(dtype)
    state["positions"], state["inv_freq"], state["sections"] = _positions(case, gen, dev), _inv_freq(case, dev), _sections(case)
    if train:
        state["dq"], state["dk"] = normal((b, s, hq, d), 0.1), normal((b, s, hk, d), 0.1)
        for name in ("q", "k", "q_weight", "k_weight"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------------------------- one pass


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_rotary(state) if state["case"]["op"] == "rotary" else _plain_norm(state)


def _run_own(state):
    ops, case = _ops(), state["case"]
    if case["op"] == "rotary":
        q, k, qw, kw = state["q"], state["k"], state["q_weight"], state["k_weight"]
        args = (q, k, state["positions"], state["inv_freq"], state["sections"], qw, kw, EPS, case["interleaved"])
        if case["mode"] == "infer":
            with torch.no_grad():
                return ops.rotary(*args)
        out = ops.rotary(*args)
        wanted = (q, k) if qw is None else (q, k, qw, kw)
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, wanted, (state["dq"], state["dk"]))
    x, r, w = state["x"], state["residual"], state["weight"]
    if case["op"] == "quant":
        with torch.no_grad():
            return ops.rms_norm_quant(x, w, r, EPS, block=case["block"])
    if case["mode"] == "infer":
        with torch.no_grad():
            return ops.rms_norm(x, w, r, EPS)
    if r is None:
        y = ops.rms_norm(x, w, None, EPS)
        return (y.detach(),) + torch.autograd.grad(y, (x, w), state["dy"])
    y, s = ops.rms_norm(x, w, r, EPS)
    return (y.detach(), s.detach()) + torch.autograd.grad((y, s), (x, r, w), (state["dy"], state["ds"]))


def _plain_norm(state):
    case, x, r, w = state["case"], state["x"], state["residual"], state["weight"].float()
    s = x.float() if r is None else x.float() + r.float()
    rstd = (s.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    n = s * rstd
    y = n * w
    stream = () if r is None else (s.to(r.dtype),)
    if case["op"] == "quant":
        rows, c, block = case["rows"], case["c"], case["block"] or case["c"]
        blocks = -(-c // block)
        whole = torch.nn.functional.pad(y, (0, blocks * block - c)).reshape(rows, blocks, block)
        scale = (whole.abs().amax(dim=-1) / E4M3_MOST).clamp_min(TINY)
        q = (whole / scale.unsqueeze(-1)).clamp(-E4M3_MOST, E4M3_MOST).reshape(rows, blocks * block)[:, :c]
        return (q.to(torch.float8_e4m3fn), scale) + stream
    if case["mode"] == "infer":
        return (y.to(x.dtype),) + stream if stream else y.to(x.dtype)
    dy = state["dy"].float()
    g = dy * w
    d = rstd * (g - n * (g * n).mean(dim=-1, keepdim=True))
    if r is not None:
        d = d + state["ds"].float()
    grads = (d.to(x.dtype),) if r is None else (d.to(x.dtype), d.to(r.dtype))
    return (y.to(x.dtype),) + stream + grads + ((dy * n).sum(dim=0).to(state["weight"].dtype),)


def _split(t, n, interleaved):
    """(first, second) of the rotary pairs in the leading 2n columns, and the columns that are left."""
    if interleaved:
        return t[..., 0:2 * n:2], t[..., 1:2 * n:2], t[..., 2 * n:]
    return t[..., :n], t[..., n:2 * n], t[..., 2 * n:]


def _joined(a, b, rest, interleaved):
    if interleaved:
        return torch.cat([torch.stack([a, b], dim=-1).flatten(-2), rest], dim=-1)
    return torch.cat([a, b, rest], dim=-1)


def _turned(t, cos, sin, interleaved):
    a, b, rest = _split(t, cos.shape[-1], interleaved)
    return _joined(a * cos - b * sin, b * cos + a * sin, rest, interleaved)


def _plain_rotary(state):
    case, inter = state["case"], state["case"]["interleaved"]
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"), torch.tensor(state["sections"], device="cuda"), output_size=sum(state["sections"]))
    angle = (state["positions"].float()[..., axis] * state["inv_freq"]).unsqueeze(2)
    cos, sin = angle.cos(), angle.sin()

    def forward(t, weight):
        t = t.float()
        if weight is None:
            return None, None, _turned(t, cos, sin, inter)
        rstd = (t.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
        n = t * rstd
        return rstd, n, _turned(n * weight.float(), cos, sin, inter)

    def backward(dout, rstd, n, weight):
        g = _turned(dout.float(), cos, -sin, inter)
        if weight is None:
            return g, None
        gw = g * weight.float()
        return rstd * (gw - n * (gw * n).mean(dim=-1, keepdim=True)), (g * n).sum(dim=(0, 1, 2)).to(weight.dtype)

    q, k, qw, kw = state["q"], state["k"], state["q_weight"], state["k_weight"]
    rq, nq, oq = forward(q, qw)
    rk, nk, ok = forward(k, kw)
    outs = (oq.to(q.dtype), ok.to(k.dtype))
    if case["mode"] == "infer":
        return outs
    dq, dqw = backward(state["dq"], rq, nq, qw)
    dk, dkw = backward(state["dk"], rk, nk, kw)
    return outs + (dq.to(q.dtype), dk.to(k.dtype)) + (() if qw is None else (dqw, dkw))


# ---------------------------------------------------------------------------------------------- what it takes


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        b, s, hq, hk, d = (case[n] for n in ("b", "s", "hq", "hk", "d"))
        elements = b * s * (hq + hk) * d
        tables = b * s * len(_sections(case)) * 8 + sum(_sections(case)) * 4
        if case["mode"] == "infer":  # q and k in, out
            return {"bytes": 2 * elements * size + tables, "flops": elements * (8 if case["norm"] else 4)}
        # ... and the gradients in, out, and q and k once more where the norm's backward needs them
        return {"bytes": (5 if case["norm"] else 4) * elements * size + 2 * tables, "flops": elements * (22 if case["norm"] else 8)}
    elements = case["rows"] * case["c"]
    wide = 4 if case["residual"] == "float32" else size
    stream = 0 if case["residual"] == "none" else wide
    weight = case["c"] * (4 if case["weight"] == "float32" else size)
    if case["op"] == "quant":  # x and residual in; codes, scales and the residual stream out
        scales = case["rows"] * (-(-case["c"] // case["block"]) if case["block"] else 1) * 4
        return {"bytes": elements * (size + 1 + 2 * stream) + scales + weight, "flops": 7 * elements}
    forward = elements * (2 * size + 2 * stream) + weight
    if case["mode"] == "infer":
        return {"bytes": forward, "flops": 5 * elements}
    # ... and dy, the stream's gradient and the stream (x itself without one) in; the gradients of x and of the residual
    # (one tensor where their types are the same) and of the weight out
    if case["residual"] == "none":
        back = 3 * size
    else:
        back = size + 2 * stream + stream + (size if wide != size else 0)
    return {"bytes": forward + elements * back + 2 * weight, "flops": 16 * elements}


# ---------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_rotary(case, state) if case["op"] == "rotary" else _exact_norm(case, state)


def _rms64(t):
    """t over its root mean square, and the reciprocal of that, along the last axis."""
    size = torch.linalg.vector_norm(t, dim=-1, keepdim=True) / math.sqrt(t.shape[-1])
    inverse = 1.0 / torch.sqrt(size * size + EPS)
    return t * inverse, inverse


def _exact_norm(case, state):
    t = state["x"].double()
    if state["residual"] is not None:
        t += state["residual"].double()
    unit, inverse = _rms64(t)
    weight = state["weight"].double()
    out = [unit * weight]
    if case["op"] == "quant":
        width = case["block"] or case["c"]
        scales = torch.stack([p.abs().amax(dim=-1) for p in out[0].split(width, dim=-1)], dim=-1) / E4M3_MOST
        scales = torch.clamp(scales, min=TINY)
        out = [out[0] / scales.repeat_interleave(width, dim=-1)[:, :case["c"]], scales]
    if state["residual"] is not None:
        out.append(t)
    if case["mode"] == "train":
        dy = state["dy"].double()
        # y_i = w_i t_i / |t|: the gradient is inverse * (w dy) less its part along t
        through = dy * weight
        along = torch.einsum("rc,rc->r", through, unit).unsqueeze(-1) / case["c"]
        d = inverse * through - inverse * along * unit
        if state["residual"] is not None:
            d += state["ds"].double()
            out.append(d)
        out.append(d)
        out.append(torch.einsum("rc,rc->c", dy, unit))
    return out[0] if len(out) == 1 else tuple(out)


def _exact_rotary(case, state):
    parts, pairs = state["sections"], sum(state["sections"])
    where = state["positions"].double()
    columns = torch.cat([where[..., a:a + 1].expand(*where.shape[:-1], p) for a, p in enumerate(parts)], dim=-1)
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), columns * state["inv_freq"].double()).unsqueeze(2)
    if case["interleaved"]:
        first = torch.arange(pairs, device="cuda") * 2
        second = first + 1
    else:
        first = torch.arange(pairs, device="cuda")
        second = first + pairs

    def rotate(t, by):
        z = torch.complex(t[..., first], t[..., second]) * by
        t = t.clone()
        t[..., first], t[..., second] = z.real, z.imag
        return t

    def head(name):
        """The output, and in training the gradients of the tensor and of its norm weight."""
        t, weight = state[name].double(), state[name + "_weight"]
        unit, inverse = _rms64(t) if weight is not None else (t, None)
        out = rotate(unit * weight.double() if weight is not None else unit, turn)
        if case["mode"] == "infer":
            return (out,)
        back = rotate(state["d" + name].double(), turn.conj())
        if weight is None:
            return out, back
        through = back * weight.double()
        along = torch.einsum("bshd,bshd->bsh", through, unit).unsqueeze(-1) / case["d"]
        return out, inverse * (through - along * unit), torch.einsum("bshd,bshd->d", back, unit)

    # (outputs, then gradients, then those of the weights)
    return tuple(value for pair in zip(head("q"), head("k")) for value in pair)
