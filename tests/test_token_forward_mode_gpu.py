"""Operators on token rows in forward mode: an error, never a result without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import channels_last_groupnorm_b200 as pkg

pytestmark = pytest.mark.gpu


CALLS = {
    "dropout of x": lambda d, e: pkg.dropout_add(d, e["x"], 0.2, 1),
    "dropout into d": lambda d, e: pkg.dropout_add(e["x"], d, 0.2, 1),
    "norm of x": lambda d, e: pkg.rms_norm(d, e["w"]),
    "norm over d": lambda d, e: pkg.rms_norm(e["x"], e["w"], d)[0],
    "norm with weight d": lambda d, e: pkg.rms_norm(e["x"], d[0]),
    "8 bits": lambda d, e: pkg.rms_norm_quant(d)[1],
    "4 bits": lambda d, e: pkg.quantize_4bit(d)[1].float(),
    "norm to 4 bits": lambda d, e: pkg.rms_norm_quant_4bit(e["x"], None, d)[2],
    "from 4 bits": lambda d, e: pkg.dequantize_4bit(*e["four"], scale=d[:1, 0]),
    "product": lambda d, e: pkg.linear_4bit(*e["four"], *e["four"], bias=d[0, :8]),
    "rotary of q": lambda d, e: pkg.rotary(d.view(1, 8, 1, 64), e["heads"], e["positions"], e["freq"], (32,))[0],
    "rotary of k": lambda d, e: pkg.rotary(e["heads"], d.view(1, 8, 1, 64), e["positions"], e["freq"], (32,))[1],
}


@pytest.mark.parametrize("name", list(CALLS))
def test_duals_are_refused(name):
    x, v = torch.randn(8, 64, device="cuda"), torch.randn(8, 64, device="cuda")
    e = {"x": x, "w": torch.rand(64, device="cuda"), "four": pkg.quantize_4bit(x), "heads": x.view(1, 8, 1, 64),
         "positions": torch.arange(8, device="cuda", dtype=torch.int32).view(1, 8, 1), "freq": torch.rand(32, device="cuda")}

    def call(d):
        return CALLS[name](d, e)

    for leaf in (x, x.clone().requires_grad_(True)):
        with torch.no_grad(), fw.dual_level(), pytest.raises(NotImplementedError):
            call(fw.make_dual(leaf, v))
    with fw.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        call(fw.make_dual(x, v))
    with pytest.raises(NotImplementedError, match="forward mode"):
        torch.func.jvp(call, (x,), (v,))
    with torch.no_grad(), fw.dual_level():  # (a level alone is no reason)
        call(x)


@pytest.mark.parametrize("op", ["dropout", "norm", "rotary"])
def test_dual_gradients_are_refused(op):
    """Forward over reverse."""
    x = torch.randn(1, 8, 2, 64, device="cuda").requires_grad_(True)
    if op == "dropout":
        out = pkg.dropout_add(x, None, 0.2, 1)
    elif op == "norm":
        out = pkg.rms_norm(x)
    else:
        out = pkg.rotary(x, None, torch.arange(8, device="cuda").view(1, 8, 1), torch.rand(32, device="cuda"), (32,))[0]
    with fw.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(out, x, fw.make_dual(torch.randn_like(x), torch.randn_like(x)))
