"""A transformer block over the tokens of a video, trained for a few steps and then served.

Feature maps come out of a convolutional stage through `GN_NHWC` (group norm with SiLU, channels-last); their pixels are the
tokens of a block with `RMSNorm` in front of attention and feed-forward (each adding the residual stream as it goes), `AxialRotary` positions
in time, height and width with the norm of each head, and torch's attention.  With `dropout` both branches drop elements as they join the
residual stream (`dropout_add`).  For serving, the norms hand 8-bit codes and scales to 8-bit products, or 4-bit ones to `Linear4bit`.

    python examples/video_block.py [--frames 4] [--size 16] [--channels 256] [--heads 4] [--steps 20] [--dropout 0.1] [--bits 4]
"""
import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from channels_last_groupnorm_b200 import GN_NHWC, AxialRotary, DropoutAdd, Linear4bit, RMSNorm  # noqa: E402


class VideoBlock(nn.Module):
    """Maps (frames, channels, height, width), channels-last, to the same; attention over all pixels of all frames."""

    def __init__(self, channels, heads, device=None, dtype=None, dropout=0.0):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.heads, self.head_dim = heads, channels // heads
        third = self.head_dim // 2 // 3
        self.norm_in = GN_NHWC(32, channels, activation="silu", **kw)
        self.norm1 = RMSNorm(channels, **kw)
        self.qkv = nn.Linear(channels, 3 * channels, bias=False, **kw)
        self.rotary = AxialRotary(self.head_dim, (self.head_dim // 2 - 2 * third, third, third), qk_norm=True, **kw)
        self.out = nn.Linear(channels, channels, bias=False, **kw)
        self.norm2 = RMSNorm(channels, **kw)
        self.up = nn.Linear(channels, 4 * channels, bias=False, **kw)
        self.down = nn.Linear(4 * channels, channels, bias=False, **kw)
        self.drop1, self.drop2 = DropoutAdd(dropout, layer=0), DropoutAdd(dropout, layer=1)

    def positions(self, frames, height, width, device):
        grid = torch.meshgrid(*(torch.arange(n, device=device) for n in (frames, height, width)), indexing="ij")
        return torch.stack(grid, dim=-1).reshape(frames * height * width, 3)

    def attention(self, qkv, positions):
        tokens = qkv.shape[0]
        qkv = qkv.view(tokens, 3, self.heads, self.head_dim)
        q, k = self.rotary(qkv[:, 0], qkv[:, 1], positions)  # (slices of the projection, read in place)
        o = F.scaled_dot_product_attention(*(t.transpose(0, 1).unsqueeze(0) for t in (q, k, qkv[:, 2])))
        return o.squeeze(0).transpose(0, 1).reshape(tokens, -1)

    def tokens_of(self, maps):
        return self.norm_in(maps).permute(0, 2, 3, 1).reshape(-1, maps.shape[1])  # a view: the maps are channels-last

    def maps_of(self, tokens, like):
        frames, channels, height, width = like.shape
        return tokens.view(frames, height, width, channels).permute(0, 3, 1, 2)

    def forward(self, maps, seed=None):
        """seed: of the step's dropout, a number or a tensor of one int64 on the device; training with dropout needs it."""
        positions = self.positions(maps.shape[0], maps.shape[2], maps.shape[3], maps.device)
        stream = self.tokens_of(maps)
        attended = self.out(self.attention(self.qkv(self.norm1(stream)), positions))
        if self.training and self.drop1.p > 0:
            stream = self.drop1(attended, stream, seed)
            return self.maps_of(self.drop2(self.down(F.gelu(self.up(self.norm2(stream)))), stream, seed), maps)
        y, stream = self.norm2(attended, stream)
        return self.maps_of(stream + self.down(F.gelu(self.up(y))), maps)

    @torch.no_grad()
    def serve(self, maps, weights):
        """The same with the norms' outputs, and the projections behind them, in 8 bits; weights: from `quantised`."""
        positions = self.positions(maps.shape[0], maps.shape[2], maps.shape[3], maps.device)
        stream = self.tokens_of(maps)
        attended = self.out(self.attention(product(*self.norm1.quantize(stream), *weights["qkv"], maps.dtype), positions))
        codes, scales, stream = self.norm2.quantize(attended, stream)
        return self.maps_of(stream + self.down(F.gelu(product(codes, scales, *weights["up"], maps.dtype))), maps)

    @torch.no_grad()
    def serve_4bit(self, maps, weights):
        """The same in 4 bits, and the other two projections too; weights: of the four projections, as `Linear4bit`."""
        block = weights["qkv"].block
        positions = self.positions(maps.shape[0], maps.shape[2], maps.shape[3], maps.device)
        stream = self.tokens_of(maps)
        attended = weights["out"](self.attention(weights["qkv"](self.norm1.quantize_4bit(stream, block=block)), positions))
        codes, scales, stream = self.norm2.quantize_4bit(attended, stream, block=block)
        return self.maps_of(stream + weights["down"](F.gelu(weights["up"]((codes, scales)))), maps)


def quantised(weight):
    """A projection's weight in e4m3 with one scale for each output."""
    scale = weight.float().abs().amax(dim=1, keepdim=True) / 448
    return (weight.float() / scale).to(torch.float8_e4m3fn), scale


def product(codes, scales, weight, weight_scale, dtype):
    """(codes * scales) times the transposed (weight * weight_scale)"""
    return torch._scaled_mm(codes, weight.t(), scale_a=scales, scale_b=weight_scale.t(), out_dtype=dtype)


def main(frames=4, size=16, channels=256, heads=4, steps=20, dtype=torch.bfloat16, dropout=0.0, bits=8):
    """Trains towards a fixed target and serves; returns the first and the last loss and how far serving in 8 or 4 bits is off."""
    torch.manual_seed(0)
    block = VideoBlock(channels, heads, device="cuda", dtype=dtype, dropout=dropout)
    maps = torch.randn(frames, channels, size, size, device="cuda").to(dtype=dtype, memory_format=torch.channels_last)
    target = torch.roll(maps, (1, 2, 3), dims=(0, 2, 3)) * 0.5
    optimizer = torch.optim.AdamW(block.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        loss = F.mse_loss(block(maps, seed=step).float(), target.float())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    block.eval()
    with torch.no_grad():
        want = block(maps).float()
        if bits == 8:
            got = block.serve(maps, {"qkv": quantised(block.qkv.weight), "up": quantised(block.up.weight)}).float()
        else:
            got = block.serve_4bit(maps, {name: Linear4bit.from_linear(getattr(block, name)) for name in ("qkv", "out", "up", "down")}).float()
    return losses[0].item(), losses[-1].item(), ((got - want).norm() / want.norm()).item()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("frames", 4), ("size", 16), ("channels", 256), ("heads", 4), ("steps", 20)):
        parser.add_argument("--" + name, type=int, default=default)
    parser.add_argument("--dropout", type=float, default=0.0)
    parser.add_argument("--bits", type=int, default=8, choices=(8, 4))
    args = parser.parse_args()
    first, last, off = main(**vars(args))
    print("loss %.4f -> %.4f; served in %d bits: %.3f off" % (first, last, args.bits, off))
