"""The masks of dropout from their definition, on the CPU."""
import numpy
import torch


def philox(at, layer, seed):
    """Words of Philox 4x32-10, counter (at, layer), key seed, 64 bits each: shape (*at, 4)."""
    u32, u64, mask = numpy.uint32, numpy.uint64, 2 ** 32 - 1
    at = numpy.asarray(at, dtype=u64)
    c = [(at & u64(mask)).astype(u32), (at >> u64(32)).astype(u32), numpy.full(at.shape, layer & mask, u32), numpy.full(at.shape, layer >> 32 & mask, u32)]
    k = [seed & mask, seed >> 32 & mask]
    for _ in range(10):
        a, b = c[0].astype(u64) * u64(0xD2511F53), c[2].astype(u64) * u64(0xCD9E8D57)
        c = [(b >> u64(32)).astype(u32) ^ c[1] ^ u32(k[0]), (b & u64(mask)).astype(u32), (a >> u64(32)).astype(u32) ^ c[3] ^ u32(k[1]), (a & u64(mask)).astype(u32)]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return numpy.stack(c, axis=-1)


def kept(n, p, seed, layer=0, begin=0, device="cpu"):
    """Whether elements begin .. begin + n (begin a multiple of 4) are kept."""
    words = philox(numpy.arange(begin // 4, (begin + n + 3) // 4), layer % 2 ** 64, seed % 2 ** 64).reshape(-1)[:n]
    return torch.from_numpy(words.astype(numpy.int64) >= round(p * 2 ** 32)).to(device)
