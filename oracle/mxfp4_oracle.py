"""CPU restatement of the MXFP4 operators in 64 bits, for the tests only.

Written from the format's definition: blocks of 32 share the power of two
``2^(floor(log2 amax) - 2)`` (at least 2^-127), values round to the nearest
E2M1 number with ties to the even code, saturating at 6; an infinity or a NaN
anywhere in a block gives it the NaN scale (byte 255) and zero codes.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP32_MAX = torch.finfo(torch.float32).max


def scale_bytes(amax: torch.Tensor) -> torch.Tensor:
    """E8M0 bytes (int64) of blocks with these fp64 largest magnitudes."""
    finite = amax <= FP32_MAX  # False for NaN
    _, e = torch.frexp(torch.where(finite, amax, torch.ones_like(amax)))  # amax = m 2^e, m in [0.5, 1)
    byte = (e.long() - 1 - 2 + 127).clamp(min=0)
    byte = torch.where(amax == 0, torch.zeros_like(byte), byte)
    return torch.where(finite, byte, torch.full_like(byte, 255))


def codes(t: torch.Tensor) -> torch.Tensor:
    """E2M1 codes (int64) of fp64 values already divided by their scale."""
    a = t.abs()
    best = torch.zeros_like(a, dtype=torch.long)
    for c in range(1, 8):
        border = (GRID[c - 1] + GRID[c]) / 2
        best = torch.where((a > border) | ((a == border) & (c % 2 == 0)), torch.full_like(best, c), best)
    return best + 8 * (torch.signbit(t)).long()


def quant(y: torch.Tensor, byte: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes [M, K], scale bytes [M, K/32])``, both int64, of fp64 ``y``."""
    m, k = y.shape
    b = y.double().reshape(m, k // 32, 32)
    mag = b.abs()
    amax = torch.where(mag.isnan().any(-1), torch.full((), math.nan, dtype=torch.float64), mag.amax(-1))
    byte = scale_bytes(amax) if byte is None else byte
    t = b * torch.exp2((127 - byte).double())[..., None]
    c = codes(t)
    c = torch.where((byte == 255)[..., None], torch.zeros_like(c), c)
    return c.reshape(m, k), byte


def pack(c: torch.Tensor) -> torch.Tensor:
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)


def unpack(data: torch.Tensor) -> torch.Tensor:
    d = data.cpu().long()
    return torch.stack([d & 15, d >> 4], dim=-1).reshape(d.shape[0], -1)


def tile(byte: torch.Tensor) -> torch.Tensor:
    """Scale bytes [R, C] to tiles, one byte at a time (the layout's words)."""
    r, c = byte.shape
    out = torch.zeros((r + 127) // 128, 2 * ((c + 7) // 8), 512, dtype=torch.uint8)
    rows = torch.arange(r)[:, None].expand(r, c)
    blk = torch.arange(c)[None, :].expand(r, c)
    out[rows // 128, blk // 4, rows % 32 * 16 + rows % 128 // 32 * 4 + blk % 4] = byte.to(torch.uint8)
    return out


def untile(tiles: torch.Tensor, r: int, c: int) -> torch.Tensor:
    t = tiles.cpu().long()
    rows = torch.arange(r)[:, None].expand(r, c)
    blk = torch.arange(c)[None, :].expand(r, c)
    return t[rows // 128, blk // 4, rows % 32 * 16 + rows % 128 // 32 * 4 + blk % 4]


def values(c: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """fp64 values of codes and scale bytes."""
    m, k = c.shape
    v = torch.tensor(GRID, dtype=torch.float64)[c & 7] * (1 - 2 * (c >> 3)).double()
    s = torch.exp2((byte - 127).double())
    s = torch.where(byte == 255, torch.full_like(s, math.nan), s)
    return (v.reshape(m, k // 32, 32) * s[..., None]).reshape(m, k)


def decode(data: torch.Tensor, tiles: torch.Tensor) -> torch.Tensor:
    c = unpack(data)
    return values(c, untile(tiles, c.shape[0], c.shape[1] // 32))


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None):
    """``(y fp64, new residual in x's type or None)``."""
    v = x.double() if residual is None else (x.float() + residual.float()).double()  # the fp32 sum
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * weight.double()
    res = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    return y, res
