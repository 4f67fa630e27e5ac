"""The block cache in 4 bits in 64 bits and plain loops: e2m1 codes under a power of two for each 32 elements of a token's head,
the layout of a block, and what append does to rows on the way (norms, rotation)."""

from __future__ import annotations

import math

import torch

from . import cache as cache8
from . import prologue

MIN_EXP, MAX_EXP = -100, 125
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def key_offset(t: int, d: int, head_dim: int) -> int:
    """Byte of token t's element d in a block's keys of one head (an even element in its lower half)."""
    return (t // 32) * 16 * head_dim + ((t // 16 % 2) * (head_dim // 32) + d // 32) * 256 + (t % 16) * 16 + d % 32 // 2


def value_offset(t: int, d: int, head_dim: int) -> int:
    return ((t // 32) * 16 * head_dim + ((d // 64) * 64 + (t // 4 % 4) * 16 + d // 2 % 16) * 16 + (d // 32 % 2) * 8
            + (t // 16 % 2) * 4 + t % 4)


def scale_offset(t: int, d: int, head_dim: int, value: bool) -> int:
    """Byte of the scale of token t's element d in a block's scales of one head."""
    at = (t // 32) * 2 * head_dim
    if value:
        return at + head_dim + (d // 32) * 32 + (t // 4 % 4) * 8 + (t // 16 % 2) * 4 + t % 4
    if head_dim == 64:
        return at + ((t // 16 % 2) * 2 + d // 32) * 16 + t % 16
    return at + ((d // 32 % 4) * 16 + t % 16) * (head_dim // 64) + (d // 128) * 2 + t // 16 % 2


def offsets(block: int, head_dim: int, value: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(block, head_dim) int64 bytes of the elements, and of their scales."""
    at = value_offset if value else key_offset
    return (torch.tensor([[at(t, d, head_dim) for d in range(head_dim)] for t in range(block)]),
            torch.tensor([[scale_offset(t, d, head_dim, value) for d in range(head_dim)] for t in range(block)]))


def exponent(largest: float) -> int:
    e = MIN_EXP
    while e < MAX_EXP and largest > 6.0 * 2.0 ** e:
        e += 1
    return e


def rounded(x: float) -> float:
    """To the nearest e2m1 value, of two equally near to the one at an even place; past the range to its end."""
    a = min(abs(x), 6.0)
    best = min(range(8), key=lambda i: (abs(GRID[i] - a), i % 2))
    return math.copysign(GRID[best], x)


def quantised(x: torch.Tensor) -> torch.Tensor:
    """(..., D) float64 as the cache holds it."""
    groups = x.reshape(-1, 32)
    out = torch.empty_like(groups)
    for i, g in enumerate(groups.tolist()):
        if any(math.isnan(v) for v in g):
            out[i] = math.nan
            continue
        e = exponent(max((abs(v) for v in g if math.isfinite(v)), default=0.0))
        out[i] = torch.tensor([rounded(v * 2.0 ** -e) * 2.0 ** e for v in g], dtype=torch.float64)
    return out.reshape(x.shape)


class Cache:
    """The elements as the float64 values that they stand for: ``values[side]`` (blocks, heads, block, D)."""

    def __init__(self, keys, values, scales, block):
        blocks, heads, n = keys.shape
        self.block, self.d = block, 2 * n // block
        grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64)
        flat_scales = scales.cpu().view(torch.uint8).reshape(blocks, heads, -1)
        self.values = []
        for side, flat in enumerate((keys, values)):
            raw = flat.cpu().view(torch.uint8)
            at, scale_at = offsets(block, self.d, bool(side))
            byte = raw[:, :, at.reshape(-1)].view(blocks, heads, block, self.d)
            odd = torch.arange(self.d) % 2 == 1
            code = torch.where(odd, byte >> 4, byte & 15)
            e = flat_scales[:, :, scale_at.reshape(-1)].view(blocks, heads, block, self.d).double()
            factor = torch.where(e == 255, torch.full_like(e, math.nan), torch.exp2(e - 127))
            self.values.append(grid[code.long()] * factor)

    def append(self, key, value, writes):
        for ident, first, row, count in writes:
            for side, new in enumerate((key, value)):
                self.values[side][ident, :, first:first + count] = quantised(new[row:row + count].cpu().double()).transpose(0, 1)

    def rows(self, table_row, start, end):
        """Keys and values (end - start, heads, D) float64 of a request's tokens; of an unknown block zeros."""
        out = []
        for full in self.values:
            got = [full[table_row[p // self.block], :, p % self.block]
                   if 0 <= table_row[p // self.block] < full.shape[0] else torch.zeros_like(full[0, :, 0])
                   for p in range(start, end)]
            out.append(torch.stack(got) if got else full.new_zeros((0, *full[0, :, 0].shape)))
        return out


attention, attention_whole = cache8.attention, cache8.attention_whole


def normed(x: torch.Tensor, norm) -> torch.Tensor:
    """float64 rows under ``norm`` (mode, weight, eps), or as they are."""
    x = x.cpu().double()
    if norm is None:
        return x
    mode, weight, eps = norm
    x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if mode == prologue.WEIGHT:
        return x * weight.cpu().double()
    return x * (1.0 + weight.cpu().double()) if mode == prologue.ONE_PLUS else x


def turned(x: torch.Tensor, rope, positions) -> tuple[torch.Tensor, torch.Tensor]:
    """(rows turned by halves, the sum of the magnitudes of what is added up in each element)."""
    if rope is None:
        return x, x.abs()
    cos, sin = (t.cpu().double() for t in rope)
    r, n = cos.shape[1], cos.shape[0]
    at = torch.arange(x.shape[0]) if positions is None else positions.cpu().long()
    known = (at >= 0) & (at < n)
    c, s = (torch.where(known[:, None], t[at.clamp(0, n - 1)], torch.full((), math.nan, dtype=torch.float64))[:, None]
            for t in (cos, sin))
    rot, rest = x[..., :r], x[..., r:]
    other = torch.cat((-rot[..., r // 2:], rot[..., :r // 2]), -1)
    return (torch.cat((rot * c + other * s, rest), -1),
            torch.cat(((rot * c).abs() + (other * s).abs(), rest.abs()), -1))
