"""The block cache's operators in 64 bits and plain loops: block tables and slots from request lengths, e4m3 codes under a
power-of-two scale per block and head, the layout of a block, and attention over the values that the codes stand for."""

from __future__ import annotations

import math

import torch

MIN_EXP, MAX_EXP = -100, 119


def reserve(table, lengths, counts, free, free_count, rows, block):
    """(table, dict) of host lists: what ``kv_cache.reserve`` writes."""
    table = [list(r) for r in table]
    n, width = len(lengths), len(table[0]) if table else 0
    out = {"q_cu": [0] * (n + 1), "lengths": list(lengths), "slots": [-1] * rows, "positions": [0] * rows, "writes": [],
           "free_left": free_count, "status": 0}
    if (any(x < 0 for x in lengths) or any(x < 0 for x in counts) or sum(counts) > rows
            or any(a + b > width * block for a, b in zip(lengths, counts)) or not 0 <= free_count <= len(free)):
        return table, {**out, "status": 11}
    if sum(-(-(a + b) // block) - -(-a // block) for a, b in zip(lengths, counts)) > free_count:
        return table, {**out, "status": 10}
    row = 0
    for i in range(n):
        for p in range(lengths[i], lengths[i] + counts[i]):
            if p % block == 0:
                free_count -= 1
                table[i][p // block] = free[free_count]
            if p % block == 0 or p == lengths[i]:
                out["writes"].append([table[i][p // block], p % block, row, 0])
            out["writes"][-1][3] += 1
            out["slots"][row] = table[i][p // block] * block + p % block
            out["positions"][row] = p
            row += 1
        out["q_cu"][i + 1] = row
        out["lengths"][i] = lengths[i] + counts[i]
    out["free_left"] = free_count
    return table, out


def key_offset(t: int, d: int, head_dim: int) -> int:
    """Byte of token t's element d in a block's keys of one head."""
    return ((t // 16) * (head_dim // 64) + d // 64) * 1024 + (t % 16) * 64 + d % 64


def value_offset(t: int, d: int, head_dim: int) -> int:
    return ((t // 32) * 32 * head_dim + (d // 32) * 1024 + (d % 16) * 64 + (t // 4 % 4) * 16 + (d // 16 % 2) * 8
            + (t // 16 % 2) * 4 + t % 4)


def offsets(block: int, head_dim: int, value: bool) -> torch.Tensor:
    """(block * head_dim) int64: the byte of token t's element d at t * head_dim + d."""
    at = value_offset if value else key_offset
    return torch.tensor([at(t, d, head_dim) for t in range(block) for d in range(head_dim)])


def e4m3_values() -> torch.Tensor:
    """(256) float64: the value of each code (sign, four exponent bits with bias 7, three mantissa bits; no infinities)."""
    out = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(-v if c & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def rounded(x: torch.Tensor) -> torch.Tensor:
    """float64 to the nearest e4m3 value, ties to even, past the range (infinities too) at its end, NaN as NaN."""
    _, power = torch.frexp(torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(x), power - 4)
    y = torch.where(torch.isfinite(x), torch.round(x / step) * step, x)
    return torch.where(torch.isnan(y), y, y.clamp(-448.0, 448.0))


def exponent(largest: float) -> int:
    e = MIN_EXP
    while e < MAX_EXP and largest > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """Codes as the float64 values they stand for, (blocks, heads, block, D), and exponents (blocks, heads, 2)."""

    def __init__(self, keys, values, scales, block):
        blocks, heads, n = keys.shape
        self.block, self.d = block, n // block
        table = e4m3_values()
        self.codes = []
        for side, flat in enumerate((keys, values)):
            rows = flat.cpu().view(torch.uint8)[:, :, offsets(block, self.d, bool(side))]
            self.codes.append(table[rows.long()].view(blocks, heads, block, self.d))
        self.exps = ((scales.cpu().view(torch.int32) >> 23) & 255) - 127

    def append(self, key, value, writes):
        for ident, first, row, count in writes:
            for side, new in enumerate((key, value)):
                codes = self.codes[side]
                for h in range(codes.shape[1]):
                    x = new[row:row + count, h].cpu().double()
                    fine = x[torch.isfinite(x)].abs()
                    e = exponent(float(fine.max()) if fine.numel() else 0.0)
                    if first > 0:
                        old = min(max(int(self.exps[ident, h, side]), MIN_EXP), MAX_EXP)
                        e = max(e, old)
                        codes[ident, h, :first] = rounded(codes[ident, h, :first] * 2.0 ** (old - e))
                    codes[ident, h, first:first + count] = rounded(x * 2.0 ** -e)
                    self.exps[ident, h, side] = e

    def rows(self, table_row, start, end):
        """Keys and values (end - start, heads, D) float64 of a request's tokens; of an unknown block zeros."""
        out = []
        for side, codes in enumerate(self.codes):
            full = codes * torch.ldexp(torch.ones((), dtype=torch.float64), self.exps[..., side])[..., None, None]
            got = [full[table_row[p // self.block], :, p % self.block]
                   if 0 <= table_row[p // self.block] < full.shape[0] else torch.zeros_like(full[0, :, 0])
                   for p in range(start, end)]
            out.append(torch.stack(got) if got else full.new_zeros((0, *full[0, :, 0].shape)))
        return out

    def attend(self, query, table, q_cu, lengths, scale, causal=True, window=-1):
        query = query.cpu().double()
        out = torch.zeros_like(query)
        for i, length in enumerate(lengths):
            qa, qb = q_cu[i], q_cu[i + 1]
            if qb <= qa or length <= 0:
                continue
            key, value = self.rows(table[i], 0, length)
            out[qa:qb] = attention(query[qa:qb], key, value, scale, causal, window)
        return out


def attention(query, key, value, scale, causal, window):
    """Softmax attention of (Lq, heads, D) over (Lk, kv heads, D), the last query at the last key; each row over the keys
    that it sees and no others (what is hidden may be NaN), zeros for a row that sees none."""
    group = query.shape[1] // key.shape[1]
    out = torch.zeros_like(query)
    for i in range(query.shape[0]):
        at = i + key.shape[0] - query.shape[0]
        last = at if causal else key.shape[0] - 1
        first = max(0, at - window) if window >= 0 else 0
        if last < first:
            continue
        k, v = key[first:last + 1], value[first:last + 1]
        q = query[i].view(key.shape[1], group, -1)
        s = torch.einsum("hgd,khd->hgk", q, k) * scale
        out[i] = torch.einsum("hgk,khd->hgd", torch.softmax(s, -1), v).reshape(query.shape[1:])
    return out


def attention_whole(query, key, value, scale, causal, window):
    """``attention`` of long runs at once, by a mask (no NaN among the keys and values)."""
    lq, heads, d = query.shape
    lk, kv_heads = key.shape[:2]
    if lk == 0:
        return torch.zeros_like(query)
    q = query.view(lq, kv_heads, -1, d).permute(1, 2, 0, 3).reshape(kv_heads, -1, d)
    s = torch.matmul(q, key.permute(1, 2, 0).contiguous()) * scale
    at = torch.arange(lq, device=query.device)[:, None] + lk - lq
    j = torch.arange(lk, device=query.device)[None, :]
    seen = (j <= at) if causal else torch.ones((lq, lk), dtype=torch.bool, device=query.device)
    if window >= 0:
        seen = seen & (j >= at - window)
    s.view(kv_heads, -1, lq, lk).masked_fill_(~seen, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)  # (a row that sees nothing)
    o = torch.matmul(p, value.transpose(0, 1).contiguous())
    return o.view(kv_heads, -1, lq, d).permute(2, 0, 1, 3).reshape(lq, heads, d)
