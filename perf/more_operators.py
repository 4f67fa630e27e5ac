"""Measured cases of what a layer does with its block cache beside plain 8-bit keys and values: appending with the norms and
the position rotation applied on the way, and a cache held in 4 bits with the attention that reads it.

``append``   the projections' keys and values into the 8-bit cache: norms, rotation, one power-of-two scale per block and head
``append4``  the same into the 4-bit cache (e2m1 codes, a power of two for each 32 elements of a token's head), and the blocks
             that got tokens read back as bf16
``read4``    the cached rows of a batch out of the 4-bit cache as packed bf16 keys and values
``attend4``  attention of new queries over the 4-bit cache: one token per request, a few, or a chunk of a prompt

Ranges that ``draw`` spreads over: 1 to 64 requests, 1 to 16,384 new tokens, cached lengths from 0 to 65,536 tokens, blocks of
32, 64 and 128 tokens, head sizes 64, 128, 256 and 512 with the head counts of this repository's workloads, whole and partial
rotations, both kinds of norm weight, keys and values of their own or out of one packed projection, with and without a window.

The 8-bit cache: ``keys`` and ``values`` (blocks, kv heads, block size * D) e4m3, ``scales`` (blocks, kv heads, 2) fp32.
The 4-bit cache: ``keys`` and ``values`` (blocks, kv heads, block size * D / 2) bytes of two e2m1 codes, ``scales`` (blocks,
kv heads, block size / 32, 2, D) e8m0: of each 32 tokens D bytes for the keys and D for the values. The orders are those in which
a lane of a matrix instruction takes them (``_key_order`` to ``_value_bytes``).
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

EPS = 1e-6
#: Exponents that a scale may have, of each format, and the format's largest value.
LIMITS = {8: (-100, 119, 448.0), 4: (-100, 125, 6.0)}


def _case(name, op, **more):
    base = {"name": name, "op": op, "requests": 1, "median": 0, "longest": 0, "new": 1, "block": 64, "heads": 32,
            "kv_heads": 16, "head_dim": 128, "window": -1, "rotated": 0, "one_plus": False, "value_norm": True,
            "packed": False, "pack": 0}
    base.update(more)
    return base


def listed():
    return [
        # the new token of each request of a batch into one global layer's 8-bit cache
        _case("append-step", "append", requests=48, median=900, longest=4096, new=48, rotated=128),
        # ragged prompt chunks that begin anywhere in a block; a layer that rotates a quarter of its head and norms no
        # values, out of a packed projection
        _case("append-chunks", "append", requests=24, median=700, longest=4096, new=2500, heads=16, kv_heads=8,
              head_dim=256, rotated=64, one_plus=True, value_norm=False, packed=True),
        # one long document into a global layer's cache
        _case("append-document", "append", new=32768, rotated=128),
        # the new token of each request into the 4-bit cache
        _case("append4-step", "append4", requests=48, median=900, longest=4096, new=48, rotated=128),
        # one long document into the 4-bit cache
        _case("append4-document", "append4", new=32768, rotated=128),
        # the cached prompts of a few requests, as rows (the 31B global layer)
        _case("read4-batch", "read4", requests=6, median=1500, longest=8192, heads=32, kv_heads=4, head_dim=512, block=32),
        # a long cached document, as rows
        _case("read4-document", "read4", median=32768, longest=32768),
        # a handful of short requests, one token each: launches count
        _case("decode4-short", "attend4", requests=4, median=250, longest=511, new=4, heads=8, kv_heads=2, head_dim=64,
              block=32),
        # a decoding step of a ragged batch
        _case("decode4-batch", "attend4", requests=48, median=900, longest=8192, new=48),
        # one long document, one token, the 31B global layer
        _case("decode4-document", "attend4", median=131072, longest=131072, new=1, heads=32, kv_heads=4, head_dim=512,
              block=128),
        # a few tokens per request to check at once, sliding layers
        _case("decode4-few-sliding", "attend4", requests=32, median=2500, longest=8192, new=128, heads=16, kv_heads=8,
              head_dim=256, window=1023),
        # a prompt chunk over what is cached of the prompt
        _case("chunk4-prefill", "attend4", median=30000, longest=30000, new=2048),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "append", "append4", "append4", "read4", "attend4", "attend4", "attend4", "attend4"])
    heads, kv_heads, head_dim, window = rng.choice([(8, 2, 64, -1), (16, 8, 128, -1), (32, 16, 128, -1),
                                                    (16, 8, 256, 1023), (16, 8, 256, 511), (32, 4, 512, -1)])
    more = {"block": rng.choice([32, 64, 128]), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "pack": rng.randrange(1 << 20)}
    if op in ("append", "append4"):
        requests = size(1, 64)
        new = requests if rng.random() < 0.4 else size(requests, 16384)
        more.update(rotated=rng.choice([head_dim, head_dim, head_dim // 2 if head_dim == 64 else head_dim // 4]),
                    one_plus=rng.random() < 0.5, value_norm=rng.random() < 0.7, packed=rng.random() < 0.5)
        case = _case("", op, requests=requests, median=size(30, 1000), longest=4096, new=new, **more)
    elif op == "read4":
        case = _case("", op, requests=size(1, 16), median=size(30, 1500), longest=2048, **more)
    else:
        kind = rng.choice(["step", "step", "few", "long", "chunk"])
        more["window"] = window
        if kind == "step":
            requests = size(1, 64)
            case = _case("", op, requests=requests, median=size(30, 1200), longest=4096, new=requests, **more)
        elif kind == "few":
            requests = size(1, 32)
            case = _case("", op, requests=requests, median=size(30, 2000), longest=4096,
                         new=requests * rng.randint(2, 8) + rng.randint(0, 3), **more)
        elif kind == "long":
            length = size(8192, 65536)
            case = _case("", op, requests=1, median=length, longest=length, new=rng.randint(1, 4), **more)
        else:
            length = size(1000, 16000)
            case = _case("", op, requests=rng.randint(1, 2), median=length, longest=length, new=size(64, 1024), **more)
    del case["name"]
    return case


# ---- layouts (from the case alone)

def _lengths(case):
    """(tokens held before the call, new tokens) of each request."""
    rng = np.random.default_rng(case["pack"] + 41)
    n = case["requests"]
    if n == 1:
        held = np.array([case["median"]], dtype=np.int64)
    else:
        held = np.exp(rng.normal(math.log(max(1, case["median"])), 1.0, size=n))
        held = np.clip(np.round(held), 0, case["longest"]).astype(np.int64)
        if n > 4:
            held[int(rng.integers(n))] = 0  # a request that begins
    if case["op"] == "read4":
        return held, np.zeros(n, dtype=np.int64)
    new = case["new"]
    if new <= n:
        return held, np.ones(n, dtype=np.int64)
    if case["op"] == "attend4":  # about the same for each
        counts = np.full(n, new // n, dtype=np.int64)
        counts[0] += new - int(counts.sum())
    else:
        share = np.exp(rng.normal(0, 1.0, size=n))
        counts = np.maximum(1, np.floor(share / share.sum() * (new - n))).astype(np.int64)
        counts[int(np.argmax(counts))] += new - int(counts.sum())
    return held, counts


def _blocks_of(tokens, block):
    return -(-tokens // block)


def _writes(case, held, counts, table):
    """(block, first slot, first row, tokens) of each block that gets tokens."""
    block, row, out = case["block"], 0, []
    for i in range(case["requests"]):
        at, end = int(held[i]), int(held[i] + counts[i])
        while at < end:
            n = min(block - at % block, end - at)
            out.append((int(table[i, at // block]), at % block, row, n))
            at, row = at + n, row + n
    return np.array(out, dtype=np.int64).reshape(-1, 4)


def _inputs(case, seed):
    """Seeded tensors of the case, the same for ``prepare`` and ``exact``."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    held, counts = _lengths(case)
    full = held + counts
    block, kv_heads, d, n = case["block"], case["kv_heads"], case["head_dim"], case["requests"]
    t = SimpleNamespace(case=case, block=block, bits=8 if case["op"] == "append" else 4)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    # the held blocks scattered over the pool, elsewhere for each seed
    blocks = _blocks_of(full, block)
    t.blocks = int(blocks.sum()) + 2
    order = torch.randperm(t.blocks, generator=gen, device="cuda").cpu().numpy()
    table, at = np.full((n, max(1, int(blocks.max())) + 2), -1, dtype=np.int64), 0
    for i, c in enumerate(blocks):
        table[i, :c] = order[at:at + c]
        at += int(c)
    t.table, t.lengths, t.rows, t.longest = i32(table), i32(full), int(full.sum()), int(full.max())

    def unit(*shape):
        x = torch.randn(shape, generator=gen, device="cuda")
        return x.mul_(torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)).bfloat16()  # what the layer's norm leaves

    t.old_keys = unit(t.blocks, kv_heads, block, d)
    t.old_values = torch.randn((t.blocks, kv_heads, block, d), generator=gen, device="cuda").bfloat16()
    if case["op"] in ("append", "append4"):
        rows = int(counts.sum())
        wide = 2 * kv_heads + (case["heads"] if case["packed"] else 0)
        # what the projections leave: heads of several sizes, and a few tokens much larger than the others
        x = torch.randn((rows, wide, d), generator=gen, device="cuda")
        x *= torch.exp2(torch.randint(-2, 3, (1, wide, 1), generator=gen, device="cuda").float())
        x *= torch.where(torch.rand((rows, 1, 1), generator=gen, device="cuda") < 0.1, 6.0, 1.0)
        x = x.bfloat16()
        first = wide - 2 * kv_heads
        t.key, t.value = x[:, first:first + kv_heads], x[:, first + kv_heads:]
        if not case["packed"]:
            t.key, t.value = t.key.contiguous(), t.value.contiguous()
        t.weight = (torch.randn(d, generator=gen, device="cuda") * 0.2 + (0.0 if case["one_plus"] else 1.0)).bfloat16()
        t.writes_host = _writes(case, held, counts, table)
        t.writes = i32(t.writes_host)
        t.positions = i32(np.concatenate([np.arange(a, b) for a, b in zip(held, full)]))
        # the rotary tables of all positions; angles of far ones need 64 bits
        r = case["rotated"]
        power = torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r
        angle = torch.arange(t.longest, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** -power
        angle = torch.cat((angle, angle), 1)
        t.cos, t.sin = torch.cos(angle).bfloat16(), torch.sin(angle).bfloat16()
        # the blocks that got tokens, as a table of their own, with what each then holds
        t.filled_host = t.writes_host[:, 1] + t.writes_host[:, 3]
        t.touched, t.filled, t.filled_rows = t.writes[:, :1], i32(t.filled_host), int(t.filled_host.sum())
    if case["op"] == "attend4":
        t.query = unit(int(counts.sum()), case["heads"], d)
        t.q_cu = i32(np.concatenate([[0], np.cumsum(counts)]))
        t.max_q, t.queries = int(counts.max()), int(counts.sum())
    return t


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def prepare(case, seed):
    """The case's inputs, and the cache as earlier steps left it."""
    t = _inputs(case, seed)
    k, v = t.old_keys.float(), t.old_values.float()
    if t.bits == 8:
        ke, ve = _exponent(_largest(k, (2, 3)), 8), _exponent(_largest(v, (2, 3)), 8)
        t.keys = _key_order8(_codes8(k, ke[:, :, None, None]))
        t.values = _value_order8(_codes8(v, ve[:, :, None, None]))
        t.scales = _power(torch.stack((ke, ve), -1)).contiguous()
    else:
        t.keys, t.values, t.scales = _packed4(k, v)
    del t.old_keys, t.old_values
    return t


# ---- the plain forms: codes and layouts

def _power(e):
    """2^e in fp32, exactly (-126 <= e <= 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _largest(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def _exponent(largest, bits):
    """The least e with largest <= 448 * 2^e (448 = 0.875 * 2^9), of 4 bits 6 * 2^e (6 = 0.75 * 2^3), within the limits."""
    low, high, _ = LIMITS[bits]
    part, power = torch.frexp(largest)
    top, shift = (0.875, 9) if bits == 8 else (0.75, 3)
    e = power - shift + (part > top).to(power.dtype)
    return torch.where(largest > 0, e, torch.full_like(e, low)).clamp(low, high)


def _scaled(x, e):
    """x / 2^e (two exact factors: 2^-e alone may be past fp32's range)."""
    half = torch.div(-e, 2, rounding_mode="floor")
    return x * _power(half) * _power(-e - half)


def _codes8(x, e):
    """x / 2^e to the nearest e4m3 value (ties to even), what is past the range at its end, NaN as NaN."""
    y = _scaled(x, e)
    return torch.where(torch.isnan(y), y, y.clamp(-448.0, 448.0)).to(torch.float8_e4m3fn)


def _codes4(x, e):
    """x / 2^e as e2m1 codes 0 .. 15 (0, 1/2, 1, 3/2, 2, 3, 4, 6, then their negatives; nearest, ties to even, what is past the
    range at its end; a NaN's code counts for nothing, its scale is NaN)."""
    y = _scaled(x, e)
    a = torch.where(torch.isnan(y), torch.zeros_like(y), y.abs().clamp(max=6.0))
    low, mid = torch.round(a * 2), torch.round(a) + 2
    code = torch.where(a < 2, low, torch.where(a < 4, mid, torch.round(a / 2) + 4))
    return (code.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3))


def _values4(code):
    """fp32 values of e2m1 codes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)
    return torch.cat((grid, -grid))[code.long()]


def _key_order8(codes):
    """(blocks, heads, tokens, D) as the 8-bit cache lays keys out: [tokens / 16][D / 64][16 tokens][64 elements]."""
    b, h, n, d = codes.shape
    x = codes.view(torch.uint8).view(b, h, n // 16, 16, d // 64, 64).permute(0, 1, 2, 4, 3, 5)
    return x.reshape(b, h, n * d).view(torch.float8_e4m3fn)


def _key_rows8(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(torch.uint8).view(b, h, n // 16, d // 64, 16, 64).permute(0, 1, 2, 4, 3, 5)
    return x.reshape(b, h, n, d).view(torch.float8_e4m3fn)


def _value_order8(codes):
    """[tokens / 32][D / 32][16 (d % 16)][4 (token / 4 % 4)][2 (d / 16 % 2)][2 (token / 16 % 2)][4 (token % 4)]."""
    b, h, n, d = codes.shape
    x = codes.view(torch.uint8).view(b, h, n // 32, 2, 4, 4, d // 32, 2, 16)  # t, q, i, dg, dh, dl
    return x.permute(0, 1, 2, 6, 8, 4, 7, 3, 5).reshape(b, h, n * d).view(torch.float8_e4m3fn)


def _value_rows8(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(torch.uint8).view(b, h, n // 32, d // 32, 16, 4, 2, 2, 4)  # dg, dl, q, dh, t, i
    return x.permute(0, 1, 2, 7, 5, 8, 3, 6, 4).reshape(b, h, n, d).view(torch.float8_e4m3fn)


def _key_order(code):
    """(blocks, heads, tokens, D) 4-bit codes as bytes in the cache's order of keys: [tokens / 16][D / 32][16 tokens][32
    elements, the even one of each byte in its lower half]."""
    b, h, n, d = code.shape
    x = (code[..., ::2] | code[..., 1::2] << 4).view(b, h, n // 16, 16, d // 32, 16)
    return x.permute(0, 1, 2, 4, 3, 5).reshape(b, h, n * d // 2)


def _key_codes(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(b, h, n // 16, d // 32, 16, 16).permute(0, 1, 2, 4, 3, 5).reshape(b, h, n, d // 2)
    return torch.stack((x & 15, x >> 4), -1).reshape(b, h, n, d)


def _value_order(code):
    """[tokens / 32][D / 64][4 (token / 4 % 4)][16 (d / 2 % 16)][2 (d / 32 % 2)][2 (token / 16 % 2)][4 (token % 4)]."""
    b, h, n, d = code.shape
    x = (code[..., ::2] | code[..., 1::2] << 4).view(b, h, n // 32, 2, 4, 4, d // 64, 2, 16)  # t, q, i, dg, g, pair
    return x.permute(0, 1, 2, 6, 4, 8, 7, 3, 5).reshape(b, h, n * d // 2)


def _value_codes(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(b, h, n // 32, d // 64, 4, 16, 2, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 6, 5)  # from dg, q, pair, g, t, i
    x = x.reshape(b, h, n, d // 2)
    return torch.stack((x & 15, x >> 4), -1).reshape(b, h, n, d)


def _key_bytes(e):
    """(blocks, heads, tokens, D / 32) as (blocks, heads, tokens / 32, D) in the cache's order of the keys' scales: [4 (d / 32 %
    4)][16 tokens][D / 128][2 (token / 16 % 2)], of head size 64 [2 (token / 16 % 2)][2 (d / 32)][16 tokens]."""
    b, h, n, g = e.shape
    if g == 2:
        return e.view(b, h, n // 32, 2, 16, 2).permute(0, 1, 2, 3, 5, 4).reshape(b, h, n // 32, 64)
    x = e.view(b, h, n // 32, 2, 16, g // 4, 4)  # t, token, dt, kb
    return x.permute(0, 1, 2, 6, 4, 5, 3).reshape(b, h, n // 32, 32 * g)


def _key_scales(flat, n, g):
    b, h = flat.shape[:2]
    if g == 2:
        return flat.view(b, h, n // 32, 2, 2, 16).permute(0, 1, 2, 3, 5, 4).reshape(b, h, n, 2)
    return flat.view(b, h, n // 32, 4, 16, g // 4, 2).permute(0, 1, 2, 6, 4, 5, 3).reshape(b, h, n, g)


def _value_bytes(e):
    """The same of the values' scales: [D / 32][4 (token / 4 % 4)][2 (token / 16 % 2)][4 (token % 4)]."""
    b, h, n, g = e.shape
    return e.view(b, h, n // 32, 2, 4, 4, g).permute(0, 1, 2, 6, 4, 3, 5).reshape(b, h, n // 32, 32 * g)


def _value_scales(flat, n, g):
    b, h = flat.shape[:2]
    return flat.view(b, h, n // 32, g, 4, 2, 4).permute(0, 1, 2, 5, 4, 6, 3).reshape(b, h, n, g)


def _quantised4(x):
    """(codes, scale bytes) of (..., D): a scale for each 32 elements."""
    groups = x.unflatten(-1, (-1, 32))
    e = _exponent(_largest(groups, -1), 4)
    code = _codes4(groups, e[..., None]).flatten(-2)
    return code, torch.where(torch.isnan(groups).any(-1), torch.full_like(e, 255), e + 127).to(torch.uint8)


def _packed4(k, v):
    """Keys and values (blocks, heads, tokens, D) as the 4-bit cache's tensors."""
    (kc, ke), (vc, ve) = _quantised4(k), _quantised4(v)
    return _key_order(kc), _value_order(vc), torch.stack((_key_bytes(ke), _value_bytes(ve)), 3).contiguous()


def _rows4(t, ident):
    """Keys and values (entries, heads, block, D) fp32 of the blocks ``ident``."""
    d, n = t.case["head_dim"], t.block

    def value(code, scale):
        factor = torch.where(scale == 255, torch.full((), math.nan, device=code.device), _power(scale.int() - 127))
        return (_values4(code).unflatten(-1, (-1, 32)) * factor[..., None]).flatten(-2)

    scales = t.scales[ident]
    return (value(_key_codes(t.keys[ident], n, d), _key_scales(scales[:, :, :, 0], n, d // 32)),
            value(_value_codes(t.values[ident], n, d), _value_scales(scales[:, :, :, 1], n, d // 32)))


# ---- the plain forms: the operators

def _normed(x, weight, one_plus):
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    return x if weight is None else x * (1.0 + weight.float() if one_plus else weight.float())


def _new_rows(t):
    """The new keys and values in 32 bits: normed, the keys rotated."""
    r = t.case["rotated"]
    key = _normed(t.key.float(), t.weight, t.case["one_plus"])
    cos, sin = t.cos[t.positions.long()].float()[:, None], t.sin[t.positions.long()].float()[:, None]
    a, b = key[..., :r // 2], key[..., r // 2:r]
    key = torch.cat((a * cos[..., :r // 2] - b * sin[..., :r // 2], b * cos[..., r // 2:] + a * sin[..., r // 2:], key[..., r:]), -1)
    return key, _normed(t.value.float(), None, False) if t.case["value_norm"] else t.value.float()


def _placed(t, new):
    """(which slots of the written blocks are new, the rows there (writes, heads, block, D), zeros elsewhere)."""
    ident, first, row, count = (x.long() for x in t.writes.unbind(-1))
    place = torch.arange(t.block, device=new.device)
    written = (place >= first[:, None]) & (place < (first + count)[:, None])
    source = (row[:, None] + place - first[:, None]).clamp(0, new.shape[0] - 1)
    x = new[source].permute(0, 2, 1, 3)
    written = written[:, None, :, None]
    return ident, first, written, torch.where(written, x, torch.zeros_like(x))


def _append_one(t, flat, scales, new, rows_of, order):
    ident, first, written, x = _placed(t, new)
    low, high, _ = LIMITS[8]
    before = rows_of(flat.view(torch.uint8)[ident], t.block, new.shape[2])
    e = _exponent(_largest(x, (2, 3)), 8)
    old = ((scales[ident].view(torch.int32) >> 23) - 127).clamp(low, high)
    e = torch.where(first[:, None] > 0, torch.maximum(e, old), e)
    fresh, again = _codes8(x, e[:, :, None, None]), _codes8(before.float(), (e - old)[:, :, None, None])
    earlier = (torch.arange(t.block, device=new.device) < first[:, None])[:, None, :, None]
    codes = torch.where(written, fresh.view(torch.uint8),
                        torch.where(earlier, again.view(torch.uint8), before.view(torch.uint8)))
    return ident, order(codes.view(torch.float8_e4m3fn)), _power(e)


def _append(t):
    key, value = _new_rows(t)
    ident, keys, k_scale = _append_one(t, t.keys, t.scales[..., 0].contiguous(), key, _key_rows8, _key_order8)
    _, values, v_scale = _append_one(t, t.values, t.scales[..., 1].contiguous(), value, _value_rows8, _value_order8)
    t.keys.view(torch.uint8)[ident] = keys.view(torch.uint8)
    t.values.view(torch.uint8)[ident] = values.view(torch.uint8)
    t.scales[ident] = torch.stack((k_scale, v_scale), -1)
    return t.keys, t.values, t.scales


def _append4(t):
    d, n = t.case["head_dim"], t.block
    key, value = _new_rows(t)
    ident, _, written, key = _placed(t, key)
    value = _placed(t, value)[3]
    scales = t.scales[ident]
    (kc, ke), (vc, ve) = _quantised4(key), _quantised4(value)
    t.keys[ident] = _key_order(torch.where(written, kc, _key_codes(t.keys[ident], n, d)))
    t.values[ident] = _value_order(torch.where(written, vc, _value_codes(t.values[ident], n, d)))
    ke = torch.where(written, ke, _key_scales(scales[:, :, :, 0], n, d // 32))
    ve = torch.where(written, ve, _value_scales(scales[:, :, :, 1], n, d // 32))
    t.scales[ident] = torch.stack((_key_bytes(ke), _value_bytes(ve)), 3)
    return _read4(t, t.touched, t.filled, t.filled_rows)


def _before(x):
    """(n + 1) sums of x's elements before each."""
    return torch.cat((torch.zeros(1, dtype=torch.int64, device=x.device), torch.cumsum(x.long(), 0)))


def _read4(t, table, lengths, rows):
    k_cu = _before(lengths)
    row = torch.arange(rows, device=table.device)
    seq = torch.searchsorted(k_cu[1:].contiguous(), row, right=True)
    position = row - k_cu[seq]
    key, value = _rows4(t, torch.arange(t.blocks, device=table.device))
    ident, inside = table[seq, position // t.block].long(), position % t.block
    return {"key": key.bfloat16()[ident, :, inside], "value": value.bfloat16()[ident, :, inside], "k_cu": k_cu.int()}


def _attend4(t):
    case = t.case
    n, width = t.lengths.numel(), _blocks_of(t.longest, t.block)
    kv_heads, d, group = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    key, value = _rows4(t, t.table[:, :width].clamp(min=0).reshape(-1).long())

    def padded(x):
        return x.view(n, width, kv_heads, t.block, d).transpose(1, 2).reshape(n, kv_heads, width * t.block, d)

    key, value = padded(key), padded(value)
    q_cu, keys = t.q_cu.long(), t.lengths.long()
    place = torch.arange(t.max_q, device=t.query.device)
    source = (q_cu[:-1, None] + place).clamp(max=t.queries - 1)
    q = t.query[source].float().view(n, t.max_q, kv_heads, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(n, kv_heads, group * t.max_q, d)
    s = torch.matmul(q, key.transpose(2, 3).contiguous()).mul_(_scale(case))
    at = place + (keys - q_cu.diff())[:, None]  # (n, max_q): each query's key coordinate
    column = torch.arange(width * t.block, device=q.device)
    seen = (column <= at[..., None]) & (column < keys[:, None, None])
    if case["window"] >= 0:
        seen &= column >= at[..., None] - case["window"]
    s.view(n, kv_heads, group, t.max_q, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    value = torch.where((column < keys[:, None])[:, None, :, None], value, torch.zeros_like(value))
    o = torch.matmul(p, value) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(n, kv_heads, group, t.max_q, d).permute(0, 3, 1, 2, 4).reshape(n, t.max_q, case["heads"], d)
    row = torch.arange(t.queries, device=q.device)
    seq = torch.searchsorted(q_cu[1:].contiguous(), row, right=True)
    return o[seq, row - q_cu[seq]].bfloat16()


# ---- one pass

def run(state):
    t = state
    op = t.case["op"]
    with torch.inference_mode():
        if own:
            from karpo_decision_amd import kv_cache, ops

            if op == "append":
                cache = kv_cache.Cache(t.keys, t.values, t.scales, t.block)
            else:
                cache = kv_cache.Cache(t.keys.view(torch.float4_e2m1fn_x2), t.values.view(torch.float4_e2m1fn_x2),
                                       t.scales.view(torch.float8_e8m0fnu), t.block)
            if op in ("append", "append4"):
                k_norm = ops.Norm(ops.NORM_ONE_PLUS if t.case["one_plus"] else ops.NORM_WEIGHT, t.weight, EPS)
                v_norm = ops.Norm(ops.NORM_PLAIN, None, EPS) if t.case["value_norm"] else None
                kv_cache.append(cache, t.key, t.value, t.writes, k_norm=k_norm, v_norm=v_norm, rope=(t.cos, t.sin),
                                positions=t.positions)
                if op == "append":
                    return t.keys, t.values, t.scales
                table, lengths, rows = t.touched, t.filled, t.filled_rows
            else:
                table, lengths, rows = t.table, t.lengths, t.rows
            if op == "attend4":
                return kv_cache.attend(t.query, cache, table, t.q_cu, lengths, t.max_q, _scale(t.case), causal=True,
                                       window=t.case["window"], total_keys=rows)
            key, value, k_cu = kv_cache.read(cache, table, lengths, rows)
            return {"key": key, "value": value, "k_cu": k_cu}
        if op == "read4":
            return _read4(t, t.table, t.lengths, t.rows)
        return {"append": _append, "append4": _append4, "attend4": _attend4}[op](t)


# ---- what a pass cannot do without

def work(case):
    held, counts = _lengths(case)
    d, kv_heads, block, rows = case["head_dim"], case["kv_heads"], case["block"], int(counts.sum())
    full = held + counts
    per_token = 2 * kv_heads * d  # elements
    if case["op"] in ("append", "append4"):
        jobs = int(((full - 1) // block - held // block + 1).sum())
        flops = 12 * rows * kv_heads * d
        moved = rows * (2 * per_token + 4 * case["rotated"] + 4) + jobs * 16
        if case["op"] == "append":
            return {"bytes": moved + rows * per_token + jobs * 8 * kv_heads, "flops": flops}
        back = int(_writes(case, held, counts, np.zeros((len(held), int(_blocks_of(full, block).max())), np.int64))[:, [1, 3]].sum())
        return {"bytes": moved + rows * per_token * 17 // 32 + back * per_token * (17 + 64) // 32, "flops": flops}
    if case["op"] == "read4":
        tokens = int(full.sum())
        return {"bytes": tokens * per_token * (17 + 64) // 32 + 4 * int(_blocks_of(full, block).sum()), "flops": tokens * per_token}
    window = case["window"]
    seen = full if window < 0 else np.minimum(full, counts + window)
    pairs = 0
    for length, count in zip(full, counts):
        at = np.arange(length - count, length, dtype=np.int64) + 1
        pairs += int((at if window < 0 else np.minimum(at, window + 1)).sum())
    return {"bytes": int(seen.sum()) * per_token * 17 // 32 + 4 * int(_blocks_of(seen, block).sum())
            + 4 * rows * case["heads"] * d, "flops": 4 * d * case["heads"] * pairs}


# ---- the same in 64 bits, written apart from the above

def exact(case, seed):
    t = _inputs(case, seed)
    block, kv_heads, d, dev = case["block"], case["kv_heads"], case["head_dim"], "cuda"
    low, high, most = LIMITS[t.bits]

    def exponent(largest):
        """The least e with largest <= most * 2^e."""
        e = torch.ceil(torch.log2(torch.where(largest > 0, largest / most, torch.ones_like(largest))))
        e = torch.where(largest <= most * torch.exp2(e - 1), e - 1, e)  # (log2 a rounding off)
        e = torch.where(largest > most * torch.exp2(e), e + 1, e)
        return torch.where(largest > 0, e, torch.full_like(e, low)).clamp(low, high)

    def rounded(x):
        """To the format's grid: 3 or 1 bits after the leading one, even steps below the least normal number."""
        least, after = (2.0 ** -6, 3) if t.bits == 8 else (1.0, 1)
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=least))) - after)
        return (torch.round(x / step) * step).clamp(-most, most)

    def fours(x):
        """(..., D) as the 4-bit cache holds it."""
        g = x.reshape(*x.shape[:-1], -1, 32)
        scale = torch.exp2(exponent(g.abs().amax(-1, keepdim=True)))
        return (rounded(g / scale) * scale).reshape(x.shape)

    new_k = new_v = None
    if case["op"] in ("append", "append4"):
        new_k, new_v = t.key.double(), t.value.double()
        new_k = new_k / torch.sqrt((new_k * new_k).sum(-1, keepdim=True) / d + EPS)
        new_k = new_k * ((1.0 if case["one_plus"] else 0.0) + t.weight.double())
        r = case["rotated"]
        c, s = (x.double()[t.positions.long()].unsqueeze(1) for x in (t.cos, t.sin))
        turned = torch.cat((-new_k[..., r // 2:r], new_k[..., :r // 2]), -1)
        new_k = torch.cat((new_k[..., :r] * c + turned * s, new_k[..., r:]), -1)
        if case["value_norm"]:
            new_v = new_v / torch.sqrt((new_v * new_v).sum(-1, keepdim=True) / d + EPS)
    old_k, old_v = t.old_keys.double(), t.old_values.double()

    if case["op"] == "append":
        ke, ve = (exponent(x.abs().amax((2, 3))) for x in (old_k, old_v))
        kc, vc = (rounded(x / torch.exp2(e)[..., None, None]) for x, e in ((old_k, ke), (old_v, ve)))
        for ident, first, row, count in t.writes_host.tolist():
            for codes, exps, new in ((kc, ke, new_k), (vc, ve, new_v)):
                x = new[row:row + count].transpose(0, 1)
                e = exponent(x.abs().amax((1, 2)))
                if first:
                    e = torch.maximum(e, exps[ident])
                    codes[ident, :, :first] = rounded(codes[ident, :, :first] / torch.exp2(e - exps[ident])[:, None, None])
                codes[ident, :, first:first + count] = rounded(x / torch.exp2(e)[:, None, None])
                exps[ident] = e
        token, elem = torch.arange(block, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
        k_at = ((token // 16) * (d // 64) + elem // 64) * 1024 + (token % 16) * 64 + elem % 64
        v_at = (token // 32) * 32 * d + (elem // 32) * 1024 + (elem % 16) * 64 + (token // 4 % 4) * 16 \
            + (elem // 16 % 2) * 8 + (token // 16 % 2) * 4 + token % 4
        flat_k, flat_v = (torch.empty((t.blocks, kv_heads, block * d), dtype=torch.float64, device=dev) for _ in "kv")
        flat_k[:, :, k_at.reshape(-1)] = kc.flatten(2)
        flat_v[:, :, v_at.reshape(-1)] = vc.flatten(2)
        return flat_k, flat_v, torch.exp2(torch.stack((ke, ve), -1))

    k, v = fours(old_k), fours(old_v)
    del old_k, old_v
    if case["op"] == "append4":
        new_k, new_v, out_k, out_v = fours(new_k), fours(new_v), [], []
        for ident, first, row, count in t.writes_host.tolist():
            for all_rows, new, out in ((k, new_k, out_k), (v, new_v, out_v)):
                out.append(torch.cat((all_rows[ident, :, :first].transpose(0, 1), new[row:row + count])))
        return {"key": torch.cat(out_k), "value": torch.cat(out_v), "k_cu": None}

    table, lengths = t.table.cpu().numpy(), t.lengths.tolist()

    def rows(x, i):
        ids = torch.tensor(table[i, :_blocks_of(lengths[i], block)], dtype=torch.int64, device=dev)
        return x[ids].transpose(1, 2).reshape(-1, kv_heads, d)[:lengths[i]]

    if case["op"] == "read4":
        return {"key": torch.cat([rows(k, i) for i in range(len(lengths))]),
                "value": torch.cat([rows(v, i) for i in range(len(lengths))]), "k_cu": None}
    q_cu, group = t.q_cu.tolist(), case["heads"] // kv_heads
    out = torch.zeros(t.query.shape, dtype=torch.float64, device=dev)
    for i, length in enumerate(lengths):
        key, value = rows(k, i).permute(1, 0, 2).contiguous(), rows(v, i).permute(1, 0, 2).contiguous()
        shift = length - (q_cu[i + 1] - q_cu[i])
        chunk = max(1, (1 << 28) // (case["heads"] * max(1, length)))
        for a in range(q_cu[i], q_cu[i + 1], chunk):
            b = min(q_cu[i + 1], a + chunk)
            q = t.query[a:b].double().view(b - a, kv_heads, group, d).permute(1, 2, 0, 3).reshape(kv_heads, -1, d)
            s = torch.matmul(q, key.transpose(1, 2).contiguous()) / math.sqrt(d)
            at = torch.arange(a - q_cu[i], b - q_cu[i], device=dev)[:, None] + shift
            j = torch.arange(length, device=dev)[None, :]
            hidden = j > at
            if case["window"] >= 0:
                hidden |= j < at - case["window"]
            s.view(kv_heads, group, b - a, -1).masked_fill_(hidden, -math.inf)
            o = torch.matmul(torch.softmax(s, -1), value)
            out[a:b] = o.view(kv_heads, group, b - a, d).permute(2, 0, 1, 3).reshape(b - a, case["heads"], d)
    return out
