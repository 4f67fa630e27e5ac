"""Measured cases of the block cache: keys and values kept between calls in 8 bits (e4m3), with one power-of-two scale
for each block of tokens and head, and the four operators of a serving step over it.

``reserve``  from request lengths: block table, slot map, positions and the list of block writes, on the GPU
``append``   new keys and values into their blocks (a block whose scale grows has its earlier tokens rounded again)
``read``     the cached rows of a batch back as packed bf16 keys and values
``attend``   attention of new queries over the cache: one token per request, a few, or a chunk of a prompt

Ranges that ``draw`` spreads over: 1 to 512 requests, 1 to 65,536 new tokens, cached lengths from 0 to 131,072 tokens,
blocks of 32, 64 and 128 tokens, head sizes 64, 128, 256 and 512 with the head counts of this repository's workloads,
with and without a window.

The cache's layout (``keys`` and ``values`` (blocks, kv heads, block size * D) e4m3, ``scales`` (blocks, kv heads, 2)
fp32): a block's keys lie in tiles of 16 tokens by 64 elements, its values in tiles of 32 tokens by 32 elements with
the tokens innermost, in the order in which a lane of a matrix instruction takes them (``_key_order``,
``_value_order``).
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

#: Exponents a block's scale may have: above, 448 * 2^e would pass bf16's range; below, everything rounds to zero.
LOW, HIGH = -100, 119
E4M3_MAX = 448.0


def _case(name, op, **more):
    base = {"name": name, "op": op, "requests": 1, "median": 0, "longest": 0, "new": 1, "block": 64, "heads": 32,
            "kv_heads": 16, "head_dim": 128, "window": -1, "pack": 0}
    base.update(more)
    return base


def listed():
    return [
        # one decoding step of a batch: one new token per request, what every layer of the step then uses
        _case("reserve-step", "reserve", requests=48, median=900, longest=4096, new=48, block=64),
        # a batch of prompts and prompt chunks admitted at once
        _case("reserve-prompts", "reserve", requests=64, median=400, longest=4096, new=65536, block=32),
        # the new token of each request into one layer's cache
        _case("append-step", "append", requests=48, median=900, longest=4096, new=48),
        # ragged prompt chunks that begin anywhere in a block, a 12B-class sliding layer
        _case("append-chunks", "append", requests=24, median=700, longest=4096, new=2500, heads=16, kv_heads=8,
              head_dim=256),
        # one long document into a global layer's cache
        _case("append-document", "append", requests=1, new=32768),
        # the cached prompts of a few requests, as rows (the 31B global layer)
        _case("read-batch", "read", requests=6, median=1500, longest=8192, heads=32, kv_heads=4, head_dim=512, block=32),
        # a long cached document, as rows
        _case("read-document", "read", requests=1, median=32768, longest=32768),
        # a handful of short requests, one token each: launches count
        _case("decode-short", "attend", requests=4, median=250, longest=511, new=4, heads=8, kv_heads=2, head_dim=64,
              block=32),
        # a decoding step of a ragged batch
        _case("decode-batch", "attend", requests=48, median=900, longest=8192, new=48),
        # one long document, one token, the 31B global layer
        _case("decode-document", "attend", requests=1, median=131072, longest=131072, new=1, heads=32, kv_heads=4,
              head_dim=512, block=128),
        # a few tokens per request to check at once, sliding layers
        _case("decode-few-sliding", "attend", requests=32, median=2500, longest=8192, new=128, heads=16, kv_heads=8,
              head_dim=256, window=1023),
        # a prompt chunk over what is cached of the prompt
        _case("chunk-prefill", "attend", requests=1, median=30000, longest=30000, new=2048),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["reserve", "append", "append", "read", "attend", "attend", "attend", "attend"])
    block = rng.choice([32, 64, 128])
    heads, kv_heads, head_dim, window = rng.choice([(8, 2, 64, -1), (16, 8, 128, -1), (32, 16, 128, -1),
                                                    (16, 8, 256, 1023), (16, 8, 256, 511), (32, 4, 512, -1)])
    more = {"block": block, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "pack": rng.randrange(1 << 20)}
    if op == "reserve":
        requests = size(1, 512)
        new = requests if rng.random() < 0.5 else size(requests, 65536)
        case = _case("", op, requests=requests, median=size(30, 2000), longest=4096, new=new, **more)
    elif op == "append":
        requests = size(1, 64)
        new = requests if rng.random() < 0.4 else size(requests, 16384)
        case = _case("", op, requests=requests, median=size(30, 1000), longest=4096, new=new, **more)
    elif op == "read":
        requests = size(1, 16)
        case = _case("", op, requests=requests, median=size(30, 1500), longest=2048, **more)
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
    rng = np.random.default_rng(case["pack"] + 17)
    n = case["requests"]
    if n == 1:
        held = np.array([case["median"]], dtype=np.int64)
    else:
        held = np.exp(rng.normal(math.log(max(1, case["median"])), 1.0, size=n))
        held = np.clip(np.round(held), 0, case["longest"]).astype(np.int64)
        if n > 4:
            held[int(rng.integers(n))] = 0  # a request that begins
    new = case["new"]
    if new <= n:
        counts = np.ones(n, dtype=np.int64)
    elif case["op"] == "attend":  # about the same for each
        counts = np.full(n, new // n, dtype=np.int64)
        counts[0] += new - int(counts.sum())
    else:
        share = np.exp(rng.normal(0, 1.0, size=n))
        counts = np.maximum(1, np.floor(share / share.sum() * (new - n))).astype(np.int64)
        counts[int(np.argmax(counts))] += new - int(counts.sum())
    return held, counts


def _blocks_of(tokens, block):
    return -(-tokens // block)


def _tables(case, held, spare):
    """(block table, ids no request holds), host arrays: the held blocks scattered over the pool."""
    rng = np.random.default_rng(case["pack"] + 29)
    block, counts = case["block"], _blocks_of(held, case["block"])
    pool = int(counts.sum()) + spare
    order = rng.permutation(pool).astype(np.int32)
    width = max(1, int(counts.max()) + spare)
    table = np.full((case["requests"], width), -1, dtype=np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += int(c)
    return table, order[at:], pool


def _inputs(case, seed):
    """Seeded tensors of the case, the same for ``prepare`` and ``exact``."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    held, counts = _lengths(case)
    block, kv_heads, d = case["block"], case["kv_heads"], case["head_dim"]
    after = held + counts
    t = SimpleNamespace(case=case, block=block)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] in ("reserve", "append"):
        fresh = int((_blocks_of(after, block) - _blocks_of(held, block)).sum())
        table, free, pool = _tables(case, held, fresh + 3)
        order = torch.randperm(len(free), generator=gen, device="cuda")
        t.table, t.free = i32(table), i32(free)[order].contiguous()
        t.free_count = i32([len(free) - 1])
        t.lengths, t.counts, t.rows = i32(held), i32(counts), int(counts.sum())
    else:
        # attend: the new tokens are in the cache already, as in a step of which append is over
        full = after if case["op"] == "attend" else held
        table, free, pool = _tables(case, full, 2)
        pick = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)  # other blocks for each seed
        table = i32(table)
        t.table = torch.where(table >= 0, pick[table.clamp(min=0).long()], table).contiguous()
        t.lengths, t.rows, t.longest = i32(full), int(full.sum()), int(full.max())
        t.q_cu = i32(np.concatenate([[0], np.cumsum(counts)]))
        t.max_q, t.queries = int(counts.max()), int(counts.sum())
    if case["op"] == "reserve":
        return t
    t.blocks = pool
    x = torch.randn((pool, kv_heads, block, d), generator=gen, device="cuda")
    x *= torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)  # what the layer's key norm leaves
    t.old_keys = x.bfloat16()
    t.old_values = x.normal_(generator=gen).bfloat16()
    if case["op"] == "append":
        rows = t.rows
        key = torch.randn((rows, kv_heads, d), generator=gen, device="cuda")
        t.key = (key * torch.rsqrt(key.pow(2).mean(-1, keepdim=True) + 1e-6)).bfloat16()
        # a few tokens are much larger than what a block holds: its scale grows
        size = torch.where(torch.rand((rows, kv_heads, 1), generator=gen, device="cuda") < 0.1, 6.0, 1.0)
        t.value = (torch.randn((rows, kv_heads, d), generator=gen, device="cuda") * size).bfloat16()
    if case["op"] == "attend":
        q = torch.randn((t.queries, case["heads"], d), generator=gen, device="cuda")
        t.query = (q * torch.rsqrt(q.pow(2).mean(-1, keepdim=True) + 1e-6)).bfloat16()
    return t


def _scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def prepare(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "reserve":
        return t
    # the cache as earlier steps left it
    ke, ve = _exponent(_largest(t.old_keys.float(), (2, 3))), _exponent(_largest(t.old_values.float(), (2, 3)))
    t.keys = _key_order(_codes(t.old_keys.float(), ke[:, :, None, None]))
    t.values = _value_order(_codes(t.old_values.float(), ve[:, :, None, None]))
    t.scales = _power(torch.stack((ke, ve), -1)).contiguous()
    del t.old_keys, t.old_values
    if case["op"] == "append":
        step = _reserve(t)
        held, counts = _lengths(case)
        t.writes = step["writes"]
        t.used = int(((held + counts - 1) // t.block - held // t.block + 1)[counts > 0].sum())
    return t


# ---- the plain forms

def _power(e):
    """2^e in fp32, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _largest(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def _exponent(largest):
    """The least e with largest <= 448 * 2^e, within LOW .. HIGH."""
    part, power = torch.frexp(largest)
    e = power - 9 + (part > 0.875).to(power.dtype)
    return torch.where(largest > 0, e, torch.full_like(e, LOW)).clamp(LOW, HIGH)


def _codes(x, e):
    """x / 2^e to the nearest e4m3 value (ties to even), what is past the range at its end, NaN as NaN."""
    y = x * _power(-e)
    return torch.where(torch.isnan(y), y, y.clamp(-E4M3_MAX, E4M3_MAX)).to(torch.float8_e4m3fn)


def _key_order(codes):
    """(blocks, heads, tokens, D) as the cache lays keys out: [tokens / 16][D / 64][16 tokens][64 elements]."""
    b, h, n, d = codes.shape
    x = codes.view(torch.uint8).view(b, h, n // 16, 16, d // 64, 64).permute(0, 1, 2, 4, 3, 5)
    return x.reshape(b, h, n * d).view(torch.float8_e4m3fn)


def _key_rows(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(torch.uint8).view(b, h, n // 16, d // 64, 16, 64).permute(0, 1, 2, 4, 3, 5)
    return x.reshape(b, h, n, d).view(torch.float8_e4m3fn)


def _value_order(codes):
    """(blocks, heads, tokens, D) as the cache lays values out: [tokens / 32][D / 32][16 (d % 16)][4 (token / 4 % 4)]
    [2 (d / 16 % 2)][2 (token / 16 % 2)][4 (token % 4)]."""
    b, h, n, d = codes.shape
    x = codes.view(torch.uint8).view(b, h, n // 32, 2, 4, 4, d // 32, 2, 16)  # t, q, i, dg, dh, dl
    return x.permute(0, 1, 2, 6, 8, 4, 7, 3, 5).reshape(b, h, n * d).view(torch.float8_e4m3fn)


def _value_rows(flat, n, d):
    b, h = flat.shape[:2]
    x = flat.view(torch.uint8).view(b, h, n // 32, d // 32, 16, 4, 2, 2, 4)  # dg, dl, q, dh, t, i
    return x.permute(0, 1, 2, 7, 5, 8, 3, 6, 4).reshape(b, h, n, d).view(torch.float8_e4m3fn)


def _before(x):
    """(n + 1) sums of x's elements before each."""
    return torch.cat((torch.zeros(1, dtype=torch.int64, device=x.device), torch.cumsum(x.long(), 0)))


def _capacity(rows, n, block):
    return min(rows, rows // block + 2 * n)


def _reserve(t):
    """Block table, slots, positions and block writes of ``counts`` new tokens per request. Blocks come from the end of
    the first ``free_count`` entries of ``free``, in the order of the tokens that need them."""
    block, rows, n = t.block, t.rows, t.lengths.numel()
    held_tokens, counts = t.lengths.long(), t.counts.long()
    after = held_tokens + counts
    held = (held_tokens + block - 1) // block
    need = (after + block - 1) // block - held
    touched = torch.where(counts > 0, (after - 1) // block - held_tokens // block + 1, torch.zeros_like(counts))
    q_cu, need_cu, write_cu = _before(counts), _before(need), _before(touched)
    left = t.free_count.long() - need_cu[-1]
    bad = (t.lengths < 0).any() | (t.counts < 0).any() | (q_cu[-1] > rows) | (after > t.table.shape[1] * block).any()
    status = torch.where(bad, 11, torch.where(left[0] < 0, 10, 0)).to(torch.int32).reshape(1)
    fine = status[0] == 0
    row = torch.arange(rows, device=t.table.device)
    seq = torch.searchsorted(q_cu[1:].contiguous(), row, right=True).clamp(max=n - 1)
    valid = (row < q_cu[-1]) & fine
    position = torch.where(valid, held_tokens[seq] + row - q_cu[seq], torch.zeros_like(row))
    at, inside = position // block, position % block
    fresh = at >= held[seq]
    taken = t.free_count.long() - 1 - (need_cu[seq] + at - held[seq])
    known = t.table[seq, at.clamp(max=t.table.shape[1] - 1)].long()
    ident = torch.where(fresh, t.free[taken.clamp(0, t.free.numel() - 1)].long(), known)
    slots = torch.where(valid, ident * block + inside, torch.full_like(row, -1))
    begins = valid & ((inside == 0) | (row == q_cu[seq]))
    table = torch.cat((t.table.reshape(-1), t.table.new_zeros(1)))
    table[torch.where(begins & fresh, seq * t.table.shape[1] + at, torch.full_like(row, table.numel() - 1))] = ident.int()
    capacity = _capacity(rows, n, block)
    writes = t.table.new_zeros((capacity + 1, 4))
    entry = torch.where(begins, write_cu[seq] + at - held_tokens[seq] // block, torch.full_like(row, capacity))
    count = torch.minimum(block - inside, q_cu[seq + 1] - row)
    writes[entry] = torch.stack((ident, inside, row, count), -1).int()
    return {"q_cu": torch.where(fine, q_cu, torch.zeros_like(q_cu)).int(),
            "lengths": torch.where(fine, after, held_tokens).int(), "slots": slots, "positions": position.int(),
            "writes": writes[:capacity], "table": table[:-1].view(t.table.shape),
            "free_left": torch.where(fine, left, t.free_count.long()).int(), "status": status}


def _append_one(flat, scales, new, writes, block, rows_of, order):
    """One of keys and values: the touched blocks with the new rows in them, and their scales."""
    d = new.shape[2]
    ident, first, row, count = (x.long() for x in writes.unbind(-1))
    before = rows_of(flat[ident], block, d)
    place = torch.arange(block, device=flat.device)
    written = (place >= first[:, None]) & (place < (first + count)[:, None])  # (writes, block)
    source = (row[:, None] + place - first[:, None]).clamp(0, new.shape[0] - 1)
    x = new[source].float().permute(0, 2, 1, 3)  # (writes, heads, block, D)
    x = torch.where(written[:, None, :, None], x, torch.zeros_like(x))
    e = _exponent(_largest(x, (2, 3)))
    old = ((scales[ident].view(torch.int32) >> 23) - 127).clamp(LOW, HIGH)
    e = torch.where(first[:, None] > 0, torch.maximum(e, old), e)
    fresh = _codes(x, e[:, :, None, None])
    again = _codes(before.float(), (e - old)[:, :, None, None])
    earlier = (place < first[:, None])[:, None, :, None]
    codes = torch.where(written[:, None, :, None], fresh.view(torch.uint8),
                        torch.where(earlier, again.view(torch.uint8), before.view(torch.uint8)))
    return ident, order(codes.view(torch.float8_e4m3fn)), _power(e)


def _append(t):
    writes = t.writes[:t.used]
    ident, keys, k_scale = _append_one(t.keys.view(torch.uint8), t.scales[..., 0].contiguous(), t.key, writes, t.block,
                                       _key_rows, _key_order)
    _, values, v_scale = _append_one(t.values.view(torch.uint8), t.scales[..., 1].contiguous(), t.value, writes,
                                     t.block, _value_rows, _value_order)
    t.keys.view(torch.uint8)[ident] = keys.view(torch.uint8)
    t.values.view(torch.uint8)[ident] = values.view(torch.uint8)
    t.scales[ident] = torch.stack((k_scale, v_scale), -1)
    return t.keys, t.values, t.scales


def _dequantised(t, ident):
    """Keys and values (entries, heads, block, D) fp32 of the blocks ``ident``."""
    d, scales = t.case["head_dim"], t.scales[ident][..., None, None]
    key = _key_rows(t.keys.view(torch.uint8)[ident], t.block, d).float() * scales[:, :, 0]
    return key, _value_rows(t.values.view(torch.uint8)[ident], t.block, d).float() * scales[:, :, 1]


def _read(t):
    k_cu = _before(t.lengths)
    row = torch.arange(t.rows, device=t.table.device)
    seq = torch.searchsorted(k_cu[1:].contiguous(), row, right=True)
    position = row - k_cu[seq]
    key, value = _dequantised(t, torch.arange(t.blocks, device=t.table.device))
    ident, inside = t.table[seq, position // t.block].long(), position % t.block
    return {"key": key.bfloat16()[ident, :, inside], "value": value.bfloat16()[ident, :, inside],
            "k_cu": k_cu.int()}


def _attend(t):
    case = t.case
    n, width = t.lengths.numel(), _blocks_of(t.longest, t.block)
    kv_heads, d, group = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    key, value = _dequantised(t, t.table[:, :width].clamp(min=0).reshape(-1).long())

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
            from karpo_decision_amd import kv_cache

            if op == "reserve":
                step = kv_cache.reserve(t.table, t.lengths, t.counts, t.free, t.free_count, t.rows, t.block)
                return {"q_cu": step.q_cu, "lengths": step.lengths, "slots": step.slots, "positions": step.positions,
                        "writes": step.writes, "table": t.table, "free_left": step.free_left, "status": step.status}
            cache = kv_cache.Cache(t.keys, t.values, t.scales, t.block)
            if op == "append":
                kv_cache.append(cache, t.key, t.value, t.writes)
                return t.keys, t.values, t.scales
            if op == "read":
                key, value, k_cu = kv_cache.read(cache, t.table, t.lengths, t.rows)
                return {"key": key, "value": value, "k_cu": k_cu}
            return kv_cache.attend(t.query, cache, t.table, t.q_cu, t.lengths, t.max_q, _scale(t.case), causal=True,
                                   window=t.case["window"], total_keys=t.rows)
        return {"reserve": _reserve, "append": _append, "read": _read, "attend": _attend}[op](t)


# ---- what a pass cannot do without

def work(case):
    held, counts = _lengths(case)
    n, d, kv_heads, block = case["requests"], case["head_dim"], case["kv_heads"], case["block"]
    rows = int(counts.sum())
    if case["op"] == "reserve":
        fresh = int((_blocks_of(held + counts, block) - _blocks_of(held, block)).sum())
        jobs = int(((held + counts - 1) // block - held // block + 1).sum())
        return {"bytes": 4 * 4 * n + 12 * rows + 8 * fresh + 16 * jobs + 4 * jobs, "flops": 0}
    if case["op"] == "append":
        jobs = int(((held + counts - 1) // block - held // block + 1).sum())
        return {"bytes": 2 * rows * kv_heads * d * 3 + jobs * (16 + 8 * kv_heads), "flops": 4 * rows * kv_heads * d}
    if case["op"] == "read":
        blocks = int(_blocks_of(held, block).sum())
        return {"bytes": 2 * int(held.sum()) * kv_heads * d * 3 + blocks * (4 + 8 * kv_heads),
                "flops": 2 * int(held.sum()) * kv_heads * d}
    full, window = held + counts, case["window"]
    seen = full if window < 0 else np.minimum(full, counts + window)
    pairs = 0
    for length, count in zip(full, counts):
        at = np.arange(length - count, length, dtype=np.int64) + 1
        pairs += int((at if window < 0 else np.minimum(at, window + 1)).sum())
    blocks = int(_blocks_of(seen, block).sum())
    return {"bytes": 2 * int(seen.sum()) * kv_heads * d + blocks * (4 + 8 * kv_heads) + 4 * rows * case["heads"] * d,
            "flops": 4 * d * case["heads"] * pairs}


# ---- the same in 64 bits, written apart from the above

def exact(case, seed):
    if case["op"] == "reserve":
        return None
    t = _inputs(case, seed)
    block, kv_heads, d = case["block"], case["kv_heads"], case["head_dim"]
    dev = "cuda"

    def exponent(x):
        """Of the largest finite magnitude over the last two dims: the least e with it <= 448 * 2^e."""
        x = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).flatten(-2).amax(-1)
        e = torch.ceil(torch.log2(torch.where(x > 0, x / 448.0, torch.ones_like(x))))
        e = torch.where(x <= 448.0 * torch.exp2(e - 1), e - 1, e)  # (log2 a rounding off)
        e = torch.where(x > 448.0 * torch.exp2(e), e + 1, e)
        return torch.where(x > 0, e, torch.full_like(e, LOW)).clamp(LOW, HIGH)

    def rounded(x):
        """To e4m3's grid: 3 bits after the leading one, steps of 2^-9 below 2^-6."""
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        return (torch.round(x / step) * step).clamp(-448.0, 448.0)

    def spread(x):
        return x[..., None, None]

    # the cache before the call: codes (blocks, heads, tokens, D) as values, and exponents
    old_k, old_v = t.old_keys.double(), t.old_values.double()
    ke, ve = exponent(old_k), exponent(old_v)
    kc, vc = rounded(old_k / spread(torch.exp2(ke))), rounded(old_v / spread(torch.exp2(ve)))
    table = t.table.cpu().numpy()
    lengths = t.lengths.cpu().numpy()
    if case["op"] == "append":
        counts, row = t.counts.cpu().numpy(), 0
        free, top = t.free.cpu().numpy(), int(t.free_count.item())
        for i in range(len(lengths)):
            at, end = int(lengths[i]), int(lengths[i] + counts[i])
            while at < end:
                b, first = at // block, at % block
                if first == 0:
                    top -= 1
                    ident = int(free[top])
                else:
                    ident = int(table[i, b])
                n = min(block - first, end - at)
                for codes, exps, new in ((kc, ke, t.key), (vc, ve, t.value)):
                    x = new[row:row + n].double().permute(1, 0, 2)
                    e = exponent(x)
                    if first:
                        e = torch.maximum(e, exps[ident])
                        codes[ident, :, :first] = rounded(codes[ident, :, :first] / spread(torch.exp2(e - exps[ident])))
                    codes[ident, :, first:first + n] = rounded(x / spread(torch.exp2(e)))
                    exps[ident] = e
                at, row = at + n, row + n
        token, elem = torch.arange(block, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
        k_at = ((token // 16) * (d // 64) + elem // 64) * 1024 + (token % 16) * 64 + elem % 64
        v_at = (token // 32) * 32 * d + (elem // 32) * 1024 + (elem % 16) * 64 + (token // 4 % 4) * 16 \
            + (elem // 16 % 2) * 8 + (token // 16 % 2) * 4 + token % 4
        flat_k, flat_v = (torch.empty((t.blocks, kv_heads, block * d), dtype=torch.float64, device=dev) for _ in "kv")
        flat_k[:, :, k_at.reshape(-1)] = kc.flatten(2)
        flat_v[:, :, v_at.reshape(-1)] = vc.flatten(2)
        return flat_k, flat_v, torch.exp2(torch.stack((ke, ve), -1))
    kc, vc = kc * spread(torch.exp2(ke)), vc * spread(torch.exp2(ve))

    def rows(x, i):
        ids = torch.tensor(table[i, :_blocks_of(int(lengths[i]), block)], dtype=torch.int64, device=dev)
        return x[ids].transpose(1, 2).reshape(-1, kv_heads, d)[:int(lengths[i])]

    if case["op"] == "read":
        return {"key": torch.cat([rows(kc, i) for i in range(len(lengths))]),
                "value": torch.cat([rows(vc, i) for i in range(len(lengths))]), "k_cu": None}
    q_cu, group = t.q_cu.tolist(), case["heads"] // kv_heads
    out = torch.zeros(t.query.shape, dtype=torch.float64, device=dev)
    for i in range(len(lengths)):
        k, v = rows(kc, i).permute(1, 0, 2).contiguous(), rows(vc, i).permute(1, 0, 2).contiguous()
        shift = int(lengths[i]) - (q_cu[i + 1] - q_cu[i])
        chunk = max(1, (1 << 28) // (case["heads"] * max(1, int(lengths[i]))))
        for a in range(q_cu[i], q_cu[i + 1], chunk):
            b = min(q_cu[i + 1], a + chunk)
            q = t.query[a:b].double().view(b - a, kv_heads, group, d).permute(1, 2, 0, 3).reshape(kv_heads, -1, d)
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
            at = torch.arange(a - q_cu[i], b - q_cu[i], device=dev)[:, None] + shift
            j = torch.arange(int(lengths[i]), device=dev)[None, :]
            hidden = j > at
            if case["window"] >= 0:
                hidden |= j < at - case["window"]
            s.view(kv_heads, group, b - a, -1).masked_fill_(hidden, -math.inf)
            o = torch.matmul(torch.softmax(s, -1), v)
            out[a:b] = o.view(kv_heads, group, b - a, d).permute(2, 0, 1, 3).reshape(b - a, case["heads"], d)
    return out
