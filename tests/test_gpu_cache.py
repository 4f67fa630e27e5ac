"""The block cache on the GPU against the oracle's loops and 64-bit sums (oracle/cache.py).

Codes, scales, tables and slots have to be equal. Attention's tolerance, per output element: the output's rounding to bf16
(2^-8 of its magnitude) plus the weights' (each at most 2^-8 off: 2^-8 times the weighted mean of |value|) plus 2^-14 of the
latter for the fp32 scores and exponentials (scores below 2^6 here, off by a few of their 2^-18 steps)."""

from __future__ import annotations

import math

import pytest
import torch

from karpo_decision_amd import kv_cache
from oracle import cache as oracle

pytestmark = pytest.mark.gpu


def ints(values, device, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=device)


def bits(t):
    return t.view(torch.uint8).cpu()


# ---- reserve

def _requests(n, block, width, seed, most=200):
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, width * block // 2, (n,), generator=gen)
    edge = torch.randint(0, 4, (n,), generator=gen)  # some at a block's border or next to it
    lengths = torch.where(edge == 0, lengths // block * block, torch.where(edge == 1, lengths // block * block + block - 1,
                                                                           lengths))
    counts = torch.randint(0, most, (n,), generator=gen)
    counts = torch.where(torch.randint(0, 3, (n,), generator=gen) == 0, torch.ones_like(counts), counts)
    counts = torch.where(torch.randint(0, 5, (n,), generator=gen) == 0, torch.zeros_like(counts), counts)
    counts = torch.minimum(counts, width * block - lengths)
    held = (lengths + block - 1) // block
    need = int(((lengths + counts + block - 1) // block - held).sum())
    pool = torch.randperm(int(held.sum()) + need + 2, generator=gen).tolist()
    table = [[pool.pop() for _ in range(h)] + [-1] * (width - h) for h in held.tolist()]
    return table, lengths.tolist(), counts.tolist(), pool


def _reserve_and_compare(device, table, lengths, counts, free, free_count, rows, block, strided=False):
    want_table, want = oracle.reserve(table, lengths, counts, free, free_count, rows, block)
    dev_table = ints(table, device)
    if strided:
        wide = torch.full((len(table), len(table[0]) + 5), -7, dtype=torch.int32, device=device)
        wide[:, :len(table[0])] = dev_table
        dev_table = wide[:, :len(table[0])]
    step = kv_cache.reserve(dev_table, ints(lengths, device), ints(counts, device), ints(free, device),
                            ints([free_count], device), rows, block)
    assert step.status.tolist() == [want["status"]]
    assert dev_table.tolist() == want_table
    if strided:
        assert (wide[:, len(table[0]):] == -7).all()
    for name in ("q_cu", "lengths", "slots", "positions"):
        assert getattr(step, name).tolist() == want[name], name
    writes = want["writes"] + [[0] * 4] * (step.writes.shape[0] - len(want["writes"]))
    assert step.writes.tolist() == writes
    assert step.free_left.tolist() == [want["free_left"]]
    return step


@pytest.mark.parametrize("n,block,width,rows_more,strided", [
    (1, 32, 8, 0, False), (7, 64, 6, 13, True), (48, 128, 5, 0, False), (300, 32, 9, 1, False), (1024, 32, 4, 0, False),
    (1025, 64, 4, 77, False), (2500, 32, 3, 0, True)])
def test_reserve(gpu, n, block, width, rows_more, strided):
    table, lengths, counts, free = _requests(n, block, width, seed=n)
    _reserve_and_compare(gpu, table, lengths, counts, free, len(free), sum(counts) + rows_more, block, strided)


def test_reserve_one_token_each(gpu):
    lengths = [0, 31, 32, 33, 63, 64, 95]
    table = [[10 * i + j if j < -(-x // 32) else -1 for j in range(4)] for i, x in enumerate(lengths)]
    step = _reserve_and_compare(gpu, table, lengths, [1] * 7, [91, 92, 93, 94, 95], 4, 7, 32)
    step.check()


def test_reserve_long_prompts(gpu):
    lengths, counts = [5, 0, 4095], [70000, 1, 60000]
    width = 2400
    table = [[i * width + j if j < -(-x // 32) else -1 for j in range(width)] for i, x in enumerate(lengths)]
    free = list(range(90000, 96000))
    _reserve_and_compare(gpu, table, lengths, counts, free, 5990, 130010, 32)


@pytest.mark.parametrize("change", [
    {"free_count": 2}, {"free_count": -1}, {"free_count": 6}, {"rows": 36}, {"counts": [40, -1, 3]}, {"lengths": [30, -1, 0]},
    {"counts": [40, 200, 3]}, {"lengths": [30, 2**31 - 1, 0]}, {"counts": [2**31 - 1] * 3}], ids=str)
def test_reserve_leaves_all_as_it_was_where_it_refuses(gpu, change):
    call = {"table": [[4, -1, -1], [5, 6, -1], [-1, -1, -1]], "lengths": [30, 40, 0], "counts": [40, 1, 3],
            "free": [1, 2, 3, 0, 7], "free_count": 5, "rows": 44, "block": 32}
    step = _reserve_and_compare(gpu, **{**call, **change})
    with pytest.raises(RuntimeError if change == {"free_count": 2} else ValueError):
        step.check()


def test_reserve_without_requests_or_tokens(gpu):
    empty = torch.empty((0, 3), dtype=torch.int32, device=gpu)
    none = torch.empty(0, dtype=torch.int32, device=gpu)
    step = kv_cache.reserve(empty, none, none, none, ints([0], gpu), 5, 64)
    assert step.q_cu.tolist() == [0] and step.slots.tolist() == [-1] * 5 and step.status.tolist() == [0]
    assert step.writes.shape == (0, 4)
    _reserve_and_compare(gpu, [[3], [4]], [7, 32], [0, 0], [], 0, 0, 32)


# ---- append

def _random_cache(device, blocks, kv_heads, head_dim, block, seed):
    """A cache whose every byte is a code (NaN among them where ``append`` has to leave it alone) with usual scales."""
    gen = torch.Generator(device=device).manual_seed(seed)
    cache = kv_cache.create(blocks, kv_heads, head_dim, block, device=device)
    for t in (cache.keys, cache.values):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=gen, device=device, dtype=torch.uint8))
    e = torch.randint(-12, -4, cache.scales.shape, generator=gen, device=device)
    cache.scales.copy_(torch.exp2(e.float()))
    return cache


def _copy(cache):
    return kv_cache.Cache(cache.keys.clone(), cache.values.clone(), cache.scales.clone(), cache.block_size)


def _append_and_compare(cache, key, value, writes):
    """The whole cache after ``append`` against the oracle's: codes as values (either zero, any NaN), scales, and the
    bytes of every slot that no write reaches."""
    before = _copy(cache)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, cache.block_size)
    want.append(key, value, writes)
    kv_cache.append(cache, key, value, ints(writes, cache.keys.device))
    got = oracle.Cache(cache.keys, cache.values, cache.scales, cache.block_size)
    assert torch.equal(got.exps, want.exps)
    reached = torch.zeros((cache.blocks, cache.block_size), dtype=torch.bool)
    for ident, first, _, count in writes:
        reached[ident, :first + count] = True
    for side in (0, 1):
        a, b = got.codes[side], want.codes[side]
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(a.nan_to_num(9e9), b.nan_to_num(9e9))
        at = oracle.offsets(cache.block_size, cache.head_dim, bool(side))
        old, new = (bits(c[side])[:, :, at].view(cache.blocks, cache.kv_heads, cache.block_size, -1)
                    for c in (before, cache))
        same = (old == new).all(-1).all(1)
        assert (same | reached).all()


@pytest.mark.parametrize("head_dim", [64, 128, 256, 512])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_append(gpu, head_dim, block):
    """Whole blocks, one token, tokens that begin and end inside a group of 32, each over leftovers of other requests."""
    cache = _random_cache(gpu, 9, 3, head_dim, block, seed=head_dim + block)
    gen = torch.Generator(device=gpu).manual_seed(1)
    rows = 2 * block + 60
    key, value = (torch.randn((rows, 3, head_dim), generator=gen, device=gpu).bfloat16() for _ in range(2))
    value[::7] *= 50  # larger than what the block holds: earlier codes are rounded again
    key[3::11] *= 300
    writes = [[2, 0, 0, block], [5, 0, block, 1], [0, 17, block + 1, 1], [7, block - 1, block + 2, 1],
              [1, 3, block + 3, 21], [3, 11, block + 24, block - 11], [8, 0, 2 * block + 13, 13], [6, 30, 2 * block + 26, 2],
              [4, 0, 2 * block + 28, 32]]
    _append_and_compare(cache, key, value, writes)


def test_append_reads_strided_rows_and_leaves_others(gpu):
    cache = _random_cache(gpu, 4, 2, 128, 32, seed=3)
    packed = torch.randn((50, 6, 160), device=gpu).bfloat16()
    key, value = packed[:, 1:3, :128], packed[:, 4:, 32:]
    assert key.stride() == (960, 160, 1)
    _append_and_compare(cache, key, value, [[1, 5, 40, 10], [3, 0, 2, 32]])


def test_append_extremes(gpu):
    """Zeros, the least and largest bf16 values, infinities and NaN; a scale that grows past all earlier codes."""
    cache = _random_cache(gpu, 8, 1, 64, 32, seed=4)
    key = torch.zeros((8, 1, 64), dtype=torch.bfloat16, device=gpu)
    key[1] = 9.2e-41
    key[2, :, ::2] = 3.3895e38
    key[3, :, 1], key[3, :, 2], key[3, :, 3], key[3, :, 4] = math.inf, -math.inf, math.nan, 0.37
    key[4] = math.inf
    key[5] = math.nan
    key[6] = -1.0e30
    key[7] = torch.linspace(-450, 450, 64)
    value = key.flip(0).contiguous()
    writes = [[i, 0 if i % 2 else 9, i, 1] for i in range(8)]
    _append_and_compare(cache, key, value, writes)


def test_append_ties_and_subnormal_codes(gpu):
    """Elements between two codes (to even), and below the least normal code."""
    cache = kv_cache.create(2, 1, 64, 32, device=gpu)
    steps = torch.arange(0, 64, device=gpu).float()
    key = torch.stack([448 - steps * 3.5, steps * 2.0 ** -10, (steps + 0.5) * 2.0 ** -9, 16 + steps / 2, 240 + steps, -steps / 64,
                       steps * 0 + 448, steps * 1.0625]).bfloat16()[:, None]
    _append_and_compare(cache, key, -key, [[1, 0, 0, 8]])


def test_append_skips_writes_out_of_range(gpu):
    """Blocks outside the pool, slots past a block, rows past the input: nothing is followed."""
    cache = _random_cache(gpu, 3, 2, 64, 32, seed=5)
    before = _copy(cache)
    rows = torch.randn((10, 2, 64), device=gpu).bfloat16()
    writes = [[3, 0, 0, 4], [-1, 0, 0, 4], [0, 30, 0, 4], [0, -1, 0, 4], [1, 0, 8, 4], [1, 0, -1, 4], [2, 0, 0, 0], [2, 0, 0, -3],
              [2**31 - 1, 0, 0, 1], [0, 32, 0, 1], [0, 0, 2**31 - 1, 2**31 - 1], [0, 2**31 - 1, 0, 2]]
    kv_cache.append(cache, rows, rows, ints(writes, gpu))
    for a, b in zip(before[:3], cache[:3]):
        assert torch.equal(bits(a), bits(b))


def test_blocks_past_32_bit_offsets(gpu):
    """Append, read and attend at a block whose codes start past 2^31 bytes."""
    block, head_dim, heads, ident = 128, 512, 4, 8500  # 262,144 bytes a block: past 2^31 from block 8,192 on
    cache = kv_cache.Cache(*(torch.empty((8503, heads, block * head_dim), dtype=torch.uint8, device=gpu)
                             .view(torch.float8_e4m3fn) for _ in range(2)),
                           torch.zeros((8503, heads, 2), device=gpu), block)
    gen = torch.Generator(device=gpu).manual_seed(6)
    key, value = (torch.randn((40, heads, head_dim), generator=gen, device=gpu).bfloat16() for _ in range(2))
    kv_cache.append(cache, key, value, ints([[ident, 0, 0, 40]], gpu))
    got_k, got_v, k_cu = kv_cache.read(cache, ints([[ident]], gpu), ints([40], gpu), 40)
    assert k_cu.tolist() == [0, 40]
    for got, x in ((got_k, key), (got_v, value)):
        # half a step of e4m3 (2^-4 of the element), or half its least step: 2^-10 of a scale below 2^-6 here
        assert ((got.float() - x.float()).abs() <= x.float().abs() * 2.0 ** -4 + 2.0 ** -16).all()
    query = torch.randn((1, 8, head_dim), generator=gen, device=gpu).bfloat16()
    with torch.inference_mode():
        out = kv_cache.attend(query, cache, ints([[ident]], gpu), ints([0, 1], gpu), ints([40], gpu), 1, 0.04)
    _close(out, query, got_k.cpu().double(), got_v.cpu().double(), 0.04)


def _close(out, query, key, value, scale, causal=True, window=-1):
    """One request's rows within the tolerance of the module's docstring (key, value: float64, what the cache holds)."""
    query = query.cpu().double()
    want = oracle.attention(query, key, value, scale, causal, window)
    size = oracle.attention(query, key, value.abs(), scale, causal, window)
    off = (out.cpu().double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -14)
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), f"off {off.max():.3e}, worst {(off / bound.clamp(min=1e-30)).max():.2f} of the bound"


# ---- read

@pytest.mark.parametrize("head_dim,block,lengths", [
    (64, 32, [1, 0, 33, 70]), (128, 64, [200, 64, 5, 0, 0, 129]), (256, 128, [31, 300]), (512, 32, [95, 1]),
    (128, 32, [(7 * i) % 90 for i in range(300)])])
def test_read(gpu, head_dim, block, lengths):
    width = max(1, -(-max(lengths) // block)) + 1
    cache = _random_cache(gpu, 40, 2, head_dim, block, seed=7)
    table = [[(i * 11 + j * 7) % 40 for j in range(width)] for i in range(len(lengths))]
    if len(table) > 2:
        table[2][0] = -1  # reads as zeros
        table[3][0] = 40
    rows = sum(lengths) + 3
    key, value, k_cu = kv_cache.read(cache, ints(table, gpu), ints(lengths, gpu), rows)
    assert key.shape == value.shape == (rows, 2, head_dim)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    at = 0
    for i, n in enumerate(lengths):
        assert k_cu[i].item() == at
        wk, wv = want.rows(table[i], 0, n)
        for got, w in ((key, wk), (value, wv)):
            g = got[at:at + n].cpu().double()
            assert torch.equal(g.nan_to_num(9e9), w.nan_to_num(9e9)) and torch.equal(torch.isnan(g), torch.isnan(w))
        at += n
    assert k_cu[-1].item() == at


def test_read_writes_no_row_past_its_bound(gpu):
    """Lengths whose sum is past ``rows``, below zero and past the table's row."""
    cache = _random_cache(gpu, 4, 1, 64, 32, seed=8)
    table = ints([[0, 1], [2, 3], [1, 2]], gpu)
    backing = torch.full((2, 200, 64), 3.0, dtype=torch.bfloat16, device=gpu)
    import ctypes

    from karpo_decision_amd import _lib, ops
    lengths, k_cu = ints([-5, 1000, 40], gpu), torch.empty(4, dtype=torch.int32, device=gpu)
    c = _lib.KarpoCache(*(t.data_ptr() for t in cache[:3]), 4, 1, 64, 32)
    args = _lib.KarpoCacheReadArgs(c, table.data_ptr(), 2, 2, 3, lengths.data_ptr(), backing[0].data_ptr(),
                                   backing[1].data_ptr(), 90, k_cu.data_ptr())
    _lib.check(_lib.load().karpo_cache_read(ctypes.byref(args), ops._current_stream(0)), "read")
    assert k_cu.tolist() == [0, 0, 64, 104]
    assert (backing[:, 90:] == 3).all() and not (backing[:, :90] == 3).all(-1).all()


# ---- attend

def _attend_case(device, head_dim, heads, kv_heads, block, lengths, counts, window=-1, causal=True, scale=None, seed=0,
                 trailing=0, wide=1, oracle_too=True):
    scale = 1 / math.sqrt(head_dim) if scale is None else scale
    width = max(1, -(-max(lengths) // block)) + wide
    gen = torch.Generator().manual_seed(seed)
    pool = torch.randperm(sum(-(-x // block) for x in lengths) + 3, generator=gen).tolist()
    blocks = len(pool)
    cache = _random_cache(device, blocks, kv_heads, head_dim, block, seed)
    cache.scales.copy_(torch.exp2(torch.randint(-9, -6, cache.scales.shape, generator=gen).float()))
    table = [[pool.pop() for _ in range(-(-x // block))] for x in lengths]
    table = [r + [-1] * (width - len(r)) for r in table]
    # the tokens in use hold no NaN (leftovers behind them do)
    for side, flat in enumerate((cache.keys, cache.values)):
        raw = flat.view(torch.uint8)
        at = oracle.offsets(block, head_dim, bool(side)).view(block, head_dim).to(device)
        for i, x in enumerate(lengths):
            for j in range(-(-x // block)):
                n = min(block, x - j * block)
                part = raw[table[i][j]][:, at[:n].reshape(-1)]
                raw[table[i][j]][:, at[:n].reshape(-1)] = torch.where((part & 127) == 127, part - 1, part)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block) if oracle_too else None
    rows = sum(counts) + trailing
    query = torch.randn((rows, heads, head_dim), generator=gen).bfloat16()
    q_cu = [0]
    for c in counts:
        q_cu.append(q_cu[-1] + c)
    return cache, want, table, query, q_cu, scale


def _attend_and_compare(device, *args, **more):
    cache, want, table, query, q_cu, scale = _attend_case(device, *args, **more)
    lengths, counts = args[4], args[5]
    causal, window = more.get("causal", True), more.get("window", -1)
    with torch.inference_mode():
        out = kv_cache.attend(query.to(device), cache, ints(table, device), ints(q_cu, device), ints(lengths, device),
                              max(counts), scale, causal=causal, window=window, total_keys=sum(lengths))
    for i, n in enumerate(lengths):
        key, value = want.rows(table[i], 0, n)
        _close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], key, value, scale, causal, window)
    return cache, out


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (128, 4, 4), (128, 16, 2), (256, 6, 2), (512, 8, 1),
                                                     (512, 3, 3), (64, 40, 1)])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_decode(gpu, head_dim, heads, kv_heads, block):
    """One token per request: lengths of one, around groups and blocks, one longer; leftovers hold NaN codes."""
    _attend_and_compare(gpu, head_dim, heads, kv_heads, block, [1, 32, 33, 31, 128, 129, 700, 0], [1] * 8)


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts", [
    (128, 8, 4, [3, 1, 0, 7]), (64, 8, 2, [5, 5, 5, 5]), (256, 16, 8, [4, 2, 1, 1]), (512, 32, 4, [2, 3, 1, 2]),
    (128, 16, 2, [13, 1, 2, 9])])
def test_a_few_tokens_each(gpu, head_dim, heads, kv_heads, counts):
    _attend_and_compare(gpu, head_dim, heads, kv_heads, 64, [100, 40, 63, 513], counts)


@pytest.mark.parametrize("window", [0, 5, 40, 100])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(gpu, window, causal):
    _attend_and_compare(gpu, 128, 4, 2, 32, [300, 64, 1, 37], [3, 1, 1, 30], window=window, causal=causal)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,window", [
    (128, 4, 2, [300, 170], [130, 170], -1), (256, 4, 2, [500], [200], 99), (64, 8, 2, [400, 0, 90], [90, 0, 90], -1),
    (512, 4, 1, [260, 33], [120, 33], -1)])
def test_chunks_of_prompts(gpu, head_dim, heads, kv_heads, lengths, counts, window):
    _attend_and_compare(gpu, head_dim, heads, kv_heads, 64, lengths, counts, window=window)


def _workspace(cache, heads, max_q, total_q, total_keys, n, width, window):
    """Bytes that the call's path asks for: the unpacked keys and values are in them, or they are not."""
    import ctypes

    from karpo_decision_amd import _lib
    c = _lib.KarpoCache(*(t.data_ptr() for t in cache[:3]), cache.blocks, cache.kv_heads, cache.head_dim, cache.block_size)
    a = _lib.KarpoCacheAttendArgs(c, 4096, 4096, 8, 8, 8, 8, 4096, 4096, 4096, width, width, n, heads, max_q, total_q,
                                  total_keys, 0.1, window, 0)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
    return need.value


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,window,causal", [
    (64, 32, 2, [5100, 3000], [1500, 900], -1, True), (128, 32, 4, [3000, 1777], [1500, 1777], -1, True),
    (128, 32, 4, [3000, 2100, 0, 40], [1500, 1000, 3, 41], 600, True), (256, 16, 2, [2500, 1900], [800, 700], -1, False),
    (256, 16, 2, [2500, 2900], [900, 800], 333, True), (512, 8, 1, [2000, 900], [700, 900], -1, True)])
def test_long_chunks(gpu, head_dim, heads, kv_heads, lengths, counts, window, causal):
    """Chunks long enough that the keys are unpacked first, against 64-bit products on the GPU."""
    block = 64
    cache, _, table, query, q_cu, scale = _attend_case(gpu, head_dim, heads, kv_heads, block, lengths, counts, oracle_too=False)
    rows = sum(lengths)
    need = _workspace(cache, heads, max(counts), sum(counts), rows, len(lengths), len(table[0]), window)
    seen = rows if window < 0 else min(rows, len(lengths) * (max(counts) + window))
    assert need > 4 * seen * kv_heads * head_dim  # the path that unpacks
    query = query.to(gpu)
    with torch.inference_mode():
        out = kv_cache.attend(query, cache, ints(table, gpu), ints(q_cu, gpu), ints(lengths, gpu), max(counts), scale,
                              causal=causal, window=window, total_keys=rows)
        key, value, k_cu = kv_cache.read(cache, ints(table, gpu), ints(lengths, gpu), rows)  # (test_read: exact)
    k_cu = k_cu.tolist()
    for i in range(len(lengths)):
        q, k, v = query[q_cu[i]:q_cu[i + 1]].double(), key[k_cu[i]:k_cu[i + 1]].double(), value[k_cu[i]:k_cu[i + 1]].double()
        want = oracle.attention_whole(q, k, v, scale, causal, window)
        size = oracle.attention_whole(q, k, v.abs(), scale, causal, window)
        off = (out[q_cu[i]:q_cu[i + 1]].double() - want).abs()
        assert (off <= want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -14)).all(), (i, off.max())


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts", [
    (64, 16, 1, [700, 41], [70, 41]), (128, 24, 2, [1100, 300], [100, 7]), (256, 12, 1, [900], [60]),
    (512, 16, 1, [500, 64], [30, 64])])
def test_many_tiles_of_queries(gpu, head_dim, heads, kv_heads, lengths, counts):
    """The split path with several workgroups for a request's query vectors, the last of them not full."""
    _attend_and_compare(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    assert max(counts) * heads // kv_heads > 64


def test_more_queries_than_tokens(gpu):
    """Queries before the first token see nothing: zeros."""
    for counts in ([9, 5], [90, 70]):
        _, out = _attend_and_compare(gpu, 64, 4, 2, 32, [4, 0], counts)
        assert (out[:counts[0] - 4] == 0).all() and (out[counts[0]:] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(gpu, scale):
    _attend_and_compare(gpu, 64, 4, 2, 32, [130, 20], [1, 2], scale=scale)


def test_a_scale_that_is_no_number(gpu):
    cache, _, table, query, q_cu, _ = _attend_case(gpu, 64, 4, 2, 32, [130, 20], [1, 1], oracle_too=False)
    with torch.inference_mode():
        out = kv_cache.attend(query.to(gpu), cache, ints(table, gpu), ints(q_cu, gpu), ints([130, 20], gpu), 1, math.nan)
    assert torch.isnan(out).all()


def test_bounds_out_of_range_write_nothing(gpu):
    """Query bounds past the query, decreasing or negative: their requests have no queries, the others theirs."""
    cache, want, table, query, q_cu, scale = _attend_case(gpu, 64, 4, 2, 32, [130, 20, 50, 60], [2, 2, 2, 2])
    import ctypes

    from karpo_decision_amd import _lib, ops
    for bounds, good in (([0, 2, 4, 6, 9], (0, 1, 2)), ([0, 2, 1, 3, 5], (0,)), ([-3, 2, 4, 6, 8], (1, 2, 3))):
        q, cu = query.to(gpu), ints(bounds, gpu)
        out = torch.full_like(q, 7.0)
        lengths, dev_table = ints([130, 20, 50, 60], gpu), ints(table, gpu)
        c = _lib.KarpoCache(*(t.data_ptr() for t in cache[:3]), cache.blocks, 2, 64, 32)
        a = _lib.KarpoCacheAttendArgs(c, q.data_ptr(), out.data_ptr(), 256, 64, 256, 64, cu.data_ptr(), lengths.data_ptr(),
                                      dev_table.data_ptr(), len(table[0]), len(table[0]), 4, 4, 2, 8, 260, scale, -1, 0)
        need = ctypes.c_size_t()
        _lib.check(_lib.load().karpo_cache_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
        workspace = torch.empty(need.value + 16, dtype=torch.uint8, device=gpu)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
        _lib.check(_lib.load().karpo_cache_attend(ctypes.byref(a), ops._current_stream(0)), "attend")
        written = torch.zeros(8, dtype=torch.bool)
        for i, n in enumerate((130, 20, 50, 60)):
            if i in good or (bounds == [0, 2, 1, 3, 5] and i in (2, 3)):
                written[bounds[i]:bounds[i + 1]] = True
            if i in good and bounds != [0, 2, 1, 3, 5]:
                rows = slice(bounds[i], bounds[i + 1])
                _close(out[rows], query[rows], *want.rows(table[i], 0, n), scale)
        assert (out[~written.to(gpu)] == 7).all()


def test_many_requests(gpu):
    lengths = [(37 * i) % 200 for i in range(600)]
    _attend_and_compare(gpu, 64, 4, 2, 32, lengths, [1 + (i % 3 == 0) for i in range(600)])


def test_one_long_request(gpu):
    _attend_and_compare(gpu, 128, 4, 2, 64, [9001], [1])


def test_strided_queries_and_tables(gpu):
    cache, want, table, query, q_cu, scale = _attend_case(gpu, 128, 4, 2, 32, [90, 40], [2, 1], wide=4)
    wide = torch.zeros((3, 6, 160), dtype=torch.bfloat16, device=gpu)
    wide[:, 1:5, 16:144] = query.to(gpu)
    tables = torch.full((2, 20), 10 ** 6, dtype=torch.int32, device=gpu)
    tables[:, :len(table[0])] = ints(table, gpu)
    with torch.inference_mode():
        out = kv_cache.attend(wide[:, 1:5, 16:144], cache, tables[:, :len(table[0])], ints(q_cu, gpu), ints([90, 40], gpu),
                              2, scale)
    for i, n in enumerate([90, 40]):
        _close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), scale)


@pytest.mark.parametrize("counts", [[1, 1], [80, 60]])
def test_unknown_blocks_read_as_zeros(gpu, counts):
    cache, want, table, query, q_cu, scale = _attend_case(gpu, 64, 4, 2, 32, [130, 100], counts)
    table[0][1], table[1][2] = -1, cache.blocks
    with torch.inference_mode():
        out = kv_cache.attend(query.to(gpu), cache, ints(table, gpu), ints(q_cu, gpu), ints([130, 100], gpu), max(counts),
                              scale)
    for i, n in enumerate([130, 100]):
        _close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), scale)


# ---- as they are used together

def _serve(device, rounds, cache, heads, seed, between=lambda: None):
    """Rounds of reserve, append and attend, eager, on the current stream: [(step, query, key, value, out)] per round."""
    gen = torch.Generator(device=device).manual_seed(seed)
    n, width = len(rounds[0]), 8
    table = torch.full((n, width), -1, dtype=torch.int32, device=device)
    lengths = torch.zeros(n, dtype=torch.int32, device=device)
    free, left = torch.arange(cache.blocks, dtype=torch.int32, device=device), ints([cache.blocks], device)
    got = []
    for counts in rounds:
        rows = sum(counts)
        key, value = (torch.randn((rows, cache.kv_heads, cache.head_dim), generator=gen, device=device).bfloat16()
                      for _ in range(2))
        query = torch.randn((rows, heads, cache.head_dim), generator=gen, device=device).bfloat16()
        step = kv_cache.reserve(table, lengths, ints(counts, device), free, left, rows, cache.block_size)
        kv_cache.append(cache, key, value, step.writes)
        out = kv_cache.attend(query, cache, table, step.q_cu, step.lengths, max(counts), 0.1)
        lengths, left = step.lengths, step.free_left
        got.append((step, query, key, value, out))
        between()
    return table, got


@pytest.mark.parametrize("head_dim,heads,kv_heads,block", [(64, 4, 2, 32), (128, 8, 2, 64)])
def test_rounds_of_a_server(gpu, head_dim, heads, kv_heads, block):
    """Prompts, then tokens one by one and a few at a time: each round's outputs against the oracle's cache, fed the same
    rows."""
    rounds = [[40, 7, 0, 65], [1, 1, 1, 1], [1, 1, 30, 0], [3, 2, 3, 1], [1, 1, 1, 1]]
    cache = kv_cache.create(20, kv_heads, head_dim, block, device=gpu)
    with torch.inference_mode():
        table, got = _serve(gpu, rounds, cache, heads, seed=9)
    fed = kv_cache.create(20, kv_heads, head_dim, block, device="cpu")
    want = oracle.Cache(fed.keys, fed.values, fed.scales, block)
    rows = table.tolist()
    for step, query, key, value, out in got:
        step.check()
        want.append(key, value, [w for w in step.writes.tolist() if w[3]])
        q_cu, lengths = step.q_cu.tolist(), step.lengths.tolist()
        for i, n in enumerate(lengths):
            k, v = want.rows(rows[i], 0, n)
            _close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], k, v, 0.1)
    have = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    for i, n in enumerate(lengths):  # (a block's slots past its tokens are not compared)
        for a, b in zip(have.rows(rows[i], 0, n), want.rows(rows[i], 0, n)):
            assert torch.equal(a, b)


def test_a_step_on_another_stream(gpu):
    rounds = [[40, 7, 9], [1, 1, 1], [2, 1, 1]]
    with torch.inference_mode():
        caches = [kv_cache.create(16, 2, 64, 32, device=gpu) for _ in range(2)]
        _, want = _serve(gpu, rounds, caches[0], 4, seed=10)
        stream = torch.cuda.Stream(gpu)
        stream.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(stream):
            _, got = _serve(gpu, rounds, caches[1], 4, seed=10)
        torch.cuda.current_stream(gpu).wait_stream(stream)
    for a, b in zip(want, got):
        assert torch.equal(a[4], b[4])
    assert torch.equal(bits(caches[0].keys), bits(caches[1].keys))


def test_a_captured_long_chunk_replays(gpu):
    """The path that unpacks, captured: each replay reads the lengths and the cache as they are then."""
    block, heads, kv_heads, head_dim, counts = 64, 32, 2, 64, [1500, 900]
    cache, _, table, query, q_cu, scale = _attend_case(gpu, head_dim, heads, kv_heads, block, [5100, 3000], counts,
                                                       oracle_too=False)
    query, table, q_cu, lengths = query.to(gpu), ints(table, gpu), ints(q_cu, gpu), ints([5100, 3000], gpu)

    def call():
        return kv_cache.attend(query, cache, table, q_cu, lengths, 1500, scale, total_keys=8200)

    with torch.inference_mode():
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        seen = []
        for change in ([5100, 3000], [4000, 3001], [1500, 899]):
            lengths.copy_(ints(change, gpu))
            query.mul_(-0.75)
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            # bit for bit (a request's 3,001st token is a leftover, NaN among its codes)
            assert torch.equal(out.view(torch.int16), want.view(torch.int16))
            seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.parametrize("counts", [[1, 1, 1], [70, 1, 33]])
def test_a_captured_step_replays(gpu, counts):
    """A step captured once: each replay reads the lengths, rows and free blocks that its inputs hold then, with eager work
    in between; the outputs are those of eager calls, bit for bit. Two graphs captured one after the other share nothing."""
    n, rows, block, heads, kv_heads, head_dim = 3, sum(counts), 32, 4, 2, 64
    width = 8
    gen = torch.Generator(device=gpu).manual_seed(11)
    free = torch.arange(40, dtype=torch.int32, device=gpu)
    state = {"table": torch.full((n, width), -1, dtype=torch.int32, device=gpu),
             "lengths": torch.zeros(n, dtype=torch.int32, device=gpu), "left": ints([40], gpu),
             "key": torch.zeros((rows, kv_heads, head_dim), dtype=torch.bfloat16, device=gpu),
             "value": torch.zeros((rows, kv_heads, head_dim), dtype=torch.bfloat16, device=gpu),
             "query": torch.zeros((rows, heads, head_dim), dtype=torch.bfloat16, device=gpu)}
    want_counts = ints(counts, gpu)

    def step(cache, s):
        got = kv_cache.reserve(s["table"], s["lengths"], want_counts, free, s["left"], rows, block)
        kv_cache.append(cache, s["key"], s["value"], got.writes)
        return got, kv_cache.attend(s["query"], cache, s["table"], got.q_cu, got.lengths, max(counts), 0.1,
                                    total_keys=n * width * block)

    with torch.inference_mode():
        captured, eager = (kv_cache.create(40, kv_heads, head_dim, block, device=gpu) for _ in range(2))
        step(captured, {**state, "table": state["table"].clone()})  # (loads the kernels)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs = step(captured, state)
            graphs.append((graph, outputs))
        mine = {k: v.clone() for k, v in state.items()}
        for i in range(3):
            for name in ("key", "value", "query"):
                fresh = torch.randn(state[name].shape, generator=gen, device=gpu).bfloat16()
                state[name].copy_(fresh)
                mine[name].copy_(fresh)
            graph, (got, out) = graphs[i % 2]
            graph.replay()
            want, want_out = step(eager, mine)
            torch.cuda.synchronize()
            assert torch.equal(out, want_out) and out.abs().max() > 0
            assert torch.equal(got.slots, want.slots) and torch.equal(got.writes, want.writes)
            assert torch.equal(state["table"], mine["table"])
            for s, r in ((state, got), (mine, want)):
                s["lengths"].copy_(r.lengths)
                s["left"].copy_(r.free_left)
            assert torch.equal(bits(captured.values), bits(eager.values))


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts", [(64, 4, 2, [6, 1]), (128, 8, 2, [9, 2]), (512, 8, 1, [2, 1]),
                                                            (256, 16, 8, [16, 3])])
def test_nan_reaches_the_queries_that_see_it_and_no_others(gpu, head_dim, heads, kv_heads, counts):
    """NaN in one element of a new token's value, and in another's key: earlier queries of the same call do not see them."""
    lengths, block = [70, 33], 32
    cache, want, table, query, q_cu, scale = _attend_case(gpu, head_dim, heads, kv_heads, block, lengths, counts)
    raw_k, raw_v = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
    at = lengths[0] - 1  # the first request's last token: its value's element 5, head 0
    raw_v[table[0][at // block], 0, oracle.value_offset(at % block, 5, head_dim)] = 0x7f
    at = lengths[1] - 1  # the second's: its key, head 0
    raw_k[table[1][at // block], 0, oracle.key_offset(at % block, 7, head_dim)] = 0xff
    with torch.inference_mode():
        out = kv_cache.attend(query.to(gpu), cache, ints(table, gpu), ints(q_cu, gpu), ints(lengths, gpu), max(counts),
                              scale, total_keys=sum(lengths))
    group = heads // kv_heads
    nan = torch.isnan(out.cpu())
    expected = torch.zeros_like(nan)
    expected[q_cu[1] - 1, :group, 5] = True
    expected[q_cu[2] - 1, :group] = True
    assert torch.equal(nan, expected)
    for i, n in enumerate(lengths):
        key, value = (x.nan_to_num(0.0) for x in want.rows(table[i], 0, n))
        rows = slice(q_cu[i], q_cu[i + 1] - 1)  # the queries before the last, which see neither
        if rows.start < rows.stop:
            _close(out[rows], query[rows], key[:n - 1], value[:n - 1], scale)
