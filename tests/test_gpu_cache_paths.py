"""The block cache on the GPU, second part: calls whose bounds, tables or scales are not what they should be, and attention on
each of its paths (a request whole in one workgroup; split, its shares joined; keys unpacked first), which the sizes choose
between: each test asks for the workspace's size to see that it runs the path it is meant for.

Attention's tolerance on the first two paths, per output element: the output's rounding to bf16 (2^-8 of its magnitude) plus
2^-14 of the weighted mean of |value|: the weights enter the products as two bf16 terms (2^-17 off), the fp32 scores (below 2^6
here, off by a few of their 2^-18 steps, so the weights by 2^-16) and sums. On the third path a weight is one bf16 term: 2^-8 of
that mean more."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from karpo_decision_amd import _lib, kv_cache
from oracle import cache as oracle

pytestmark = pytest.mark.gpu

WHOLE, SPLIT, UNPACKED = "whole", "split", "unpacked"


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def path_of(cache, heads, counts, rows, n, width, window=-1, total_keys=None, max_q=None):
    """The path that a call of these sizes takes, by the workspace it asks for."""
    max_q = max(counts) if max_q is None else max_q
    total = n * width * cache.block_size if total_keys is None else total_keys
    c = _lib.KarpoCache(*(t.data_ptr() for t in cache[:3]), cache.blocks, cache.kv_heads, cache.head_dim, cache.block_size)
    a = _lib.KarpoCacheAttendArgs(c, 4096, 4096, 8, 8, 8, 8, 4096, 4096, 4096, width, width, n, heads, max_q, rows, total,
                                  0.1, window, 0)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
    if need.value == 0:
        return WHOLE
    # the split path's: the units before each request, and for every share two partials of a tile's vectors in fp32
    d, vectors = cache.head_dim, max_q * heads // cache.kv_heads
    most = 4 if d <= 128 else 2 if d == 256 else 1
    nt = next(t for t in (1, 2, 4) if t == most or vectors <= 16 * t)
    waves = 4 if nt == 1 and d <= 128 else 3 if (d, nt) == (64, 2) else 2 if d <= 128 or (d, nt) == (256, 1) else 1
    y = cache.kv_heads * -(-vectors // (16 * nt))
    split = -(-4 * (n + 1) // 256) * 256 + y * max(1, 256 * waves // y) * 2 * 16 * nt * (d + 2) * 4
    return SPLIT if need.value == split else UNPACKED


def make(device, head_dim, heads, kv_heads, block, lengths, counts, seed=0, width=None):
    """(cache, table, query, q_cu): codes of any value but NaN in the tokens in use, NaN among the leftovers behind them."""
    gen = torch.Generator().manual_seed(seed)
    used = [-(-x // block) for x in lengths]
    width = max(1, max(used)) if width is None else width
    pool = (torch.randperm(sum(used) + 3, generator=gen) + 1).tolist()  # block 0 is nobody's
    cache = kv_cache.create(sum(used) + 4, kv_heads, head_dim, block, device=device)
    table = [[pool.pop() for _ in range(u)] for u in used]
    for side, flat in enumerate((cache.keys, cache.values)):
        raw = torch.randint(0, 256, flat.shape, generator=gen, dtype=torch.uint8)
        at = oracle.offsets(block, head_dim, bool(side)).view(block, head_dim)
        for row, x in zip(table, lengths):
            for j, ident in enumerate(row):
                mine = at[:min(block, x - j * block)].reshape(-1)
                part = raw[ident][:, mine]
                raw[ident][:, mine] = torch.where((part & 127) == 127, part - 1, part)
        flat.view(torch.uint8).copy_(raw)
    cache.scales.copy_(torch.exp2(torch.randint(-9, -6, cache.scales.shape, generator=gen).float()))
    table = [r + [-1] * (width - len(r)) for r in table]
    query = torch.randn((sum(counts), heads, head_dim), generator=gen).bfloat16()
    q_cu = [0]
    for c in counts:
        q_cu.append(q_cu[-1] + c)
    return cache, table, query, q_cu


def attend(device, cache, table, query, q_cu, lengths, max_q, scale, **more):
    with torch.inference_mode():
        return kv_cache.attend(query.to(device), cache, ints(table, device), ints(q_cu, device), ints(lengths, device),
                               max_q, scale, **more)


def close(out, query, key, value, scale, causal=True, window=-1, weights=0.0):
    """One request's rows within the tolerance of the module's docstring (``weights``: what the path's weights are off)."""
    query, key, value = (t.to(out.device).double() for t in (query, key, value))
    want = oracle.attention_whole(query, key, value, scale, causal, window)
    size = oracle.attention_whole(query, key, value.abs(), scale, causal, window)
    off = (out.double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size * (weights + 2.0 ** -14)
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), f"off {off.max():.3e}, worst {(off / bound.clamp(min=1e-30)).max():.2f} of the bound"


# ---- blocks that are not of the pool

@pytest.mark.parametrize("head_dim", [64, 128, 256, 512])
def test_read_of_unknown_blocks_beside_a_block_without_scales(gpu, head_dim):
    """Block 0, never written, has NaN for scales: entries outside the pool read as zeros all the same."""
    cache, table, _, _ = make(gpu, head_dim, 2, 2, 32, [70, 33], [1, 1])
    cache.scales[0] = math.nan
    table[0][1], table[1][0] = -1, cache.blocks
    key, value, _ = kv_cache.read(cache, ints(table, gpu), ints([70, 33], gpu), 103)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for i, (a, b) in enumerate(((0, 70), (70, 103))):
        for got, w in zip((key, value), want.rows(table[i], 0, b - a)):
            assert torch.equal(got[a:b].cpu().double(), w)


@pytest.mark.parametrize("head_dim,heads,lengths,counts,path", [
    (64, 4, [130, 100], [1, 2], WHOLE), (64, 4, [900, 100], [1, 2], SPLIT), (128, 4, [900, 100], [1, 2], SPLIT),
    (256, 4, [900, 100], [2, 1], SPLIT), (512, 4, [300, 100], [1, 1], SPLIT), (64, 16, [3000, 2900], [2000, 1900], UNPACKED)])
def test_attend_of_unknown_blocks_beside_a_block_without_scales(gpu, head_dim, heads, lengths, counts, path):
    cache, table, query, q_cu = make(gpu, head_dim, heads, 2, 32, lengths, counts)
    assert path_of(cache, heads, counts, sum(counts), 2, len(table[0])) == path
    cache.scales[0] = math.nan
    table[0][1], table[1][2] = -1, cache.blocks
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1,
              weights=2.0 ** -8 if path == UNPACKED else 0.0)


# ---- bounds that do not hold

def attend_into(device, out, cache, table, query, q_cu, lengths, max_q, scale, total_keys):
    """``attend`` by the C ABI, into ``out`` (contiguous)."""
    from karpo_decision_amd import ops
    q, cu, n, dev_table = query.to(device), ints(q_cu, device), ints(lengths, device), ints(table, device)
    rows, heads, d = q.shape
    c = _lib.KarpoCache(*(t.data_ptr() for t in cache[:3]), cache.blocks, cache.kv_heads, d, cache.block_size)
    a = _lib.KarpoCacheAttendArgs(c, q.data_ptr(), out.data_ptr(), heads * d, d, heads * d, d, cu.data_ptr(), n.data_ptr(),
                                  dev_table.data_ptr(), len(table[0]), len(table[0]), len(table), heads, max_q, rows,
                                  total_keys, scale, -1, 0)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
    workspace = torch.empty(need.value + 16, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
    _lib.check(_lib.load().karpo_cache_attend(ctypes.byref(a), ops._current_stream(0)), "attend")
    return out


CHUNKS = (64, 16, 2, 64, [3000, 2900], [2000, 1900])  # the path that unpacks


@pytest.mark.parametrize("change", ["total_keys", "max_q", "past the query", "out of order", "negative"])
def test_a_long_chunk_with_bounds_that_do_not_hold_is_nan(gpu, change):
    """Nothing is computed then: the requests' rows are NaN, and no others are written."""
    lengths, counts = CHUNKS[4:]
    cache, table, query, q_cu = make(gpu, *CHUNKS)
    query = torch.cat((query, query[:7]))  # rows behind the last request
    total, max_q, known = sum(lengths), max(counts), torch.ones(query.shape[0], dtype=torch.bool)
    known[sum(counts):] = False
    if change == "total_keys":
        total -= 1
    elif change == "max_q":
        max_q -= 1
    elif change == "past the query":
        q_cu[2] = query.shape[0] + 1
        known[q_cu[1]:] = False
    elif change == "out of order":
        q_cu[1], q_cu[2] = q_cu[1] - 1, 1
        known[q_cu[1]:] = False
    else:
        q_cu[0] = -1
        known[:q_cu[1]] = False
    assert path_of(cache, 16, counts, query.shape[0], 2, len(table[0]), total_keys=total, max_q=max_q) == UNPACKED
    out = attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, q_cu, lengths,
                      max_q, 0.1, total)
    assert torch.isnan(out[known.to(gpu)]).all() and (out[~known.to(gpu)] == 7).all()
    if change in ("total_keys", "max_q"):
        assert torch.isnan(attend(gpu, cache, table, query, q_cu, lengths, max_q, 0.1, total_keys=total)[:sum(counts)]).all()


def test_a_long_chunk_with_bounds_that_hold_again(gpu):
    """Strided output, requests without queries among more than a workgroup's 256: the bounds' check finds nothing."""
    lengths, counts = [40] * 300 + [3000], [0, 3] * 150 + [2000]
    cache, table, query, q_cu = make(gpu, 64, 16, 2, 64, lengths, counts)
    assert path_of(cache, 16, counts, sum(counts), 301, len(table[0]), total_keys=sum(lengths)) == UNPACKED
    out = attend(gpu, cache, table, query, q_cu, lengths, 2000, 0.1, total_keys=sum(lengths))
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 64)
    for i in (1, 3, 149, 255, 257, 299, 300):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, lengths[i]), 0.1, weights=2.0 ** -8)
    q_cu[150] = q_cu[151] + 1  # one request out of order: all NaN, those of the other 255 too
    out = attend(gpu, cache, table, query, q_cu, lengths, 2000, 0.1, total_keys=sum(lengths))
    assert torch.isnan(out[:q_cu[149]]).all() and torch.isnan(out[q_cu[200]:]).all()


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,max_q,path", [
    (64, 4, 2, [130, 100], [5, 2], 2, WHOLE), (64, 80, 2, [130, 100], [1, 7], 2, WHOLE), (512, 4, 2, [100, 60], [9, 1], 1, WHOLE),
    (64, 4, 2, [900, 100, 0], [5, 3, 3], 2, SPLIT), (64, 80, 2, [900, 700], [7, 2], 2, SPLIT),
    (256, 4, 2, [900, 100], [1, 40], 33, SPLIT), (512, 4, 2, [300, 100], [9, 9], 1, SPLIT)])
def test_queries_past_max_q_are_nan(gpu, head_dim, heads, kv_heads, lengths, counts, max_q, path):
    """A request's first ``max_q`` rows are right, the others NaN (and nothing else is written)."""
    n = len(lengths)
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    query = torch.cat((query, query[:3]))
    assert path_of(cache, heads, counts, query.shape[0], n, len(table[0]), max_q=max_q) == path
    out = attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, q_cu, lengths,
                      max_q, 0.1, n * len(table[0]) * 32)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for i, tokens in enumerate(lengths):
        a, b, served = q_cu[i], q_cu[i + 1], min(counts[i], max_q)
        assert torch.isnan(out[a + served:b]).all()
        key, value = (x[:tokens - counts[i] + served] if tokens else x for x in want.rows(table[i], 0, tokens))
        close(out[a:a + served], query[a:a + served], key, value, 0.1)
    assert (out[q_cu[-1]:] == 7).all()


def test_more_tokens_than_total_keys_are_no_matter_where_nothing_is_unpacked(gpu):
    lengths, counts = [900, 100], [2, 2]
    cache, table, query, q_cu = make(gpu, 64, 4, 2, 32, lengths, counts)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for total in (0, 999):
        out = attend(gpu, cache, table, query, q_cu, lengths, 2, 0.1, total_keys=total)
        for i, n in enumerate(lengths):
            close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1)


def test_queries_without_a_bound_are_nan(gpu):
    cache, table, query, q_cu = make(gpu, 64, 4, 2, 32, [40], [2])
    assert torch.isnan(attend(gpu, cache, table, query, q_cu, [40], 0, 0.1)).all()


# ---- a scale that is no number

@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,path", [
    (64, 4, 2, [130, 0, 20], [2, 1, 30], WHOLE), (128, 4, 2, [900, 0, 20], [2, 1, 30], SPLIT),
    (64, 16, 2, [3000, 0, 20, 2900], [2000, 5, 30, 1900], UNPACKED)])
def test_a_scale_that_is_no_number_on_each_path(gpu, head_dim, heads, kv_heads, lengths, counts, path):
    """NaN for every request that holds tokens, zeros for the one that holds none, nothing behind the last."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 64, lengths, counts)
    query = torch.cat((query, query[:3]))
    total = sum(lengths)
    assert path_of(cache, heads, counts, query.shape[0], len(lengths), len(table[0]), total_keys=total) == path
    out = attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, q_cu, lengths,
                      max(counts), math.nan, total)
    for i, n in enumerate(lengths):
        rows = out[q_cu[i]:q_cu[i + 1]]
        assert torch.isnan(rows).all() if n else (rows == 0).all()
    assert (out[q_cu[-1]:] == 7).all()


# ---- the split path (shares of the keys, joined)

def attend_and_compare(device, path, head_dim, heads, kv_heads, block, lengths, counts, window=-1, causal=True, seed=0, width=None):
    cache, table, query, q_cu = make(device, head_dim, heads, kv_heads, block, lengths, counts, seed, width)
    n, scale = len(lengths), 1 / math.sqrt(head_dim)
    assert path_of(cache, heads, counts, sum(counts), n, len(table[0]), window) == path
    out = attend(device, cache, table, query, q_cu, lengths, max(counts), scale, causal=causal, window=window)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    for i, tokens in enumerate(lengths):
        if counts[i]:
            close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, tokens), scale, causal, window,
                  2.0 ** -8 if path == UNPACKED else 0.0)
    return out


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts", [
    (64, 4, 2, [1, 1, 1, 1, 1]), (64, 24, 2, [1, 2, 1, 0, 1]), (64, 24, 2, [5, 2, 1, 1, 4]), (128, 8, 4, [3, 1, 1, 7, 2]),
    (128, 40, 2, [1, 1, 1, 1, 0]), (128, 16, 2, [7, 1, 2, 5, 1]), (256, 6, 2, [4, 1, 1, 1, 5]), (256, 24, 2, [2, 1, 2, 1, 2]),
    (512, 8, 1, [1, 1, 2, 1, 1]), (512, 40, 2, [2, 1, 0, 1, 1]), (64, 80, 1, [2, 1, 1, 1, 1])])
def test_split(gpu, head_dim, heads, kv_heads, counts):
    """Every size of a workgroup's tile of query vectors, full and not: requests of one group and of many, one empty."""
    attend_and_compare(gpu, SPLIT, head_dim, heads, kv_heads, 32, [1300, 0, 33, 7, 800], counts)


@pytest.mark.parametrize("head_dim,heads,kv_heads,window", [(64, 4, 2, 700), (128, 4, 2, 651), (256, 4, 2, 1000), (512, 2, 1, 170),
                                                            (512, 4, 2, 200)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [5, 1, 32, 0, 9]])
def test_split_with_a_window(gpu, head_dim, heads, kv_heads, window, causal, counts):
    """Requests whose first groups no query sees, others within the window."""
    attend_and_compare(gpu, SPLIT, head_dim, heads, kv_heads, 64, [1500, 64, 1201, 0, 900], counts, window=window,
                       causal=causal)


def test_split_of_many_requests(gpu):
    """More than a workgroup's 256 threads take at once, twice: empty requests and requests without queries at those borders."""
    lengths, counts = [(37 * i) % 200 for i in range(700)], [1 + (i % 3 == 0) for i in range(700)]
    for i in (0, 254, 255, 256, 511, 512, 699):
        lengths[i] = 0
    for i in (1, 253, 255, 257, 510, 512, 513, 698, 699):
        counts[i] = 0
    lengths[300], lengths[514] = 900, 777
    attend_and_compare(gpu, SPLIT, 64, 4, 2, 32, lengths, counts)


@pytest.mark.parametrize("first,last", [(0, 256), (256, 512), (100, 101), (300, 300)])
def test_split_where_few_of_many_requests_have_queries(gpu, first, last):
    """Whole chunks of 256 requests without any, and a call without any at all."""
    lengths = [40] * 600
    lengths[0] = 700
    counts = [1 if first <= i < last else 0 for i in range(600)]
    cache, table, query, q_cu = make(gpu, 128, 4, 2, 32, lengths, counts or [0])
    query = torch.cat((query, torch.ones((2, 4, 128)).bfloat16()))
    assert path_of(cache, 4, [1], query.shape[0], 600, len(table[0])) == SPLIT
    out = attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, q_cu, lengths, 1,
                      0.1, 600 * len(table[0]) * 32)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for i in range(first, last, 7):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, lengths[i]), 0.1)
    assert torch.isfinite(out).all() and (out[q_cu[-1]:] == 7).all()


def test_split_without_tokens(gpu):
    """Queries of requests that hold nothing, in a table that could: zeros."""
    out = attend_and_compare(gpu, SPLIT, 128, 4, 2, 32, [0, 0, 0], [2, 1, 5], width=40)
    assert (out == 0).all()


def test_split_with_more_queries_than_tokens(gpu):
    out = attend_and_compare(gpu, SPLIT, 64, 4, 2, 32, [4, 900], [9, 2])
    assert (out[:5] == 0).all()


def test_split_bounds_out_of_range_write_nothing(gpu):
    """Query bounds past the query, decreasing or negative: their requests have no queries, the others theirs."""
    lengths = [900, 20, 800, 60]
    cache, table, query, _ = make(gpu, 64, 4, 2, 32, lengths, [2, 2, 2, 2])
    assert path_of(cache, 4, [2], 8, 4, len(table[0])) == SPLIT
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for bounds, good in (([0, 2, 4, 6, 9], (0, 1, 2)), ([-3, 2, 4, 6, 8], (1, 2, 3)), ([0, 2, 4, 3, 5], (0, 1, 3)),
                         ([9, 2, 4, 4, 2**31 - 1], (1,))):
        out = attend_into(gpu, torch.full_like(query, 7.0, device=gpu), cache, table, query, bounds, lengths, 2, 0.1, 4000)
        written = torch.zeros(8, dtype=torch.bool)
        for i in good:
            rows = slice(bounds[i], bounds[i + 1])
            written[rows] = True
            overlaps = bounds == [0, 2, 4, 3, 5] and i in (1, 3)  # (row 3 is two requests')
            if not overlaps:
                close(out[rows], query[rows], *want.rows(table[i], 0, lengths[i]), 0.1)
        assert (out[~written.to(gpu)] == 7).all()


def test_split_of_strided_queries_and_tables(gpu):
    lengths = [900, 40]
    cache, table, query, q_cu = make(gpu, 128, 4, 2, 32, lengths, [2, 1])
    wide = torch.zeros((3, 6, 160), dtype=torch.bfloat16, device=gpu)
    wide[:, 1:5, 16:144] = query.to(gpu)
    tables = torch.full((2, 50), 10 ** 6, dtype=torch.int32, device=gpu)
    tables[:, :len(table[0])] = ints(table, gpu)
    with torch.inference_mode():
        out = kv_cache.attend(wide[:, 1:5, 16:144], cache, tables[:, :len(table[0])], ints(q_cu, gpu), ints(lengths, gpu), 2, 0.1)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1)


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts,window", [(64, 4, 2, [6, 1], -1), (128, 8, 2, [9, 2], 700),
                                                                   (512, 8, 1, [2, 1], -1), (256, 16, 8, [16, 3], 650)])
def test_split_nan_reaches_the_queries_that_see_it_and_no_others(gpu, head_dim, heads, kv_heads, counts, window):
    """NaN in one element of a last token's value, and in another's key; with a window also in tokens that no query sees."""
    lengths, block = [1100, 833], 32
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, block, lengths, counts)
    assert path_of(cache, heads, counts, sum(counts), 2, len(table[0]), window) == SPLIT
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    raw_k, raw_v = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
    at = lengths[0] - 1
    raw_v[table[0][at // block], 0, oracle.value_offset(at % block, 5, head_dim)] = 0x7f
    at = lengths[1] - 1
    raw_k[table[1][at // block], 0, oracle.key_offset(at % block, 7, head_dim)] = 0xff
    if window >= 0:
        for i in range(2):  # the last token before every query's window
            at = lengths[i] - counts[i] - window - 1
            raw_v[table[i][at // block], :, oracle.value_offset(at % block, 3, head_dim)] = 0xff
            raw_k[table[i][at // block], :, oracle.key_offset(at % block, 9, head_dim)] = 0x7f
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, window=window)
    group = heads // kv_heads
    expected = torch.zeros(out.shape, dtype=torch.bool)
    expected[q_cu[1] - 1, :group, 5] = True
    expected[q_cu[2] - 1, :group] = True
    assert torch.equal(torch.isnan(out.cpu()), expected)
    for i, n in enumerate(lengths):
        rows = slice(q_cu[i], q_cu[i + 1] - 1)  # the queries before the last, which see neither
        if rows.start < rows.stop:
            key, value = want.rows(table[i], 0, n)
            close(out[rows], query[rows], key[:n - 1], value[:n - 1], 0.1, window=window)


def test_split_on_another_stream_and_beside_another_call(gpu):
    lengths, counts = [2000, 5, 900], [1, 2, 1]
    cache, table, query, q_cu = make(gpu, 128, 8, 2, 64, lengths, counts)
    assert path_of(cache, 8, counts, 4, 3, len(table[0])) == SPLIT
    args = (query.to(gpu), cache, ints(table, gpu), ints(q_cu, gpu), ints(lengths, gpu), 2, 0.1)
    with torch.inference_mode():
        want = kv_cache.attend(*args)
        streams = [torch.cuda.Stream(gpu) for _ in range(2)]
        got = []
        for i in range(8):
            with torch.cuda.stream(streams[i % 2]):
                if i < 2:
                    streams[i].wait_stream(torch.cuda.default_stream(gpu))
                got.append(kv_cache.attend(*args))
        torch.cuda.synchronize()
    for out in got:
        assert torch.equal(out, want)


@pytest.mark.parametrize("head_dim,heads,kv_heads,window", [(128, 8, 2, -1), (256, 4, 2, 700)])
def test_captured_split_calls_replay(gpu, head_dim, heads, kv_heads, window):
    """Two graphs of one call after another: each replay reads the lengths, bounds and queries of then."""
    most, counts = [2000, 1500, 900], [2, 1, 1]
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 64, most, counts)
    assert path_of(cache, heads, counts, 4, 3, len(table[0]), window) == SPLIT
    query, table, q_cu, lengths = query.to(gpu), ints(table, gpu), ints(q_cu, gpu), ints(most, gpu)

    def call():
        return kv_cache.attend(query, cache, table, q_cu, lengths, 2, 0.1, window=window)

    with torch.inference_mode():
        call()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = call()
            graphs.append((graph, out))
        seen = []
        for i, (change, bounds) in enumerate(((most, [0, 2, 3, 4]), ([1999, 0, 33], [0, 1, 3, 4]), ([32, 1500, 1], [0, 2, 2, 3]),
                                              ([0, 0, 5], [0, 0, 2, 4]), (most, [0, 2, 3, 4]))):
            lengths.copy_(ints(change, gpu))
            q_cu.copy_(ints(bounds, gpu))
            query.mul_(-0.75)
            graph, out = graphs[i % 2]
            out.zero_()
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(out[:bounds[-1]], want[:bounds[-1]]) and (out[bounds[-1]:] == 0).all()
            seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2]) and not torch.equal(seen[0], seen[4])


# ---- sums that cannot hide a mistake

def one_code(exponent):
    """The e4m3 code of 2^-exponent (tensor), -8 .. 6."""
    return ((7 - exponent) << 3).to(torch.uint8)


@pytest.mark.parametrize("head_dim,heads,kv_heads,block,lengths,counts", [
    (64, 1024, 1024, 64, [9000, 8300], [1, 1]), (512, 64, 64, 32, [9000, 8225], [64, 1]), (256, 512, 256, 128, [9000], [16]),
    (128, 512, 512, 32, [17000, 16600], [1, 1]), (128, 8, 2, 64, [20011, 700, 9001], [2, 1, 3]),
    (512, 4, 4, 128, [16001], [1])])
def test_each_group_of_tokens_counts(gpu, head_dim, heads, kv_heads, block, lengths, counts):
    """Equal scores, and values that are one in an element of their group's own: a group of 32 tokens left out, or read under
    another block's scale (they differ from block to block and head to head), shows in its element. In all but the last two
    cases a workgroup's share of one request is over 256 groups, 64 a wave, after which it looks up the table again."""
    assert max(counts) * heads // kv_heads <= 64 and max(lengths) > 640  # the split path
    gen = torch.Generator(device=gpu).manual_seed(1)
    used = [-(-x // block) for x in lengths]
    cache = kv_cache.create(sum(used), kv_heads, head_dim, block, device=gpu)
    exps = torch.randint(-8, 7, (sum(used), kv_heads, 2), generator=gen, device=gpu)
    cache.scales.copy_(torch.exp2(exps.float()))
    order = torch.randperm(sum(used), generator=gen, device=gpu).tolist()
    table = [[order.pop() for _ in range(u)] for u in used]
    keys, values = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
    tokens = range(block)
    keys[:, :, offsets_of(oracle.key_offset, tokens, [0] * block, head_dim, gpu)] = one_code(exps[..., :1])
    for row in table:
        for j, ident in enumerate(row):
            own = [(j * block + t) // 32 % head_dim for t in tokens]
            values[ident][:, offsets_of(oracle.value_offset, tokens, own, head_dim, gpu)] = one_code(exps[ident, :, 1:])
    query = torch.randn((sum(counts), heads, head_dim), generator=gen, device=gpu).bfloat16()
    query[..., 0] = 4.0
    width = max(used)
    table = [r + [-1] * (width - len(r)) for r in table]
    q_cu = [0]
    for c in counts:
        q_cu.append(q_cu[-1] + c)
    assert path_of(cache, heads, counts, sum(counts), len(lengths), width) == SPLIT
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 1.0).double()
    for i, n in enumerate(lengths):
        for r in range(counts[i]):
            sees = n - counts[i] + r + 1
            element = torch.arange(sees, device=gpu) // 32 % head_dim
            want = torch.bincount(element, minlength=head_dim).double() / sees
            off = (out[q_cu[i] + r] - want).abs()
            assert (off <= want * (2.0 ** -8 + 2.0 ** -14)).all(), (i, r, off.max())


def offsets_of(at, tokens, elements, head_dim, device):
    return torch.tensor([at(t, d, head_dim) for t, d in zip(tokens, elements)], device=device)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,path", [
    (64, 4, 2, [40, 90], WHOLE), (128, 8, 2, [40, 90], WHOLE), (256, 4, 4, [40, 90], WHOLE), (512, 4, 4, [40, 90], WHOLE),
    (64, 4, 2, [1000, 90], SPLIT), (128, 8, 2, [40, 1000], SPLIT), (256, 4, 2, [700, 90], SPLIT), (512, 4, 4, [40, 300], SPLIT),
    (64, 64, 2, [1000, 90], SPLIT), (128, 120, 2, [40, 1000], SPLIT), (256, 64, 2, [700, 90], SPLIT)])
def test_weights_are_as_fine_as_the_output(gpu, head_dim, heads, kv_heads, lengths, path):
    """Two tokens of nearly one score whose values cancel, in one group: a weight rounded to one bf16 term (2^-8 off) shows in
    the difference (tests/test_cache.py plants it), two terms (2^-17) do not."""
    block = 32
    cache, table, _, _ = make(gpu, head_dim, heads, kv_heads, block, lengths, [1, 1])
    keys, values = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
    keys.zero_(), values.zero_()
    cache.scales.fill_(1.0)
    for i in range(2):
        at = lengths[i] // 2 // 2 * 2
        ident, t = table[i][at // block], at % block
        keys[ident, :, oracle.key_offset(t, 0, head_dim)] = 0x38       # 1
        keys[ident, :, oracle.key_offset(t + 1, 0, head_dim)] = 0x36   # 7 / 8
        for d in range(head_dim):
            values[ident, :, oracle.value_offset(t, d, head_dim)] = 0x38
            values[ident, :, oracle.value_offset(t + 1, d, head_dim)] = 0xb8
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    assert path_of(cache, heads, [1, 1], 2, 2, len(table[0])) == path
    query = torch.zeros((2, heads, head_dim), dtype=torch.bfloat16)
    for start in (0.5, 1.7):
        query[..., 0] = start + torch.arange(2 * heads).view(2, heads) / 32
        out = attend(gpu, cache, table, query, [0, 1, 2], lengths, 1, 1.0)
        for i, n in enumerate(lengths):
            close(out[i:i + 1], query[i:i + 1], *want.rows(table[i], 0, n), 1.0)


# ---- the uses that the cache is for

@pytest.mark.parametrize("head_dim,heads,kv_heads,counts,path", [
    (128, 8, 2, [1] * 16, SPLIT), (128, 8, 2, [1] * 15 + [5], SPLIT), (64, 32, 2, [900] + [1] * 15, UNPACKED),
    (512, 8, 1, [2] * 16, SPLIT)])
def test_branches_over_one_prompt(gpu, head_dim, heads, kv_heads, counts, path):
    """Requests that share the whole blocks of one prompt, and each go on in blocks of their own."""
    block, prompt = 32, 31 * 32
    own = [max(counts[i], 1) + 3 * i for i in range(16)]
    lengths = [prompt + x for x in own]
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, block, lengths, counts)
    for row in table[1:]:
        row[:31] = table[0][:31]
    total = sum(lengths)
    assert path_of(cache, heads, counts, sum(counts), 16, len(table[0]), total_keys=total) == path
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, total_keys=total)
    want = oracle.Cache(cache.keys, cache.values, cache.scales, block)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1,
              weights=2.0 ** -8 if path == UNPACKED else 0.0)


def test_a_branch_that_copies_the_block_it_shares_in_part(gpu):
    """A second request over 80 tokens of a first, in blocks of 32: two blocks shared, the third, half full, copied; then both go
    on by tokens of their own, larger than the block's, so that its scale grows in one and not in the other."""
    block, heads, kv_heads, d = 32, 4, 2, 64
    cache = kv_cache.create(8, kv_heads, d, block, device=gpu)
    gen = torch.Generator().manual_seed(2)
    key, value = (torch.randn((80 + 2, kv_heads, d), generator=gen).bfloat16() for _ in range(2))
    key[81] *= 40
    value[81] *= 40
    table = torch.full((2, 4), -1, dtype=torch.int32, device=gpu)
    free, left = ints([0, 1, 2, 3, 4, 5, 6, 7], gpu), ints([8], gpu)
    with torch.inference_mode():
        first = kv_cache.reserve(table, ints([0, 0], gpu), ints([80, 0], gpu), free, left, 80, block)
        kv_cache.append(cache, key[:80].to(gpu), value[:80].to(gpu), first.writes)
        a, b = int(table[0, 2]), 0  # (block 0 is free: blocks are taken from the list's end)
        table[1, :2], table[1, 2] = table[0, :2], b
        for t in (cache.keys.view(torch.uint8), cache.values.view(torch.uint8), cache.scales):
            t[b] = t[a]
        second = kv_cache.reserve(table, ints([80, 80], gpu), ints([1, 1], gpu), free[1:].contiguous(), first.free_left - 1, 2, block)
        second.check()
        kv_cache.append(cache, key[80:].to(gpu), value[80:].to(gpu), second.writes)
        query = torch.randn((2, heads, d), generator=gen).bfloat16()
        out = kv_cache.attend(query.to(gpu), cache, table, second.q_cu, second.lengths, 1, 0.1)
    fed = kv_cache.create(8, kv_heads, d, block, device="cpu")
    want = oracle.Cache(fed.keys, fed.values, fed.scales, block)
    want.append(key[:80], value[:80], [[7, 0, 0, 32], [6, 0, 32, 32], [5, 0, 64, 16], [4, 0, 64, 16]])
    want.append(key[80:], value[80:], [[5, 16, 0, 1], [4, 16, 1, 1]])
    for i, blocks in enumerate(([7, 6, 5], [7, 6, 4])):
        close(out[i:i + 1], query[i:i + 1], *want.rows(blocks, 0, 81), 0.1)


@pytest.mark.parametrize("head_dim,heads,kv_heads,chunk,window", [(64, 4, 2, 200, -1), (64, 32, 2, 1000, -1), (256, 16, 8, 300, 511),
                                                                  (128, 8, 2, 40, 700)])
def test_a_chunk_among_single_tokens(gpu, head_dim, heads, kv_heads, chunk, window):
    lengths, counts = [1300, 40, 1, 900, 333], [chunk, 1, 1, 1, 0]
    cache, table, *_ = make(gpu, head_dim, heads, kv_heads, 64, lengths, counts)
    path = path_of(cache, heads, counts, sum(counts), 5, len(table[0]), window)
    attend_and_compare(gpu, path, head_dim, heads, kv_heads, 64, lengths, counts, window=window)


def test_append_converts_every_bf16_value(gpu):
    """All 65,536 bf16 values, in their order of magnitude, into blocks that hold one of nine scales already: codes and scales
    are those of the definition."""
    bits = torch.arange(65536, dtype=torch.int32)
    order = (bits & 0x7fff) * 2 + (bits >> 15)  # by magnitude, signs side by side
    x = bits[order.argsort()].to(torch.int16).view(torch.bfloat16).view(-1, 1, 64)  # 1,024 rows of 64
    writes = [[w, 1, 31 * w, min(31, 1024 - 31 * w)] for w in range(-(-1024 // 31))]
    for old in (-100, -61, -30, -9, -8, 0, 7, 60, 119):
        cache = kv_cache.create(len(writes), 1, 64, 32, device=gpu)
        cache.scales.fill_(2.0 ** old)
        want = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
        want.append(x, -x, writes)
        kv_cache.append(cache, x.to(gpu), (-x).to(gpu), ints(writes, gpu))
        got = oracle.Cache(cache.keys, cache.values, cache.scales, 32)
        assert torch.equal(got.exps, want.exps), old
        for a, b in zip(got.codes, want.codes):
            assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(9e9), b.nan_to_num(9e9)), old


def test_a_compiled_step_gives_what_the_calls_give(gpu):
    """torch.compile breaks its graph around the calls: each sees the tensors of its own step, not those of the traced one."""
    def step(cache, table, lengths, counts, free, left, key, value, query):
        got = kv_cache.reserve(table, lengths, counts, free, left, 47, 32)
        kv_cache.append(cache, key * 2, value, got.writes)
        k, v, _ = kv_cache.read(cache, table, got.lengths, 47)
        return kv_cache.attend(query + 1, cache, table, got.q_cu, got.lengths, 40, 0.1) * 2, k + 1, v

    def inputs(seed):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        rows = [torch.randn((47, h, 64), generator=gen, device=gpu).bfloat16() for h in (2, 2, 4)]
        return (kv_cache.create(20, 2, 64, 32, device=gpu), torch.full((2, 6), -1, dtype=torch.int32, device=gpu),
                ints([0, 0], gpu), ints([40, 7], gpu), torch.arange(20, dtype=torch.int32, device=gpu), ints([20], gpu), *rows)

    torch._dynamo.reset()
    compiled, kept = torch.compile(step, backend="eager"), []
    with torch.inference_mode():
        for seed in range(3):
            kept.append(inputs(seed))  # (kept, so that the next step's tensors lie elsewhere)
            for a, b in zip(compiled(*kept[-1]), step(*inputs(seed))):
                assert torch.equal(a, b)
