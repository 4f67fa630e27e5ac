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
    # the unpacked rows, two bytes an element, keys and values; the split path's partials are vectors of fp32: its size is
    # the same for any number of keys past the bound of the first path
    a.total_keys, more = total + 4096, ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(more)), "bytes")
    if window >= 0:
        return UNPACKED if need.value > 4 * min(total, n * (max_q + window)) * cache.kv_heads * cache.head_dim else SPLIT
    return SPLIT if more.value == need.value else UNPACKED


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
