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


def path_of(cache, heads, counts, rows, n, width, window=-1, total_keys=None):
    """The path that a call of these sizes takes, by the workspace it asks for."""
    max_q = max(counts)
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
