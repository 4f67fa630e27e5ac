"""Caches in 4 bits, calls over them and attention's tolerance, for the GPU tests of the block cache in 4 bits."""

from __future__ import annotations

import ctypes

import torch

from karpo_decision_amd import _lib, kv_cache
from oracle import cache4 as oracle

WHOLE, SPLIT, UNPACKED = "whole", "split", "unpacked"


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def raw(t):
    return t.view(torch.uint8)


def random_cache(device, blocks, kv_heads, head_dim, block, seed):
    """Every byte a code or a scale, some scales NaN."""
    gen = torch.Generator().manual_seed(seed)
    cache = kv_cache.create(blocks, kv_heads, head_dim, block, device=device, bits=4)
    for t in cache[:2]:
        raw(t).copy_(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
    e = torch.randint(117, 123, cache.scales.shape, generator=gen, dtype=torch.uint8)
    e[torch.rand(e.shape, generator=gen) < 0.02] = 255
    raw(cache.scales).copy_(e)
    return cache


def copy_of(cache):
    return kv_cache.Cache(*(raw(t).clone().view(t.dtype) for t in cache[:3]), cache.block_size)


def make(device, head_dim, heads, kv_heads, block, lengths, counts, seed=0, width=None):
    """(cache, table, query, q_cu): no NaN in the tokens in use, NaN among the leftovers behind them and in unused blocks."""
    gen = torch.Generator().manual_seed(seed)
    used = [-(-x // block) for x in lengths]
    width = max(1, max(used)) if width is None else width
    pool = (torch.randperm(sum(used) + 3, generator=gen) + 1).tolist()  # block 0 is nobody's
    cache = random_cache(device, sum(used) + 4, kv_heads, head_dim, block, seed + 1)
    table = [[pool.pop() for _ in range(u)] for u in used]
    scales = raw(cache.scales).cpu().view(cache.blocks, kv_heads, -1)
    scales[torch.rand(scales.shape, generator=gen) < 0.3] = 255
    for value in (False, True):
        at = oracle.offsets(block, head_dim, value)[1][:, ::32]
        for row, x in zip(table, lengths):
            for j, ident in enumerate(row):
                mine = at[:min(block, x - j * block)].reshape(-1)
                scales[ident][:, mine] = torch.randint(118, 121, (kv_heads, len(mine)), generator=gen, dtype=torch.uint8)
    raw(cache.scales).copy_(scales.view(cache.scales.shape))
    table = [r + [-1] * (width - len(r)) for r in table]
    query = torch.randn((sum(counts), heads, head_dim), generator=gen).bfloat16()
    q_cu = [0]
    for c in counts:
        q_cu.append(q_cu[-1] + c)
    return cache, table, query, q_cu


def values_of(cache):
    return oracle.Cache(cache.keys, cache.values, cache.scales, cache.block_size)


def path_of(cache, heads, max_q, rows, n, width, window=-1, total_keys=None):
    """The path that a call of these sizes takes, by the workspace it asks for."""
    total = n * width * cache.block_size if total_keys is None else total_keys
    c = _lib.KarpoCache4(*(t.data_ptr() for t in cache[:3]), cache.blocks, cache.kv_heads, cache.head_dim, cache.block_size)
    a = _lib.KarpoCache4AttendArgs(c, 4096, 4096, 8, 8, 8, 8, 4096, 4096, 4096, width, width, n, heads, max_q, rows, total,
                                   0.1, window, 0)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache4_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
    if need.value == 0:
        return WHOLE
    # the split path's: the units before each request, and for every share two partials of a tile's vectors in fp32
    d, vectors = cache.head_dim, max_q * heads // cache.kv_heads
    most = 4 if d <= 128 else 2 if d == 256 else 1
    nt = next(t for t in (1, 2, 4) if t == most or vectors <= 16 * t)
    waves = 4 if (d, nt) == (64, 1) else 3 if (d, nt) in ((64, 2), (128, 1)) else 2 if d <= 128 or (d, nt) == (256, 1) else 1
    y = cache.kv_heads * -(-vectors // (16 * nt))
    split = -(-4 * (n + 2) // 256) * 256 + y * max(1, 256 * waves // y) * 2 * 16 * nt * (d + 2) * 4
    return SPLIT if need.value == split else UNPACKED


def attend(device, cache, table, query, q_cu, lengths, max_q, scale, **more):
    with torch.inference_mode():
        return kv_cache.attend(query.to(device), cache, ints(table, device), ints(q_cu, device), ints(lengths, device),
                               max_q, scale, **more)


def close(out, query, key, value, scale, causal=True, window=-1, weights=0.0):
    """One request's rows within, per element, the output's rounding to bf16 (2^-8 of its magnitude) plus 2^-14 of the weighted
    mean of |value|: the weights enter the products as two bf16 terms (2^-17 off); the scores (below 2^6 here) are off by a few of
    their 2^-18 steps and by the queries' second e4m3 term, 2^-22 of the largest of 32 elements of a query times the sum of
    their keys' magnitudes (below 2^-22 * 4 * 32 * 2^-4 * 16 groups here), so the weights by less than 2^-15. ``weights``: what
    the path's weights are off (2^-8 where they are one bf16 term)."""
    if query.shape[0] == 0:
        return
    query, key, value = (t.to(out.device).double() for t in (query, key, value))
    want = oracle.attention_whole(query, key, value, scale, causal, window)
    size = oracle.attention_whole(query, key, value.abs(), scale, causal, window)
    off = (out.double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + size * (weights + 2.0 ** -14)
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), f"off {off.max():.3e}, worst {(off / bound.clamp(min=1e-30)).max():.2f} of the bound"


def check_attend(device, head_dim, heads, kv_heads, block, lengths, counts, path=None, window=-1, causal=True, scale=None, seed=0,
                 total_keys=True):
    scale = head_dim ** -0.5 if scale is None else scale
    cache, table, query, q_cu = make(device, head_dim, heads, kv_heads, block, lengths, counts, seed)
    total = sum(lengths) if total_keys else None
    took = path_of(cache, heads, max(counts), sum(counts), len(lengths), len(table[0]), window, total)
    assert path is None or took == path, took
    out = attend(device, cache, table, query, q_cu, lengths, max(counts), scale, causal=causal, window=window, total_keys=total)
    want = values_of(cache)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), scale, causal, window,
              weights=2.0 ** -8 if took == UNPACKED else 0.0)
    return cache, table, query, q_cu, out
