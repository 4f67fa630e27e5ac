"""The block cache in 4 bits on the GPU against the oracle's loops and 64-bit sums (oracle/cache4.py). Codes and scales of bf16
rows have to be equal; attention's tolerance is ``cache4_cases.close``'s."""

from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from cache4_cases import (SPLIT, UNPACKED, WHOLE, attend, check_attend, close, copy_of, ints, make, path_of, random_cache, raw,
                          values_of)
from karpo_decision_amd import _lib, kv_cache
from oracle import cache4 as oracle

pytestmark = pytest.mark.gpu


# ---- append

def _same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(9e9), b.nan_to_num(9e9))


def _append_and_compare(cache, key, value, writes):
    """The whole cache after ``append`` against the oracle's, and the bytes of what no write names."""
    before, want = copy_of(cache), values_of(cache)
    want.append(key, value, writes)
    kv_cache.append(cache, key, value, ints(writes, cache.keys.device))
    got = values_of(cache)
    reached = torch.zeros((cache.blocks, cache.block_size), dtype=torch.bool)
    for ident, first, _, count in writes:
        reached[ident, first:first + count] = True
    for side in (0, 1):
        assert _same(got.values[side], want.values[side])
        at, scale_at = oracle.offsets(cache.block_size, cache.head_dim, bool(side))
        for old, new, where in ((before[side], cache[side], at), (before.scales, cache.scales, scale_at)):
            old, new = (raw(t).cpu().reshape(cache.blocks, cache.kv_heads, -1)[:, :, where.reshape(-1)]
                        .view(cache.blocks, cache.kv_heads, cache.block_size, -1) for t in (old, new))
            assert ((old == new).all(-1).all(1) | reached).all()


@pytest.mark.parametrize("head_dim", [64, 128, 256, 512])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_append(gpu, head_dim, block):
    """Whole blocks, one token, tokens that begin and end inside a group of 32, each over leftovers of other requests."""
    cache = random_cache(gpu, 9, 3, head_dim, block, seed=head_dim + block)
    gen = torch.Generator(device=gpu).manual_seed(1)
    rows = 2 * block + 60
    key, value = (torch.randn((rows, 3, head_dim), generator=gen, device=gpu).bfloat16() for _ in range(2))
    value[::7] *= 50
    key[3::11] *= 300
    writes = [[2, 0, 0, block], [5, 0, block, 1], [0, 17, block + 1, 1], [7, block - 1, block + 2, 1],
              [1, 3, block + 3, 21], [3, 11, block + 24, block - 11], [8, 0, 2 * block + 13, 13], [6, 30, 2 * block + 26, 2],
              [4, 0, 2 * block + 28, 32]]
    _append_and_compare(cache, key, value, writes)


def test_append_reads_strided_rows_and_leaves_others(gpu):
    cache = random_cache(gpu, 4, 2, 128, 32, seed=3)
    packed = torch.randn((50, 6, 160), device=gpu).bfloat16()
    key, value = packed[:, 1:3, :128], packed[:, 4:, 32:]
    assert key.stride() == (960, 160, 1)
    _append_and_compare(cache, key, value, [[1, 5, 40, 10], [3, 0, 2, 32]])


def test_append_extremes(gpu):
    """Zeros, the least and largest bf16 values, infinities and NaN."""
    cache = random_cache(gpu, 9, 1, 64, 32, seed=4)
    key = torch.zeros((9, 1, 64), dtype=torch.bfloat16, device=gpu)
    key[1] = 9.2e-41
    key[2, :, ::2] = 3.3895e38
    key[3, :, 1], key[3, :, 2], key[3, :, 3], key[3, :, 4] = math.inf, -math.inf, math.nan, 0.37
    key[4] = math.inf
    key[5] = math.nan
    key[6] = -1.0e30
    key[7] = torch.linspace(-7, 7, 64)
    key[8, :, 40], key[8, :, 41], key[8, :, 42] = math.inf, 0.01, -0.003
    _append_and_compare(cache, key, key.flip(0).contiguous(), [[i, 0 if i % 2 else 9, i, 1] for i in range(9)])


def test_append_rounds_every_bf16_value(gpu):
    """All finite bf16 values, under the scale of 6 * 2^e for several e, ties and the borders of the range among them."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    fine = every[torch.isfinite(every.float())]
    for e in (0, -60, 100):
        top = torch.tensor(6.0 * 2.0 ** e).bfloat16()
        part = fine[(fine.float().abs() <= top.float()) & (fine.float().abs() >= 2.0 ** (e - 4))]
        part = torch.cat((part, part.new_zeros(-part.numel() % 31))).view(-1, 31)
        x = torch.cat((part, top.expand(part.shape[0], 1)), 1)
        x = torch.cat((x, x.new_zeros((-x.shape[0] % 2, 32)))).view(-1, 1, 64)
        cache = kv_cache.create(-(-x.shape[0] // 32), 1, 64, 32, device=gpu, bits=4)
        writes = [[i, 0, 32 * i, min(32, x.shape[0] - 32 * i)] for i in range(cache.blocks)]
        _append_and_compare(cache, x.to(gpu), -x.to(gpu), writes)


def test_append_skips_writes_out_of_range(gpu):
    cache = random_cache(gpu, 3, 2, 64, 32, seed=5)
    before = copy_of(cache)
    rows = torch.randn((10, 2, 64), device=gpu).bfloat16()
    writes = [[3, 0, 0, 4], [-1, 0, 0, 4], [0, 30, 0, 4], [0, -1, 0, 4], [1, 0, 8, 4], [1, 0, -1, 4], [2, 0, 0, 0], [2, 0, 0, -3],
              [2**31 - 1, 0, 0, 1], [0, 32, 0, 1], [0, 0, 2**31 - 1, 2**31 - 1], [0, 2**31 - 1, 0, 2]]
    kv_cache.append(cache, rows, rows, ints(writes, gpu))
    for a, b in zip(before[:3], cache[:3]):
        assert torch.equal(raw(a), raw(b))


@pytest.mark.parametrize("n", [1, 7, 8, 9, 17])
def test_append_of_several_writes(gpu, n):
    cache = random_cache(gpu, n, 2, 64, 32, seed=n)
    rows = torch.randn((3 * n, 2, 64), device=gpu).bfloat16()
    _append_and_compare(cache, rows, rows * 2, [[n - 1 - i, i % 30, 3 * i, 1 + i % 3] for i in range(n)])


def test_append_without_rows_or_writes(gpu):
    cache = random_cache(gpu, 2, 2, 64, 32, seed=6)
    before = copy_of(cache)
    none = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device=gpu)
    kv_cache.append(cache, none, none, ints([[0, 0, 0, 1]], gpu))
    kv_cache.append(cache, none, none, torch.zeros((0, 4), dtype=torch.int32, device=gpu))
    for a, b in zip(before[:3], cache[:3]):
        assert torch.equal(raw(a), raw(b))


def test_blocks_past_32_bit_offsets(gpu):
    """Append, read and attend at a block whose codes start past 2^31 bytes."""
    block, head_dim, heads, ident = 128, 512, 4, 16500  # 131,072 bytes a block: past 2^31 from block 16,384 on
    cache = kv_cache.Cache(*(torch.empty((16503, heads, block * head_dim // 2), dtype=torch.uint8, device=gpu)
                             .view(torch.float4_e2m1fn_x2) for _ in range(2)),
                           torch.empty((16503, heads, block // 32, 2, head_dim), dtype=torch.uint8, device=gpu)
                           .view(torch.float8_e8m0fnu), block)
    gen = torch.Generator(device=gpu).manual_seed(6)
    key, value = (torch.randn((40, heads, head_dim), generator=gen, device=gpu).bfloat16() for _ in range(2))
    kv_cache.append(cache, key, value, ints([[ident, 0, 0, 40]], gpu))
    got_k, got_v, k_cu = kv_cache.read(cache, ints([[ident]], gpu), ints([40], gpu), 40)
    assert k_cu.tolist() == [0, 40]
    for got, x in ((got_k, key), (got_v, value)):
        assert torch.equal(got.cpu().double(), oracle.quantised(x.cpu().double()))
    query = torch.randn((1, 8, head_dim), generator=gen, device=gpu).bfloat16()
    out = attend(gpu, cache, [[ident]], query, [0, 1], [40], 1, 0.04)
    close(out, query, got_k, got_v, 0.04)


# ---- read

@pytest.mark.parametrize("head_dim,block,lengths", [
    (64, 32, [1, 0, 33, 70]), (128, 64, [200, 64, 5, 0, 0, 129]), (256, 128, [31, 300]), (512, 32, [95, 1]),
    (128, 32, [(7 * i) % 90 for i in range(300)])])
def test_read(gpu, head_dim, block, lengths):
    width = max(1, -(-max(lengths) // block)) + 1
    cache = random_cache(gpu, 40, 2, head_dim, block, seed=7)
    table = [[(i * 11 + j * 7) % 40 for j in range(width)] for i in range(len(lengths))]
    if len(table) > 2:
        table[2][0] = -1  # reads as zeros
        table[3][0] = 40
    rows = sum(lengths) + 3
    key, value, k_cu = kv_cache.read(cache, ints(table, gpu), ints(lengths, gpu), rows)
    assert key.shape == value.shape == (rows, 2, head_dim)
    want, at = values_of(cache), 0
    for i, n in enumerate(lengths):
        assert k_cu[i].item() == at
        for got, w in zip((key, value), want.rows(table[i], 0, n)):
            assert _same(got[at:at + n].cpu().double(), w)
        at += n
    assert k_cu[-1].item() == at


def test_read_writes_no_row_past_its_bound(gpu):
    """Lengths whose sum is past ``rows``, below zero and past the table's row."""
    from karpo_decision_amd import ops
    cache = random_cache(gpu, 4, 1, 64, 32, seed=8)
    table = ints([[0, 1], [2, 3], [1, 2]], gpu)
    backing = torch.full((2, 200, 64), 3.125, dtype=torch.bfloat16, device=gpu)  # (no value of the cache)
    lengths, k_cu = ints([-5, 1000, 40], gpu), torch.empty(4, dtype=torch.int32, device=gpu)
    c = _lib.KarpoCache4(*(t.data_ptr() for t in cache[:3]), 4, 1, 64, 32)
    args = _lib.KarpoCache4ReadArgs(c, table.data_ptr(), 2, 2, 3, lengths.data_ptr(), backing[0].data_ptr(),
                                    backing[1].data_ptr(), 90, k_cu.data_ptr())
    _lib.check(_lib.load().karpo_cache4_read(ctypes.byref(args), ops._current_stream(0)), "read")
    assert k_cu.tolist() == [0, 0, 64, 104]
    assert (backing[:, 90:] == 3.125).all() and not (backing[:, :90] == 3.125).any()


def test_read_of_many_rows(gpu):
    """More rows than the L2 caches hold are stored through them."""
    cache = random_cache(gpu, 140, 8, 128, 128, seed=9)
    table = [list(range(139, -1, -1))]
    key, value, _ = kv_cache.read(cache, ints(table, gpu), ints([140 * 128 - 5], gpu), 140 * 128 - 5)
    assert 4 * key.numel() > 32 << 20
    want = values_of(cache)
    for got, full in zip((key, value), want.values):
        rows = full.flip(0).transpose(1, 2).reshape(-1, 8, 128)[:key.shape[0]]
        assert _same(got.cpu().double(), rows)


# ---- attend

@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (128, 4, 4), (128, 16, 2), (256, 6, 2), (512, 8, 1),
                                                     (512, 3, 3), (64, 40, 1)])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_decode(gpu, head_dim, heads, kv_heads, block):
    """One token per request: lengths of one, around groups and blocks, one longer; leftovers hold NaN scales."""
    check_attend(gpu, head_dim, heads, kv_heads, block, [1, 32, 33, 31, 64, 65, 128, 129, 700, 0], [1] * 10, SPLIT, total_keys=False)


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (128, 4, 4), (256, 6, 2), (512, 8, 1)])
@pytest.mark.parametrize("block", [32, 64])
def test_decode_of_short_requests(gpu, head_dim, heads, kv_heads, block):
    """Requests that one workgroup takes whole."""
    check_attend(gpu, head_dim, heads, kv_heads, block, [1, 32, 33, 31, 64, 65, 97, 0, 128], [1] * 9, WHOLE)


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts", [
    (128, 8, 4, [3, 1, 0, 7]), (64, 8, 2, [5, 5, 5, 5]), (256, 16, 8, [4, 2, 1, 1]), (512, 32, 4, [2, 3, 1, 2]),
    (128, 16, 2, [13, 1, 2, 9]), (64, 4, 1, [7, 16, 3, 12])])
def test_a_few_tokens_each(gpu, head_dim, heads, kv_heads, counts):
    check_attend(gpu, head_dim, heads, kv_heads, 64, [100, 40, 63, 913], counts, SPLIT, total_keys=False)


@pytest.mark.parametrize("window", [0, 5, 40, 63, 64, 100])
@pytest.mark.parametrize("causal", [True, False])
def test_windows(gpu, window, causal):
    check_attend(gpu, 128, 4, 2, 32, [300, 64, 1, 37], [3, 1, 1, 30], window=window, causal=causal)
    check_attend(gpu, 64, 4, 2, 32, [300, 64, 1, 37], [1, 1, 1, 1], window=window, causal=causal)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,window", [
    (128, 4, 2, [300, 170], [130, 170], -1), (256, 4, 2, [500], [200], 99), (64, 8, 2, [400, 0, 90], [90, 0, 90], -1),
    (512, 4, 1, [260, 33], [120, 33], -1)])
def test_chunks_of_prompts(gpu, head_dim, heads, kv_heads, lengths, counts, window):
    check_attend(gpu, head_dim, heads, kv_heads, 64, lengths, counts, window=window)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,window,causal", [
    (64, 32, 2, [5100, 3000], [1500, 900], -1, True), (128, 32, 4, [3000, 1777], [1500, 1777], -1, True),
    (128, 32, 4, [3000, 2100, 0, 40], [1500, 1000, 3, 41], 600, True), (256, 16, 2, [2500, 1900], [800, 700], -1, False),
    (256, 16, 2, [2500, 2900], [900, 800], 333, True), (512, 8, 1, [2000, 900], [700, 900], -1, True)])
def test_long_chunks(gpu, head_dim, heads, kv_heads, lengths, counts, window, causal):
    """Chunks long enough that the keys are unpacked first."""
    check_attend(gpu, head_dim, heads, kv_heads, 64, lengths, counts, UNPACKED, window=window, causal=causal)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts", [
    (64, 16, 1, [700, 41], [70, 41]), (128, 24, 2, [1100, 300], [100, 7]), (256, 12, 1, [900], [60]),
    (512, 16, 1, [500, 64], [30, 64])])
def test_many_tiles_of_queries(gpu, head_dim, heads, kv_heads, lengths, counts):
    """The split path with several workgroups for a request's query vectors, the last of them not full."""
    check_attend(gpu, head_dim, heads, kv_heads, 32, lengths, counts, SPLIT, total_keys=False)
    assert max(counts) * heads // kv_heads > 64


def test_more_queries_than_tokens(gpu):
    """Queries before the first token see nothing: zeros."""
    for counts in ([9, 5], [90, 70]):
        out = check_attend(gpu, 64, 4, 2, 32, [4, 0], counts)[4]
        assert (out[:counts[0] - 4] == 0).all() and (out[counts[0]:] == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_scales(gpu, scale, head_dim):
    check_attend(gpu, head_dim, 4, 2, 32, [130, 20], [1, 2], scale=scale)


def test_a_scale_that_is_no_number(gpu):
    for lengths, counts, heads in (([130, 20], [1, 1], 4), ([900, 20], [1, 1], 4), ([3000, 2900], [2000, 1900], 16)):
        cache, table, query, q_cu = make(gpu, 64, heads, 2, 32, lengths, counts)
        out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), math.nan, total_keys=sum(lengths))
        assert torch.isnan(out).all()


def test_many_requests(gpu):
    lengths = [(37 * i) % 200 for i in range(600)]
    check_attend(gpu, 64, 4, 2, 32, lengths, [1 + (i % 3 == 0) for i in range(600)])
    check_attend(gpu, 64, 4, 2, 32, lengths[:-1] + [1500], [1 + (i % 3 == 0) for i in range(600)], SPLIT, total_keys=False)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths", [(64, 8, 2, [257, 260, 640, 31, 0, 511]), (128, 3, 3, [640, 300, 1]),
                                                             (256, 8, 1, [290, 640, 639])])
@pytest.mark.parametrize("window", [-1, 0, 290])
def test_whole_requests_by_twice_the_waves(gpu, head_dim, heads, kv_heads, lengths, window):
    """One workgroup of eight waves a request, some without a group of 32 tokens; the window's begin inside a group."""
    check_attend(gpu, head_dim, heads, kv_heads, 32, lengths, [1] * len(lengths), WHOLE, window=window, total_keys=False)
    check_attend(gpu, head_dim, heads, kv_heads, 64, lengths, [2] * len(lengths), WHOLE, window=window, causal=False)


@pytest.mark.parametrize("head_dim,kv_heads,requests,more", [(64, 2, 70, 1), (128, 3, 48, 4), (256, 1, 130, 1), (512, 4, 33, 3)])
def test_long_walks_of_many_requests(gpu, head_dim, kv_heads, requests, more):
    """Workgroups that take up to 1,024 tokens whole, 1,280 of head sizes below 512."""
    longest = 1024 if head_dim == 512 else 1280
    lengths = [(337 * i) % (longest + 1) for i in range(requests - 1)] + [longest]
    counts = [i % (more + 1) for i in range(requests - 1)] + [more]
    check_attend(gpu, head_dim, 2 * kv_heads, kv_heads, 64, lengths, counts, WHOLE, total_keys=False)


@pytest.mark.parametrize("seed", range(int(os.environ.get("KARPO_RANDOM_BATCHES", "16"))))
def test_random_batches(gpu, seed):
    """Requests of every kind together: empty ones, short and long ones, none, one or many queries, with and without a window."""
    gen = torch.Generator().manual_seed(1000 + seed)

    def one_of(*choices):
        return choices[int(torch.randint(len(choices), (1,), generator=gen))]

    def up_to(most):  # evenly over the logarithm
        return int(2.0 ** (torch.rand(1, generator=gen).item() * math.log2(most + 1))) - 1

    head_dim, kv_heads, group, block = one_of(64, 128, 256, 512), one_of(1, 2, 3), one_of(1, 2, 5, 8), one_of(32, 64, 128)
    requests, longest, most = 1 + up_to(400), one_of(90, 1100, 5000), one_of(1, 1, 4, 40)
    lengths, counts = [], []
    while len(lengths) < requests and sum(lengths) < 40000:
        lengths.append(up_to(longest))
        counts.append(min(one_of(0, 1, 1, most), lengths[-1] + 1))
    counts[0] = max(1, counts[0])
    check_attend(gpu, head_dim, kv_heads * group, kv_heads, block, lengths, counts, window=one_of(-1, -1, 0, 100, 1000),
                 causal=one_of(True, True, False), seed=seed, total_keys=one_of(True, False))


@pytest.mark.parametrize("head_dim,kv_heads", [(64, 2), (128, 2), (256, 1), (512, 1)])
def test_one_long_request(gpu, head_dim, kv_heads):
    check_attend(gpu, head_dim, 4, kv_heads, 64, [9001], [1], SPLIT)


@pytest.mark.parametrize("head_dim", [64, 128, 256, 512])
def test_each_group_of_a_long_request_shows(gpu, head_dim):
    """Scores so even that every token counts, and values of one sign: a group left out or taken twice is off by 1/140."""
    lengths, counts = [4480 + 37], [2]
    cache, table, query, q_cu = make(gpu, head_dim, 4, 1, 64, lengths, counts)
    raw(cache.values).bitwise_and_(0x77)
    out = attend(gpu, cache, table, query, q_cu, lengths, 2, 1e-4)
    key, value = values_of(cache).rows(table[0], 0, lengths[0])
    close(out, query, key, value, 1e-4)


def test_queries_of_all_magnitudes(gpu):
    """Elements from 2^-20 to 2^6 side by side in a query: the two e4m3 terms hold those that matter."""
    lengths, counts = [300, 70], [1, 2]
    cache, table, query, q_cu = make(gpu, 128, 4, 2, 32, lengths, counts)
    gen = torch.Generator().manual_seed(5)
    query = (query.float() * torch.exp2(torch.randint(-20, 5, query.shape, generator=gen).float())).bfloat16()
    out = attend(gpu, cache, table, query, q_cu, lengths, 2, 0.02)
    want = values_of(cache)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.02)


def test_strided_queries_and_tables(gpu):
    cache, table, query, q_cu = make(gpu, 128, 4, 2, 32, [90, 40], [2, 1], width=7)
    wide = torch.zeros((3, 6, 160), dtype=torch.bfloat16, device=gpu)
    wide[:, 1:5, 16:144] = query.to(gpu)
    tables = torch.full((2, 20), 10 ** 6, dtype=torch.int32, device=gpu)
    tables[:, :7] = ints(table, gpu)
    with torch.inference_mode():
        out = kv_cache.attend(wide[:, 1:5, 16:144], cache, tables[:, :7], ints(q_cu, gpu), ints([90, 40], gpu), 2, 0.1)
    want = values_of(cache)
    for i, n in enumerate([90, 40]):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1)


@pytest.mark.parametrize("head_dim,heads,lengths,counts,path", [
    (64, 4, [130, 100], [1, 2], WHOLE), (128, 4, [400, 300], [2, 1], WHOLE), (64, 4, [900, 100], [1, 2], SPLIT),
    (128, 4, [900, 100], [1, 1], SPLIT),
    (256, 4, [900, 100], [2, 1], SPLIT), (512, 4, [300, 100], [1, 1], SPLIT), (64, 16, [3000, 2900], [2000, 1900], UNPACKED)])
def test_unknown_blocks_read_as_zeros(gpu, head_dim, heads, lengths, counts, path):
    """Beside a block 0 all of whose scales are NaN."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, 2, 32, lengths, counts)
    assert path_of(cache, heads, max(counts), sum(counts), 2, len(table[0])) == path
    raw(cache.scales)[0] = 255
    table[0][1], table[1][2] = -1, cache.blocks
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1)
    want = values_of(cache)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1,
              weights=2.0 ** -8 if path == UNPACKED else 0.0)


def _attend_into(device, out, cache, table, query, q_cu, lengths, max_q, scale, total_keys):
    """``attend`` by the C ABI, into ``out`` (contiguous)."""
    from karpo_decision_amd import ops
    q, cu, n, dev_table = query.to(device), ints(q_cu, device), ints(lengths, device), ints(table, device)
    rows, heads, d = q.shape
    c = _lib.KarpoCache4(*(t.data_ptr() for t in cache[:3]), cache.blocks, cache.kv_heads, d, cache.block_size)
    a = _lib.KarpoCache4AttendArgs(c, q.data_ptr(), out.data_ptr(), heads * d, d, heads * d, d, cu.data_ptr(), n.data_ptr(),
                                   dev_table.data_ptr(), len(table[0]), len(table[0]), len(table), heads, max_q, rows,
                                   total_keys, scale, -1, 0)
    need = ctypes.c_size_t()
    _lib.check(_lib.load().karpo_cache4_attend_workspace_bytes(ctypes.byref(a), ctypes.byref(need)), "bytes")
    workspace = torch.empty(need.value + 16, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need.value
    _lib.check(_lib.load().karpo_cache4_attend(ctypes.byref(a), ops._current_stream(0)), "attend")
    return out


@pytest.mark.parametrize("bounds,good", [([0, 2, 4, 6, 9], (0, 1, 2)), ([-3, 2, 4, 6, 8], (1, 2, 3))])
def test_bounds_out_of_range_write_nothing(gpu, bounds, good):
    """Query bounds past the query or negative: their requests have no queries, the others theirs."""
    lengths = [130, 20, 50, 60]
    cache, table, query, _ = make(gpu, 64, 4, 2, 32, lengths, [2] * 4)
    out = _attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, bounds, lengths,
                       2, 0.1, 260)
    want, written = values_of(cache), torch.zeros(8, dtype=torch.bool, device=gpu)
    for i in good:
        rows = slice(bounds[i], bounds[i + 1])
        written[rows] = True
        close(out[rows], query[rows], *want.rows(table[i], 0, lengths[i]), 0.1)
    assert (out[~written] == 7).all()


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,max_q,path", [
    (64, 4, 2, [130, 100], [5, 2], 2, WHOLE), (256, 4, 2, [530, 400, 0], [5, 2, 3], 2, WHOLE), (512, 4, 2, [100, 60], [9, 1], 1, WHOLE),
    (64, 4, 2, [900, 100, 0], [5, 3, 3], 2, SPLIT), (64, 80, 2, [900, 700], [7, 2], 2, SPLIT),
    (256, 4, 2, [900, 100], [1, 40], 33, SPLIT), (512, 4, 2, [300, 100], [9, 9], 1, SPLIT)])
def test_queries_past_max_q_are_nan(gpu, head_dim, heads, kv_heads, lengths, counts, max_q, path):
    n = len(lengths)
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    query = torch.cat((query, query[:3]))
    assert path_of(cache, heads, max_q, query.shape[0], n, len(table[0])) == path
    out = _attend_into(gpu, torch.full(query.shape, 7.0, dtype=torch.bfloat16, device=gpu), cache, table, query, q_cu, lengths,
                       max_q, 0.1, n * len(table[0]) * 32)
    want = values_of(cache)
    for i, length in enumerate(lengths):
        done = min(max_q, counts[i])
        rows = slice(q_cu[i], q_cu[i] + done)
        key, value = want.rows(table[i], 0, length)
        # the queries sit at the request's last tokens, of all its rows
        full = oracle.attention_whole(query[q_cu[i]:q_cu[i + 1]].double(), key, value, 0.1, True, -1)[:done]
        size = oracle.attention_whole(query[q_cu[i]:q_cu[i + 1]].double(), key, value.abs(), 0.1, True, -1)[:done]
        assert ((out[rows].cpu().double() - full).abs() <= full.abs() * 2.0 ** -8 + size * 2.0 ** -14).all()
        assert torch.isnan(out[q_cu[i] + done:q_cu[i + 1]]).all()
    assert (out[q_cu[-1]:] == 7).all()


@pytest.mark.parametrize("change", ["total_keys", "max_q"])
def test_a_long_chunk_with_bounds_that_do_not_hold_is_nan(gpu, change):
    lengths, counts = [3000, 2900], [2000, 1900]
    cache, table, query, q_cu = make(gpu, 64, 16, 2, 64, lengths, counts)
    total, max_q = sum(lengths) - (change == "total_keys"), 2000 - (change == "max_q")
    assert path_of(cache, 16, max_q, sum(counts), 2, len(table[0]), total_keys=total) == UNPACKED
    assert torch.isnan(attend(gpu, cache, table, query, q_cu, lengths, max_q, 0.1, total_keys=total)).all()


@pytest.mark.parametrize("head_dim,heads,kv_heads,counts", [(64, 4, 2, [6, 1]), (128, 8, 2, [9, 2]), (128, 2, 2, [3, 1]),
                                                            (512, 8, 1, [2, 1]), (256, 16, 8, [16, 3])])
@pytest.mark.parametrize("more", [0, 350, 900])
def test_nan_reaches_the_queries_that_see_it_and_no_others(gpu, head_dim, heads, kv_heads, counts, more):
    """A NaN scale of 32 elements of a new token's value, and of another's key: earlier queries of the call do not see them."""
    lengths, block = [70 + more, 33], 32
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, block, lengths, counts)
    scales = raw(cache.scales).view(cache.blocks, kv_heads, -1)
    at = lengths[0] - 1  # the first request's last token: its value's elements 32 .. 63, head 0
    scales[table[0][at // block], 0, oracle.scale_offset(at % block, 37, head_dim, True)] = 255
    at = lengths[1] - 1  # the second's: its key, head 0
    scales[table[1][at // block], 0, oracle.scale_offset(at % block, 7, head_dim, False)] = 255
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1)
    group, nan = heads // kv_heads, torch.isnan(out.cpu())
    expected = torch.zeros_like(nan)
    expected[q_cu[1] - 1, :group, 32:64] = True
    expected[q_cu[2] - 1, :group] = True
    assert torch.equal(nan, expected)
    want = values_of(cache)
    for i, n in enumerate(lengths):
        key, value = (x.nan_to_num(0.0) for x in want.rows(table[i], 0, n))
        rows = slice(q_cu[i], q_cu[i + 1] - 1)  # the queries before the last, which see neither
        if rows.start < rows.stop:
            close(out[rows], query[rows], key[:n - 1], value[:n - 1], 0.1)


# ---- as they are used together

def _serve(device, rounds, cache, heads, seed):
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
    return table, got


@pytest.mark.parametrize("head_dim,heads,kv_heads,block", [(64, 4, 2, 32), (128, 8, 2, 64), (256, 2, 1, 128)])
def test_rounds_of_a_server(gpu, head_dim, heads, kv_heads, block):
    """Prompts, then tokens one by one and a few at a time: each round's outputs against the oracle's cache, fed the same rows."""
    rounds = [[40, 7, 0, 65], [1, 1, 1, 1], [1, 1, 30, 0], [3, 2, 3, 1], [1, 1, 1, 1]]
    cache = kv_cache.create(20, kv_heads, head_dim, block, device=gpu, bits=4)
    with torch.inference_mode():
        table, got = _serve(gpu, rounds, cache, heads, seed=9)
    want = values_of(kv_cache.create(20, kv_heads, head_dim, block, device="cpu", bits=4))
    rows = table.tolist()
    for step, query, key, value, out in got:
        step.check()
        want.append(key, value, [w for w in step.writes.tolist() if w[3]])
        q_cu, lengths = step.q_cu.tolist(), step.lengths.tolist()
        for i, n in enumerate(lengths):
            close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(rows[i], 0, n), 0.1)
    have = values_of(cache)
    for i, n in enumerate(lengths):
        for a, b in zip(have.rows(rows[i], 0, n), want.rows(rows[i], 0, n)):
            assert torch.equal(a, b)


def test_a_step_on_another_stream(gpu):
    rounds = [[40, 7, 9], [1, 1, 1], [2, 1, 1]]
    with torch.inference_mode():
        caches = [kv_cache.create(16, 2, 64, 32, device=gpu, bits=4) for _ in range(2)]
        _, want = _serve(gpu, rounds, caches[0], 4, seed=10)
        stream = torch.cuda.Stream(gpu)
        stream.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(stream):
            _, got = _serve(gpu, rounds, caches[1], 4, seed=10)
        torch.cuda.current_stream(gpu).wait_stream(stream)
    for a, b in zip(want, got):
        assert torch.equal(a[4], b[4])
    for a, b in zip(caches[0][:3], caches[1][:3]):
        assert torch.equal(raw(a), raw(b))


@pytest.mark.parametrize("counts,heads,width", [([1, 1, 1], 4, 8), ([70, 1, 33], 4, 9), ([1, 1, 1], 4, 64)])
def test_a_captured_step_replays(gpu, counts, heads, width):
    """A step captured once: each replay reads the lengths, rows and free blocks that its inputs hold then, with eager work
    in between; the outputs are those of eager calls, bit for bit. Two graphs captured one after the other share nothing. (Four
    rounds of 70 tokens need nine blocks of 32.)"""
    n, rows, block, kv_heads, head_dim = 3, sum(counts), 32, 2, 64
    gen = torch.Generator(device=gpu).manual_seed(11)
    free = torch.arange(60, dtype=torch.int32, device=gpu)
    state = {"table": torch.full((n, width), -1, dtype=torch.int32, device=gpu),
             "lengths": torch.zeros(n, dtype=torch.int32, device=gpu), "left": ints([60], gpu),
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
        captured, eager = (kv_cache.create(60, kv_heads, head_dim, block, device=gpu, bits=4) for _ in range(2))
        step(captured, {**state, "table": state["table"].clone()})  # (loads the kernels)
        raw(captured.keys).zero_(), raw(captured.values).zero_(), raw(captured.scales).zero_()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs = step(captured, state)
            graphs.append((graph, outputs))
        mine = {k: v.clone() for k, v in state.items()}
        for i in range(4):
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
            for s, r in ((state, got), (mine, want)):
                s["lengths"].copy_(r.lengths)
                s["left"].copy_(r.free_left)
            for a, b in zip(captured[:3], eager[:3]):
                assert torch.equal(raw(a), raw(b))


def test_results_repeat_bit_for_bit(gpu):
    for lengths, counts, heads in (([3000, 70, 900], [1, 1, 1], 8), ([900, 700], [5, 2], 80), ([3000, 2900], [2000, 1900], 16)):
        cache, table, query, q_cu = make(gpu, 64, heads, 2, 64, lengths, counts)
        a, b = (attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, total_keys=sum(lengths)) for _ in range(2))
        assert torch.equal(a, b)


def test_branches_over_one_prompt_and_a_copied_block(gpu):
    """Two requests share a prompt's whole blocks; the partly filled one is copied before either appends to it."""
    cache = kv_cache.create(8, 2, 64, 32, device=gpu, bits=4)
    gen = torch.Generator(device=gpu).manual_seed(3)
    key, value = (torch.randn((50, 2, 64), generator=gen, device=gpu).bfloat16() for _ in range(2))
    kv_cache.append(cache, key, value, ints([[3, 0, 0, 32], [5, 0, 32, 18]], gpu))
    for t in cache[:3]:
        raw(t)[6] = raw(t)[5]
    more = torch.randn((2, 2, 2, 64), generator=gen, device=gpu).bfloat16()
    kv_cache.append(cache, more[0], more[1], ints([[5, 18, 0, 1], [6, 18, 1, 1]], gpu))
    query = torch.randn((2, 4, 64), generator=gen, device=gpu).bfloat16()
    out = attend(gpu, cache, [[3, 5], [3, 6]], query, [0, 1, 2], [51, 51], 1, 0.1)
    for i in range(2):
        k, v = (oracle.quantised(torch.cat((x, m[i:i + 1])).cpu().double()) for x, m in ((key, more[0]), (value, more[1])))
        close(out[i:i + 1], query[i:i + 1], k, v, 0.1)
