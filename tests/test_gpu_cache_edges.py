"""The block caches on the GPU where few numbers of real use lie: slots that no append wrote, queries and values at the end of
bf16's range, sums in which each group of tokens shows. Tolerances are ``cache4_cases.close``'s."""

from __future__ import annotations

import math

import pytest
import torch

from cache4_cases import SPLIT, UNPACKED, WHOLE, attend, close, ints, make, path_of, raw, values_of
from karpo_decision_amd import kv_cache, ops
from oracle import cache4 as oracle
from test_gpu_cache4 import _append_and_compare
from test_gpu_cache_rope import _server

pytestmark = pytest.mark.gpu


# ---- slots that no append wrote

def _leave_garbage(cache, table, written, seed):
    """Scales of 2^126, 2^127 and NaN and any codes wherever no token of ``written`` (first, end of each request) is."""
    gen = torch.Generator().manual_seed(seed)
    block, d = cache.block_size, cache.head_dim
    scales = raw(cache.scales).cpu().view(cache.blocks, cache.kv_heads, -1)
    kept = scales.clone()
    scales.copy_(torch.randint(253, 256, scales.shape, generator=gen, dtype=torch.uint8))
    for value in (False, True):
        at = oracle.offsets(block, d, value)[1][:, ::32]
        for row, (first, end) in zip(table, written):
            for j, ident in enumerate(row):
                tokens = range(max(0, first - j * block), max(0, min(block, end - j * block)))
                if len(tokens):
                    mine = at[list(tokens)].reshape(-1)
                    scales[ident][:, mine] = kept[ident][:, mine]
    raw(cache.scales).copy_(scales.view(cache.scales.shape))


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,path", [
    (64, 4, 2, [1, 33, 70, 0, 130], [1, 1, 1, 1, 1], WHOLE), (128, 4, 2, [1, 33, 70, 0, 130], [1, 2, 1, 1, 3], WHOLE),
    (256, 2, 1, [1, 33, 70, 0, 130], [1, 2, 1, 1, 3], WHOLE), (512, 2, 2, [1, 33, 70, 0, 250], [1, 2, 1, 1, 3], WHOLE),
    (64, 8, 2, [257, 500, 31, 0], [1, 2, 1, 1], WHOLE), (128, 3, 3, [257, 500, 31, 0], [1, 2, 1, 1], WHOLE),
    (256, 4, 2, [257, 500, 31, 0], [1, 2, 1, 1], WHOLE), (64, 8, 2, [1300, 77, 1], [1, 1, 1], SPLIT),
    (64, 8, 2, [1300, 77, 9], [7, 8, 9], SPLIT), (64, 16, 1, [1300, 77], [30, 7], SPLIT), (128, 4, 2, [1300, 77, 1], [1, 1, 1], SPLIT),
    (128, 8, 2, [1300, 77, 9], [7, 8, 9], SPLIT), (128, 16, 1, [1300, 77], [30, 7], SPLIT), (256, 4, 2, [1300, 77, 1], [1, 1, 1], SPLIT),
    (256, 8, 1, [1300, 77, 9], [7, 8, 9], SPLIT), (512, 4, 2, [1300, 77, 1], [1, 1, 1], SPLIT),
    (512, 8, 1, [1300, 77, 9], [7, 8, 9], SPLIT), (64, 16, 2, [3001, 2901], [2000, 1900], UNPACKED)])
@pytest.mark.parametrize("block", [32, 64])
def test_slots_that_nothing_wrote_reach_no_query(gpu, head_dim, heads, kv_heads, lengths, counts, path, block):
    """Scales that append never writes (2^126 and 2^127, under which codes pass bf16's range) behind the requests' tokens."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, block, lengths, counts)
    _leave_garbage(cache, table, [(0, n) for n in lengths], seed=head_dim)
    n, total = len(lengths), sum(lengths)
    assert path_of(cache, heads, max(counts), sum(counts), n, len(table[0]), total_keys=total) == path
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, total_keys=total)
    want = values_of(cache)
    for i, length in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, length), 0.1,
              weights=2.0 ** -8 if path == UNPACKED else 0.0)


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts,window,path", [
    (64, 4, 2, [300, 120], [1, 1], 40, WHOLE), (128, 8, 2, [300, 120], [3, 2], 40, WHOLE), (256, 4, 2, [600, 120], [1, 1], 300, WHOLE),
    (512, 4, 2, [300, 120], [3, 1], 40, WHOLE), (128, 8, 2, [2000, 120], [9, 1], 900, SPLIT), (64, 8, 2, [2000, 1900], [60, 9], 900, SPLIT),
    (256, 8, 1, [2000, 120], [40, 1], 900, SPLIT), (512, 8, 2, [2000, 120], [40, 1], 900, SPLIT)])
def test_blocks_behind_a_window_reach_no_query(gpu, head_dim, heads, kv_heads, lengths, counts, window, path):
    """Tokens that every query's window has left, in blocks that nothing wrote (a table that still names blocks given back); more
    than one tile of query vectors, of which the later ones meet groups that only the earlier ones see."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    firsts = [max(0, n - c - window) for n, c in zip(lengths, counts)]  # the first token that a query sees
    _leave_garbage(cache, table, list(zip(firsts, lengths)), seed=head_dim)
    assert path_of(cache, heads, max(counts), sum(counts), 2, len(table[0]), window, sum(lengths)) == path
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, window=window, total_keys=sum(lengths))
    want = values_of(cache)
    for i, (first, length) in enumerate(zip(firsts, lengths)):
        key, value = want.rows(table[i], 0, length)
        key[:first], value[:first] = 0.0, 0.0
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], key, value, 0.1, window=window)


# ---- queries and values at the end of bf16's range

PATHS = [(64, 4, 2, [200, 33], [1, 2]), (64, 4, 2, [1500, 33], [1, 2]), (128, 16, 2, [200, 33], [5, 2]), (128, 16, 2, [1500, 33], [5, 2]),
         (256, 4, 2, [500, 33], [1, 1]), (256, 8, 1, [1500, 33], [3, 2]), (512, 4, 1, [200, 33], [1, 2]), (512, 4, 1, [1500, 33], [1, 2])]


@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts", PATHS)
def test_the_largest_queries(gpu, head_dim, heads, kv_heads, lengths, counts):
    """Finite elements up to (2 - 2^-7) * 2^127, each of the last sixteen numbers of bf16 and of the binade before among them, over
    keys under the least scale, so that the scores (some 2^28) are as far from the ends as any."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    at = oracle.offsets(32, head_dim, False)[1].reshape(-1).unique()
    scales = raw(cache.scales).view(cache.blocks, kv_heads, -1)
    scales[:, :, at.to(gpu)] = 27  # 2^-100
    gen = torch.Generator().manual_seed(3)
    bits = torch.randint(0x7ef0, 0x7f80, query.shape, generator=gen)  # from 1.875 * 2^126 to the last
    bits = torch.where(torch.rand(query.shape, generator=gen) < 0.3, torch.randint(0x7f70, 0x7f80, query.shape, generator=gen), bits)
    bits |= torch.randint(0, 2, query.shape, generator=gen) << 15
    query = (bits - (bits >> 15 << 16)).to(torch.int16).view(torch.bfloat16)
    assert torch.isfinite(query.float()).all() and query.float().abs().max() == 255 * 2.0 ** 120
    out = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 2.0 ** -31, total_keys=sum(lengths))
    want = values_of(cache)
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 2.0 ** -31)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts", PATHS)
def test_queries_that_are_no_numbers(gpu, head_dim, heads, kv_heads, lengths, counts, bad):
    """One element of one head of one query: that head's row is NaN, and no other."""
    cache, table, query, q_cu = make(gpu, head_dim, heads, kv_heads, 32, lengths, counts)
    bad_query = query.clone()
    bad_query[-1, 1, 5] = bad
    out = attend(gpu, cache, table, bad_query, q_cu, lengths, max(counts), 0.1, total_keys=sum(lengths)).clone()
    assert torch.isnan(out[-1, 1]).all()
    want = values_of(cache)
    out[-1, 1] = attend(gpu, cache, table, query, q_cu, lengths, max(counts), 0.1, total_keys=sum(lengths))[-1, 1]
    for i, n in enumerate(lengths):
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], *want.rows(table[i], 0, n), 0.1)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("head_dim,kv_heads,tokens", [(64, 2, 140), (128, 2, 140), (256, 1, 140), (512, 1, 140), (64, 2, 400), (128, 2, 400),
                                                      (256, 1, 400), (64, 16, 20000), (128, 16, 20000), (256, 8, 20000), (512, 4, 20000)])
@pytest.mark.parametrize("count", [1, 9])
def test_large_values_under_growing_scores(gpu, bits, head_dim, kv_heads, tokens, count):
    """Values of 1.5 * 2^121 everywhere, scores that grow by 2^7 from one token to a later one: weights above 1 would take the sums
    past fp32's range. The scores are 0 at every 512th token, 7 (in powers of two) 256 tokens (128 where there are no more) behind
    it, and -42 elsewhere, so that 39 weights of 1 are the most that is summed up: below 2^127."""
    hot = 128 if tokens < 256 else 256
    cache = kv_cache.create(-(-tokens // 64), kv_heads, head_dim, 64, device=gpu, bits=bits)
    key = torch.zeros((tokens, kv_heads, head_dim), device=gpu)
    key[:, :, 0] = -6.0
    key[::512, :, 0], key[hot::512, :, 0] = 0.0, 1.0
    value = torch.full_like(key, 1.5 * 2.0 ** 121)
    writes = [[j, 0, 64 * j, min(64, tokens - 64 * j)] for j in range(cache.blocks)]
    kv_cache.append(cache, key.bfloat16(), value.bfloat16(), ints(writes, gpu))
    query = torch.zeros((count, 2 * kv_heads, head_dim))
    query[:, :, 0] = 1.0
    out = attend(gpu, cache, [list(range(cache.blocks))], query.bfloat16(), [0, count], [tokens], count, 7 * math.log(2.0),
                 total_keys=tokens)
    assert ((out.float() / 2.0 ** 121 - 1.5).abs() <= 1.5 * 2.0 ** -8).all()


# ---- each group of tokens shows

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("head_dim,heads,kv_heads,lengths,counts", [
    (64, 4, 2, [4517, 90], [2, 1]), (128, 8, 2, [4517, 90], [2, 1]), (256, 4, 1, [4517, 90], [2, 1]), (512, 4, 1, [4517, 90], [2, 1]),
    (128, 32, 16, [20001, 4000, 700], [1, 1, 1]), (64, 40, 1, [2100, 70], [9, 2]), (128, 4, 2, [640, 333], [1, 2]),
    (256, 4, 2, [640, 333], [1, 2]), (512, 4, 2, [250, 100], [1, 2])])
def test_no_group_is_left_out_or_taken_twice(gpu, bits, head_dim, heads, kv_heads, lengths, counts):
    """Element d of a token's value is 1 where the token's group of 32 is d modulo the head size, and 0 elsewhere, under scores
    so even that every token counts alike: an element holds its own groups' share, and one of them left out or taken twice
    moves it by a tenth at least (of at most ten groups)."""
    block = 64
    gen = torch.Generator().manual_seed(head_dim)
    blocks = [-(-n // block) for n in lengths]
    ids = torch.randperm(sum(blocks), generator=gen).tolist()
    cache = kv_cache.create(sum(blocks), kv_heads, head_dim, block, device=gpu, bits=bits)
    table, q_cu = [], [0]
    keys, values = [], []
    for n, c, b in zip(lengths, counts, blocks):
        table.append([ids.pop() for _ in range(b)])
        q_cu.append(q_cu[-1] + c)
        group = torch.arange(n) // 32
        value = torch.zeros((n, kv_heads, head_dim))
        value[torch.arange(n), :, group % head_dim] = 1.0
        key = torch.randn((n, kv_heads, head_dim), generator=gen).bfloat16()
        kv_cache.append(cache, key.to(gpu), value.bfloat16().to(gpu),
                        ints([[ident, 0, block * j, min(block, n - block * j)] for j, ident in enumerate(table[-1])], gpu))
        keys.append(oracle.quantised(key.double()) if bits == 4 else None)
        values.append(value.double())
    assert max(lengths) <= 10 * 32 * head_dim
    query = torch.randn((q_cu[-1], heads, head_dim), generator=gen).bfloat16()
    width = max(blocks)
    padded = [row + [-1] * (width - len(row)) for row in table]
    out = attend(gpu, cache, padded, query, q_cu, lengths, max(counts), 1e-4, total_keys=sum(lengths))
    for i, n in enumerate(lengths):
        if bits == 8:
            keys[i] = kv_cache.read(cache, ints([padded[i]], gpu), ints([n], gpu), n)[0].cpu().double()
        close(out[q_cu[i]:q_cu[i + 1]], query[q_cu[i]:q_cu[i + 1]], keys[i], values[i], 1e-4)


# ---- append and rounds of a server

@pytest.mark.parametrize("e", [0, -60, 100, -100, -104])
def test_append_rounds_small_elements_beside_large_ones(gpu, e):
    """Every finite bf16 value of at most 6 * 2^e, zeros, subnormal numbers and what rounds to nothing among them, 31 at a time
    beside 6 * 2^e (below 2^-100 the scale is the least one)."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    top = torch.tensor(6.0 * 2.0 ** e).bfloat16()
    part = every[every.float().abs() <= top.float()]
    part = torch.cat((part, part.new_zeros(-part.numel() % 31))).view(-1, 31)
    x = torch.cat((part, top.expand(part.shape[0], 1)), 1)
    x = torch.cat((x, x.new_zeros((-x.shape[0] % 2, 32)))).view(-1, 1, 64)
    cache = kv_cache.create(-(-x.shape[0] // 32), 1, 64, 32, device=gpu, bits=4)
    writes = [[i, 0, 32 * i, min(32, x.shape[0] - 32 * i)] for i in range(cache.blocks)]
    _append_and_compare(cache, x.to(gpu), -x.to(gpu), writes)


@pytest.mark.parametrize("heads,kv_heads,d,block,rotated", [(4, 2, 64, 32, 64), (16, 2, 128, 64, 64), (2, 1, 256, 128, 256)])
def test_rounds_of_a_server_in_8_bits_to_the_output_s_rounding(gpu, heads, kv_heads, d, block, rotated):
    """Calls of at most 64 query vectors a key head are never unpacked: their weights are two bf16 terms, and the outputs lie within
    the tolerance of the 4-bit cache's, without a term for weights of one."""
    most = 64 * kv_heads // heads
    rounds = [[min(c, most) for c in counts] for counts in ([40, 7, 0, 65], [1, 1, 1, 1], [1, 1, 30, 0], [3, 2, 3, 1], [1, 1, 1, 1])]
    gen = torch.Generator(device=gpu).manual_seed(6)
    server = _server(gpu, 8, heads, kv_heads, d, block, rotated)
    with torch.inference_mode():
        for counts in rounds:
            n = sum(counts)
            query = torch.randn((n, heads, d), generator=gen, device=gpu).bfloat16()
            key, value = (torch.randn((n, kv_heads, d), generator=gen, device=gpu).bfloat16() for _ in range(2))
            step, out, turned = server.round(ints(counts, gpu), n, max(counts), query, key, value)
            step.check()
            held = step.lengths.tolist()
            keys, values, k_cu = kv_cache.read(server.cache, server.table, step.lengths, sum(held))
            q_cu, k_cu = step.q_cu.tolist(), k_cu.tolist()
            for i in range(4):
                close(out[q_cu[i]:q_cu[i + 1]], turned[q_cu[i]:q_cu[i + 1]], keys[k_cu[i]:k_cu[i + 1]].double(),
                      values[k_cu[i]:k_cu[i + 1]].double(), 0.1)


@pytest.mark.parametrize("bits", [4, 8])
def test_weights_and_tables_at_any_address(gpu, bits):
    """Out of the middle of larger tensors, not at a multiple of 16 bytes: as their copies, in ``append`` and ``norm_rope``."""
    gen = torch.Generator(device=gpu).manual_seed(7)
    key, value = (torch.randn((9, 2, 64), generator=gen, device=gpu).bfloat16() for _ in range(2))
    weight, cos, sin = (torch.randn(n + 3, generator=gen, device=gpu).bfloat16()[3:] for n in (64, 9 * 64, 9 * 64))
    assert all(t.data_ptr() % 16 for t in (weight, cos, sin))
    got = []
    with torch.inference_mode():
        for w, c, s in ((weight, cos, sin), (weight.clone(), cos.clone(), sin.clone())):
            cache = kv_cache.create(1, 2, 64, 32, device=gpu, bits=bits)
            norm, rope = ops.Norm(ops.NORM_WEIGHT, w, 1e-6), (c.view(9, 64), s.view(9, 64))
            kv_cache.append(cache, key, value, ints([[0, 0, 0, 9]], gpu), k_norm=norm, v_norm=norm, rope=rope)
            got.append([*(raw(t) for t in cache[:3]), ops.norm_rope(key, norm, rope)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_compiled_step_with_norms_and_rotation(gpu, bits):
    """torch.compile breaks its graph around the calls: each sees the tensors of its own step, not those of the traced one."""
    def step(cache, table, lengths, counts, free, left, key, value, query, weight, cos, sin):
        got = kv_cache.reserve(table, lengths, counts, free, left, 47, 32)
        kv_cache.append(cache, key * 2, value, got.writes, k_norm=ops.Norm(ops.NORM_WEIGHT, weight, 1e-6), rope=(cos, sin),
                        positions=got.positions)
        k, v, _ = kv_cache.read(cache, table, got.lengths, 47)
        return kv_cache.attend(query + 1, cache, table, got.q_cu, got.lengths, 40, 0.1) * 2, k + 1, v

    def inputs(seed):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        rows = [torch.randn(shape, generator=gen, device=gpu).bfloat16()
                for shape in ((47, 2, 64), (47, 2, 64), (47, 4, 64), (64,), (50, 64), (50, 64))]
        return (kv_cache.create(20, 2, 64, 32, device=gpu, bits=bits), torch.full((2, 6), -1, dtype=torch.int32, device=gpu),
                ints([0, 0], gpu), ints([40, 7], gpu), torch.arange(20, dtype=torch.int32, device=gpu), ints([20], gpu), *rows)

    torch._dynamo.reset()
    compiled, kept = torch.compile(step, backend="eager"), []
    with torch.inference_mode():
        for seed in range(3):
            kept.append(inputs(seed))  # (kept, so that the next step's tensors lie elsewhere)
            for a, b in zip(compiled(*kept[-1]), step(*inputs(seed))):
                assert torch.equal(a, b)
