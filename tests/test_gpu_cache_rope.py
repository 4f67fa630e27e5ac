"""``kv_cache.append`` with norms and rotation on the way, into both caches, against the formulas in 64 bits.

y64 is the row in 64 bits, size the sum of the magnitudes that the rotation adds up. The kernel's y in fp32: the sum of squares
(2 log2 D + 8 roundings at most, all terms positive) and the root and reciprocal (correctly rounded or one step off) put r at most
2^-20 off; three more roundings: |y - y64| <= 2^-19 size. A stored element is y rounded to a step of its scale, half a step off,
and y's own error may take it over a border between two codes, which changes nothing in that bound: |got - y64| <= half a step
+ 2^-19 size. The scale's exponent is that of the largest |y|, with the largest |y64| a share of 2^-18 up or down."""

from __future__ import annotations

import math

import pytest
import torch

from cache4_cases import close, copy_of, ints, random_cache, raw, values_of
from karpo_decision_amd import kv_cache, ops
from oracle import cache as oracle8
from oracle import cache4 as oracle

pytestmark = pytest.mark.gpu

NORMS = {"weight": ops.NORM_WEIGHT, "one_plus": ops.NORM_ONE_PLUS, "plain": ops.NORM_PLAIN}


def _norm(kind, d, device, gen, eps=1e-6):
    if kind is None:
        return None
    weight = (torch.randn(d, generator=gen) * 0.3 + (1.0 if kind == "weight" else 0.0)).bfloat16().to(device)
    return ops.Norm(NORMS[kind], None if kind == "plain" else weight, eps)


def _tables(n, r, gen, device, stride=None):
    angle = torch.rand((n, r // 2), generator=gen) * 6.28
    angle = torch.cat((angle, angle), 1)
    out = []
    for t in (angle.cos(), angle.sin()):
        wide = torch.zeros((n, r if stride is None else stride), dtype=torch.bfloat16, device=device)
        wide[:, :r] = t.bfloat16()
        out.append(wide[:, :r])
    return tuple(out)


def _cache(bits, device, blocks, kv_heads, d, block, seed):
    if bits == 4:
        return random_cache(device, blocks, kv_heads, d, block, seed)
    cache = kv_cache.create(blocks, kv_heads, d, block, device=device)
    gen = torch.Generator().manual_seed(seed)
    for t in cache[:2]:
        raw(t).copy_(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
    cache.scales.copy_(torch.exp2(torch.randint(-12, -4, cache.scales.shape, generator=gen).float()))
    return cache


def _wanted(key, value, k_norm, v_norm, rope, positions):
    """[(y64, size)] of keys and values."""
    def plain(n):
        return None if n is None else (n.mode, n.weight, n.eps)

    v = oracle.normed(value, plain(v_norm))
    return [oracle.turned(oracle.normed(key, plain(k_norm)), rope, positions), (v, v.abs())]


def _exponents(bits, y, size):
    """The least and the largest exponent that the scale of rows ``y`` (all of them under one) can have."""
    fine = torch.isfinite(y)
    top = float(y[fine].abs().max()) if fine.any() else 0.0
    slack = float(size[fine].max()) * 2.0 ** -18 if fine.any() else 0.0
    of = oracle.exponent if bits == 4 else oracle8.exponent
    return of(max(0.0, top - slack)), of(top + slack)


def _close(got, y, size, bits, e):
    """``got`` (float64) is y under the scale 2^e."""
    assert torch.equal(torch.isnan(got), torch.isnan(y)), "NaN"
    most, least, after = (6.0, 1.0, 1) if bits == 4 else (448.0, 2.0 ** -6, 3)
    scale = 2.0 ** e
    want = torch.where(torch.isfinite(y), y, torch.sign(y).nan_to_num() * math.inf).clamp(-most * scale, most * scale)
    step = torch.exp2(torch.floor(torch.log2((want.abs() / scale).clamp(min=least))) - after) * scale
    off = (got - want).abs()
    bound = step / 2 + size.nan_to_num(posinf=0.0) * 2.0 ** -19
    bad = ~(off <= bound) & ~torch.isnan(y)
    assert not bad.any(), (got[bad][:4], want[bad][:4], e)


def _append_and_compare(cache, key, value, writes, k_norm=None, v_norm=None, rope=None, positions=None):
    bits, d, block = cache.bits, cache.head_dim, cache.block_size
    before = copy_of(cache) if bits == 4 else kv_cache.Cache(*(t.clone() for t in cache[:3]), block)
    wanted = _wanted(key, value, k_norm, v_norm, rope, positions)
    with torch.inference_mode():
        kv_cache.append(cache, key, value, ints(writes, cache.keys.device), k_norm=k_norm, v_norm=v_norm, rope=rope,
                        positions=positions)
    touched = torch.zeros((cache.blocks, block), dtype=torch.bool)
    have = values_of(cache) if bits == 4 else oracle8.Cache(cache.keys, cache.values, cache.scales, block)
    old = values_of(before) if bits == 4 else oracle8.Cache(before.keys, before.values, before.scales, block)
    for ident, first, row, count in writes:
        touched[ident, first:first + count] = True
        for side, (y, size) in enumerate(wanted):
            for h in range(cache.kv_heads):
                mine, far = y[row:row + count, h], size[row:row + count, h]
                if bits == 4:
                    got = have.values[side][ident, h, first:first + count]
                    at = oracle.offsets(block, d, bool(side))[1][first:first + count]
                    e = raw(cache.scales).cpu().view(cache.blocks, cache.kv_heads, -1)[ident, h, at.reshape(-1)]
                    e = e.view(count, d).double() - 127
                    for t in range(count):
                        for g in range(0, d, 32):
                            part = slice(g, g + 32)
                            if torch.isnan(mine[t, part]).any():
                                assert torch.isnan(got[t, part]).all()
                                continue
                            lo, hi = _exponents(4, mine[t, part], far[t, part])
                            exp = int(e[t, g])
                            assert lo <= exp <= hi and (e[t, part] == exp).all()
                            _close(got[t, part], mine[t, part], far[t, part], 4, exp)
                else:
                    lo, hi = _exponents(8, mine, far)
                    if first > 0:
                        was = min(max(int(old.exps[ident, h, side]), -100), 119)
                        lo, hi = max(lo, was), max(hi, was)
                    exp = int(have.exps[ident, h, side])
                    assert lo <= exp <= hi
                    _close(have.codes[side][ident, h, first:first + count] * 2.0 ** exp, mine, far, 8, exp)
                    if first > 0:  # the earlier tokens, rounded again where the scale grew
                        again = oracle8.rounded(old.codes[side][ident, h, :first] * 2.0 ** (was - exp))
                        assert torch.equal(again.nan_to_num(9e9), have.codes[side][ident, h, :first].nan_to_num(9e9))
                        touched[ident, :first] = True
    for side in (0, 1):
        at = oracle.offsets(block, d, bool(side))[0] if bits == 4 else oracle8.offsets(block, d, bool(side)).view(block, d)
        a, b = (raw(c[side]).cpu().view(cache.blocks, cache.kv_heads, -1)[:, :, at.reshape(-1)]
                .view(cache.blocks, cache.kv_heads, block, d) for c in (before, cache))
        assert ((a == b).all(-1).all(1) | touched).all()


def _writes(block):
    return [[2, 0, 0, block], [5, 0, block, 1], [0, 17, block + 1, 1], [7, block - 1, block + 2, 1], [1, 3, block + 3, 21],
            [3, 11, block + 24, block - 11], [6, 30, 2 * block + 13, 2]]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,block,r,k_kind,v_kind", [
    (64, 32, 64, "weight", "plain"), (64, 128, 32, "one_plus", None), (128, 64, 128, "weight", "plain"),
    (128, 32, 64, "plain", "weight"), (128, 128, 32, None, "one_plus"), (256, 64, 64, "one_plus", None),
    (256, 32, 256, "weight", "plain"), (512, 32, 512, "weight", "plain"), (512, 128, 128, None, None),
    (256, 128, 96, "plain", None)])
def test_append(gpu, bits, d, block, r, k_kind, v_kind):
    """Norms and rotations of every kind, whole blocks, single tokens and pieces of blocks over leftovers."""
    gen = torch.Generator().manual_seed(d + block)
    cache = _cache(bits, gpu, 8, 2, d, block, seed=block)
    rows = 2 * block + 15
    key, value = ((torch.randn((rows, 2, d), generator=gen) * 3).bfloat16().to(gpu) for _ in range(2))
    key[::7] *= 20
    positions = torch.randint(0, 300, (rows,), generator=gen, dtype=torch.int32).to(gpu)
    _append_and_compare(cache, key, value, _writes(block), _norm(k_kind, d, gpu, gen), _norm(v_kind, d, gpu, gen),
                        _tables(300, r, gen, gpu), positions)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("seed", range(6))
def test_append_of_random_writes(gpu, bits, seed):
    gen = torch.Generator().manual_seed(seed)

    def one_of(*choices):
        return choices[int(torch.randint(len(choices), (1,), generator=gen))]

    d, block, heads, blocks = one_of(64, 128, 256, 512), one_of(32, 64, 128), one_of(1, 2, 3), 9
    r = 32 * int(torch.randint(1, d // 32 + 1, (1,), generator=gen))
    cache = _cache(bits, gpu, blocks, heads, d, block, seed=seed)
    writes, rows = [], 0
    for ident in torch.randperm(blocks, generator=gen)[:one_of(1, 4, blocks)].tolist():
        first = one_of(0, 0, int(torch.randint(block, (1,), generator=gen)))
        count = one_of(1, block - first, 1 + int(torch.randint(block - first, (1,), generator=gen)))
        writes.append([ident, first, rows, count])
        rows += count + one_of(0, 2)  # (rows that no write names)
    key, value = (torch.randn((rows, heads, d), generator=gen).bfloat16().to(gpu) for _ in range(2))
    positions = torch.randint(0, 77, (rows,), generator=gen, dtype=torch.int32).to(gpu)
    kinds = [one_of(None, "weight", "one_plus", "plain") for _ in range(2)]
    _append_and_compare(cache, key, value, writes, *(_norm(kind, d, gpu, gen) for kind in kinds), _tables(77, r, gen, gpu), positions)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rope", [False, True])
def test_rows_without_positions_or_rotation(gpu, bits, rope):
    """Row i takes the tables' row i; or nothing but the norms."""
    gen = torch.Generator().manual_seed(5)
    cache = _cache(bits, gpu, 8, 2, 128, 64, seed=1)
    key, value = (torch.randn((150, 2, 128), generator=gen).bfloat16().to(gpu) for _ in range(2))
    tables = _tables(150 if rope else 1, 128, gen, gpu)
    _append_and_compare(cache, key, value, _writes(64), _norm("weight", 128, gpu, gen), _norm("plain", 128, gpu, gen),
                        tables if rope else None)


@pytest.mark.parametrize("bits", [4, 8])
def test_strided_rows_and_tables(gpu, bits):
    """Keys and values out of one packed projection, tables whose rows are wider than what is turned, in fp32 and three-dimensional."""
    gen = torch.Generator().manual_seed(6)
    packed = torch.randn((80, 8, 128), generator=gen).bfloat16().to(gpu)
    tables = _tables(90, 64, gen, gpu, stride=96)
    positions = torch.randint(0, 90, (80,), generator=gen, dtype=torch.int32).to(gpu)
    norm = _norm("one_plus", 128, gpu, gen)
    writes = [[1, 5, 40, 10], [3, 0, 2, 32], [0, 31, 70, 1]]
    caches = [_cache(bits, gpu, 4, 2, 128, 32, seed=2) for _ in range(2)]
    _append_and_compare(caches[0], packed[:, 4:6], packed[:, 6:], writes, norm, None, tables, positions)
    with torch.inference_mode():
        kv_cache.append(caches[1], packed[:, 4:6], packed[:, 6:], ints(writes, gpu),
                        k_norm=ops.Norm(norm.mode, norm.weight.float(), norm.eps), rope=tuple(t.float()[None] for t in tables),
                        positions=positions)
    for a, b in zip(caches[0][:3], caches[1][:3]):
        assert torch.equal(raw(a), raw(b))


@pytest.mark.parametrize("bits", [4, 8])
def test_positions_outside_the_tables_give_nan(gpu, bits):
    gen = torch.Generator().manual_seed(7)
    cache = _cache(bits, gpu, 4, 2, 128, 32, seed=3)
    key, value = (torch.randn((12, 2, 128), generator=gen).bfloat16().to(gpu) for _ in range(2))
    positions = ints([0, 1, 9, 10, -1, 2**31 - 1, -2**31, 3, 4, 5, 6, 7], gpu)
    _append_and_compare(cache, key, value, [[1, 0, 0, 9], [2, 7, 9, 3]], None, None, _tables(10, 64, gen, gpu), positions)
    key, _, _ = kv_cache.read(cache, ints([[1]], gpu), ints([9], gpu), 9)
    nan = torch.isnan(key).cpu()
    assert nan[3:7, :, :64].all() and not nan[:, :, 64:].any() and not nan[[0, 1, 2, 7, 8]].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 256])
def test_rows_with_infinities_and_nan(gpu, bits, d):
    """Without a norm an infinity is stored at the range's end and NaN as NaN; a norm of such a row is NaN, or zero beside."""
    gen = torch.Generator().manual_seed(8)
    cache = _cache(bits, gpu, 6, 1, d, 32, seed=4)
    key = torch.randn((6, 1, d), generator=gen).bfloat16()
    key[0, 0, 3], key[1, 0, 5], key[2] = math.inf, math.nan, 0.0
    key[3] = 0.0
    key[3, 0, 7] = -math.inf
    key = key.to(gpu)
    _append_and_compare(cache, key, key.flip(0).contiguous(), [[i, 0, i, 1] for i in range(6)], None, None, None, None)
    # y = x * r * w with r = 1 / sqrt(inf) = 0: zeros beside inf * 0 = NaN
    norm = ops.Norm(ops.NORM_PLAIN, None, 1e-6)
    with torch.inference_mode():
        kv_cache.append(cache, key, key, ints([[i, 0, i, 1] for i in range(6)], gpu), k_norm=norm, v_norm=norm)
    got = kv_cache.read(cache, ints([[i] for i in range(6)], gpu), ints([1] * 6, gpu), 6)
    for side in got[:2]:
        assert torch.isnan(side[0, 0, 3]) and torch.isnan(side[1]).all() and torch.isnan(side[3, 0, 7])
        assert (side[2] == 0).all() and torch.isfinite(side[4:]).all()
        assert (side[0, 0, 32:] == 0).all() and (side[3, 0, 32:] == 0).all()


def test_fp32_maximum_at_the_scales_border(gpu):
    """8 bits: a largest element of exactly 448 * 2^e keeps e, the next fp32 number above it takes the next; 4 bits: 6 * 2^e."""
    for bits, most in ((8, 448.0), (4, 6.0)):
        # y = x * w without rounding, r = 1 / sqrt(eps) with x^2 / D far below eps: r = 1 for eps = 1
        for factor, grows in ((1.0, False), (1.0 + 2.0 ** -7, True), (1.0 - 2.0 ** -8, False)):
            cache = kv_cache.create(1, 1, 64, 32, device=gpu, bits=bits)
            key = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device=gpu)
            key[0, 0, 0] = most * factor * 2.0 ** -30
            with torch.inference_mode():
                kv_cache.append(cache, key, key, ints([[0, 0, 0, 1]], gpu), k_norm=ops.Norm(ops.NORM_PLAIN, None, 1.0))
            e = (int(math.log2(cache.scales[0, 0, 0].item())) if bits == 8
                 else int(raw(cache.scales).view(-1)[oracle.scale_offset(0, 0, 64, False)]) - 127)
            assert e == -30 + grows, (bits, factor)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_captured_append_reads_its_inputs_at_each_replay(gpu, bits):
    gen = torch.Generator(device=gpu).manual_seed(9)
    cache, eager = (kv_cache.create(6, 2, 128, 32, device=gpu, bits=bits) for _ in range(2))
    key, value = (torch.randn((40, 2, 128), generator=gen, device=gpu).bfloat16() for _ in range(2))
    cpu = torch.Generator().manual_seed(1)
    tables, norm = _tables(100, 128, cpu, gpu), _norm("weight", 128, gpu, cpu)
    positions, writes = ints(list(range(40)), gpu), ints([[1, 0, 0, 32], [2, 0, 32, 8]], gpu)

    def call(c):
        kv_cache.append(c, key, value, writes, k_norm=norm, v_norm=ops.Norm(ops.NORM_PLAIN, None, 1e-6), rope=tables,
                        positions=positions)

    with torch.inference_mode():
        call(cache)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(cache)
        for t in cache[:3]:
            raw(t).zero_()
        for i in range(3):
            key.mul_(-1.5)
            value.add_(0.25)
            positions.add_(7)
            writes[:, 0] = writes[:, 0] % 5 + 1
            graph.replay()
            call(eager)
            torch.cuda.synchronize()
            for a, b in zip(cache[:3], eager[:3]):
                assert torch.equal(raw(a), raw(b)), i


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,kv_heads,block,rope", [(64, 13, 64, True), (128, 6, 128, True), (256, 3, 32, False), (512, 9, 64, True),
                                                   (512, 4, 128, True), (512, 5, 32, True), (256, 5, 128, True)])
def test_many_rows_at_once_and_in_pieces(gpu, bits, d, kv_heads, block, rope):
    """Over 96 MiB of rows, where a workgroup takes several heads: the same bits as in calls of few blocks each, which
    the other tests compare with the formulas. Ragged writes, some of one token."""
    gen = torch.Generator().manual_seed(11)
    blocks = -(-(104 << 20) // (4 * kv_heads * d * block))
    counts = torch.randint(block - 3, block + 1, (blocks,), generator=gen)
    counts[::9] = 1
    firsts = torch.minimum(torch.randint(0, 4, (blocks,), generator=gen), block - counts)
    starts = torch.cumsum(counts, 0) - counts
    ids = torch.randperm(blocks, generator=gen)
    writes = torch.stack((ids, firsts, starts, counts), 1).int().to(gpu)
    rows = -(-(97 << 20) // (4 * kv_heads * d))
    rows = max(rows, int(counts.sum()))
    key, value = (torch.randn((rows, kv_heads, d), generator=gen).bfloat16().to(gpu) for _ in range(2))
    assert 4 * rows * kv_heads * d > 96 << 20
    tables = _tables(500, d, gen, gpu) if rope else None
    positions = torch.randint(0, 500, (rows,), generator=gen, dtype=torch.int32).to(gpu) if rope else None
    norm = _norm("weight", d, gpu, gen)
    one, two = (_cache(bits, gpu, blocks, kv_heads, d, block, seed=5) for _ in range(2))
    with torch.inference_mode():
        kv_cache.append(one, key, value, writes, k_norm=norm, v_norm=norm, rope=tables, positions=positions)
        for i in range(0, blocks, 8):
            part = writes[i:i + 8].clone()
            a, b = int(part[0, 2]), int(part[-1, 2] + part[-1, 3])
            part[:, 2] -= a
            assert 4 * (b - a) * kv_heads * d <= 96 << 20
            kv_cache.append(two, key[a:b], value[a:b], part, k_norm=norm, v_norm=norm, rope=tables,
                            positions=None if positions is None else positions[a:b])
    for a, b in zip(one[:3], two[:3]):
        assert torch.equal(raw(a), raw(b))


@pytest.mark.parametrize("bits", [4, 8])
def test_near_norm_rope_and_a_plain_append(gpu, bits):
    """The two calls it stands for round to bf16 twice more, after the norm and after the rotation. The first puts what is added up
    2^-8 off, the second the sum: the rows are less than 2^-7 size apart (the rotation may cancel: not 2^-7 of the sum). Each is
    then rounded by half a step at most."""
    gen = torch.Generator(device=gpu).manual_seed(10)
    cpu = torch.Generator().manual_seed(2)
    key, value = (torch.randn((64, 2, 128), generator=gen, device=gpu).bfloat16() for _ in range(2))
    tables, norm = _tables(64, 128, cpu, gpu), _norm("weight", 128, gpu, cpu)
    plain = ops.Norm(ops.NORM_PLAIN, None, 1e-6)
    one, two = (kv_cache.create(1, 2, 128, 64, device=gpu, bits=bits) for _ in range(2))
    writes, table = ints([[0, 0, 0, 64]], gpu), ints([[0]], gpu)
    with torch.inference_mode():
        kv_cache.append(one, key, value, writes, k_norm=norm, v_norm=plain, rope=tables)
        kv_cache.append(two, ops.norm_rope(key, norm, tables), ops.norm_rope(value, plain), writes)
    sizes = [size.to(gpu) for _, size in _wanted(key, value, norm, plain, tables, None)]
    for a, b, size in zip(kv_cache.read(one, table, ints([64], gpu), 64)[:2], kv_cache.read(two, table, ints([64], gpu), 64)[:2],
                          sizes):
        a, b = a.double(), b.double()
        if bits == 8:  # half a step: 2^-4 of an element, or 2^-10 * 2^e, of which 448 * 2^e is less than twice the largest
            half = torch.maximum(torch.maximum(a.abs(), b.abs()) * 2.0 ** -4, torch.maximum(a.abs().max(), b.abs().max()) * 2.0 ** -17)
        else:  # a quarter of an element, or 2^e / 4, of which 6 * 2^e is less than four times the largest of its 32
            most = torch.maximum(a.abs(), b.abs()).view(64, 2, 4, 32).amax(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(a.shape)
            half = torch.maximum(torch.maximum(a.abs(), b.abs()) / 4, most / 6)
        assert ((a - b).abs() <= 2 * half + 2.0 ** -7 * size).all()


# ---- as they are used together

class _Server:
    """Four requests over a cache, their table, lengths and free list; ``round`` is one step of one layer."""

    def __init__(self, device, bits, heads, kv_heads, d, block, tables, norms):
        self.cache = kv_cache.create(24, kv_heads, d, block, device=device, bits=bits)
        self.heads, self.tables, self.norms = heads, tables, norms
        self.table = torch.full((4, 8), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(4, dtype=torch.int32, device=device)
        self.free, self.left = torch.arange(24, dtype=torch.int32, device=device), ints([24], device)

    def round(self, counts, rows, most, query, key, value):
        """(step, out, the queries as the attention takes them)"""
        step = kv_cache.reserve(self.table, self.lengths, counts, self.free, self.left, rows, self.cache.block_size)
        kv_cache.append(self.cache, key, value, step.writes, k_norm=self.norms[1], v_norm=self.norms[2], rope=self.tables,
                        positions=step.positions)
        at = step.positions.long()
        turned = ops.norm_rope(query, self.norms[0], tuple(t[at] for t in self.tables))
        out = kv_cache.attend(turned, self.cache, self.table, step.q_cu, step.lengths, most, 0.1)
        self.lengths.copy_(step.lengths)
        self.left.copy_(step.free_left)
        return step, out, turned


def _server(device, bits, heads, kv_heads, d, block, rotated):
    gen = torch.Generator().manual_seed(3)
    norms = [_norm(kind, d, device, gen) for kind in ("one_plus", "one_plus", "plain")]
    return _Server(device, bits, heads, kv_heads, d, block, _tables(200, rotated, gen, device), norms)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,kv_heads,d,block,rotated", [(4, 2, 64, 32, 64), (16, 2, 128, 64, 64), (2, 1, 256, 128, 256)])
def test_rounds_of_a_server(gpu, bits, heads, kv_heads, d, block, rotated):
    """Prompts, then tokens one by one and a few at a time. Each round's new rows in the cache are, bit for bit, those of a second
    cache that gets them with their own tables' rows, and its outputs those of the rows that ``read`` finds."""
    rounds = [[40, 7, 0, 65], [1, 1, 1, 1], [1, 1, 30, 0], [3, 2, 3, 1], [1, 1, 1, 1]]
    gen = torch.Generator(device=gpu).manual_seed(4)
    server = _server(gpu, bits, heads, kv_heads, d, block, rotated)
    twin = copy_of(server.cache)
    had = [0] * 4
    with torch.inference_mode():
        for counts in rounds:
            n = sum(counts)
            query = torch.randn((n, heads, d), generator=gen, device=gpu).bfloat16()
            key, value = (torch.randn((n, kv_heads, d), generator=gen, device=gpu).bfloat16() for _ in range(2))
            step, out, turned = server.round(ints(counts, gpu), n, max(counts), query, key, value)
            step.check()
            at = [p for h, c in zip(had, counts) for p in range(h, h + c)]
            had = [h + c for h, c in zip(had, counts)]
            assert step.lengths.tolist() == had
            kv_cache.append(twin, key, value, step.writes, k_norm=server.norms[1], v_norm=server.norms[2],
                            rope=tuple(t[at] for t in server.tables))
            for a, b in zip(server.cache[:3], twin[:3]):
                assert torch.equal(raw(a), raw(b))
            keys, values, k_cu = (t.tolist() if i == 2 else t.cpu().double() for i, t in enumerate(
                kv_cache.read(server.cache, server.table, step.lengths, sum(had))))
            q_cu = step.q_cu.tolist()
            for i in range(4):
                close(out[q_cu[i]:q_cu[i + 1]], turned[q_cu[i]:q_cu[i + 1]], keys[k_cu[i]:k_cu[i + 1]],
                      values[k_cu[i]:k_cu[i + 1]], 0.1, weights=2.0 ** -8 if bits == 8 else 0.0)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_captured_round_goes_on_from_replay_to_replay(gpu, bits):
    """A captured step of one token each, its lengths and free list carried on by itself, against eager steps."""
    gen = torch.Generator(device=gpu).manual_seed(5)
    heads, kv_heads, d, block = 8, 2, 128, 32
    captured, eager = (_server(gpu, bits, heads, kv_heads, d, block, 128) for _ in range(2))

    def rows(n):
        return (torch.randn((n, heads, d), generator=gen, device=gpu).bfloat16(),
                *(torch.randn((n, kv_heads, d), generator=gen, device=gpu).bfloat16() for _ in range(2)))

    with torch.inference_mode():
        prompt, ones = rows(90), ints([1] * 4, gpu)
        for s in (captured, eager):
            s.round(ints([31, 0, 32, 27], gpu), 90, 32, *prompt)
        fixed = rows(4)
        # (a first call outside the graph, over another server)
        _server(gpu, bits, heads, kv_heads, d, block, 128).round(ones, 4, 1, *fixed)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step, out, _ = captured.round(ones, 4, 1, *fixed)
        for i in range(5):
            for a, b in zip(fixed, rows(4)):
                a.copy_(b)
            graph.replay()
            want_step, want, _ = eager.round(ones, 4, 1, *fixed)
            torch.cuda.synchronize()
            want_step.check()
            assert torch.equal(out, want) and torch.equal(step.lengths, want_step.lengths), i
            for a, b in zip(captured.cache[:3], eager.cache[:3]):
                assert torch.equal(raw(a), raw(b)), i
