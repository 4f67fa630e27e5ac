"""The block cache on the CPU: what ``kv_cache`` and the C ABI refuse, before anything reaches a GPU, and the oracle that
the GPU tests compare with, pinned by torch's own e4m3 conversion and by closed forms."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from karpo_decision_amd import _lib, kv_cache
from oracle import cache as oracle

HEADER = Path(__file__).resolve().parents[1] / "include" / "karpo_cache.h"


def test_library_exports_every_declared_function():
    names = set(re.findall(r"^\s*(?:int|int64_t)\s+(karpo_cache_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(_lib.CACHE_EXPORTS)
    for name in names:
        assert hasattr(_lib.load(), name), name


@pytest.mark.parametrize("packed,named", [
    (kv_cache._RESERVE, _lib.KarpoCacheReserveArgs), (kv_cache._APPEND, _lib.KarpoCacheAppendArgs),
    (kv_cache._READ, _lib.KarpoCacheReadArgs), (kv_cache._ATTEND, _lib.KarpoCacheAttendArgs)], ids=lambda x: "")
def test_packed_arguments_are_the_structures(packed, named):
    def leaves(s):
        for name, kind in s._fields_:
            if issubclass(kind, ctypes.Structure):
                yield from leaves(getattr(s, name))
            else:
                yield getattr(s, name)

    assert packed.size == ctypes.sizeof(named)
    count = len(list(leaves(named())))
    values = list(range(1, count + 1))
    assert list(leaves(named.from_buffer_copy(packed.pack(*values)))) == values


# ---- the oracle

def test_oracle_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mine = oracle.e4m3_values()
    assert torch.equal(torch.isnan(codes), torch.isnan(mine))
    assert torch.equal(codes.nan_to_num(7e9), mine.nan_to_num(7e9))


def test_oracle_rounds_as_torch_does():
    values = oracle.e4m3_values()
    values = values[torch.isfinite(values)]
    x = torch.cat([torch.randn(4096, dtype=torch.float64) * s for s in (1e-3, 1e-2, 1.0, 100.0)]
                  + [(values[:, None] + values[None, :]).reshape(-1) / 2])  # the ties among them
    x = x.clamp(-448, 448).float()
    assert torch.equal(oracle.rounded(x.double()), x.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("largest,want", [(0.0, -100), (448.0, 0), (448.1, 1), (1.75, -8), (1.7578125, -7), (1e-38, -100),
                                          (3.3e38, 119), (1.0, -8), (2.0, -7)])
def test_oracle_exponents(largest, want):
    assert oracle.exponent(largest) == want


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("block", [32, 64])
def test_layout_is_a_permutation(head_dim, block):
    for value in (False, True):
        at = oracle.offsets(block, head_dim, value)
        assert torch.equal(at.sort().values, torch.arange(block * head_dim))


def test_oracle_reserve_by_hand():
    table, out = oracle.reserve([[5, -1, -1], [7, 2, -1], [-1, -1, -1]], [30, 64, 0], [3, 1, 33], [9, 4, 8, 6, 3], 4, 40, 32)
    assert table == [[5, 6, -1], [7, 2, 8], [4, 9, -1]]
    assert out["writes"] == [[5, 30, 0, 2], [6, 0, 2, 1], [8, 0, 3, 1], [4, 0, 4, 32], [9, 0, 36, 1]]
    assert out["slots"][:5] == [190, 191, 192, 256, 128] and out["slots"][36] == 288 and out["slots"][37:] == [-1] * 3
    assert out["positions"][:5] == [30, 31, 32, 64, 0] and out["q_cu"] == [0, 3, 4, 37]
    assert out["free_left"] == 0 and out["lengths"] == [33, 65, 33]


@pytest.mark.parametrize("causal,window", [(True, -1), (False, -1), (True, 3), (False, 0)])
def test_oracle_attention_row_by_row_and_whole(causal, window):
    gen = torch.Generator().manual_seed(0)
    query, key, value = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64) for n, h in ((9, 4), (7, 2), (7, 2)))
    a = oracle.attention(query, key, value, 0.5, causal, window)
    b = oracle.attention_whole(query, key, value, 0.5, causal, window)
    assert torch.allclose(a, b, atol=1e-12)
    assert not causal or (a[:2] == 0).all()


# ---- refusals of the Python entry points (nothing here has a GPU: a call that passes the checks ends at the device's)

def _cache(blocks=4, kv_heads=2, head_dim=64, block=32):
    return kv_cache.create(blocks, kv_heads, head_dim, block, device="cpu")


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def _reserve(**change):
    call = {"table": torch.full((2, 4), -1, dtype=torch.int32), "lengths": _ints(0, 5), "counts": _ints(3, 1),
            "free": _ints(0, 1, 2), "free_count": _ints(3), "rows": 4, "block_size": 32}
    return kv_cache.reserve(**{**call, **change})


def test_calls_on_the_cpu_are_refused():
    cache, table = _cache(), torch.zeros((1, 2), dtype=torch.int32)
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="MI355X"):
        _reserve()
    with pytest.raises(ValueError, match="MI355X"):
        kv_cache.append(cache, rows, rows, torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(ValueError, match="MI355X"):
        kv_cache.read(cache, table, _ints(3), 3)
    with pytest.raises(ValueError, match="MI355X"):
        kv_cache.attend(rows, cache, table, _ints(0, 3), _ints(3), 3, 0.125)


@pytest.mark.parametrize("change", [
    {"table": torch.zeros(4, dtype=torch.int32)}, {"table": torch.zeros((2, 4), dtype=torch.int64)},
    {"table": torch.zeros((2, 0), dtype=torch.int32)}, {"table": torch.zeros((4, 2), dtype=torch.int32).t()},
    {"table": torch.zeros((1, 4), dtype=torch.int32).expand(2, 4)},
    {"lengths": _ints(0)}, {"lengths": torch.zeros(2, dtype=torch.int64)}, {"counts": _ints(1, 2, 3)},
    {"counts": _ints(1, 0, 2, 0)[::2]}, {"free": torch.zeros((1, 3), dtype=torch.int32)}, {"free_count": _ints(1, 2)},
    {"rows": -1}, {"rows": 1 << 31}, {"block_size": 16}, {"block_size": 48}], ids=str)
def test_reserve_refuses(change):
    with pytest.raises(ValueError) as e:
        _reserve(**change)
    assert "MI355X" not in str(e.value)


@pytest.mark.parametrize("args", [(0, 2, 64, 32), (4, 0, 64, 32), (4, 2, 96, 32), (4, 2, 64, 16)])
def test_create_refuses(args):
    with pytest.raises(ValueError):
        kv_cache.create(*args, device="cpu")


@pytest.mark.parametrize("change", [
    {"keys": torch.zeros((4, 2, 2048), dtype=torch.uint8)}, {"values": torch.zeros((4, 2, 4096)).to(torch.float8_e4m3fn)},
    {"scales": torch.zeros((4, 2))}, {"scales": torch.zeros((4, 2, 2), dtype=torch.float64)}, {"block_size": 64},
    {"block_size": 33}, {"scales": torch.zeros((4, 2, 4))[..., ::2]}], ids=str)
def test_caches_that_do_not_fit_are_refused(change):
    cache = _cache()._replace(**change)
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    for call in (lambda: kv_cache.append(cache, rows, rows, torch.zeros((1, 4), dtype=torch.int32)),
                 lambda: kv_cache.read(cache, torch.zeros((1, 2), dtype=torch.int32), _ints(3), 3),
                 lambda: kv_cache.attend(rows, cache, torch.zeros((1, 2), dtype=torch.int32), _ints(0, 3), _ints(3), 3,
                                         0.125)):
        with pytest.raises(ValueError) as e:
            call()
        assert "MI355X" not in str(e.value)


@pytest.mark.parametrize("key,value,writes", [
    (torch.zeros((3, 2, 64)), None, None), (torch.zeros((3, 1, 64), dtype=torch.bfloat16), None, None),
    (torch.zeros((3, 2, 128), dtype=torch.bfloat16), None, None), (torch.zeros((3, 128), dtype=torch.bfloat16), None, None),
    (None, torch.zeros((4, 2, 64), dtype=torch.bfloat16), None),
    (torch.zeros((3, 2, 128), dtype=torch.bfloat16)[..., ::2], None, None),
    (torch.zeros((3, 2, 65), dtype=torch.bfloat16)[..., :64], None, None),
    (None, None, torch.zeros((1, 3), dtype=torch.int32)), (None, None, torch.zeros((1, 4), dtype=torch.int64)),
    (None, None, torch.zeros((4, 4), dtype=torch.int32).t())], ids=lambda t: "" if t is None else str(tuple(t.shape)))
def test_append_refuses(key, value, writes):
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError) as e:
        kv_cache.append(_cache(), rows if key is None else key, rows if value is None else value,
                        torch.zeros((1, 4), dtype=torch.int32) if writes is None else writes)
    assert "MI355X" not in str(e.value)


def test_append_and_attend_refuse_an_autograd_call():
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache.append(_cache(), rows, rows.detach(), torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache.attend(rows, _cache(), torch.zeros((1, 2), dtype=torch.int32), _ints(0, 3), _ints(3), 3, 0.125)


@pytest.mark.parametrize("change", [
    {"query": torch.zeros((3, 4, 64))}, {"query": torch.zeros((3, 3, 64), dtype=torch.bfloat16)},
    {"query": torch.zeros((3, 4, 128), dtype=torch.bfloat16)},
    {"query": torch.zeros((3, 4, 128), dtype=torch.bfloat16)[..., ::2]}, {"q_cu": _ints(0, 1, 3)},
    {"q_cu": torch.zeros(2, dtype=torch.int64)}, {"lengths": _ints(3, 3)}, {"max_q": -1}, {"max_q": 1 << 31},
    {"window": -2}, {"window": 1 << 31},
    {"total_keys": -1}, {"total_keys": 1 << 31},
    {"table": torch.zeros((1, 2), dtype=torch.int64)}], ids=str)
def test_attend_refuses(change):
    call = {"query": torch.zeros((3, 4, 64), dtype=torch.bfloat16), "cache": _cache(),
            "table": torch.zeros((1, 2), dtype=torch.int32), "q_cu": _ints(0, 3), "lengths": _ints(3), "max_q": 3,
            "scale": 0.125, "window": -1}
    with pytest.raises(ValueError) as e:
        kv_cache.attend(**{**call, **change})
    assert "MI355X" not in str(e.value)


# ---- refusals of the C ABI (the pointers are never followed)

def _c_cache(**change):
    c = _lib.KarpoCache(0x100000, 0x200000, 0x300000, 4, 2, 64, 32)
    for name, value in change.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change,status", [
    ({"head_dim": 96}, _lib.ERR_HEAD_DIM), ({"kv_heads": 0}, _lib.ERR_HEADS), ({"kv_heads": 8193}, _lib.ERR_HEADS), ({"block_size": 16}, _lib.ERR_ARG),
    ({"blocks": 0}, _lib.ERR_ARG), ({"blocks": 1 << 31}, _lib.ERR_ARG), ({"keys": None}, 1), ({"values": None}, 1),
    ({"scales": None}, 1), ({"keys": 4100}, _lib.ERR_LAYOUT), ({"scales": 4100}, _lib.ERR_LAYOUT)], ids=str)
def test_c_abi_refuses_caches(change, status):
    lib, c = _lib.load(), _c_cache(**change)
    append = _lib.KarpoCacheAppendArgs(c, 4096, 4096, 128, 64, 128, 64, 3, 4096, 1)
    read = _lib.KarpoCacheReadArgs(c, 4096, 2, 2, 1, 4096, 4096, 4096, 3, 4096)
    attend = _lib.KarpoCacheAttendArgs(c, 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 2, 2, 1, 2, 3, 3, 3, 0.1, -1, 0)
    assert lib.karpo_cache_append(ctypes.byref(append), None) == status
    assert lib.karpo_cache_read(ctypes.byref(read), None) == status
    assert lib.karpo_cache_attend(ctypes.byref(attend), None) == status
    assert lib.karpo_cache_attend_workspace_bytes(ctypes.byref(attend), ctypes.byref(ctypes.c_size_t())) == status


@pytest.mark.parametrize("change,status", [
    ({"block_size": 8}, _lib.ERR_ARG), ({"rows": -1}, _lib.ERR_ARG), ({"rows": 1 << 31}, _lib.ERR_ARG),
    ({"n_seq": -1}, _lib.ERR_ARG), ({"width": 0}, _lib.ERR_ARG), ({"table_stride": 3}, _lib.ERR_ARG),
    ({"width": 1 << 22, "table_stride": 1 << 22}, _lib.ERR_ARG), ({"free_capacity": -1}, _lib.ERR_ARG),
    ({"writes_capacity": 3}, _lib.ERR_ARG), ({"table": None}, 1), ({"lengths": None}, 1), ({"counts": None}, 1),
    ({"free_blocks": None}, 1), ({"free_count": None}, 1), ({"q_cu": None}, 1), ({"new_lengths": None}, 1),
    ({"slots": None}, 1), ({"positions": None}, 1), ({"writes": None}, 1), ({"free_left": None}, 1), ({"status": None}, 1),
    ({"writes": 0x90008}, _lib.ERR_LAYOUT), ({"slots": 0x70004}, _lib.ERR_LAYOUT),
    ({"new_lengths": 0x20000}, _lib.ERR_ARG),  # would be read by one workgroup while another writes it
    ({"free_left": 0x50000}, _lib.ERR_ARG), ({"status": 0x60000}, _lib.ERR_ARG)], ids=str)
def test_c_abi_reserve_refuses(change, status):
    a = _lib.KarpoCacheReserveArgs(0x10000, 4, 4, 2, 0x20000, 0x30000, 0x40000, 0x50000, 3, 32, 4, 0x60000, 0x65000, 0x70000,
                                   0x80000, 0x90000, 4, 0xa0000, 0xb0000)
    for name, value in change.items():
        setattr(a, name, value)
    assert _lib.load().karpo_cache_reserve(ctypes.byref(a), None) == status
    assert _lib.load().karpo_cache_reserve(None, None) == 1


@pytest.mark.parametrize("rows,n,block,want", [(48, 48, 64, 48), (0, 5, 32, 0), (65536, 64, 32, 2176), (10, 1, 32, 2),
                                               (2, 1, 32, 2), (-1, 1, 32, 0), (5, 1, 16, 0), (1 << 31, 1, 32, 0)])
def test_writes_capacity(rows, n, block, want):
    assert _lib.load().karpo_cache_writes_capacity(rows, n, block) == want


@pytest.mark.parametrize("change,status", [
    ({"heads": 3}, _lib.ERR_HEADS), ({"heads": 0}, _lib.ERR_HEADS), ({"window_left": -2}, _lib.ERR_WINDOW),
    ({"window_right": -2}, _lib.ERR_WINDOW), ({"max_q": -1}, _lib.ERR_ARG), ({"total_q": -1}, _lib.ERR_ARG),
    ({"total_keys": -1}, _lib.ERR_ARG), ({"total_keys": 1 << 31}, _lib.ERR_ARG), ({"n_seq": -1}, _lib.ERR_ARG),
    ({"n_seq": 1 << 23}, _lib.ERR_ARG), ({"table_stride": 255}, _lib.ERR_ARG),
    ({"table": None}, 1), ({"lengths": None}, 1), ({"q": None}, 1), ({"o": None}, 1), ({"q_cu": None}, 1),
    ({"q": 4104}, _lib.ERR_LAYOUT), ({"q_stride_tok": 4}, _lib.ERR_LAYOUT), ({"o_stride_head": 60}, _lib.ERR_LAYOUT),
    ({"workspace": None}, 5), ({"workspace_bytes": 16}, 5), ({"workspace": 4104}, 5)], ids=str)
def test_c_abi_attend_refuses(change, status):
    a = _lib.KarpoCacheAttendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 256, 256, 1, 4, 3, 3, 8000, 0.1,
                                  -1, 0, 4096, 1 << 40)
    for name, value in change.items():
        setattr(a, name, value)
    assert _lib.load().karpo_cache_attend(ctypes.byref(a), None) == status


def test_c_abi_append_refuses_keys_and_values_of_one_memory():
    a = _lib.KarpoCacheAppendArgs(_c_cache(values=0x100000 + 16), 4096, 4096, 128, 64, 128, 64, 3, 4096, 1)
    assert _lib.load().karpo_cache_append(ctypes.byref(a), None) == _lib.ERR_ARG


def test_c_abi_calls_without_rows_launch_nothing():
    lib = _lib.load()
    a = _lib.KarpoCacheAppendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 0, 4096, 1)
    assert lib.karpo_cache_append(ctypes.byref(a), None) == 0
    b = _lib.KarpoCacheAttendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 2, 2, 1, 4, 3, 0, 3, 0.1, -1, 0)
    assert lib.karpo_cache_attend(ctypes.byref(b), None) == 0
    b.total_q, b.max_q = 3, 0
    assert lib.karpo_cache_attend(ctypes.byref(b), None) == 0


def _calls_with(rows):
    """``append`` of keys, of values, and ``attend`` of queries."""
    plain, writes = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros((1, 4), dtype=torch.int32)
    return (lambda: kv_cache.append(_cache(), rows, plain, writes), lambda: kv_cache.append(_cache(), plain, rows, writes),
            lambda: kv_cache.attend(rows, _cache(), torch.zeros((1, 2), dtype=torch.int32), _ints(0, 3), _ints(3), 3, 0.125))


@pytest.mark.parametrize("grad", [True, False])
def test_append_and_attend_refuse_inputs_with_a_tangent(grad):
    """A tangent would be lost without a word: refused, also where no backward is recorded; not under inference_mode, which
    carries none."""
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(rows, torch.ones_like(rows))
        with torch.set_grad_enabled(grad):
            for call in _calls_with(dual):
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call()
            for call in _calls_with(rows):
                with pytest.raises(ValueError, match="MI355X"):
                    call()
        with torch.inference_mode():
            for call in _calls_with(dual):
                with pytest.raises(ValueError, match="MI355X"):
                    call()


def test_attend_refuses_a_function_transform():
    def f(rows):
        return _calls_with(rows)[2]()

    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(f, (rows,), (rows,))
    with pytest.raises(RuntimeError, match="no backward"):
        torch.func.grad(lambda x: f(x).sum())(rows)


def test_fake_tensors_are_refused():
    """They have no memory to give to a kernel."""
    with torch._subclasses.FakeTensorMode():
        cache = kv_cache.create(4, 2, 64, 32, device="cuda")
        rows = torch.empty((3, 2, 64), dtype=torch.bfloat16, device="cuda")
        table, one, two = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((1, 2), (1,), (2,)))
        for call in (lambda: kv_cache.reserve(table, one, one, two, one, 3, 32),
                     lambda: kv_cache.append(cache, rows, rows, torch.empty((1, 4), dtype=torch.int32, device="cuda")),
                     lambda: kv_cache.read(cache, table, one, 3),
                     lambda: kv_cache.attend(rows, cache, table, two, one, 3, 0.125)):
            with pytest.raises(RuntimeError, match="real tensors"):
                call()


@pytest.mark.parametrize("tokens", [40, 90, 1000])
def test_the_tolerance_of_attentions_weights_tells_one_bf16_term_from_two(tokens):
    """The GPU test's two tokens of nearly one score whose values cancel: with the weights planted here as one bf16 term the
    difference is outside the output's rounding plus 2^-14 of the weighted |value|, with two terms inside."""
    inside = {1: True, 2: True}
    for i in range(16):
        x = (0.5 + torch.tensor(i / 32)).bfloat16().double()
        score, value = torch.zeros(tokens, dtype=torch.float64), torch.zeros(tokens, dtype=torch.float64)
        score[0], score[1], value[0], value[1] = x, 0.875 * x, 1.0, -1.0
        w = torch.exp(score - score.max())
        want, size = (w * value).sum() / w.sum(), (w * value.abs()).sum() / w.sum()
        high = w.bfloat16().double()
        for terms, p in ((1, high), (2, high + (w - high).bfloat16().double())):
            out = ((p * value).sum() / w.sum()).bfloat16().double()
            inside[terms] &= bool((out - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -14)
    assert inside == {1: False, 2: True}
