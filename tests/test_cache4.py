"""The block cache in 4 bits, and append's norms and rotation, on the CPU: what ``kv_cache`` and the C ABI refuse before anything
reaches a GPU, and the oracle that the GPU tests compare with, pinned by known answers."""

from __future__ import annotations

import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

from karpo_decision_amd import _lib, build, kv_cache, ops
from oracle import cache4 as oracle

HEADER = Path(__file__).resolve().parents[1] / "include" / "karpo_cache4.h"


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_library_exports_every_declared_function():
    names = set(re.findall(r"^\s*(?:int|int64_t)\s+(karpo_cache4_\w+)\s*\(", HEADER.read_text(), re.M))
    assert names == set(_lib.CACHE4_EXPORTS)
    for name in names:
        assert hasattr(_lib.load(), name), name


@pytest.mark.parametrize("packed,named", [
    (kv_cache._APPEND_ROWS, _lib.KarpoCacheAppendRopeArgs), (kv_cache._APPEND_ROWS, _lib.KarpoCache4AppendArgs),
    (kv_cache._READ, _lib.KarpoCache4ReadArgs), (kv_cache._ATTEND, _lib.KarpoCache4AttendArgs)], ids=lambda x: "")
def test_packed_arguments_are_the_structures(packed, named):
    def leaves(s):
        for name, kind in s._fields_:
            if issubclass(kind, ctypes.Structure):
                yield from leaves(getattr(s, name))
            else:
                yield getattr(s, name)

    assert packed.size == ctypes.sizeof(named)
    values = list(range(1, len(list(leaves(named()))) + 1))
    assert list(leaves(named.from_buffer_copy(packed.pack(*values)))) == values


# ---- the oracle

@pytest.mark.parametrize("x,want", [(0.0, 0.0), (0.24, 0.0), (0.25, 0.0), (0.26, 0.5), (0.75, 1.0), (1.25, 1.0), (1.26, 1.5),
                                    (1.75, 2.0), (2.5, 2.0), (2.51, 3.0), (3.5, 4.0), (5.0, 4.0), (5.1, 6.0), (6.9, 6.0),
                                    (-0.3, -0.5), (-5.0, -4.0), (math.inf, 6.0), (-math.inf, -6.0)])
def test_oracle_rounds(x, want):
    assert oracle.rounded(x) == want


@pytest.mark.parametrize("largest,want", [(0.0, -100), (6.0, 0), (6.1, 1), (1.5, -2), (1.51, -1), (1e-38, -100), (3.3e38, 125),
                                          (3.0, -1)])
def test_oracle_exponents(largest, want):
    assert oracle.exponent(largest) == want


@pytest.mark.parametrize("head_dim", [64, 128, 256, 512])
@pytest.mark.parametrize("block", [32, 64])
def test_layout_is_a_permutation(head_dim, block):
    """Each byte has two elements, each scale 32, keys' and values' scales apart."""
    scales = []
    for value in (False, True):
        at, scale_at = oracle.offsets(block, head_dim, value)
        assert torch.equal(at.reshape(-1).sort().values, torch.arange(block * head_dim // 2).repeat_interleave(2))
        assert torch.equal(at[:, ::2], at[:, 1::2])
        assert (scale_at.view(block, -1, 32) == scale_at.view(block, -1, 32)[..., :1]).all()
        scales.append(scale_at[:, ::32].reshape(-1))
    assert torch.equal(torch.cat(scales).sort().values, torch.arange(block * head_dim // 16))


def test_oracle_prologue_by_hand():
    x = torch.tensor([[[3.0, 4.0] + [0.0] * 30]])
    out = oracle.normed(x, (ops.NORM_PLAIN, None, 0.0))
    assert torch.allclose(out[0, 0, :2], torch.tensor([3.0, 4.0], dtype=torch.float64) / math.sqrt(25 / 32))
    turn, size = oracle.turned(torch.arange(4.0, dtype=torch.float64).view(1, 1, 4) + 1,
                               (torch.zeros(3, 2), torch.ones(3, 2)), torch.tensor([2]))
    assert turn.tolist() == [[[-2.0, 1.0, 3.0, 4.0]]] and size.tolist() == [[[2.0, 1.0, 3.0, 4.0]]]
    assert torch.isnan(oracle.turned(torch.ones(1, 1, 4).double(), (torch.zeros(3, 2), torch.ones(3, 2)),
                                     torch.tensor([3]))[0][..., :2]).all()


# ---- refusals of the Python entry points

def _cache(blocks=4, kv_heads=2, head_dim=64, block=32, bits=4):
    return kv_cache.create(blocks, kv_heads, head_dim, block, device="cpu", bits=bits)


def _rows(n=3, heads=2, d=64):
    return torch.zeros((n, heads, d), dtype=torch.bfloat16)


def _writes():
    return torch.zeros((1, 4), dtype=torch.int32)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("head_dim,block", [(64, 32), (128, 64), (512, 128)])
def test_create(bits, head_dim, block):
    cache = _cache(3, 2, head_dim, block, bits)
    assert (cache.bits, cache.blocks, cache.kv_heads, cache.head_dim, cache.block_size) == (bits, 3, 2, head_dim, block)
    if bits == 4:
        total = sum(t.view(torch.uint8).numel() for t in cache[:3])
        assert total * 32 == 3 * 2 * 2 * head_dim * block * 17  # 4.25 bits an element


@pytest.mark.parametrize("args", [(0, 2, 64, 32), (4, 0, 64, 32), (4, 2, 96, 32), (4, 2, 64, 16)])
def test_create_refuses(args):
    with pytest.raises(ValueError):
        kv_cache.create(*args, device="cpu", bits=4)


@pytest.mark.parametrize("bits", [2, 16, 0])
def test_create_refuses_other_bits(bits):
    with pytest.raises(ValueError, match="bits"):
        kv_cache.create(4, 2, 64, 32, device="cpu", bits=bits)


def test_calls_on_the_cpu_are_refused():
    cache, table = _cache(), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: kv_cache.append(cache, _rows(), _rows(), _writes()),
                 lambda: kv_cache.append(_cache(bits=8), _rows(), _rows(), _writes(), k_norm=ops.Norm(ops.NORM_PLAIN, None, 1e-6)),
                 lambda: kv_cache.read(cache, table, _ints(3), 3),
                 lambda: kv_cache.attend(_rows(), cache, table, _ints(0, 3), _ints(3), 3, 0.125)):
        with pytest.raises(ValueError, match="MI355X"):
            call()


E8M0 = torch.float8_e8m0fnu


@pytest.mark.parametrize("change", [
    {"values": torch.zeros((4, 2, 1024), dtype=torch.uint8)}, {"values": torch.zeros((4, 2, 2048)).to(torch.float8_e4m3fn)},
    {"keys": torch.zeros((4, 2, 2048), dtype=torch.uint8).view(torch.float4_e2m1fn_x2)},
    {"scales": torch.zeros((4, 2, 2))}, {"scales": torch.zeros((4, 2, 1, 2, 64), dtype=torch.uint8)},
    {"scales": torch.zeros((4, 2, 2, 2, 32), dtype=torch.uint8).view(E8M0)},
    {"scales": torch.zeros((4, 2, 1, 64, 2), dtype=torch.uint8).view(E8M0).transpose(3, 4)},
    {"block_size": 64}, {"block_size": 33}], ids=str)
def test_caches_that_do_not_fit_are_refused(change):
    cache = _cache()._replace(**change)
    for call in (lambda: kv_cache.append(cache, _rows(), _rows(), _writes()),
                 lambda: kv_cache.read(cache, torch.zeros((1, 2), dtype=torch.int32), _ints(3), 3),
                 lambda: kv_cache.attend(_rows(), cache, torch.zeros((1, 2), dtype=torch.int32), _ints(0, 3), _ints(3), 3, 0.1)):
        with pytest.raises(ValueError) as e:
            call()
        assert "MI355X" not in str(e.value)


def _tables(n=8, r=64):
    return torch.ones((n, r), dtype=torch.bfloat16), torch.zeros((n, r), dtype=torch.bfloat16)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("more", [
    {"k_norm": ops.Norm(ops.NORM_WEIGHT, torch.ones(32), 1e-6)}, {"k_norm": ops.Norm(ops.NORM_WEIGHT, None, 1e-6)},
    {"v_norm": ops.Norm(ops.NORM_ONE_PLUS, torch.ones(2, 64), 1e-6)}, {"v_norm": ops.Norm(ops.NORM_ONE_PLUS, None, 1e-6)},
    {"positions": _ints(0, 1, 2)}, {"rope": _tables(2)}, {"rope": _tables(8, 96)}, {"rope": _tables(8, 16)},
    {"rope": (_tables()[0], _tables(8, 32)[1])}, {"rope": (_tables()[0][0], _tables()[1][0])},
    {"rope": _tables(), "positions": _ints(0, 1)}, {"rope": _tables(), "positions": torch.zeros(3, dtype=torch.int64)},
    {"rope": _tables(), "positions": torch.zeros((3, 1), dtype=torch.int32)},
    {"rope": _tables(), "positions": _ints(0, 1, 2, 3, 4, 5)[::2]}, {"rope": _tables(0)}], ids=lambda m: ",".join(m))
def test_append_refuses_prologues(bits, more):
    with pytest.raises(ValueError) as e:
        kv_cache.append(_cache(bits=bits), _rows(), _rows(), _writes(), **more)
    assert "MI355X" not in str(e.value)


@pytest.mark.parametrize("bits", [4, 8])
def test_append_refuses_weights_and_tables_that_require_a_gradient(bits):
    weight = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16))
    for more in ({"k_norm": ops.Norm(ops.NORM_WEIGHT, weight, 1e-6)}, {"v_norm": ops.Norm(ops.NORM_ONE_PLUS, weight, 1e-6)},
                 {"rope": (_tables()[0].requires_grad_(), _tables()[1])}):
        with pytest.raises(RuntimeError, match="no backward"):
            kv_cache.append(_cache(bits=bits), _rows(), _rows(), _writes(), **more)
        with torch.no_grad(), pytest.raises(ValueError, match="MI355X"):
            kv_cache.append(_cache(bits=bits), _rows(), _rows(), _writes(), **more)


def test_append_and_attend_refuse_an_autograd_call():
    rows = _rows().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache.append(_cache(), rows, _rows(), _writes())
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache.attend(rows, _cache(), torch.zeros((1, 2), dtype=torch.int32), _ints(0, 3), _ints(3), 3, 0.125)


def test_fake_tensors_are_refused():
    with torch._subclasses.FakeTensorMode():
        cache = kv_cache.create(4, 2, 64, 32, device="cuda", bits=4)
        rows = torch.empty((3, 2, 64), dtype=torch.bfloat16, device="cuda")
        table, one, two = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((1, 2), (1,), (2,)))
        for call in (lambda: kv_cache.append(cache, rows, rows, torch.empty((1, 4), dtype=torch.int32, device="cuda")),
                     lambda: kv_cache.read(cache, table, one, 3),
                     lambda: kv_cache.attend(rows, cache, table, two, one, 3, 0.125)):
            with pytest.raises(RuntimeError, match="real tensors"):
                call()


@pytest.mark.parametrize("first", [1, 3, 4, 8])
def test_tables_at_any_address_are_taken(first):
    """Weights and tables that begin anywhere in a larger tensor: the kernels load 16 bytes at once."""
    whole = torch.arange(9 * 64 + 8, dtype=torch.float32).bfloat16()
    for t in (whole[first:first + 64], whole[first:first + 9 * 64].view(9, 64)):
        got = ops._bf16_table(t, t.device)
        assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, t)
        assert got.data_ptr() == t.data_ptr() or t.data_ptr() % 16


# ---- refusals of the C ABI (the pointers are never followed)

def _c_cache(**change):
    c = _lib.KarpoCache4(0x100000, 0x200000, 0x300000, 4, 2, 64, 32)
    for name, value in change.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change,status", [
    ({"head_dim": 96}, _lib.ERR_HEAD_DIM), ({"kv_heads": 0}, _lib.ERR_HEADS), ({"kv_heads": 8193}, _lib.ERR_HEADS),
    ({"block_size": 16}, _lib.ERR_ARG), ({"blocks": 0}, _lib.ERR_ARG), ({"blocks": 1 << 31}, _lib.ERR_ARG), ({"keys": None}, 1),
    ({"values": None}, 1), ({"scales": None}, 1), ({"keys": 4100}, _lib.ERR_LAYOUT), ({"scales": 4104}, _lib.ERR_LAYOUT)], ids=str)
def test_c_abi_refuses_caches(change, status):
    lib, c = _lib.load(), _c_cache(**change)
    append = _lib.KarpoCache4AppendArgs(c, 4096, 4096, 128, 64, 128, 64, 3, 4096, 1)
    read = _lib.KarpoCache4ReadArgs(c, 4096, 2, 2, 1, 4096, 4096, 4096, 3, 4096)
    attend = _lib.KarpoCache4AttendArgs(c, 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 2, 2, 1, 2, 3, 3, 3, 0.1, -1, 0)
    assert lib.karpo_cache4_append(ctypes.byref(append), None) == status
    assert lib.karpo_cache4_read(ctypes.byref(read), None) == status
    assert lib.karpo_cache4_attend(ctypes.byref(attend), None) == status
    assert lib.karpo_cache4_attend_workspace_bytes(ctypes.byref(attend), ctypes.byref(ctypes.c_size_t())) == status


@pytest.mark.parametrize("change,status", [
    ({"heads": 3}, _lib.ERR_HEADS), ({"window_left": -2}, _lib.ERR_WINDOW), ({"max_q": -1}, _lib.ERR_ARG),
    ({"total_keys": 1 << 31}, _lib.ERR_ARG), ({"n_seq": 1 << 23}, _lib.ERR_ARG), ({"table_stride": 255}, _lib.ERR_ARG),
    ({"table": None}, 1), ({"q": None}, 1), ({"q_cu": None}, 1), ({"q": 4104}, _lib.ERR_LAYOUT),
    ({"workspace": None}, 5), ({"workspace_bytes": 16}, 5), ({"workspace": 4104}, 5)], ids=str)
def test_c_abi_attend_refuses(change, status):
    a = _lib.KarpoCache4AttendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 256, 256, 1, 4, 3, 3, 8000, 0.1,
                                   -1, 0, 4096, 1 << 40)
    for name, value in change.items():
        setattr(a, name, value)
    assert _lib.load().karpo_cache4_attend(ctypes.byref(a), None) == status


GOOD = {"k_norm": 1, "k_norm_eps": 1e-6, "k_norm_weight": 0x5000, "v_norm": 3, "rope_cos": 0x6000, "rope_sin": 0x7000,
        "rope_stride": 64, "rope_rows": 3, "rope_dim": 64}


@pytest.mark.parametrize("change", [
    {"k_norm": 4}, {"k_norm": -1}, {"v_norm": 1}, {"v_norm": 2}, {"k_norm_weight": None}, {"k_norm_weight": 0x5008},
    {"rope_sin": None}, {"rope_cos": None}, {"rope_dim": 16}, {"rope_dim": 0}, {"rope_dim": 96}, {"rope_dim": 40},
    {"rope_stride": 32}, {"rope_stride": 68}, {"rope_cos": 0x6004}, {"rope_rows": 0}, {"rope_rows": 2},
    {"positions": 0x8002}], ids=str)
def test_c_abi_append_refuses_prologues(change):
    prologue = _lib.KarpoCachePrologue(**{**GOOD, **change})
    four = _lib.KarpoCache4AppendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 3, 4096, 1, prologue)
    eight = _lib.KarpoCacheAppendRopeArgs(_lib.KarpoCacheAppendArgs(
        _lib.KarpoCache(0x100000, 0x200000, 0x300000, 4, 2, 64, 32), 4096, 4096, 128, 64, 128, 64, 3, 4096, 1), prologue)
    assert _lib.load().karpo_cache4_append(ctypes.byref(four), None) == _lib.ERR_PROLOGUE
    assert _lib.load().karpo_cache_append_rope(ctypes.byref(eight), None) == _lib.ERR_PROLOGUE


def test_c_abi_append_refuses_keys_and_values_of_one_memory():
    """(a block's codes are half of its elements in bytes: 4 blocks x 2 heads x 32 tokens x 64 / 2)"""
    for values, status in ((0x100000 + 16, _lib.ERR_ARG), (0x100000 + 8192 - 16, _lib.ERR_ARG), (0x100000 + 8192, 0)):
        a = _lib.KarpoCache4AppendArgs(_c_cache(values=values), 4096, 4096, 128, 64, 128, 64, 0, 4096, 1)
        assert _lib.load().karpo_cache4_append(ctypes.byref(a), None) == status


def test_c_abi_calls_without_rows_launch_nothing():
    lib = _lib.load()
    a = _lib.KarpoCache4AppendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 0, 4096, 1)
    assert lib.karpo_cache4_append(ctypes.byref(a), None) == 0
    b = _lib.KarpoCache4AttendArgs(_c_cache(), 4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 2, 2, 1, 4, 3, 0, 3, 0.1, -1, 0)
    assert lib.karpo_cache4_attend(ctypes.byref(b), None) == 0
    for fn in (lib.karpo_cache4_append, lib.karpo_cache4_read, lib.karpo_cache4_attend, lib.karpo_cache_append_rope):
        assert fn(None, None) == 1


def test_workspaces_go_by_the_format_of_the_call_alone():
    """80 requests of 1,000 tokens are split in 8 bits and taken whole in 4; what a call of the other format before it left on the
    stack changes neither."""
    lib, more = _lib.load(), (4096, 4096, 128, 64, 128, 64, 4096, 4096, 4096, 32, 32, 80, 4, 1, 80, 1000, 0.1, -1, 0)
    eight = _lib.KarpoCacheAttendArgs(_lib.KarpoCache(0x100000, 0x200000, 0x300000, 4, 2, 64, 32), *more)
    four = _lib.KarpoCache4AttendArgs(_c_cache(), *more)
    got = []
    for _ in range(4):
        for fn, a in ((lib.karpo_cache_attend_workspace_bytes, eight), (lib.karpo_cache4_attend_workspace_bytes, four)):
            need = ctypes.c_size_t()
            assert fn(ctypes.byref(a), ctypes.byref(need)) == 0
            a.workspace, a.workspace_bytes = 4096, need.value
            got.append(need.value)
    assert got == got[:2] * 4 and got[0] > 0 and got[1] == 0


def test_read_takes_lds_as_the_type_that_was_written(tmp_path):
    """The reading kernels' byte arrays in LDS hold integers (and vectors, which may alias anything). A scalar access of another
    type is one that the compiler may move across theirs, by its type tag in the compiled kernels' IR."""
    ir = tmp_path / "kernels.ll"
    subprocess.run([build.hipcc(), *build.HIP_FLAGS, "--cuda-device-only", "-S", "-emit-llvm", str(build.CSRC / "cache.hip"),
                    "-o", str(ir)], check=True, capture_output=True)
    text = ir.read_text()
    nodes = dict(re.findall(r"^(!\d+) = (.*)$", text, re.M))
    kinds = set()
    for line in text.splitlines():
        tag = re.search(r"\b(?:load|store) \w+\b.*addrspace\(3\).*!tbaa (!\d+)", line)
        if tag:
            kinds.add(nodes[re.match(r"!\{(!\d+)", nodes[tag[1]])[1]].split('"')[1])
    assert kinds == {"int"}
