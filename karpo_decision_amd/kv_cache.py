"""A block cache on MI355X: keys and values kept between calls in 8 or 4 bits, and the packed attention that reads them.

A serving step over requests that hold cached tokens (a prompt that more rounds or branches follow, an answer that grows):

    step = reserve(table, lengths, counts, free, free_count, rows, cache.block_size)  # once per step, for all layers
    append(cache, key, value, step.writes)                                            # each layer's own cache
    # or out of the projections: append(..., k_norm=ops.gemma_norm(attn.k_norm), rope=(cos, sin), positions=step.positions)
    out = attend(query, cache, table, step.q_cu, step.lengths, max_q, scale, total_keys=total)  # total: of step.lengths

``hip_attention.attend`` reads keys that live for one call; here they live in a pool of blocks of 32, 64 or 128 tokens
(``Cache``), found through a block table. An element is stored as an e4m3 code times a power of two that its block and
head share (8 bits), or as an e2m1 code times a power of two of its own for each 32 elements of a token's head (4.25 bits;
``create(bits=4)``), so a cached element is a bf16 value exactly, and ``read`` and ``attend`` work on the same numbers. All
calls take either cache.
Blocks that several requests' tables share are read only: a request appends to blocks of its own.

Lengths, bounds, tables and free lists are read on the device when the kernels run: nothing syncs, calls go on the
current stream of the tensors' device and capture into graphs. All of it is forward only. The calls are no torch operators:
torch.compile breaks its graph around them, and what has to record them whole (fullgraph, export) cannot.
"""

from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple

import torch
from torch import Tensor
from torch._subclasses import FakeTensor
from torch.autograd import forward_ad

from . import _lib
from .ops import NORM_NONE, NORM_ONE_PLUS, NORM_WEIGHT, Norm, _bf16_table, _current_stream, _on_device

BLOCK_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128, 256, 512)
_MOST = (1 << 31) - 1
_MOST_ROWS = _MOST - (1 << 16)

# The argument structures of karpo_cache.h, field by field (_lib has them by name): packing them costs a third of what
# building them by name does, and a small call's time is its host path. Those of karpo_cache4.h have the same layout.
_CACHE = "PPPqiii4x"
_RESERVE = struct.Struct("@PqiiPPPPiiqPPPPPqPP")
_APPEND = struct.Struct("@" + _CACHE + "PPqqqqqPq")
_APPEND_ROWS = struct.Struct("@" + _CACHE + "PPqqqqqPq" + "ifPifPPPqqi4xP")  # KarpoCacheAppendRopeArgs, KarpoCache4AppendArgs
_READ = struct.Struct("@" + _CACHE + "PqiiPPPqP")
_ATTEND = struct.Struct("@" + _CACHE + "PPqqqqPPPqiiiiqqfii4xPN")


_FP8, _FP4, _E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


class Cache(NamedTuple):
    """One layer's keys and values. In 8 bits: ``keys`` and ``values`` (blocks, kv heads, block_size * D) float8_e4m3fn, laid
    out as ``karpo_cache.h`` says, and ``scales`` (blocks, kv heads, 2) fp32, the powers of two of a block's keys and values. In
    4 bits: ``keys`` and ``values`` (blocks, kv heads, block_size * D / 2) float4_e2m1fn_x2 and ``scales`` (blocks, kv heads,
    block_size / 32, 2, D) float8_e8m0fnu, laid out as ``karpo_cache4.h`` says."""

    keys: Tensor
    values: Tensor
    scales: Tensor
    block_size: int

    @property
    def blocks(self) -> int:
        return self.keys.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.keys.shape[1]

    @property
    def head_dim(self) -> int:
        return self.keys.shape[2] * (8 // self.bits) // self.block_size

    @property
    def bits(self) -> int:
        return 4 if self.keys.dtype is _FP4 else 8


class Step(NamedTuple):
    """What ``reserve`` gives a step: ``q_cu`` (requests + 1) int32 bounds of the packed new tokens, ``lengths``
    (requests) int32 with the new tokens, ``slots`` (rows) int64 and ``positions`` (rows) int32 of each new token (-1 and
    0 behind the last), ``writes`` (n, 4) int32 (block, first slot, first row, tokens) for ``append``, ``free_left`` (1)
    int32, and ``status`` (1) int32: 0, or why nothing was reserved (then the table is untouched, the bounds are 0 and
    there are no writes)."""

    q_cu: Tensor
    lengths: Tensor
    slots: Tensor
    positions: Tensor
    writes: Tensor
    free_left: Tensor
    status: Tensor

    def check(self) -> None:
        """Waits for the device and raises where nothing was reserved: RuntimeError without enough free blocks,
        ValueError for lengths and counts out of range."""
        status = int(self.status.item())
        if status == _lib.CACHE_NO_BLOCKS:
            raise RuntimeError("reserve: not enough free blocks for the new tokens")
        if status:
            raise ValueError("reserve: lengths and counts must be non-negative, the counts within `rows`, a request's "
                             "tokens within its row of the table, and free_count within the free list")


def create(blocks: int, kv_heads: int, head_dim: int, block_size: int = 64,
           device: torch.device | str = "cuda", bits: int = 8) -> Cache:
    """An empty cache of ``blocks`` blocks, in 8 or 4 bits (an element is up to 2^-4 of its magnitude off in 8 bits; in 4, up to
    a quarter, or a twelfth of the largest of its 32 elements: 12% of the 2-norm for normally distributed ones)."""
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be 32, 64 or 128, not {block_size}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128, 256 or 512, not {head_dim}")
    if blocks < 1 or kv_heads < 1:
        raise ValueError(f"a cache has at least one block and one head, not {blocks} and {kv_heads}")
    if bits not in (4, 8):
        raise ValueError(f"bits must be 8 or 4, not {bits}")
    if bits == 4:
        keys, values = (torch.zeros((blocks, kv_heads, block_size * head_dim // 2), dtype=torch.uint8, device=device).view(_FP4)
                        for _ in range(2))
        scales = torch.zeros((blocks, kv_heads, block_size // 32, 2, head_dim), dtype=torch.uint8, device=device)
        return Cache(keys, values, scales.view(_E8M0), block_size)
    keys, values = (torch.zeros((blocks, kv_heads, block_size * head_dim), dtype=torch.uint8, device=device)
                    .view(torch.float8_e4m3fn) for _ in range(2))
    return Cache(keys, values, torch.zeros((blocks, kv_heads, 2), dtype=torch.float32, device=device), block_size)


def _cache_fields(cache: Cache, index: int) -> tuple[int, ...]:
    """The cache's fields of an argument structure; ``index``: the other tensors' device."""
    keys, values, scales, block = cache
    shape, fp8 = keys.shape, _FP8
    if keys.dtype is _FP4:
        return _cache4_fields(cache, index)
    if len(shape) == 3 and block in BLOCK_SIZES:  # all is well: one pass
        blocks, heads, size = shape
        head_dim = size // block
        if (head_dim in HEAD_DIMS and size == head_dim * block and values.shape == shape and blocks > 0 and heads > 0
                and scales.shape == (blocks, heads, 2) and keys.dtype is fp8 and values.dtype is fp8
                and scales.dtype is torch.float32 and keys.is_contiguous() and values.is_contiguous()
                and scales.is_contiguous() and keys.get_device() == values.get_device() == scales.get_device() == index):
            return keys.data_ptr(), values.data_ptr(), scales.data_ptr(), blocks, heads, head_dim, block
    # the refusal's message
    if keys.dtype != fp8 or values.dtype != fp8 or scales.dtype != torch.float32:
        raise ValueError(f"a cache has float8_e4m3fn keys and values and float32 scales, not {keys.dtype}, "
                         f"{values.dtype} and {scales.dtype}")
    if not keys.get_device() == values.get_device() == scales.get_device() == index:
        raise ValueError(f"the cache is on {keys.device}, {values.device} and {scales.device}, the other tensors elsewhere")
    raise ValueError(f"a cache has contiguous keys and values (blocks, kv heads, block_size * head_dim) and scales (blocks, "
                     f"kv heads, 2), block_size 32, 64 or 128 and head_dim 64, 128, 256 or 512, not {tuple(shape)}, "
                     f"{tuple(values.shape)}, {tuple(scales.shape)} and {block}")


def _cache4_fields(cache: Cache, index: int) -> tuple[int, ...]:
    keys, values, scales, block = cache
    shape = keys.shape
    if len(shape) == 3 and block in BLOCK_SIZES:
        blocks, heads, size = shape
        head_dim = 2 * size // block
        if (head_dim in HEAD_DIMS and 2 * size == head_dim * block and values.shape == shape and blocks > 0 and heads > 0
                and scales.shape == (blocks, heads, block // 32, 2, head_dim) and values.dtype is _FP4
                and scales.dtype is _E8M0 and keys.is_contiguous() and values.is_contiguous() and scales.is_contiguous()
                and keys.get_device() == values.get_device() == scales.get_device() == index):
            return keys.data_ptr(), values.data_ptr(), scales.data_ptr(), blocks, heads, head_dim, block
    if values.dtype != _FP4 or scales.dtype != _E8M0:
        raise ValueError(f"a cache in 4 bits has float4_e2m1fn_x2 keys and values and float8_e8m0fnu scales, not {keys.dtype}, "
                         f"{values.dtype} and {scales.dtype}")
    if not keys.get_device() == values.get_device() == scales.get_device() == index:
        raise ValueError(f"the cache is on {keys.device}, {values.device} and {scales.device}, the other tensors elsewhere")
    raise ValueError(f"a cache in 4 bits has contiguous keys and values (blocks, kv heads, block_size * head_dim / 2) and scales "
                     f"(blocks, kv heads, block_size / 32, 2, head_dim), block_size 32, 64 or 128 and head_dim 64, 128, 256 or "
                     f"512, not {tuple(shape)}, {tuple(values.shape)}, {tuple(scales.shape)} and {block}")


def _check_ints(index: int, **tensors: Tensor) -> None:
    """The refusal of device numbers (``_ints`` finds that there is one)."""
    for name, t in tensors.items():
        if t.dtype != torch.int32 or t.dim() != 1 or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 1-D int32 tensor on the other tensors' device")


def _ints(t: Tensor, index: int) -> bool:
    return t.dtype is torch.int32 and t.dim() == 1 and t.get_device() == index and t.is_contiguous()


def _table_fields(table: Tensor, lengths: Tensor, index: int) -> tuple[int, int, int, int]:
    """(pointer, row stride, blocks of a row, requests) of a block table that fits ``lengths``."""
    shape, strides = table.shape, table.stride()
    if len(shape) != 2 or table.dtype is not torch.int32 or table.get_device() != index:
        raise ValueError("table must be a (requests, blocks) int32 tensor on the other tensors' device")
    (n, width), (stride, inner) = shape, strides
    if width < 1 or inner != 1 or (stride < width and n > 1):
        raise ValueError(f"table must have contiguous rows of at least one block, not {(n, width)} with strides "
                         f"{(stride, inner)}")
    if not _ints(lengths, index):
        _check_ints(index, lengths=lengths)
    if lengths.numel() != n:
        raise ValueError(f"the table has {n} requests, lengths {lengths.numel()}")
    return table.data_ptr(), stride if stride >= width else width, width, n


def _on_gpu(what: str, index: int) -> None:
    if index < 0:
        raise ValueError(f"{what} runs on an MI355X GPU, not on the CPU")


def _real(what: str, t: Tensor) -> None:
    if type(t) is not Tensor and isinstance(t, FakeTensor):  # (has no memory, and these are no operators to record)
        raise RuntimeError(f"kv_cache.{what} runs on real tensors: a tracer cannot record it")


def _no_grad(what: str, *tensors: Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"kv_cache.{what} has no backward: call it under torch.inference_mode() or torch.no_grad()")
    # (without a dual level, nearly always, no tensor has a tangent: 0.07 us in place of 0.3 a tensor)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"kv_cache.{what} has no forward-mode derivative: call it under torch.inference_mode(), or with "
                           "tensors without tangents")


def reserve(table: Tensor, lengths: Tensor, counts: Tensor, free: Tensor, free_count: Tensor, rows: int,
            block_size: int) -> Step:
    """Room for ``counts[i]`` new tokens of each request i behind the ``lengths[i]`` it holds (int32 on the device): the
    entries of new blocks in ``table`` ((requests, blocks) int32, written in place), taken in the tokens' order from the
    end of the first ``free_count[0]`` entries of ``free``, and what the step's layers need (``Step``). ``rows`` bounds
    the counts' sum and is the packed new tokens' row count. The inputs but the table are left as they are: the free
    list goes on with ``free_left``, the requests with ``Step.lengths``."""
    _real("reserve", table)
    index = table.get_device()
    fields = _table_fields(table, lengths, index)
    n, rows = fields[3], int(rows)
    if not (_ints(counts, index) and _ints(free, index) and _ints(free_count, index)):
        _check_ints(index, counts=counts, free=free, free_count=free_count)
    if counts.numel() != n or free_count.numel() != 1:
        raise ValueError(f"counts must hold {n} requests and free_count one number, not {counts.numel()} and "
                         f"{free_count.numel()}")
    if not 0 <= rows <= _MOST_ROWS or block_size not in BLOCK_SIZES:
        raise ValueError(f"rows must lie in 0 .. {_MOST_ROWS} and block_size be 32, 64 or 128, not {rows} and {block_size}")
    _on_gpu("reserve", index)
    lib = _lib.load()
    jobs = lib.karpo_cache_writes_capacity(rows, n, block_size)
    # one allocation for the step: writes (16-byte aligned) and slots first
    buffer = table.new_empty(4 * jobs + 3 * rows + 2 * n + 3)
    writes, slots, positions, q_cu, new, left, status = torch.split_with_sizes(
        buffer, (4 * jobs, 2 * rows, rows, n + 1, n, 1, 1))
    at = buffer.data_ptr()
    slots_at = at + 16 * jobs
    positions_at = slots_at + 8 * rows
    q_at = positions_at + 4 * rows
    new_at = q_at + 4 * n + 4
    left_at = new_at + 4 * n
    args = _RESERVE.pack(*fields, lengths.data_ptr(), counts.data_ptr(), free.data_ptr(), free_count.data_ptr(),
                         free.numel(), block_size, rows, q_at, new_at, slots_at, positions_at, at, jobs, left_at,
                         left_at + 4)
    with _on_device(index):
        _lib.check(lib.karpo_cache_reserve(args, _current_stream(index)), "reserve")
    return Step(q_cu, new, slots.view(torch.int64), positions, writes.view(jobs, 4), left, status)


def _table_address(t: Tensor, index: int) -> int:
    """The address of a weight or table that is as the kernel takes it, or 0."""
    at = t.data_ptr()
    return at if t.dtype is torch.bfloat16 and t.get_device() == index and t.is_contiguous() and not at & 15 else 0


def _norm_fields(name: str, norm: Norm | None, key: Tensor, index: int, head_dim: int, keep: list) -> tuple[int, float, int]:
    """(mode, eps, weight's pointer) of one of ``append``'s norms."""
    if norm is None or norm.mode == NORM_NONE:
        return 0, 0.0, 0
    mode, weight = norm.mode, norm.weight
    if mode != NORM_WEIGHT and mode != NORM_ONE_PLUS:
        return mode, norm.eps, 0
    if weight is None or weight.shape != (head_dim,):
        raise ValueError(f"{name}'s weight must have shape ({head_dim},), not {None if weight is None else tuple(weight.shape)}")
    at = _table_address(weight, index)
    if not at:
        keep.append(_bf16_table(weight, key.device))
        at = keep[-1].data_ptr()
    return mode, norm.eps, at


def _rope_fields(rope: tuple[Tensor, Tensor] | None, positions: Tensor | None, key: Tensor, index: int, head_dim: int,
                 keep: list) -> tuple[int, ...]:
    """(cos, sin, stride, rows, rotated elements, positions) of ``append``'s rotation."""
    if rope is None:
        if positions is not None:
            raise ValueError("positions are rows of the rope tables: pass rope=(cos, sin) with them")
        return 0, 0, 0, 0, 0, 0
    cos, sin = rope
    shape = cos.shape
    if len(shape) == 2 and _table_address(cos, index) and _table_address(sin, index):
        stride = shape[1]
    else:
        cos, sin = (_bf16_table(t, key.device) for t in rope)
        shape = cos.shape
        if len(shape) == 2:
            stride = cos.stride(0)
            if stride != sin.stride(0) or stride < shape[1] or shape[0] == 1:
                cos, sin, stride = cos.contiguous(), sin.contiguous(), shape[1]
        keep += (cos, sin)
    if len(shape) != 2 or sin.shape != shape or shape[0] < 1 or shape[1] % 32 or not 0 < shape[1] <= head_dim:
        raise ValueError(f"rope tables must be two (positions, rotated) tables of one shape, rotated a multiple of 32 up to "
                         f"{head_dim}, not {tuple(shape)} and {tuple(sin.shape)}")
    at, rows = 0, key.shape[0]
    if positions is None:
        if shape[0] < rows:
            raise ValueError(f"without positions the rope tables need a row for each of {rows} rows, not {shape[0]}")
    else:
        if not _ints(positions, index):
            _check_ints(index, positions=positions)
        if positions.numel() != rows:
            raise ValueError(f"positions must hold a number for each of {rows} rows, not {positions.numel()}")
        at = positions.data_ptr()
    return cos.data_ptr(), sin.data_ptr(), stride, shape[0], shape[1], at


def append(cache: Cache, key: Tensor, value: Tensor, writes: Tensor, *, k_norm: Norm | None = None, v_norm: Norm | None = None,
           rope: tuple[Tensor, Tensor] | None = None, positions: Tensor | None = None) -> None:
    """New keys and values (rows, kv heads, D) bf16 into the blocks that ``writes`` lists (``Step.writes``; no block
    twice). In 8 bits a block's scale is the least power of two that holds what it got; where new tokens need a larger one, the
    block's earlier tokens are rounded again to it. In 4 bits each 32 elements have their own, and a NaN among them makes all of
    them NaN. What lies past the format's range at the largest scale, infinities too, is stored at the range's end, NaN as NaN.
    Rows and slots that no write names are left as they were.

    ``k_norm`` and ``v_norm`` (``ops.gemma_norm``, ``ops.qwen_norm``) norm the rows on the way, ``rope`` then turns the keys by
    halves over their first R elements: bf16 tables (cos, sin) of shape (positions, R), of which row i's is row ``positions[i]``
    (int32, ``Step.positions``), or row i without. All in fp32, rounded once, to the cache's codes (``ops.norm_rope`` before a
    plain append rounds to bf16 twice more). A key whose position is outside the tables gets NaN for what is turned."""
    _real("append", key)
    _no_grad("append", key, value)
    index, bf16 = key.get_device(), torch.bfloat16
    fields = _cache_fields(cache, index)
    heads, head_dim = fields[4], fields[5]
    shape, sk, sv = key.shape, key.stride(), value.stride()
    if (len(shape) != 3 or value.shape != shape or shape[1] != heads or shape[2] != head_dim or key.dtype is not bf16
            or value.dtype is not bf16 or value.get_device() != index):
        raise ValueError(f"append takes bf16 keys and values (rows, {heads}, {head_dim}) on one device, not {tuple(shape)} "
                         f"{key.dtype} on {key.device} and {tuple(value.shape)} {value.dtype} on {value.device}")
    if sk[2] != 1 or sv[2] != 1 or (sk[0] | sk[1] | sv[0] | sv[1]) & 7:
        raise ValueError(f"keys and values need a contiguous head_dim and row/head strides that are multiples of 8 "
                         f"(strides {sk}, {sv})")
    if (writes.dim() != 2 or writes.shape[1] != 4 or writes.dtype is not torch.int32 or writes.get_device() != index
            or not writes.is_contiguous()):
        raise ValueError("writes must be a contiguous (n, 4) int32 tensor on the other tensors' device")
    call = (*fields, key.data_ptr(), value.data_ptr(), sk[0], sk[1], sv[0], sv[1], shape[0], writes.data_ptr(), writes.shape[0])
    four = cache.keys.dtype is _FP4
    if not four and k_norm is None and v_norm is None and rope is None and positions is None:
        _on_gpu("append", index)
        with _on_device(index):
            _lib.check(_lib.load().karpo_cache_append(_APPEND.pack(*call), _current_stream(index)), "append")
        return
    _no_grad("append", *(n.weight for n in (k_norm, v_norm) if n is not None and n.weight is not None), *(rope or ()))
    keep: list[Tensor] = []  # (converted tables go back to the stream-ordered allocator after the launch)
    args = (*call, *_norm_fields("k_norm", k_norm, key, index, head_dim, keep),
            *_norm_fields("v_norm", v_norm, key, index, head_dim, keep),
            *_rope_fields(rope, positions, key, index, head_dim, keep))
    _on_gpu("append", index)
    lib = _lib.load()
    with _on_device(index):
        run = lib.karpo_cache4_append if four else lib.karpo_cache_append_rope
        _lib.check(run(_APPEND_ROWS.pack(*args), _current_stream(index)), "append")


def read(cache: Cache, table: Tensor, lengths: Tensor, rows: int) -> tuple[Tensor, Tensor, Tensor]:
    """(key, value, k_cu): the first ``lengths[i]`` cached tokens of each request as packed bf16 keys and values
    (``rows``, kv heads, D), request i's at k_cu[i]:k_cu[i + 1] (int32 on the device), what ``hip_attention.attend``
    takes. ``rows`` bounds the lengths' sum; rows behind the last request are not written."""
    _real("read", table)
    index = table.get_device()
    fields = _cache_fields(cache, index)
    rows_fields = _table_fields(table, lengths, index)
    rows = int(rows)
    if not 0 <= rows <= _MOST_ROWS:
        raise ValueError(f"rows must lie in 0 .. {_MOST_ROWS}, not {rows}")
    _on_gpu("read", index)
    shape = (rows, fields[4], fields[5])
    key, value = table.new_empty(shape, dtype=torch.bfloat16), table.new_empty(shape, dtype=torch.bfloat16)
    k_cu = table.new_empty(rows_fields[3] + 1)
    args = _READ.pack(*fields, *rows_fields, lengths.data_ptr(), key.data_ptr(), value.data_ptr(), rows, k_cu.data_ptr())
    with _on_device(index):
        lib = _lib.load()
        run = lib.karpo_cache4_read if cache.keys.dtype is _FP4 else lib.karpo_cache_read
        _lib.check(run(args, _current_stream(index)), "read")
    return key, value, k_cu


def attend(query: Tensor, cache: Cache, table: Tensor, q_cu: Tensor, lengths: Tensor, max_q: int, scale: float, *,
           causal: bool = True, window: int = -1, total_keys: int | None = None) -> Tensor:
    """(Lq, heads, D) bf16: ``hip_attention.attend`` over cached keys. Request i has the query rows q_cu[i]:q_cu[i + 1] of
    ``query`` ((Lq, heads, D) bf16) and ``lengths[i]`` cached tokens, its queries' own among them: the last query sits
    at the last token. Query head h reads key/value head h // (heads / kv heads). Visible tokens: all of the request's,
    or with ``causal`` those up to the query's own, narrowed by ``window`` (how many earlier tokens stay visible; -1 for
    all); a query that sees none gets zeros. A NaN reaches the queries that see its token, and in long chunks (whose keys
    are unpacked for the packed attention first) it can reach others of its tile, as there. The softmax weights enter the
    second product as two bf16 terms, in long chunks as one, as there: 2.3e-3 of the 2-norm off against 1.7e-3, the
    output's own rounding; values from 2^119 on may become infinite in long chunks. ``max_q`` bounds every request's
    query count, ``total_keys`` the lengths' sum. Long chunks unpack up to ``total_keys`` tokens into a workspace (4 *
    kv heads * D bytes each), so give it where the table is wide: the default is all that the table can hold, 51.6 GB
    for 48 requests in a table for 131,072 tokens, 16 heads of 128. Where one of the two does not hold, rows that were
    not computed are NaN: those of a request past its first ``max_q``, or, in long chunks, those of all requests. A NaN
    ``scale`` makes the rows of requests with tokens NaN. Rows behind the last request are not written."""
    _real("attend", query)
    _no_grad("attend", query)
    index = query.get_device()
    fields = _cache_fields(cache, index)
    heads, head_dim = fields[4], fields[5]
    shape, sq = query.shape, query.stride()
    if (len(shape) != 3 or query.dtype is not torch.bfloat16 or shape[2] != head_dim or shape[1] < 1
            or shape[1] % heads):
        raise ValueError(f"attend takes a (rows, heads, {head_dim}) bf16 query, its heads a multiple of {heads}, not "
                         f"{tuple(shape)} {query.dtype}")
    if sq[2] != 1 or (sq[0] | sq[1]) & 7:
        raise ValueError(f"query needs a contiguous head_dim and row/head strides that are multiples of 8 (strides {sq})")
    rows_fields = _table_fields(table, lengths, index)
    n = rows_fields[3]
    if not _ints(q_cu, index):
        _check_ints(index, q_cu=q_cu)
    if q_cu.numel() != n + 1:
        raise ValueError(f"the table has {n} requests, q_cu {q_cu.numel()} bounds")
    if not 0 <= max_q <= _MOST or not -1 <= window <= _MOST:
        raise ValueError(f"max_q must lie in 0 .. {_MOST} and window in -1 .. {_MOST}, not {max_q} and {window}")
    if total_keys is None:
        total_keys = min(n * rows_fields[2] * cache.block_size, _MOST)
    elif not 0 <= total_keys <= _MOST:
        raise ValueError(f"total_keys must lie in 0 .. {_MOST}, not {total_keys}")
    _on_gpu("attend", index)
    lib = _lib.load()
    out = query.new_empty(shape)
    if shape[0] == 0:
        return out
    if max_q == 0:  # (the C call writes nothing)
        return out.fill_(math.nan)
    call = (*fields, query.data_ptr(), out.data_ptr(), sq[0], sq[1], shape[1] * head_dim, head_dim, q_cu.data_ptr(),
            lengths.data_ptr(), *rows_fields, shape[1], int(max_q), shape[0], int(total_keys), float(scale),
            int(window), 0 if causal else -1)
    need = ctypes.c_size_t()
    size_of, run = ((lib.karpo_cache4_attend_workspace_bytes, lib.karpo_cache4_attend) if cache.keys.dtype is _FP4 else
                    (lib.karpo_cache_attend_workspace_bytes, lib.karpo_cache_attend))
    _lib.check(size_of(_ATTEND.pack(*call, 0, 0), need), "attend")
    size, at = need.value, 0
    with _on_device(index):
        if size:  # from the caching allocator (stream-ordered reuse)
            workspace = table.new_empty(size, dtype=torch.uint8)
            at = workspace.data_ptr()
        _lib.check(run(_ATTEND.pack(*call, at, size), _current_stream(index)), "attend")
    return out
