"""A block cache on MI355X: keys and values kept between calls in 8 bits, and the packed attention that reads them.

A serving step over requests that hold cached tokens (a prompt that more rounds or branches follow, an answer that grows):

    step = reserve(table, lengths, counts, free, free_count, rows, cache.block_size)  # once per step, for all layers
    append(cache, key, value, step.writes)                                            # each layer's own cache
    out = attend(query, cache, table, step.q_cu, step.lengths, max_q, scale, total_keys=total)  # total: of step.lengths

``hip_attention.attend`` reads keys that live for one call; here they live in a pool of blocks of 32, 64 or 128 tokens
(``Cache``), found through a block table. An element is stored as an e4m3 code times a power of two that its block and
head share, so a cached element is a bf16 value exactly, and ``read`` and ``attend`` work on the same numbers.
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
from .ops import _current_stream, _on_device

BLOCK_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128, 256, 512)
_MOST = (1 << 31) - 1
_MOST_ROWS = _MOST - (1 << 16)

# The argument structures of karpo_cache.h, field by field (_lib has them by name): packing them costs a third of what
# building them by name does, and a small call's time is its host path.
_CACHE = "PPPqiii4x"
_RESERVE = struct.Struct("@PqiiPPPPiiqPPPPPqPP")
_APPEND = struct.Struct("@" + _CACHE + "PPqqqqqPq")
_READ = struct.Struct("@" + _CACHE + "PqiiPPPqP")
_ATTEND = struct.Struct("@" + _CACHE + "PPqqqqPPPqiiiiqqfii4xPN")


class Cache(NamedTuple):
    """One layer's keys and values: ``keys`` and ``values`` (blocks, kv heads, block_size * D) float8_e4m3fn, laid out as
    ``karpo_cache.h`` says, and ``scales`` (blocks, kv heads, 2) fp32, the powers of two of a block's keys and values."""

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
        return self.keys.shape[2] // self.block_size


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
           device: torch.device | str = "cuda") -> Cache:
    """An empty cache of ``blocks`` blocks."""
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be 32, 64 or 128, not {block_size}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128, 256 or 512, not {head_dim}")
    if blocks < 1 or kv_heads < 1:
        raise ValueError(f"a cache has at least one block and one head, not {blocks} and {kv_heads}")
    keys, values = (torch.zeros((blocks, kv_heads, block_size * head_dim), dtype=torch.uint8, device=device)
                    .view(torch.float8_e4m3fn) for _ in range(2))
    return Cache(keys, values, torch.zeros((blocks, kv_heads, 2), dtype=torch.float32, device=device), block_size)


def _cache_fields(cache: Cache, index: int) -> tuple[int, ...]:
    """The cache's fields of an argument structure; ``index``: the other tensors' device."""
    keys, values, scales, block = cache
    shape, fp8 = keys.shape, torch.float8_e4m3fn
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


def append(cache: Cache, key: Tensor, value: Tensor, writes: Tensor) -> None:
    """New keys and values (rows, kv heads, D) bf16 into the blocks that ``writes`` lists (``Step.writes``; no block
    twice). A block's scale is the least power of two that holds what it got; where new tokens need a larger one, the
    block's earlier tokens are rounded again to it. What lies past e4m3's range at the largest scale, infinities too, is
    stored at the range's end, NaN as NaN. Rows and slots that no write names are left as they were."""
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
    _on_gpu("append", index)
    args = _APPEND.pack(*fields, key.data_ptr(), value.data_ptr(), sk[0], sk[1], sv[0], sv[1], shape[0],
                        writes.data_ptr(), writes.shape[0])
    with _on_device(index):
        _lib.check(_lib.load().karpo_cache_append(args, _current_stream(index)), "append")


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
        _lib.check(_lib.load().karpo_cache_read(args, _current_stream(index)), "read")
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
    output's own rounding. ``max_q`` bounds every request's query count, ``total_keys`` the lengths' sum. Long chunks
    unpack up to ``total_keys`` tokens into a workspace (4 * kv heads * D bytes each), so give it where the table is wide:
    the default is all that the table can hold, 51.6 GB for 48 requests in a table for 131,072 tokens, 16 heads of 128.
    Where one of the two does not hold, rows that were not computed are NaN: those of a request past its first ``max_q``,
    or, in long chunks, those of all requests. A NaN ``scale`` makes the rows of requests with tokens NaN. Rows behind the
    last request are not written."""
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
    _lib.check(lib.karpo_cache_attend_workspace_bytes(_ATTEND.pack(*call, 0, 0), need), "attend")
    size, at = need.value, 0
    with _on_device(index):
        if size:  # from the caching allocator (stream-ordered reuse)
            workspace = table.new_empty(size, dtype=torch.uint8)
            at = workspace.data_ptr()
        _lib.check(lib.karpo_cache_attend(_ATTEND.pack(*call, at, size), _current_stream(index)), "attend")
    return out
