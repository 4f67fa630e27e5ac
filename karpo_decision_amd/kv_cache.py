"""A block cache on MI355X: keys and values kept between calls in 8 bits, and the packed attention that reads them.

A serving step over requests that hold cached tokens (a prompt that more rounds or branches follow, an answer that grows):

    step = reserve(table, lengths, counts, free, free_count, rows, cache.block_size)  # once per step, for all layers
    append(cache, key, value, step.writes)                                            # each layer's own cache
    out = attend(query, cache, table, step.q_cu, step.lengths, max_q, scale)

``hip_attention.attend`` reads keys that live for one call; here they live in a pool of blocks of 32, 64 or 128 tokens
(``Cache``), found through a block table. An element is stored as an e4m3 code times a power of two that its block and
head share, so a cached element is a bf16 value exactly, and ``read`` and ``attend`` work on the same numbers.

Lengths, bounds, tables and free lists are read on the device when the kernels run: nothing syncs, calls go on the
current stream of the tensors' device and capture into graphs. All of it is forward only.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from .ops import _current_stream, _on_device

BLOCK_SIZES = (32, 64, 128)
HEAD_DIMS = (64, 128, 256, 512)
_MOST = (1 << 31) - 1


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


def _cache_args(cache: Cache, device: torch.device) -> _lib.KarpoCache:
    keys, values, scales, block = cache
    shape, fp8 = keys.shape, torch.float8_e4m3fn
    if len(shape) == 3 and block in BLOCK_SIZES:  # all is well: one pass
        blocks, heads, size = shape
        head_dim = size // block
        if (head_dim in HEAD_DIMS and size == head_dim * block and values.shape == shape and blocks > 0 and heads > 0
                and scales.shape == (blocks, heads, 2) and keys.dtype is fp8 and values.dtype is fp8
                and scales.dtype is torch.float32 and keys.is_contiguous() and values.is_contiguous()
                and scales.is_contiguous() and keys.device == device and values.device == device
                and scales.device == device):
            return _lib.KarpoCache(keys.data_ptr(), values.data_ptr(), scales.data_ptr(), blocks, heads, head_dim, block)
    # the refusal's message
    if keys.dtype != fp8 or values.dtype != fp8 or scales.dtype != torch.float32:
        raise ValueError(f"a cache has float8_e4m3fn keys and values and float32 scales, not {keys.dtype}, "
                         f"{values.dtype} and {scales.dtype}")
    if keys.device != device or values.device != device or scales.device != device:
        raise ValueError(f"the cache is on {keys.device}, {values.device} and {scales.device}, the other tensors on {device}")
    raise ValueError(f"a cache has contiguous keys and values (blocks, kv heads, block_size * head_dim) and scales (blocks, "
                     f"kv heads, 2), block_size 32, 64 or 128 and head_dim 64, 128, 256 or 512, not {tuple(shape)}, "
                     f"{tuple(values.shape)}, {tuple(scales.shape)} and {block}")


def _check_ints(device: torch.device, tensors: dict[str, Tensor]) -> None:
    for name, t in tensors.items():
        if t.dtype is not torch.int32 or t.dim() != 1 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 1-D int32 tensor on {device}")


def _check_table(table: Tensor, lengths: Tensor, device: torch.device) -> tuple[int, int, int]:
    """(requests, blocks of a row, row stride) of a block table that fits ``lengths``."""
    if table.dim() != 2 or table.dtype is not torch.int32 or table.device != device:
        raise ValueError(f"table must be a (requests, blocks) int32 tensor on {device}")
    (n, width), (stride, inner) = table.shape, table.stride()
    if width < 1 or inner != 1 or (stride < width and n > 1):
        raise ValueError(f"table must have contiguous rows of at least one block, not {(n, width)} with strides "
                         f"{(stride, inner)}")
    if lengths.numel() != n:
        raise ValueError(f"the table has {n} requests, lengths {lengths.numel()}")
    return n, width, stride if stride >= width else width


def _on_gpu(what: str, t: Tensor) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{what} runs on an MI355X GPU, not on {t.device}")


def _no_grad(what: str, *tensors: Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"kv_cache.{what} has no backward: call it under torch.inference_mode() or torch.no_grad()")


def reserve(table: Tensor, lengths: Tensor, counts: Tensor, free: Tensor, free_count: Tensor, rows: int,
            block_size: int) -> Step:
    """Room for ``counts[i]`` new tokens of each request i behind the ``lengths[i]`` it holds (int32 on the device): the
    entries of new blocks in ``table`` ((requests, blocks) int32, written in place), taken in the tokens' order from the
    end of the first ``free_count[0]`` entries of ``free``, and what the step's layers need (``Step``). ``rows`` bounds
    the counts' sum and is the packed new tokens' row count. The inputs but the table are left as they are: the free
    list goes on with ``free_left``, the requests with ``Step.lengths``."""
    device = table.device
    n, width, stride = _check_table(table, lengths, device)
    _check_ints(device, {"lengths": lengths, "counts": counts, "free": free, "free_count": free_count})
    rows, capacity = int(rows), free.numel()
    if counts.numel() != n or free_count.numel() != 1:
        raise ValueError(f"counts must hold {n} requests and free_count one number, not {counts.numel()} and "
                         f"{free_count.numel()}")
    if rows < 0 or block_size not in BLOCK_SIZES:
        raise ValueError(f"rows must be non-negative and block_size 32, 64 or 128, not {rows} and {block_size}")
    _on_gpu("reserve", table)
    lib = _lib.load()
    jobs = lib.karpo_cache_writes_capacity(rows, n, block_size)
    # one allocation for the step: writes (16-byte aligned) and slots first
    buffer = torch.empty(4 * jobs + 3 * rows + 2 * n + 3, dtype=torch.int32, device=device)
    writes, slots, positions, q_cu, new, left, status = torch.split_with_sizes(
        buffer, (4 * jobs, 2 * rows, rows, n + 1, n, 1, 1))
    at = buffer.data_ptr()
    slots_at = at + 16 * jobs
    positions_at = slots_at + 8 * rows
    q_at = positions_at + 4 * rows
    new_at = q_at + 4 * n + 4
    left_at = new_at + 4 * n
    args = _lib.KarpoCacheReserveArgs(
        table.data_ptr(), stride, width, n, lengths.data_ptr(), counts.data_ptr(), free.data_ptr(),
        free_count.data_ptr(), capacity, block_size, rows, q_at, new_at, slots_at, positions_at, at, jobs, left_at,
        left_at + 4)
    index = device.index
    with _on_device(index):
        _lib.check(lib.karpo_cache_reserve(ctypes.byref(args), _current_stream(index)), "reserve")
    return Step(q_cu, new, slots.view(torch.int64), positions, writes.view(jobs, 4), left, status)


def append(cache: Cache, key: Tensor, value: Tensor, writes: Tensor) -> None:
    """New keys and values (rows, kv heads, D) bf16 into the blocks that ``writes`` lists (``Step.writes``; no block
    twice). A block's scale is the least power of two that holds what it got; where new tokens need a larger one, the
    block's earlier tokens are rounded again to it. What lies past e4m3's range at the largest scale, infinities too, is
    stored at the range's end, NaN as NaN. Rows and slots that no write names are left as they were."""
    _no_grad("append", key, value)
    device, bf16 = key.device, torch.bfloat16
    c = _cache_args(cache, device)
    shape, sk, sv = key.shape, key.stride(), value.stride()
    if (len(shape) != 3 or value.shape != shape or shape[1] != c.kv_heads or shape[2] != c.head_dim
            or key.dtype is not bf16 or value.dtype is not bf16 or value.device != device):
        raise ValueError(f"append takes bf16 keys and values (rows, {c.kv_heads}, {c.head_dim}) on {device}, not "
                         f"{tuple(shape)} {key.dtype} and {tuple(value.shape)} {value.dtype} on {value.device}")
    if sk[2] != 1 or sv[2] != 1 or (sk[0] | sk[1] | sv[0] | sv[1]) & 7:
        raise ValueError(f"keys and values need a contiguous head_dim and row/head strides that are multiples of 8 "
                         f"(strides {sk}, {sv})")
    if (writes.dim() != 2 or writes.shape[1] != 4 or writes.dtype != torch.int32 or writes.device != device
            or not writes.is_contiguous()):
        raise ValueError(f"writes must be a contiguous (n, 4) int32 tensor on {device}")
    _on_gpu("append", key)
    args = _lib.KarpoCacheAppendArgs(c, key.data_ptr(), value.data_ptr(), sk[0], sk[1], sv[0], sv[1], shape[0],
                                     writes.data_ptr(), writes.shape[0])
    with _on_device(device.index):
        _lib.check(_lib.load().karpo_cache_append(ctypes.byref(args), _current_stream(device.index)), "append")


def read(cache: Cache, table: Tensor, lengths: Tensor, rows: int) -> tuple[Tensor, Tensor, Tensor]:
    """(key, value, k_cu): the first ``lengths[i]`` cached tokens of each request as packed bf16 keys and values
    (``rows``, kv heads, D), request i's at k_cu[i]:k_cu[i + 1] (int32 on the device), what ``hip_attention.attend``
    takes. ``rows`` bounds the lengths' sum; rows behind the last request are not written."""
    device = table.device
    c = _cache_args(cache, device)
    n, width, stride = _check_table(table, lengths, device)
    _check_ints(device, {"lengths": lengths})
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"rows must be non-negative, not {rows}")
    _on_gpu("read", table)
    key, value = (torch.empty((rows, c.kv_heads, c.head_dim), dtype=torch.bfloat16, device=device) for _ in range(2))
    k_cu = torch.empty(n + 1, dtype=torch.int32, device=device)
    args = _lib.KarpoCacheReadArgs(c, table.data_ptr(), stride, width, n, lengths.data_ptr(), key.data_ptr(),
                                   value.data_ptr(), rows, k_cu.data_ptr())
    with _on_device(device.index):
        _lib.check(_lib.load().karpo_cache_read(ctypes.byref(args), _current_stream(device.index)), "read")
    return key, value, k_cu


def attend(query: Tensor, cache: Cache, table: Tensor, q_cu: Tensor, lengths: Tensor, max_q: int, scale: float, *,
           causal: bool = True, window: int = -1, total_keys: int | None = None) -> Tensor:
    """(Lq, heads, D) bf16: ``hip_attention.attend`` over cached keys. Request i has the query rows q_cu[i]:q_cu[i + 1] of
    ``query`` ((Lq, heads, D) bf16) and ``lengths[i]`` cached tokens, its queries' own among them: the last query sits
    at the last token. Query head h reads key/value head h // (heads / kv heads). Visible tokens: all of the request's,
    or with ``causal`` those up to the query's own, narrowed by ``window`` (how many earlier tokens stay visible; -1 for
    all); a query that sees none gets zeros. ``max_q`` bounds every request's query count, ``total_keys`` the lengths'
    sum (default: all that the table can hold; it sizes the workspace of long query runs). Rows behind the last request
    are not written."""
    _no_grad("attend", query)
    device = query.device
    c = _cache_args(cache, device)
    shape = query.shape
    if (len(shape) != 3 or query.dtype is not torch.bfloat16 or shape[2] != c.head_dim or shape[1] < 1
            or shape[1] % c.kv_heads):
        raise ValueError(f"attend takes a (rows, heads, {c.head_dim}) bf16 query, its heads a multiple of {c.kv_heads}, "
                         f"not {tuple(shape)} {query.dtype}")
    sq = query.stride()
    if sq[2] != 1 or (sq[0] | sq[1]) & 7:
        raise ValueError(f"query needs a contiguous head_dim and row/head strides that are multiples of 8 (strides {sq})")
    n, width, stride = _check_table(table, lengths, device)
    _check_ints(device, {"lengths": lengths, "q_cu": q_cu})
    if q_cu.numel() != n + 1:
        raise ValueError(f"the table has {n} requests, q_cu {q_cu.numel()} bounds")
    if max_q < 0 or window < -1:
        raise ValueError(f"max_q must be non-negative and window at least -1, not {max_q} and {window}")
    if total_keys is None:
        total_keys = min(n * width * c.block_size, _MOST)
    elif not 0 <= total_keys <= _MOST:
        raise ValueError(f"total_keys must lie in 0 .. {_MOST}, not {total_keys}")
    _on_gpu("attend", query)
    lib = _lib.load()
    out = torch.empty(shape, dtype=torch.bfloat16, device=device)
    if shape[0] == 0:
        return out
    so = out.stride()
    args = _lib.KarpoCacheAttendArgs(
        c, query.data_ptr(), out.data_ptr(), sq[0], sq[1], so[0], so[1], q_cu.data_ptr(), lengths.data_ptr(),
        table.data_ptr(), stride, width, n, shape[1], int(max_q), shape[0], int(total_keys), float(scale), int(window),
        0 if causal else -1)
    pointer, need = ctypes.byref(args), ctypes.c_size_t()
    _lib.check(lib.karpo_cache_attend_workspace_bytes(pointer, ctypes.byref(need)), "attend")
    index = device.index
    with _on_device(index):
        # from the caching allocator (stream-ordered reuse)
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need.value
        _lib.check(lib.karpo_cache_attend(pointer, _current_stream(index)), "attend")
    return out
