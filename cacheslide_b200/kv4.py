"""The paged KV cache in 4 bits.

A pool of 4-bit records holds three and a half times the tokens of a 16-bit
one, and a decode step, which is bound by reading them, takes that much less
time:

* ``PagedKV4`` / ``empty_pool`` -- the pool;
* ``append``    -- keys (normed and rotated, as ``rotary.qk_norm_rope`` leaves
  them) and values into their slots, a scale and a lowest value a group;
* ``gather``    -- the values that records stand for, in 16 bits again;
* ``attention`` -- decodes, drafted tokens and whole questions over the pool,
  through block tables and lengths on the device.

``tables.step_maps`` makes the slots and tables.  The reference keeps 16-bit
records only (``NativePagedKV``, paged.py:57-128); slots, blocks and what a
request sees mean the same here.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from . import _native as N
from .prefix import _overlap

UNIT = 16  # tokens of a unit: their codes and scales of one head, contiguous
_TYPES = (torch.float16, torch.bfloat16)


def unit_bytes(head_dim: int, group: int) -> int:
    """Bytes of 16 tokens of one head."""
    return UNIT * head_dim + 8 * UNIT * (head_dim // group)


class PagedKV4:
    """A pool of 4-bit records over ``storage``, uint8 [block, kv_head,
    block_size / 16, ``unit_bytes(head_dim, group)``], contiguous.

    A group of ``group`` elements of a head is 4-bit codes with a scale and a
    lowest value in ``dtype`` (float16 or bfloat16), which is also the type of
    the rows that go in and come out.  ``head_dim`` 64 or 128, ``group`` 32, 64
    or 128 and at most ``head_dim``; the block size is a multiple of 16.  The
    layout within a unit is documented at ``cs_kv4_pool``."""

    def __init__(self, storage: Tensor, head_dim: int, dtype: torch.dtype, group: int = 64):
        if dtype not in _TYPES:
            raise ValueError("a 4-bit pool's dtype must be float16 or bfloat16")
        if head_dim not in (64, 128) or group not in (32, 64, 128) or group > head_dim:
            raise ValueError("head dim must be 64 or 128, group 32, 64 or 128 and at most that")
        if not isinstance(storage, Tensor) or storage.dtype is not torch.uint8 or \
                storage.dim() != 4 or storage.shape[3] != unit_bytes(head_dim, group) or \
                storage.shape[1] < 1 or storage.shape[2] < 1 or not storage.is_contiguous():
            raise ValueError("storage must be contiguous uint8 [block, kv_head, block_size / 16, "
                             f"{unit_bytes(head_dim, group)}]")
        if storage.data_ptr() % 16:
            raise ValueError("storage must be 16-byte aligned")
        self.storage, self.head_dim, self.dtype, self.group = storage, head_dim, dtype, group
        self.num_blocks, self.kv_heads = storage.shape[0], storage.shape[1]
        self.block_size = UNIT * storage.shape[2]
        self.device = storage.device
        self.view = N.KV4Pool(storage.data_ptr(), self.num_blocks, self.kv_heads, self.block_size,
                              head_dim, group, N.DTYPES[dtype])


def empty_pool(num_blocks: int, kv_heads: int, block_size: int, head_dim: int,
               dtype: torch.dtype, device: torch.device | str = "cuda",
               group: int = 64) -> PagedKV4:
    """A pool of zeros (records that stand for zero keys and values)."""
    if type(block_size) is not int or block_size < UNIT or block_size % UNIT:
        raise ValueError(f"block_size must be a multiple of {UNIT}")
    if head_dim not in (64, 128) or group not in (32, 64, 128):
        raise ValueError("head dim must be 64 or 128, group 32, 64 or 128 and at most that")
    storage = torch.zeros(num_blocks, kv_heads, block_size // UNIT, unit_bytes(head_dim, group),
                          dtype=torch.uint8, device=device)
    return PagedKV4(storage, head_dim, dtype, group)


def _slots(slots: Tensor, pool: PagedKV4) -> int:
    if (slots.dim() != 1 or slots.dtype is not torch.int64
            or slots.get_device() != pool.storage.get_device()
            or slots.shape[0] > 1 and slots.stride(0) != 1):
        raise ValueError("slots must be a contiguous int64 vector on the pool's device")
    return slots.shape[0]


def _pool(pool: PagedKV4) -> int:
    if not isinstance(pool, PagedKV4):
        raise ValueError("pool must be a PagedKV4")
    return pool.storage.get_device()


def append(pool: PagedKV4, slots: Tensor, key: Tensor, value: Tensor, *,
           status: N.Status | None = None) -> None:
    """The records of ``slots`` (int64 [token]) become ``key`` and ``value``
    [token, kv_head, dim] in 4 bits.

    Each group's codes are the nearest of its sixteen values by their float32
    difference to the lowest, ties to the even code; a group that holds an
    infinity or a NaN stands for NaN throughout.  Slot -1 is padding and is not
    written; any other slot outside the pool is skipped and sets
    ``ST_SLOT_RANGE`` in ``status``.  Distinct tokens need distinct slots.  A
    serving operator without a derivative."""
    device = _pool(pool)
    n = _slots(slots, pool)
    shape = (n, pool.kv_heads, pool.head_dim)
    for name, x in (("key", key), ("value", value)):
        if x.shape != shape or x.dtype is not pool.dtype or x.get_device() != device:
            raise ValueError(f"{name} must be {pool.dtype} [token, {pool.kv_heads}, "
                             f"{pool.head_dim}] on the pool's device")
    ks, vs = key.stride(), value.stride()
    if ks[2] != 1:
        key = key.contiguous()
        ks = key.stride()
    if vs[2] != 1:
        value = value.contiguous()
        vs = value.stride()
    status_ptr = N.status_ptr(status, device)
    if device < 0:
        N.require_cuda(pool.storage)
    N.launch("cs_kv4_append", pool.device, pool.view, slots.data_ptr(), n, key.data_ptr(), ks[0],
             ks[1], value.data_ptr(), vs[0], vs[1], status_ptr)


def gather(pool: PagedKV4, slots: Tensor, *,
           status: N.Status | None = None) -> tuple[Tensor, Tensor]:
    """The keys and values [token, kv_head, dim] that the records of ``slots``
    stand for, rounded to the pool's dtype.  Slot -1 gives zeros, and so does
    any other slot outside the pool, which sets ``ST_SLOT_RANGE`` in
    ``status``."""
    device = _pool(pool)
    n = _slots(slots, pool)
    status_ptr = N.status_ptr(status, device)
    if device < 0:
        N.require_cuda(pool.storage)
    key, value = torch.empty(2, n, pool.kv_heads, pool.head_dim, dtype=pool.dtype,
                             device=pool.device).unbind(0)
    st = key.stride()
    N.launch("cs_kv4_gather", pool.device, pool.view, slots.data_ptr(), n, key.data_ptr(), st[0],
             st[1], value.data_ptr(), st[0], st[1], status_ptr)
    return key, value


def _ints(name: str, x: Tensor, count: int, device: int) -> int:
    if (x.shape != (count,) or x.dtype is not torch.int32 or x.get_device() != device
            or count > 1 and x.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 vector of {count} on the pool's "
                         "device")
    return x.data_ptr()


def attention(query: Tensor, pool: PagedKV4, tables: Tensor, lengths: Tensor,
              starts: Tensor | None = None, *, scale: float | None = None,
              out: Tensor | None = None, return_lse: bool = False,
              status: N.Status | None = None) -> Tensor | tuple[Tensor, Tensor]:
    """Causal softmax attention of a batch over a 4-bit pool.

    Request ``b``'s keys are its positions ``0 .. lengths[b] - 1`` (int32
    [request]) through row ``b`` of ``tables`` (int32 [request, block]); its
    queries are rows ``starts[b] .. starts[b + 1] - 1`` of ``query`` [token,
    q_head, dim] (``StepMaps.starts``; without ``starts``, row ``b`` alone),
    the newest of those positions: query ``i`` of ``n`` sees keys up to
    ``lengths[b] - n + i``.  Their own keys are appended before the call.
    Lengths, starts and tables are read on the device, so a captured call
    follows them.  ``scale`` defaults to ``dim ** -0.5``.

    Returns [token, q_head, dim] in ``out`` (which may overlap ``query``: it is
    then copied first) or a new tensor and, with ``return_lse``, the float32
    log of each row's softmax denominator.  A row that sees no key gives zeros
    and -inf.  Rows that belong to no request are left as they were in ``out``,
    and are such empty rows in a new tensor (and in the lse with it).

    A block outside the pool reads as zero keys and values and sets
    ``ST_SLOT_RANGE`` in ``status``; a length past the tables' width is cut
    there, and a request is left out whose first row lies below an earlier one's
    or whose rows fall or leave the query's; both set ``ST_CAPACITY``.  Rows of
    a request that is left out belong to none.  A serving operator without a
    derivative."""
    device = _pool(pool)
    if query.dim() != 3 or query.dtype is not pool.dtype or query.get_device() != device or \
            query.shape[2] != pool.head_dim or query.shape[1] < 1 or \
            query.shape[1] % pool.kv_heads:
        raise ValueError(f"query must be {pool.dtype} [token, q_head, {pool.head_dim}] on the "
                         "pool's device, its heads a multiple of the pool's")
    if tables.dim() != 2 or tables.dtype is not torch.int32 or tables.get_device() != device or \
            tables.shape[1] > 1 and tables.stride(1) != 1:
        raise ValueError("tables must be int32 [request, block] with contiguous rows on the "
                         "pool's device")
    requests, width = tables.shape
    if requests > 1 and tables.stride(0) < width:
        raise ValueError("the rows of tables must not overlap")
    tokens, q_heads, _ = shape = query.shape
    p_lengths = _ints("lengths", lengths, requests, device)
    p_starts = None
    if starts is not None:
        p_starts = _ints("starts", starts, requests + 1, device)
    elif tokens != requests:
        raise ValueError("without starts there is one query row a request")
    if scale is None:
        scale = pool.head_dim ** -0.5
    elif not math.isfinite(ctypes.c_float(scale).value):
        raise ValueError("scale must be finite")
    status_ptr = N.status_ptr(status, device)
    if query.stride(2) != 1:
        query = query.contiguous()
    fresh = out is None
    if fresh:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not pool.dtype or out.get_device() != device or \
            out.stride(2) != 1:
        raise ValueError("out must match query, with a contiguous last dimension")
    elif tokens and _overlap(out, query):  # blocks read queries after others have written
        query = query.clone(memory_format=torch.contiguous_format)
    if device < 0:
        N.require_cuda(pool.storage)
    lse = None
    if return_lse:
        lse = torch.empty(shape[:2], dtype=torch.float32, device=pool.device)
        if not fresh and starts is not None:
            lse.fill_(-math.inf)
    qs, os = query.stride(), out.stride()
    p = N.KV4AttnParams(
        query.data_ptr(), qs[0], qs[1], tokens, q_heads, requests, pool.view, tables.data_ptr(),
        tables.stride(0), width, fresh, p_lengths, p_starts, scale, out.data_ptr(), os[0], os[1],
        N.ptr(lse), status_ptr)
    size = N.load().cs_kv4_attn_workspace(p)
    workspace = torch.empty(size, dtype=torch.uint8, device=pool.device)
    N.launch("cs_kv4_attn", pool.device, p, workspace.data_ptr())
    return (out, lse) if return_lse else out
