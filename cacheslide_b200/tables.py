"""Block tables and slot maps of a serving step, built on the GPU.

A step's slots follow from the requests' lengths and block tables.  Where those
live on the device -- a captured decode loop, a batch whose lengths a kernel
advances -- ``step_maps`` makes the step's positions and slots there in one
launch, takes the blocks that requests grow into from a stack of free ones, and
lists the slots of every request's keys for the attention that reads by slots.

The reference builds these on the host, token by token (the block tables of
``NativePagedKV``, paged.py:57-128); slots mean the same here.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import _native as N


class StepMaps(NamedTuple):
    """Where a step's tokens go (``step_maps``)."""

    starts: Tensor      #: int32 [requests + 1]: first row of each request's tokens; the total
    positions: Tensor   #: int64 [tokens]; 0 in rows past the last request's
    slots: Tensor       #: int64 [tokens]; -1 there
    key_starts: Tensor | None  #: int64 [requests + 1], with ``keys``
    key_slots: Tensor | None   #: int64 [keys], with ``keys``; -1 past the last
    free_left: Tensor | None   #: int32 [1], with ``free``


def _vector(name: str, x: Tensor, count: int | None, device: int) -> int:
    if (x.dim() != 1 or x.dtype is not torch.int32 or x.get_device() != device
            or count is not None and x.shape[0] != count
            or x.shape[0] > 1 and x.stride(0) != 1):
        many = "" if count is None else f" of {count}"
        raise ValueError(f"{name} must be a contiguous int32 vector{many} on the tables' device")
    return x.data_ptr()


def _whole(name: str, value: int, low: int, high: int = 1 << 31) -> int:
    if type(value) is not int or not low <= value < high:
        raise ValueError(f"{name} must be an integer of at least {low} and below {high}")
    return value


def step_maps(lengths: Tensor, new: Tensor, tables: Tensor, block_size: int, num_blocks: int, *,
              tokens: int, keys: int = 0, offset: int = 0, free: Tensor | None = None,
              free_count: Tensor | None = None, status: N.Status | None = None) -> StepMaps:
    """Slots and positions of a step from lengths on the device.

    Request ``b`` holds ``lengths[b]`` tokens after the step, the newest
    ``new[b]`` of which the step brings (int32 vectors; 0 new tokens: idle).
    Position ``p`` lies in slot ``tables[b, p // block_size] * block_size + p %
    block_size`` of a pool of ``num_blocks`` blocks.  ``tables`` is int32
    [request, block].  ``tokens`` is the number of rows that the step's arrays
    hold: the sum of ``new``, or more (the rest is padding: slot -1, position
    0).  With ``keys`` the slots of every request's positions are listed too,
    request after request; ``offset`` is added to the positions alone.

    With ``free`` (int32 block ids) and ``free_count`` (int32 [1], how many of
    them are valid) the blocks that a request needs beyond those of its older
    positions come from the end of the valid ids, requests in order, and are
    written into ``tables``; ``free_left`` is what remains.  Calling again with
    the same inputs does the same again.  Without them the tables are complete.

    All or nothing: a negative length, ``new > lengths``, too narrow a table,
    more rows than ``tokens`` (or keys than ``keys``), too few free blocks or a
    ``free_count`` that is negative or past ``free``
    sets ``ST_CAPACITY`` in ``status``, and then every slot is -1, every
    position and start 0 and the tables are left alone.  A block outside the
    pool gives slot -1 and sets ``ST_SLOT_RANGE``.  Nothing waits on the host."""
    if not isinstance(tables, Tensor) or tables.dim() != 2 or tables.dtype is not torch.int32 or \
            tables.shape[1] > 1 and tables.stride(1) != 1:
        raise ValueError("tables must be int32 [request, block] with contiguous rows")
    device = tables.get_device()
    requests, width = tables.shape
    p_lengths = _vector("lengths", lengths, requests, device)
    p_new = _vector("new", new, requests, device)
    _whole("block_size", block_size, 1)
    _whole("num_blocks", num_blocks, 0, 1 << 62)
    _whole("tokens", tokens, 0, (1 << 31) - 1)
    _whole("keys", keys, 0, 1 << 62)
    _whole("offset", offset, 0)
    if (free is None) != (free_count is None):
        raise ValueError("free and free_count come together")
    if requests > 1 and tables.stride(0) < width:
        raise ValueError("the rows of tables must not overlap")
    p_free = p_count = None
    if free is not None:
        p_free = _vector("free", free, None, device)
        p_count = _vector("free_count", free_count, 1, device)
        if free.shape[0] == 0:  # an empty tensor has no address, and is not read
            p_free = p_count
    status_ptr = N.status_ptr(status, device)
    if device < 0:
        N.require_cuda(tables)
    on = tables.device
    positions, slots = torch.empty(2, tokens, dtype=torch.int64, device=on).unbind(0)
    starts = torch.empty(requests + 1, dtype=torch.int32, device=on)
    left = key_starts = key_slots = None
    if free is not None:
        left = torch.empty(1, dtype=torch.int32, device=on)
    if keys:
        key_slots = torch.empty(keys, dtype=torch.int64, device=on)
        key_starts = torch.empty(requests + 1, dtype=torch.int64, device=on)
    p = N.StepMapsParams(
        p_lengths, p_new, requests, block_size, num_blocks, tables.data_ptr(), tables.stride(0),
        width, offset, p_free, p_count, N.ptr(left), 0 if free is None else free.shape[0], tokens,
        keys, starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), N.ptr(key_starts),
        N.ptr(key_slots), status_ptr)
    N.launch("cs_step_maps", on, p)
    return StepMaps(starts, positions, slots, key_starts, key_slots, left)
