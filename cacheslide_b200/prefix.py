"""Attention of a batch whose requests share a long prefix in the paged pool.

Retrieval batches, chat tenants and several samples of one document keep the
common part of their prompts in the pool once (shared blocks in their block
tables).  Decoding, verifying drafted tokens or prefilling the questions then
reads that part once for the whole batch, and each request's own keys once
for that request: ``SharedPrefixAttention`` is the rotary layers' counterpart
of the per-request attention of runtime.py:490-508 (causal softmax attention
over ``NativePagedKV``'s records, paged.py:205-240).

The batch's lengths become a plan once (``cs_prefix_plan``), reused by every
layer of the step; each call is a launch or two on the current stream,
without host synchronisation.
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Sequence

import torch
from torch import Tensor

from . import _native as N
from .paged import NativePagedKV
from .rotary import pool_view

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _lens(name: str, values: Sequence[int]) -> tuple[ctypes.Array, int]:
    values = list(values)
    if any(type(v) is not int or not 0 <= v < 1 << 31 for v in values):
        raise ValueError(f"{name} must be nonnegative integers below 2^31")
    return (ctypes.c_int64 * max(1, len(values)))(*values), sum(values)


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether the spans of memory from first to last element meet."""
    def span(t: Tensor) -> tuple[int, int]:
        first = t.data_ptr()
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return first, first + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


class SharedPrefixAttention:
    """The attention of one batch layout; call it once per layer.

    ``query_lens[b]`` query tokens of request ``b`` are the newest of its
    ``suffix_lens[b]`` own keys: query ``i`` of ``n`` sees its group's whole
    prefix and own keys up to ``suffix_len - n + i`` (its own position).  A
    request may have fewer own keys than queries (the first queries then see
    only the prefix).  The requests form consecutive groups of
    ``group_sizes``, group ``g`` sharing ``prefix_lens[g]`` keys; by default
    one group holds them all.  The lengths stay on the plan under these names:
    a call compares only their sums with its tensors, so a caller that keeps
    plans compares the lengths."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, dtype: torch.dtype,
                 device: torch.device | str, *, query_lens: Sequence[int],
                 suffix_lens: Sequence[int], prefix_lens: Sequence[int],
                 group_sizes: Sequence[int] | None = None):
        if dtype not in _TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        if min(q_heads, kv_heads, head_dim) < 1 or q_heads % kv_heads:
            raise ValueError("query heads must be a multiple of KV heads")
        if group_sizes is None:
            group_sizes = [len(query_lens)]
        if len(query_lens) != len(suffix_lens) or len(prefix_lens) != len(group_sizes):
            raise ValueError("one query and suffix length a request, one prefix length a group")
        queries, self.tokens = _lens("query_lens", query_lens)
        suffixes, self.suffix_keys = _lens("suffix_lens", suffix_lens)
        prefixes, self.prefix_keys = _lens("prefix_lens", prefix_lens)
        sizes, members = _lens("group_sizes", group_sizes)
        if members != len(query_lens):
            raise ValueError("group_sizes must add up to the requests")
        self.query_lens, self.suffix_lens = tuple(query_lens), tuple(suffix_lens)
        self.prefix_lens, self.group_sizes = tuple(prefix_lens), tuple(group_sizes)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.shape = torch.Size((self.tokens, q_heads, head_dim))
        self.dtype, self.device = dtype, torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        shape = N.PrefixShape(
            q_heads, kv_heads, head_dim, N.DTYPES[dtype], len(prefix_lens), len(query_lens),
            ctypes.addressof(prefixes), ctypes.addressof(sizes), ctypes.addressof(queries),
            ctypes.addressof(suffixes))
        self.info = N.PrefixPlanInfo()
        lib = N.load()
        capacity = 16 * self.tokens + 4096
        while True:
            words = torch.empty(capacity, dtype=torch.int32)
            rc = lib.cs_prefix_plan(ctypes.byref(shape), ctypes.byref(self.info),
                                    words.data_ptr(), capacity)
            if rc != N.CS_ERR_TOO_LARGE or self.info.words <= capacity:
                break
            capacity = self.info.words
        N.check(rc, "cs_prefix_plan")
        self.words = words[:self.info.words].to(self.device)
        self._stream = N.stream_of(self.device) if self.device.type == "cuda" else None

    def __call__(self, query: Tensor, kv: Tensor | NativePagedKV | N.PagedKV,
                 prefix_slots: Tensor, suffix_slots: Tensor, *, scale: float | None = None,
                 out: Tensor | None = None, return_lse: bool = False,
                 status: N.Status | None = None) -> Tensor | tuple[Tensor, Tensor]:
        """``query`` [token, q_head, dim] of all requests in order;
        ``prefix_slots`` / ``suffix_slots`` (int64) the pool slots of the
        groups' prefixes and the requests' own keys, concatenated.  ``scale``
        defaults to ``dim ** -0.5``.  ``out`` may overlap ``query`` (which is then
        copied first).  Returns [token, q_head, dim] (and, with
        ``return_lse``, the float32 log of each row's softmax denominator,
        -inf for a row that sees no key, whose output is zero).

        A slot outside the pool reads as a zero key and value and sets
        ``ST_SLOT_RANGE`` in ``status``.  A serving operator: it has no
        derivative of either mode, and its outputs are constants to autograd."""
        shape, device = self.shape, self.device
        index = device.index
        if query.shape != shape or query.dtype is not self.dtype or query.get_device() != index:
            raise ValueError(f"query must be {self.dtype} {tuple(shape)} on {device}")
        for name, slots, count in (("prefix_slots", prefix_slots, self.prefix_keys),
                                   ("suffix_slots", suffix_slots, self.suffix_keys)):
            if slots.shape != (count,) or slots.dtype is not torch.int64 or \
                    slots.get_device() != index or count > 1 and slots.stride(0) != 1:
                raise ValueError(f"{name} must be a contiguous int64 vector of {count} slots")
        qs = query.stride()
        if qs[2] != 1:
            query = query.contiguous()
            qs = query.stride()
        view = pool_view(kv)
        N.require_pool_on(view, index)
        status_ptr = N.status_ptr(status, index)
        if view.dtype != N.DTYPES[self.dtype] or view.kv_heads != self.kv_heads \
                or view.head_dim != self.head_dim:
            raise ValueError("the pool's dtype, KV heads and head dim must be the plan's")
        if scale is None:
            scale = self.head_dim ** -0.5
        elif not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if out is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        elif out.shape != shape or out.dtype is not self.dtype or out.get_device() != index \
                or out.stride(2) != 1:
            raise ValueError("out must match query, with a contiguous last dimension")
        elif _overlap(out, query):  # blocks read queries after others have written
            query = query.clone(memory_format=torch.contiguous_format)
            qs = query.stride()
        os = out.stride()
        lse = torch.empty(shape[:2], dtype=torch.float32, device=device) if return_lse else None
        p = N.PrefixParams(
            query.data_ptr(), qs[0], qs[1], view, prefix_slots.data_ptr(),
            suffix_slots.data_ptr(), self.q_heads, scale, out.data_ptr(), os[0], os[1],
            N.ptr(lse), status_ptr)
        if N.stream_of(device) != self._stream:  # the plan may be dropped before the call has run
            self.words.record_stream(torch.cuda.current_stream(device))
        workspace = None
        if self.info.workspace:
            workspace = torch.empty(self.info.workspace, dtype=torch.uint8, device=device)
        N.launch("cs_prefix_attn", device, p, self.info, self.words.data_ptr(),
                 N.ptr(workspace))
        return (out, lse) if return_lse else out
