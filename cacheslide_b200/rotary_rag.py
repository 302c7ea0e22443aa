"""A retrieval batch of a rotary layer, its documents resident once.

The rotary counterpart of ``rag.RagStep`` for one layer: a shared prefix (the
retrieved chunks in one order, or a system prompt) lies in the paged pool
once; every request owns blocks for its question and answer.  The layer's
three calls run as a model runner would make them:

* ``write_prefix``  the document's keys, normed and rotated at positions
  0 .. n-1, and values into the prefix slots (``rotary.append_rotated``);
* ``step``          new tokens of every request -- the whole questions, one
  decoded token each, or drafted ones -- with their keys appended behind the
  request's own and their queries attending over prefix and own keys
  (``append_rotated`` and ``prefix.SharedPrefixAttention``).

A step's plan depends on the lengths alone: build it once (``plan``) and pass
it to every layer; a plan of other lengths is refused.  The prefill of the document itself is ordinary causal
attention over ``rotary.qk_norm_rope``'s output.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from . import _native as N
from .prefix import SharedPrefixAttention
from .rotary import append_rotated, rotary_tables
from .tables import step_maps


class RotaryRagBatch:
    """Block ownership and positions of one layer's batch over a pool
    ``[blocks, kv_heads, block_size, 2 * dim]`` of the caller."""

    def __init__(self, pool: Tensor, q_heads: int, prefix_length: int, requests: int,
                 max_own: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                 eps: float = 1e-6, interleaved: bool = False,
                 block_ids: Sequence[int] | None = None):
        if pool.ndim != 4 or pool.device.type != "cuda" or pool.dtype not in N.DTYPES:
            raise ValueError("pool must be a CUDA tensor [blocks, kv_heads, block_size, 2 * dim]")
        blocks, _, block, width = pool.shape
        for name, value, low in (("prefix_length", prefix_length, 0), ("requests", requests, 1),
                                 ("max_own", max_own, 1)):
            if type(value) is not int or value < low:
                raise ValueError(f"{name} must be an integer of at least {low}")
        per_prefix, per_request = -(-prefix_length // block), -(-max_own // block)
        need = per_prefix + requests * per_request
        ids = list(range(blocks)) if block_ids is None else list(block_ids)
        if len(ids) < need or len(set(ids)) != len(ids) or \
                any(type(b) is not int or not 0 <= b < blocks for b in ids):
            raise ValueError(f"the batch needs {need} distinct blocks of the pool")
        table = torch.tensor(ids[:need], dtype=torch.int64, device=pool.device)
        offset = torch.arange(block, dtype=torch.int64, device=pool.device)
        slots = (table[:, None] * block + offset).reshape(-1)
        self.pool, self.q_heads, self.requests, self.max_own = pool, q_heads, requests, max_own
        self.prefix_slots = slots[:prefix_length].contiguous()
        self.own_slots = slots[per_prefix * block:].view(requests, -1)
        self.own_table = table[per_prefix:].view(requests, -1).int()
        self.lengths = [0] * requests
        self.cos, self.sin = rotary_tables(prefix_length + max_own,
                                           width // 2 if rotary_dim is None else rotary_dim,
                                           base=base, device=pool.device)
        self.q_weight, self.k_weight, self.eps = q_weight, k_weight, eps
        self.interleaved = interleaved
        self.status = N.Status(pool.device)

    def _append(self, key: Tensor, value: Tensor, query: Tensor | None = None,
                plan: SharedPrefixAttention | None = None) -> tuple[Tensor | None, Tensor | None]:
        """The prefix's keys and values into its slots or, with a plan, a step's
        new ones into their requests': the slots and positions of the new tokens
        and the slots of every own key come from the plan's lengths on the
        device.  Returns the turned queries and the own keys' slots."""
        own = q_weight = None
        if plan is None:
            slots = self.prefix_slots
            positions = torch.arange(key.shape[0], device=self.pool.device)
        else:
            blocks, _, block, _ = self.pool.shape
            new_lens, own_lens = plan.device_lens
            maps = step_maps(own_lens, new_lens, self.own_table, block, blocks,
                             tokens=plan.tokens, keys=plan.suffix_keys,
                             offset=self.prefix_slots.numel(), status=self.status)
            slots, positions, q_weight = maps.slots, maps.positions, self.q_weight
            own = slots[:0] if maps.key_slots is None else maps.key_slots
        turned = append_rotated(self.pool, slots, key, value, positions, self.cos, self.sin,
                                query=query, q_weight=q_weight, k_weight=self.k_weight,
                                eps=self.eps, interleaved=self.interleaved, status=self.status)
        return turned, own

    def write_prefix(self, key: Tensor, value: Tensor) -> None:
        """The prefix's keys (as projected, neither normed nor rotated) and
        values, [prefix, kv_head, dim]."""
        self._append(key, value)

    def _own(self, query_lens: Sequence[int]) -> list[int]:
        """Each request's own keys after a step."""
        own = [have + new for have, new in zip(self.lengths, query_lens, strict=True)]
        if max(own) > self.max_own:
            raise ValueError("a request's own keys pass its blocks")
        return own

    def plan(self, query_lens: Sequence[int]) -> SharedPrefixAttention:
        """The attention of a step in which request b brings query_lens[b] tokens."""
        own = self._own(query_lens)
        return SharedPrefixAttention(
            self.q_heads, self.pool.shape[1], self.pool.shape[3] // 2, self.pool.dtype,
            self.pool.device, query_lens=query_lens, suffix_lens=own,
            prefix_lens=[self.prefix_slots.numel()])

    def step(self, query: Tensor, key: Tensor, value: Tensor, query_lens: Sequence[int],
             plan: SharedPrefixAttention | None = None) -> Tensor:
        """One layer of a step: ``query`` [token, q_head, dim] and ``key`` /
        ``value`` [token, kv_head, dim] of the new tokens, requests in order.
        Returns the attention's output [token, q_head, dim].  Everything that
        the attention would refuse is refused before the keys are written."""
        if plan is None:
            plan = self.plan(query_lens)
        else:
            pool = self.pool
            mine = (tuple(query_lens), tuple(self._own(query_lens)),
                    (self.prefix_slots.numel(),), (self.requests,), self.q_heads, pool.shape[1],
                    pool.shape[3] // 2, pool.dtype, pool.device)
            if mine != (plan.query_lens, plan.suffix_lens, plan.prefix_lens, plan.group_sizes,
                        plan.q_heads, plan.kv_heads, plan.head_dim, plan.dtype, plan.device):
                raise ValueError("the plan is of other lengths, heads or pool than this step")
        if query.shape != plan.shape or query.dtype is not plan.dtype:
            raise ValueError(f"query must be {plan.dtype} {tuple(plan.shape)}")
        turned, own = self._append(key, value, query, plan)
        out = plan(turned, self.pool, self.prefix_slots, own, status=self.status)
        self.lengths = list(plan.suffix_lens)
        return out

    def check(self) -> None:
        """Raise if any launch so far reported a status bit (waits for them)."""
        bits = self.status.read()
        if bits & (N.ST_SLOT_RANGE | N.ST_POS_RANGE):
            raise ValueError("a slot outside the pool or a position outside the tables")
        if bits:
            raise RuntimeError(f"device status bits set: {bits:#x}")
