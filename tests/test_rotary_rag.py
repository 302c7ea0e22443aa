"""The retrieval batch of a rotary layer without a GPU: which plans a step
takes.  The batch's fields are filled by hand on the CPU and its append is
recorded, so nothing is launched."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200.prefix import SharedPrefixAttention
from cacheslide_b200.rotary_rag import RotaryRagBatch


class _Appended(Exception):
    pass


def batch(lengths, max_own=20, block=16, prefix=40, dtype=torch.float32):
    b = RotaryRagBatch.__new__(RotaryRagBatch)
    per = -(-max_own // block) * block
    b.pool = torch.zeros(32, 2, block, 16, dtype=dtype)
    b.q_heads, b.requests, b.max_own = 4, len(lengths), max_own
    b.prefix_slots = torch.arange(prefix)
    b.own_slots = 48 + torch.arange(len(lengths) * per).view(len(lengths), per)
    b.lengths = list(lengths)

    def appended(*args):
        raise _Appended

    b._append = appended
    return b


def plan(queries, own, prefix=40, heads=(4, 2, 8), dtype=torch.float32, **kw):
    return SharedPrefixAttention(*heads, dtype, "cpu", query_lens=queries, suffix_lens=own,
                                 prefix_lens=[prefix], **kw)


def step(b, queries, plan=None):
    n = sum(queries)
    return b.step(torch.zeros(n, 4, 8), torch.zeros(n, 2, 8), torch.zeros(n, 2, 8), queries, plan)


def test_a_step_takes_the_plan_of_its_lengths():
    for given in (None, plan([2, 1, 3], [5, 1, 7])):
        with pytest.raises(_Appended):
            step(batch([3, 0, 4]), [2, 1, 3], given)


@pytest.mark.parametrize("queries,own,kw", [
    ([1, 2, 3], [5, 1, 7], {}),                      # the same sums, other requests
    ([2, 1, 3], [4, 2, 7], {}),                      # other histories of the same sum
    ([2, 1, 3], [5, 1, 7], dict(prefix=39)),
    ([2, 1], [5, 1], {}),
    ([2, 1, 3], [5, 1, 7], dict(heads=(8, 2, 8))),
    ([2, 1, 3], [5, 1, 7], dict(heads=(4, 4, 8))),
    ([2, 1, 3], [5, 1, 7], dict(heads=(4, 2, 16))),
    ([2, 1, 3], [5, 1, 7], dict(dtype=torch.float16)),
])
def test_a_step_refuses_another_plan_before_it_writes(queries, own, kw):
    b = batch([3, 0, 4])
    with pytest.raises(ValueError, match="plan"):
        step(b, [2, 1, 3], plan(queries, own, **kw))
    assert b.lengths == [3, 0, 4]


def test_a_step_refuses_a_plan_of_several_groups():
    with pytest.raises(ValueError, match="plan"):
        step(batch([3, 0]), [2, 1], SharedPrefixAttention(
            4, 2, 8, torch.float32, "cpu", query_lens=[2, 1], suffix_lens=[5, 1],
            prefix_lens=[20, 20], group_sizes=[1, 1]))


@pytest.mark.parametrize("given", [False, True])
def test_a_step_past_the_own_keys_of_a_request(given):
    """Blocks hold 32 keys, the tables' positions end at 20."""
    with pytest.raises(ValueError, match="own keys"):
        step(batch([18, 0]), [3, 1], plan([3, 1], [21, 1]) if given else None)


@pytest.mark.parametrize("given", [False, True])
def test_a_step_refuses_lengths_that_are_no_counts(given):
    for queries in ([-1, 3], [2], [2, 1, 1]):
        with pytest.raises(ValueError):
            step(batch([3, 0]), queries, plan([2, 1], [5, 1]) if given else None)


def test_a_step_refuses_queries_of_another_shape_before_it_writes():
    b = batch([3, 0])
    z = torch.zeros
    with pytest.raises(ValueError, match="query"):
        b.step(z(4, 4, 8), z(3, 2, 8), z(3, 2, 8), [2, 1])
    with pytest.raises(ValueError, match="query"):
        b.step(z(3, 4, 8, dtype=torch.float16), z(3, 2, 8), z(3, 2, 8), [2, 1])
