"""The C entries of the attention behind shared prefixes without a GPU: lengths
that no plan holds, plans of other heads, scales that float32 does not hold."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200.prefix import SharedPrefixAttention

HUGE = (1 << 63) - 1


def c_plan(prefix_lens, group_sizes, query_lens, suffix_lens, heads=(32, 8, 128),
           dtype=N.CS_BF16):
    vec = lambda v: (ctypes.c_int64 * max(1, len(v)))(*v)  # noqa: E731
    arrays = [vec(v) for v in (prefix_lens, group_sizes, query_lens, suffix_lens)]
    shape = N.PrefixShape(*heads, dtype, len(prefix_lens), len(query_lens),
                          *(ctypes.addressof(v) for v in arrays))
    info, words = N.PrefixPlanInfo(), (ctypes.c_int32 * 4096)()
    rc = N.load().cs_prefix_plan(ctypes.byref(shape), ctypes.byref(info), words, 4096)
    return rc, info


@pytest.mark.parametrize("lens", [
    ([5], [2], [1, HUGE], [3, 3]), ([5], [2], [1, 1], [3, HUGE]), ([5], [2], [1, 1], [HUGE, 3]),
    ([5, HUGE], [1, 1], [1, 1], [3, 3]), ([5, 1 << 32], [1, 1], [1, 1], [3, 3]),
    ([5], [2], [1, 1 << 33], [3, 3]), ([5], [2], [1, 1], [3, 1 << 31]),
])
def test_lengths_whose_sums_pass_64_bits(lens):
    assert c_plan(*lens)[0] == N.CS_ERR_UNSUPPORTED


@pytest.mark.parametrize("sizes", [[HUGE, HUGE, 4], [2, HUGE], [1 << 32, 2], [-1, 3]])
def test_group_sizes_that_only_add_up_modulo_64_bits(sizes):
    assert c_plan([5] * len(sizes), sizes, [1, 1], [3, 3])[0] == N.CS_ERR_INVALID
