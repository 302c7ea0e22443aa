"""The C entries of the attention behind shared prefixes without a GPU: lengths
that no plan holds, plans of other heads, scales that float32 does not hold."""

from __future__ import annotations

import ctypes

import pytest

from cacheslide_b200 import _native as N

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


def c_call(info, heads=(32, 8, 128), dtype=N.CS_BF16, workspace=16, scale=0.1):
    """cs_prefix_attn up to its checks: no argument is a place in memory."""
    kv = N.PagedKV(cache=16, num_blocks=4, kv_heads=heads[1], block_size=16, head_dim=heads[2],
                   stride_block=heads[1] * 32 * heads[2], stride_head=32 * heads[2],
                   stride_offset=2 * heads[2], stride_elem=1, dtype=dtype)
    p = N.PrefixParams(q=16, paged=kv, prefix_slots=16, suffix_slots=16, q_heads=heads[0],
                       scale=scale, out=16)
    return N.load().cs_prefix_attn(ctypes.byref(p), ctypes.byref(info), 16, workspace, None)


@pytest.mark.parametrize("heads,dtype", [
    ((64, 8, 128), N.CS_BF16), ((64, 16, 128), N.CS_BF16), ((32, 4, 128), N.CS_BF16),
    ((32, 8, 64), N.CS_BF16), ((32, 8, 80), N.CS_BF16), ((32, 8, 128), N.CS_F32),
])
def test_a_call_refuses_a_plan_of_other_heads(heads, dtype):
    rc, info = c_plan([3000], [4], [1] * 4, [30] * 4)
    assert rc == N.CS_OK and info.variant > 0 and info.workspace > 0
    assert c_call(info, heads, dtype) == N.CS_ERR_INVALID
    assert c_call(info, workspace=None) == N.CS_ERR_INVALID


def test_a_call_refuses_a_row_plan_of_other_groups():
    rc, info = c_plan([3000], [4], [1] * 4, [30] * 4, dtype=N.CS_F32)
    assert rc == N.CS_OK and info.variant == 0
    assert c_call(info, (32, 4, 128), N.CS_F32) == N.CS_ERR_INVALID


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -1e300])
def test_a_call_refuses_scales_that_are_not_finite_floats(scale):
    _, info = c_plan([3000], [4], [1] * 4, [30] * 4)
    assert c_call(info, scale=scale) == N.CS_ERR_INVALID
