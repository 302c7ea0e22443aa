"""Attention behind shared prefixes where values are not finite: which columns
of which rows a key's infinity or NaN may reach, bit for bit."""

from __future__ import annotations

import pytest
import torch

from test_gpu_prefix import BF, HF, LAYOUTS, batch, bounds, plan_of
from oracle import prefix as oprefix

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
HEADS = [(8, 2, 128, BF), (32, 8, 128, HF), (8, 2, 64, HF), (8, 8, 64, BF)]


def last_own_slots(s, lens):
    """Per request with queries and own keys: its newest token and its slot,
    which only that token sees."""
    out, t, k0 = [], 0, 0
    for n, m in zip(lens["query_lens"], lens["suffix_lens"]):
        if n and m:
            out.append((t + n - 1, int(s["suffix_slots"][k0 + m - 1])))
        t, k0 = t + n, k0 + m
    return out


@pytest.mark.parametrize("name", ["wide batch", "wide ragged", "drafts"])
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
@pytest.mark.parametrize("column", ["first", "last"])
def test_a_hidden_value_in_one_half_leaves_the_other_half_alone(cuda, name, hq, hk, d, dtype,
                                                                column):
    """Rows that do not see the key keep, in the columns of the half of the head
    without it, the bits that they have without the infinity; the columns of
    its half are computed again (within the tolerance); equal calls give equal
    bits."""
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    plan = plan_of(s, lens)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    clean = plan(*args)
    c = 3 if column == "first" else d - 2
    other = slice(d // 2, d) if column == "first" else slice(0, d // 2)
    sees = torch.zeros(s["query"].shape[0], dtype=torch.bool, device=cuda)
    for i, (token, slot) in enumerate(last_own_slots(s, lens)):
        s["cache"][slot // 16, :, slot % 16, d + c] = (NAN, INF, -INF)[i % 3]
        sees[token] = True
    got = plan(*args)
    for _ in range(5):
        assert torch.equal(plan(*args)[~sees], got[~sees])
    if plan.info.variant == 2:
        assert torch.equal(got[~sees][..., other], clean[~sees][..., other])
    tol = bounds(dtype, d, lens, *oprefix.attention(
        s["query"], s["cache"].nan_to_num(0, 0, 0), s["prefix_slots"], s["suffix_slots"], **lens))[0]
    off = (got.double() - clean.double()).abs()[~sees]
    assert (off <= 2 * tol[~sees]).all()
    # those that see it: that column alone is not finite
    assert not torch.isfinite(got[sees][..., c]).any()
    rest = torch.arange(d, device=cuda) != c
    assert torch.isfinite(got[sees][..., rest]).all()
