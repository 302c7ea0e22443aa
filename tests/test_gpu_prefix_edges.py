"""Attention behind shared prefixes where values are not finite: which columns
of which rows a key's infinity or NaN may reach, bit for bit."""

from __future__ import annotations

import pytest
import torch

from test_gpu_prefix import BF, HF, LAYOUTS, batch, plan_of

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


def put(s, slots, values, d):
    """values[k][column] written to the V half of slot k's records, every head."""
    for slot, row in zip(slots, values):
        for c, x in row.items():
            s["cache"][slot // 16, :, slot % 16, d + c] = x


NAMES = ["decode", "drafts", "groups", "questions", "wide batch", "wide ragged"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
@pytest.mark.parametrize("columns", ["first half", "last half", "all"])
def test_a_hidden_value_leaves_no_trace(cuda, name, hq, hk, d, dtype, columns):
    """Rows that do not see the key have the bits that they have without the
    infinity, also in repeated calls, and in the row that sees it the other
    columns are finite."""
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    plan = plan_of(s, lens)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    sees = torch.zeros(s["query"].shape[0], dtype=torch.bool, device=cuda)
    cols = dict([("first half", [3]), ("last half", [d - 2]), ("all", range(d))])[columns]
    last = last_own_slots(s, lens)
    put(s, [slot for _, slot in last], [dict.fromkeys(cols, 0.0)] * len(last), d)
    clean, clean_lse = plan(*args, return_lse=True)
    put(s, [slot for _, slot in last],
        [dict.fromkeys(cols, (NAN, INF, -INF)[i % 3]) for i in range(len(last))], d)
    sees[[token for token, _ in last]] = True
    for _ in range(4):
        got, lse = plan(*args, return_lse=True)
        assert torch.equal(got[~sees], clean[~sees]) and torch.equal(lse, clean_lse)
    hit = torch.zeros(d, dtype=torch.bool, device=cuda)
    hit[list(cols)] = True
    for i, (token, _) in enumerate(last):
        if i % 3 == 0:
            assert torch.isnan(got[token][:, hit]).all()
        else:
            assert (got[token][:, hit] == (INF, -INF)[i % 3 - 1]).all()
        assert torch.equal(got[token][:, ~hit], clean[token][:, ~hit])


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
def test_values_in_the_prefix_reach_their_columns_alone(cuda, name, hq, hk, d, dtype):
    """NaN, infinities of one sign and of both: what a sum of positive weights
    times such values is, and the bits without them in every other column."""
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    plan = plan_of(s, lens)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    where = [int(s["prefix_slots"][i]) for i in (0, 66, 100)]
    values = [{0: NAN, 5: INF, 6: -INF, 7: INF}, {7: -INF, d - 1: NAN, d // 2: INF},
              {0: INF, 5: INF, d // 2 + 1: -INF}]
    put(s, where, [dict.fromkeys(row, 0.0) for row in values], d)
    clean, clean_lse = plan(*args, return_lse=True)
    put(s, where, values, d)
    want = clean.clone()
    sees = torch.zeros(s["query"].shape[0], dtype=torch.bool, device=cuda)
    sees[:sum(lens["query_lens"][:(lens["group_sizes"] or [len(lens["query_lens"])])[0]])] = True
    for c, x in ((0, NAN), (5, INF), (6, -INF), (7, NAN), (d - 1, NAN), (d // 2, INF),
                 (d // 2 + 1, -INF)):
        want[sees, :, c] = x
    got, lse = plan(*args, return_lse=True)
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    assert torch.equal(lse, clean_lse)


@pytest.mark.parametrize("name", ["decode", "wide batch"])
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
def test_values_of_keys_that_weigh_nothing(cuda, name, hq, hk, d, dtype):
    """A score of -inf weighs nothing, whatever its value holds."""
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    plan = plan_of(s, lens)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    s["query"][..., 0] = 1.0
    first = s["prefix_slots"][30:130]
    s["cache"][first // 16, :, first % 16, 0] = -INF
    s["cache"][first // 16, :, first % 16, d:] = 0.0
    clean = plan(*args)
    s["cache"][first // 16, :, first % 16, d:] = NAN
    assert torch.equal(plan(*args), clean)


@pytest.mark.parametrize("name", ["decode", "questions", "wide ragged"])
def test_values_in_strided_outputs_and_odd_queries(cuda, name):
    """The same where outputs are not stored in vectors."""
    s, lens = batch(cuda, 8, 2, 128, BF, *LAYOUTS[name])
    plan = plan_of(s, lens)
    tokens = s["query"].shape[0]
    slot = int(s["prefix_slots"][70])
    put(s, [slot], [{2: 0.0, 100: 0.0}], 128)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    want = plan(*args)
    put(s, [slot], [{2: NAN, 100: INF}], 128)
    want[..., 2], want[..., 100] = NAN, INF
    out = torch.zeros(tokens, 8, 129, dtype=BF, device=cuda)
    odd = torch.zeros(tokens, 8 * 128 + 1, dtype=BF, device=cuda)[:, 1:].unflatten(1, (8, 128))
    odd.copy_(s["query"])
    got = plan(odd, *args[1:], out=out[..., 1:])
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    assert not out[..., 0].any()


@pytest.mark.parametrize("hq,hk,d,dtype", HEADS + [(4, 2, 80, BF), (4, 2, 64, torch.float32)])
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_part_of_little_weight_keeps_what_is_not_finite(cuda, hq, hk, d, dtype, value):
    """Scores far below the row's largest (here by some 2000) still weigh more
    than nothing: a NaN or infinite value among them makes its column not
    finite, wherever the plan cuts the keys."""
    s, lens = batch(cuda, hq, hk, d, dtype, [1] * 3, [40] * 3, [4000])
    plan = plan_of(s, lens)
    s["query"][..., 0] = 160.0
    slots = s["prefix_slots"]
    s["cache"][..., 0] = 0.0
    s["cache"][slots[:1000] // 16, :, slots[:1000] % 16, 0] = 160.0
    far = int(slots[3000])
    put(s, [far], [{9: value}], d)
    got = plan(s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"])
    assert not torch.isfinite(got[..., 9]).any()
    rest = torch.arange(d, device=cuda) != 9
    assert torch.isfinite(got[..., rest]).all()


@pytest.mark.parametrize("name,block,scattered", [("drafts", 16, 1.0), ("wide ragged", 5, 0.0),
                                                  ("wide ragged", 16, 0.2), ("decode", 1, 0.0)])
@pytest.mark.parametrize("scale", [None, -0.1])
def test_values_in_relocated_slots_and_in_a_graph(cuda, name, block, scattered, scale):
    """Keys copied row by row, negative scales, and calls that follow each
    other closely."""
    s, lens = batch(cuda, 8, 2, 128, BF, *LAYOUTS[name], block=block, scattered=scattered)
    plan = plan_of(s, lens)
    hidden = [slot for _, slot in last_own_slots(s, lens)]
    seen = int(s["prefix_slots"][77])
    sees = torch.zeros(s["query"].shape[0], dtype=torch.bool, device=cuda)
    sees[[token for token, _ in last_own_slots(s, lens)]] = True

    def fill(value):
        for slot in hidden:
            s["cache"][slot // block, :, slot % block, 128 + 40] = value
        s["cache"][seen // block, :, seen % block, 128 + 90] = value

    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    fill(0.0)
    want = plan(*args, scale=scale)
    want[..., 90] = NAN
    want[sees, :, 40] = NAN
    fill(NAN)
    got = plan(*args, scale=scale)
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    outs = [torch.empty_like(got) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for out in outs:
            plan(*args, scale=scale, out=out)
    graph.replay()
    for out in outs:
        torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("name", ["decode", "questions", "wide batch"])
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS + [(4, 2, 80, BF)])
@pytest.mark.parametrize("shift", [0, 1])
def test_output_over_the_queries(cuda, name, hq, hk, d, dtype, shift):
    """``out`` may be the queries' own memory, or overlap it, whatever the
    values hold."""
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    plan = plan_of(s, lens)
    for _, slot in last_own_slots(s, lens):
        s["cache"][slot // 16, :, slot % 16, d + 3] = NAN
    rest = s["cache"], s["prefix_slots"], s["suffix_slots"]
    want = plan(s["query"], *rest)
    tokens = s["query"].shape[0]
    both = torch.zeros(tokens + shift, hq, d, dtype=dtype, device=cuda)
    query, out = both[:tokens].copy_(s["query"]), both[shift:]
    assert plan(query, *rest, out=out).data_ptr() == out.data_ptr()
    torch.testing.assert_close(out, want, rtol=0, atol=0, equal_nan=True)
