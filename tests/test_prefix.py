"""Attention behind shared prefixes without a GPU: the plan's ranges, and the
refusals."""

from __future__ import annotations

import random

import pytest
import torch

from cacheslide_b200.prefix import SharedPrefixAttention


def plan(queries, suffixes, prefixes, sizes=None, heads=(32, 8, 128), dtype=torch.bfloat16):
    return SharedPrefixAttention(*heads, dtype, "cpu", query_lens=queries, suffix_lens=suffixes,
                                 prefix_lens=prefixes, group_sizes=sizes)


def ranges(queries, suffixes, prefixes, sizes=None):
    """Per token: the prefix keys and own keys it sees."""
    out, b, p0, k0 = [], 0, 0, 0
    for length, members in zip(prefixes, [len(queries)] if sizes is None else sizes):
        for _ in range(members):
            n, m = queries[b], suffixes[b]
            out += [(p0, p0 + length, k0, k0 + max(0, m - n + i + 1)) for i in range(n)]
            k0, b = k0 + m, b + 1
        p0 += length
    return out


def random_batch(r):
    groups = r.randint(1, 4)
    sizes = [r.randint(0, 9) for _ in range(groups)]
    top = r.choice([1, 4, 40, 300])
    queries = [r.randint(0 if r.random() < 0.2 else 1, top) for _ in range(sum(sizes))]
    suffixes = [max(0, n + r.randint(-3, 700)) for n in queries]
    return queries, suffixes, [r.choice([0, 1, r.randint(2, 6000)]) for _ in sizes], sizes


@pytest.mark.parametrize("seed", range(30))
def test_tokens_see_what_the_definition_says(seed):
    case = random_batch(random.Random(seed))
    p = plan(*case)
    got = p.words[:4 * p.tokens].view(-1, 4).tolist()
    want = ranges(*case)
    for g, w in zip(got, want):
        assert g[:2] == list(w[:2]) and g[2:] == list(w[2:])
    assert len(got) == len(want)


@pytest.mark.parametrize("change", [
    dict(heads=(32, 5, 128)), dict(heads=(0, 8, 128)), dict(heads=(32, 8, 0)),
    dict(heads=(32, 8, 1024)), dict(dtype=torch.float64), dict(dtype=torch.int32),
    dict(queries=[1]), dict(queries=[1, -1]), dict(queries=[1, 2.0]), dict(suffixes=[1, 1 << 31]),
    dict(suffixes=[1 << 30, 1 << 30]), dict(prefixes=[1, 2]), dict(prefixes=[]),
    dict(sizes=[1]), dict(sizes=[1, 1]), dict(queries=[1 << 29, 1]),
])
def test_plan_refuses(change):
    good = dict(queries=[1, 2], suffixes=[3, 4], prefixes=[5], sizes=None)
    with pytest.raises(ValueError):
        plan(**{**good, **change})


def test_call_refuses_cpu_tensors():
    p = plan([1], [1], [4])
    z = torch.zeros(1, 32, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        p(z, torch.zeros(1, 8, 16, 256, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64),
          torch.zeros(1, dtype=torch.int64))


def items_of(p):
    i = p.info
    rows = p.words[i.item_off:i.item_off + 8 * i.n_items].view(-1, 8).tolist()
    join = p.words[i.join_off:i.join_off + 4 * i.n_join].view(-1, 4).tolist()
    return rows, join, p.words[i.list_off:].tolist()


@pytest.mark.parametrize("heads", [(32, 8, 128), (8, 8, 64), (24, 2, 64), (128, 1, 128)])
@pytest.mark.parametrize("seed", range(25))
def test_items_cover_every_seen_key_once(seed, heads):
    """Each (token, key) pair that the definition allows lies in exactly one
    item of that token, items fit their row tiles, and each token's partial
    results are joined once each or written by its only item."""
    case = random_batch(random.Random(100 + seed))
    p = plan(*case, heads=heads)
    items, join, entries = items_of(p)
    want = ranges(*case)
    per = 128 // (heads[0] // heads[1]) * p.info.variant
    pieces = [[] for _ in want]
    for tok0, ntok, a0, a1, b0, b1, part, _ in items:
        assert 0 < ntok <= per and a0 <= a1 and b0 <= b1 and (a1 > a0 or b1 > b0)
        for k in range(ntok):
            pieces[tok0 + k].append((a0, a1, b0, b1, -1 if part < 0 else part + k))
    joined = {}
    for token, first, count, _ in join:
        assert token not in joined
        joined[token] = sorted(entries[first:first + count])
    seen_parts = [e for v in joined.values() for e in v]
    assert len(seen_parts) == len(set(seen_parts))
    assert all(0 <= e < p.info.part_tokens for e in seen_parts)
    for token, (p0, p1, lo, hi) in enumerate(want):
        mine = pieces[token]
        for which, (start, end) in ((0, (p0, p1)), (2, (lo, hi))):
            spans = sorted((max(x[which], start), min(x[which + 1], end)) for x in mine)
            spans = [x for x in spans if x[1] > x[0]]
            at = start
            for s0, s1 in spans:
                assert s0 == at
                at = s1
            assert at == end
        for x in mine:  # an item's prefix range lies inside its tokens' prefix
            assert x[0] == x[1] or p0 <= x[0] and x[1] <= p1
        parts = sorted(x[4] for x in mine)
        if token in joined:
            assert parts == joined[token]
        else:
            assert parts == [-1]


def test_plan_spreads_a_long_prefix_over_the_machine():
    """Few rows over many keys: enough parts for every SM, none of them long."""
    p = plan([1] * 8, [30] * 8, [65536], heads=(64, 8, 128))
    items, _, _ = items_of(p)
    assert len(items) * 8 >= 148
    assert max(-(-(i[3] - i[2]) // 128) for i in items) <= 512 * 8 // 148 + 1


def test_plan_of_types_without_tensor_cores_has_no_items():
    for heads, dtype in (((4, 2, 80), torch.bfloat16), ((4, 2, 128), torch.float32),
                         ((256, 1, 128), torch.bfloat16)):
        p = plan([1, 2], [3, 4], [5], heads=heads, dtype=dtype)
        assert p.info.variant == 0 and p.info.n_items == 0 and p.info.workspace == 0
