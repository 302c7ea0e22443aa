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
