"""Attention over the 4-bit pool with starts that are none: the requests that are
left out, and every row of the output, new or given."""

from __future__ import annotations

import math
import random

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4
from test_gpu_kv4 import _batch, _check

pytestmark = pytest.mark.gpu


def _kept(starts, tokens):
    """The requests that have rows, and the requests that are in order."""
    rows, kept, floor = [], 0, 0
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        if lo >= floor and lo <= hi <= tokens:
            rows += [(b, lo, hi)] if hi > lo else []
            kept += 1
        floor = max(floor, lo)
    return rows, kept


def _dirty(cuda):
    """Memory that a new tensor may get next."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 22):
        torch.full((n,), math.nan, device=cuda)


def _try(cuda, starts, tokens, lengths, seed=2, dim=128, hq=8, hk=2):
    pool, table, q, _ = _batch(cuda, seed, [tokens] + [0] * (len(lengths) - 1), lengths, hq, hk,
                               dim, 64, 16, torch.bfloat16)
    rows, kept = _kept(starts, tokens)
    args = (q.to(cuda), pool, table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
            torch.tensor(starts, dtype=torch.int32, device=cuda))
    _dirty(cuda)
    status = N.Status(cuda)
    got, lse = kv4.attention(*args, return_lse=True, status=status)
    assert status.read() == (0 if kept == len(lengths) else N.ST_CAPACITY)
    free = torch.ones(tokens, dtype=torch.bool)
    wide = tokens * (hq // hk) // len(lengths) > 32
    for b, lo, hi in rows:
        free[lo:hi] = False
        _check(got[lo:hi], lse[lo:hi], pool, table[b:b + 1], q[lo:hi], [0, hi - lo], [lengths[b]],
               dim ** -0.5, wide)
    assert got[free].eq(0).all() and lse[free].eq(-math.inf).all()
    for _ in range(3):
        _dirty(cuda)
        again, again_lse = kv4.attention(*args, return_lse=True)
        assert torch.equal(again, got) and torch.equal(again_lse, lse)
    out = torch.full_like(got, 7.0)
    kv4.attention(*args, out=out)
    assert torch.equal(out[~free], got[~free]) and out[free].eq(7).all()


@pytest.mark.parametrize("starts", [
    [0, 9], [-1, 8], [0, 100, 4], [0, 5, 3], [0, 5, 3, 8], [8, 8], [3, 6], [5, 2, 8], [0, 8, 0, 8],
    [-5, -3, 2, 8], [2, 1, 0], [0, 3, 100, 3, 8], [4, 4, 2, 4, 8], [0, 2, -2147483648, 8],
    [0, 2147483647, 8], [2147483647, -2147483648]])
def test_a_few_rows(cuda, starts):
    _try(cuda, starts, 8, [20 + 31 * b for b in range(len(starts) - 1)])


@pytest.mark.parametrize("starts", [
    [0, 301], [-1, 150, 300], [0, 200, 100, 300], [0, 200, 100], [0, 100, 90, 95, 300],
    [5, 70, 290], [100, 50, 300], [0, 300, 0, 300], [0, 150, 1000, 150, 300]])
def test_many_rows(cuda, starts):
    _try(cuda, starts, 300, [320 + 91 * b for b in range(len(starts) - 1)])


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("tokens,requests", [(700, 500), (9000, 200)])
def test_many_requests(cuda, seed, tokens, requests):
    r = random.Random(seed)
    starts = sorted(r.randrange(tokens + 1) for _ in range(requests + 1))
    for _ in range(seed):
        starts[r.randrange(requests + 1)] = r.choice([-3, 0, tokens, tokens + 1, tokens // 2])
    _try(cuda, starts, tokens, [r.randrange(60) for _ in range(requests)], dim=64, hq=4, hk=1)


def test_rows_without_requests(cuda):
    pool, table, q, _ = _batch(cuda, 2, [8], [20], 8, 2, 128, 64, 16, torch.bfloat16)
    _dirty(cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    got, lse = kv4.attention(q.to(cuda), pool, table[:0].to(cuda), none,
                             torch.zeros(1, dtype=torch.int32, device=cuda), return_lse=True)
    assert got.eq(0).all() and lse.eq(-math.inf).all()
