"""Attention over the 4-bit pool gives the same bits whatever a call before left in
shared memory or lies behind the last tokens."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import kv4
from test_gpu_kv4 import FORMS, TYPES, _batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("new,hq", [(1, 2), (1, 6), (3, 6), (5, 6), (40, 6)])
def test_the_same_bits_after_anything(cuda, dtype, dim, group, new, hq):
    """Rows that a tile lacks and keys that a unit lacks see what was there before:
    large scales, infinities, NaN, ordinary numbers."""
    lengths = [max(new, n) for n in (1, 5, 16, 18, 33, 50, 130, 260, 700)]
    pool, table, q, starts = _batch(cuda, 12, [new] * 9, lengths, hq, 2, dim, group, 16, dtype)
    args = (table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda))
    want, want_lse = kv4.attention(q.to(cuda), pool, *args, return_lse=True)
    full = torch.full((9,), 16 * table.shape[1], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    other = kv4.empty_pool(pool.num_blocks, 2, 16, dim, dtype, cuda, group)
    for fill in (0x7B, 0xFF, 0x7C, 0x00, None, None, None):
        if fill is None:
            other.storage.random_(0, 256, generator=g)
        else:
            other.storage.fill_(fill)
        kv4.attention(q.to(cuda), other, args[0].clamp(min=0), full, args[2])
        got, lse = kv4.attention(q.to(cuda), pool, *args, return_lse=True)
        assert torch.equal(got, want) and torch.equal(lse, want_lse), fill
        # and behind the last tokens
        dirty = kv4.empty_pool(pool.num_blocks, 2, 16, dim, dtype, cuda, group)
        dirty.storage.copy_(other.storage)
        row, pair = dim // 2, 4 * (dim // group)
        for b, length in enumerate(lengths):
            for j in range(-(-length // 16)):
                rows, block = min(16, length - 16 * j), int(table[b, j])
                base = 0
                for size in (row, row, pair, pair):
                    part = slice(base, base + rows * size)
                    dirty.storage[block, :, 0, part] = pool.storage[block, :, 0, part]
                    base += 16 * size
        got, lse = kv4.attention(q.to(cuda), dirty, *args, return_lse=True)
        assert torch.equal(got, want) and torch.equal(lse, want_lse), fill
