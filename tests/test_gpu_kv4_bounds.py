"""Attention over the 4-bit pool within the tight bounds of oracle/kv4.py, in the
most and in the mean square: mistakes of one key, one unit or one operand part lie
outside (tests/test_kv4_bounds.py)."""

from __future__ import annotations

import math

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4
from oracle import kv4 as okv4
from test_gpu_kv4 import FORMS, TYPES, _batch, _wide

pytestmark = pytest.mark.gpu
MEAN = 1.15  # of some thousand rows' squares; an operand part that is lost gives 1.5 and more


def _tight(cuda, new, lengths, hq, hk, dim, group, block, dtype, seed=0, scale=None, scale_k=1.0):
    pool, table, q, starts = _batch(cuda, seed, new, lengths, hq, hk, dim, group, block, dtype,
                                    scale_k=scale_k)
    status = N.Status(cuda)
    got, lse = kv4.attention(
        q.to(cuda), pool, table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
        starts.to(cuda), scale=scale, return_lse=True, status=status)
    assert status.read() == 0
    wide = _wide(new, hq // hk)
    storage, got, lse = pool.storage.cpu(), got.cpu().double(), lse.cpu().double()
    eps, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal
    square = off = 0.0
    for b, length in enumerate(lengths):
        lo, hi = int(starts[b]), int(starts[b + 1])
        if lo == hi:
            continue
        want = okv4.bounds(q[lo:hi], storage, table[b], length, hi - lo, group,
                           dim ** -0.5 if scale is None else scale, wide)
        error = (got[lo:hi] - want.out).abs()
        assert (error <= want.err + eps * (want.out.abs() + want.err) + tiny * eps).all(), b
        far = (lse[lo:hi] - want.lse).abs()
        assert ((far <= want.lse_err) | (lse[lo:hi] == want.lse)).all(), (b, far.nan_to_num().max())
        off += (error ** 2).sum()
        square += (want.var + (okv4.ROUNDING * eps * want.out) ** 2).sum()
    assert math.sqrt(off / square) <= MEAN, math.sqrt(off / square)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", FORMS)
def test_questions(cuda, dtype, dim, group):
    _tight(cuda, [129, 64, 40, 150], [600, 64, 90, 333], 8, 2, dim, group, 48, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("new", [1, 3])
def test_decodes_and_drafts(cuda, dtype, dim, group, new):
    _tight(cuda, [new] * 40, [max(new, 37 * b % 700 + 1) for b in range(40)], 16, 4, dim, group, 16,
           dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[1] * 12, [2] * 12, [200, 3, 100]])
def test_cut_and_joined(cuda, dtype, new):
    _tight(cuda, new, [9001 - 700 * b for b in range(len(new))], 8, 2, 128, 64, 16, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_decodes_beside_a_chunk(cuda, dtype):
    _tight(cuda, [1] * 20 + [300], [100 + 90 * b for b in range(20)] + [700], 8, 2, 128, 64, 16,
           dtype)


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("scale_k", [1e-6, 1e5])
def test_small_and_large_keys(cuda, scale_k, new):
    _tight(cuda, [new] * 9, [77 + 30 * b for b in range(9)], 8, 2, 128, 64, 16, torch.bfloat16,
           scale=0.1 / scale_k, scale_k=scale_k)
