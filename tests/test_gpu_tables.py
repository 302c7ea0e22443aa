"""Slot maps built on the GPU against the token-by-token restatement."""

from __future__ import annotations

import random

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200.tables import step_maps
from oracle import kv4 as okv4

pytestmark = pytest.mark.gpu


def _batch(seed, requests, block, new_max, length_max, spare=3):
    r = random.Random(seed)
    new = [r.randint(0, new_max) for _ in range(requests)]
    lengths = [r.randint(n, max(n, length_max)) for n in new]
    width = max([1] + [-(-a // block) for a in lengths]) + 1
    need = sum(-(-a // block) for a in lengths)
    ids = list(range(need + spare))
    r.shuffle(ids)
    tables, at = [], 0
    for a, n in zip(lengths, new):
        held = -(-(a - n) // block)
        tables.append(ids[at:at + held] + [-7] * (width - held))
        at += held
    free = ids[at:]
    return lengths, new, tables, free, need + spare


def _dev(x, cuda, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device=cuda)
    return t if shape is None else t.reshape(shape)


@pytest.mark.parametrize("requests,block,new_max,length_max",
                         [(1, 16, 1, 1), (3, 16, 40, 100), (32, 16, 1, 700), (257, 3, 5, 60),
                          (300, 1, 2, 9), (1000, 32, 7, 200), (5, 128, 2000, 4000), (2, 16, 0, 0)])
def test_maps_equal_the_restatement(cuda, requests, block, new_max, length_max):
    lengths, new, tables, free, blocks = _batch(requests, requests, block, new_max, length_max)
    for extra_t, extra_k, offset in ((0, 0, 0), (5, 3, 77)):
        tokens, keys = sum(new) + extra_t, sum(lengths) + extra_k
        want = okv4.step_maps(lengths, new, tables, block, blocks, tokens, keys, offset, free,
                              len(free))
        held = _dev(tables, cuda, (requests, -1))
        status = N.Status(cuda)
        for _ in range(2):  # the same again
            m = step_maps(_dev(lengths, cuda), _dev(new, cuda), held, block, blocks,
                          tokens=tokens, keys=keys, offset=offset, free=_dev(free + [0], cuda),
                          free_count=_dev([len(free)], cuda), status=status)
            assert m.starts.tolist() == want["starts"]
            assert m.positions.tolist() == want["positions"]
            assert m.slots.tolist() == want["slots"]
            if keys:
                assert m.key_starts.tolist() == want["key_starts"]
                assert m.key_slots.tolist() == want["key_slots"]
            assert m.free_left.tolist() == [want["left"]]
            assert held.tolist() == want["tables"]
        assert status.read() == 0
        # complete tables, without the free ones
        m = step_maps(_dev(lengths, cuda), _dev(new, cuda), held, block, blocks, tokens=tokens)
        assert m.slots.tolist() == want["slots"] and m.free_left is None and m.key_slots is None


def test_slots_pass_32_bits(cuda):
    table = _dev([[1 << 30, (1 << 30) + 5]], cuda)
    m = step_maps(_dev([20], cuda), _dev([20], cuda), table, 16, 1 << 31, tokens=20, keys=20)
    want = [(1 << 34) + i for i in range(16)] + [(1 << 34) + 80 + i for i in range(4)]
    assert m.slots.tolist() == want == m.key_slots.tolist()


@pytest.mark.parametrize("change", ["negative", "more new", "narrow", "rows", "keys", "free",
                                    "count past the stack", "negative count"])
def test_all_or_nothing(cuda, change):
    lengths, new, tables, free, blocks = _batch(11, 40, 16, 9, 300)
    tokens, keys, count = sum(new), sum(lengths), len(free)
    if change == "negative":
        new[5] = -1
    elif change == "more new":
        lengths[7], new[7] = 3, 4
        tokens += 9
    elif change == "narrow":
        lengths[39] = 16 * len(tables[0]) + 1
        keys += lengths[39]
    elif change == "rows":
        tokens -= 1
    elif change == "keys":
        keys -= 1
    elif change == "count past the stack":
        count += 1
    elif change == "negative count":
        count = -1
        new, lengths = [0] * 40, [16] * 40
        keys = 640
    else:
        need = sum(-(-a // 16) - -(-(a - n) // 16) for a, n in zip(lengths, new))
        count = need - 1
    held = _dev(tables, cuda)
    status = N.Status(cuda)
    m = step_maps(_dev(lengths, cuda), _dev(new, cuda), held, 16, blocks, tokens=tokens,
                  keys=keys, free=_dev(free, cuda), free_count=_dev([count], cuda),
                  status=status)
    assert status.read() == N.ST_CAPACITY
    assert m.slots.eq(-1).all() and m.key_slots.eq(-1).all()
    assert m.positions.eq(0).all() and m.starts.eq(0).all() and m.key_starts.eq(0).all()
    assert m.free_left.tolist() == [count] and held.tolist() == tables


def test_a_block_outside_the_pool(cuda):
    status = N.Status(cuda)
    table = _dev([[2, 9], [-1, 0]], cuda)
    m = step_maps(_dev([20, 17], cuda), _dev([4, 17], cuda), table, 16, 9, tokens=21,
                  status=status)
    assert status.read() == N.ST_SLOT_RANGE
    assert m.slots.tolist() == [-1] * 4 + [-1] * 16 + [0]
    assert m.positions.tolist() == [16, 17, 18, 19] + list(range(17))


def test_captured_steps_follow_the_device_lengths(cuda):
    """A decode loop in a graph: lengths advance, blocks are taken, on a side stream."""
    lengths, new = _dev([0, 30, 47], cuda), _dev([1, 1, 1], cuda)
    table = _dev([[0] * 6, [1, 2, 0, 0, 0, 0], [3, 4, 5, 0, 0, 0]], cuda)
    free, count = _dev(list(range(6, 20)), cuda), _dev([14], cuda)
    out = torch.zeros(40, 3, dtype=torch.int64, device=cuda)
    status = N.Status(cuda)
    at = torch.zeros(1, dtype=torch.int64, device=cuda)

    def step():
        lengths.add_(1)
        m = step_maps(lengths, new, table, 16, 20, tokens=3, free=free, free_count=count,
                      status=status)
        count.copy_(m.free_left)
        out.index_copy_(0, at, m.slots[None])
        at.add_(1)

    start = [t.clone() for t in (lengths, table, count)]
    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        step()
        for t, s in zip((lengths, table, count), start):
            t.copy_(s)
        at.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(40):
            graph.replay()
    stream.synchronize()
    have, tabs, left = [0, 30, 47], [list(t) for t in start[1].tolist()], 14
    for i in range(40):
        have = [a + 1 for a in have]
        want = okv4.step_maps(have, [1, 1, 1], tabs, 16, 20, 3, free=list(range(6, 20)),
                              free_count=left)
        tabs, left = want["tables"], want["left"]
        assert out[i].tolist() == want["slots"], i
    assert table.tolist() == tabs and count.tolist() == [left] and status.read() == 0
