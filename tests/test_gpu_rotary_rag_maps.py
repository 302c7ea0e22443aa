"""The retrieval batch's slots and positions, made on the device: those of its
blocks, and a step captured with its plan follows the same buffers."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import rotary_rag
from cacheslide_b200.rotary_rag import RotaryRagBatch

pytestmark = pytest.mark.gpu


def _batch(cuda, requests=5, prefix=37, max_own=40):
    pool = torch.zeros(40, 2, 16, 256, dtype=torch.bfloat16, device=cuda)
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(2)).tolist()
    return RotaryRagBatch(pool, 4, prefix, requests, max_own, block_ids=ids)


def _rows(cuda, n, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, h, 128, generator=g).bfloat16().to(cuda) for h in (4, 2, 2)]


def test_places_of_a_step(cuda, monkeypatch):
    batch = _batch(cuda)
    batch.write_prefix(*_rows(cuda, 37, 0)[1:])
    seen = []
    real = rotary_rag.append_rotated

    def append(pool, slots, key, value, positions, *args, **kw):
        seen.append((slots.tolist(), positions.tolist()))
        return real(pool, slots, key, value, positions, *args, **kw)

    monkeypatch.setattr(rotary_rag, "append_rotated", append)
    have = [0] * 5
    for i, counts in enumerate(([3, 0, 17, 1, 40], [1, 0, 0, 2, 0], [0, 9, 4, 0, 0])):
        batch.step(*_rows(cuda, sum(counts), i), counts)
        slots, positions = [], []
        for b, n in enumerate(counts):
            slots += batch.own_slots[b, have[b]:have[b] + n].tolist()
            positions += list(range(37 + have[b], 37 + have[b] + n))
            have[b] += n
        assert seen[-1] == (slots, positions) and batch.lengths == have
    batch.check()


def test_a_step_without_tokens_keeps_the_batch(cuda):
    batch = _batch(cuda)
    batch.write_prefix(*_rows(cuda, 37, 0)[1:])
    assert batch.step(*_rows(cuda, 0, 0), [0] * 5).shape == (0, 4, 128)
    assert batch.lengths == [0] * 5
    batch.check()


def test_a_captured_step(cuda):
    counts = [2, 1, 3, 1, 1]
    eager, captured = _batch(cuda), _batch(cuda)
    for b in (eager, captured):
        b.write_prefix(*_rows(cuda, 37, 0)[1:])
    plan = captured.plan(counts)
    rows = _rows(cuda, 8, 1)
    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        captured.step(*rows, counts, plan)  # first uses outside the capture
        captured.lengths = [0] * 5
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = captured.step(*rows, counts, plan)
        graph.replay()
    stream.synchronize()
    assert torch.equal(out, eager.step(*rows, counts))
    assert torch.equal(captured.pool, eager.pool)
    captured.check()
