"""Captured attention over the 4-bit pool follows the lengths, starts and tables that
it finds at each replay, in both kernels, beside other replays and eager calls."""

from __future__ import annotations

import random

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4
from test_gpu_kv4 import _batch

pytestmark = pytest.mark.gpu


def _captured(cuda, seed, tokens, requests, dtype):
    """A graph of one call over a pool of its own, and the buffers that it reads."""
    pool, table, q, _ = _batch(cuda, seed, [tokens] + [0] * (requests - 1), [400] * requests, 8, 2,
                               128, 64, 16, dtype)
    s = dict(q=q.to(cuda), tables=table.to(cuda), status=N.Status(cuda),
             lengths=torch.zeros(requests, dtype=torch.int32, device=cuda),
             starts=torch.zeros(requests + 1, dtype=torch.int32, device=cuda))

    def call():
        return kv4.attention(s["q"], pool, s["tables"], s["lengths"], s["starts"], return_lse=True,
                             status=s["status"])

    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s["out"], s["lse"] = call()
    stream.synchronize()
    return s | dict(graph=graph, stream=stream, call=call)


def _change(s, r):
    """Other lengths, starts (in order, or not) and tables."""
    requests, tokens = s["lengths"].shape[0], s["q"].shape[0]
    starts = sorted(r.randrange(tokens + 1) for _ in range(requests + 1))
    if r.random() < 0.5:
        starts[0], starts[-1] = 0, tokens
    if r.random() < 0.3:
        starts[r.randrange(requests + 1)] = r.choice([-1, 0, tokens, tokens + 7])
    s["starts"].copy_(torch.tensor(starts, dtype=torch.int32))
    s["lengths"].copy_(torch.tensor([r.randrange(401) for _ in range(requests)],
                                    dtype=torch.int32))
    order = torch.randperm(requests, generator=torch.Generator().manual_seed(r.randrange(1 << 30)))
    s["tables"].copy_(s["tables"][order.to(s["tables"].device)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,requests", [(12, 12), (30, 9), (500, 6)])
def test_replays_follow_their_buffers(cuda, dtype, tokens, requests):
    r, s = random.Random(tokens), _captured(cuda, 3, tokens, requests, dtype)
    for i in range(12):
        with torch.cuda.stream(s["stream"]):
            _change(s, r)
            s["graph"].replay()
        s["stream"].synchronize()
        out, lse = s["call"]()
        assert torch.equal(out, s["out"]) and torch.equal(lse, s["lse"]), i
    assert s["status"].read() & ~N.ST_CAPACITY == 0


def test_replays_side_by_side(cuda):
    """Graphs of both kernels on streams of their own, with eager calls among them."""
    r = random.Random(5)
    all_ = [_captured(cuda, i, t, n, torch.bfloat16)
            for i, (t, n) in enumerate(((9, 9), (40, 10), (300, 4), (700, 11)))]
    for s in all_:
        _change(s, r)
    torch.cuda.synchronize()
    want = [tuple(x.clone() for x in s["call"]()) for s in all_]
    torch.cuda.synchronize()
    for i in range(20):
        for s in all_:
            s["out"].fill_(7)
        torch.cuda.synchronize()
        for s in all_:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        eager = [s["call"]() for s in all_]
        torch.cuda.synchronize()
        for s, (out, lse), (a, b) in zip(all_, want, eager):
            assert torch.equal(s["out"], out) and torch.equal(s["lse"], lse), i
            assert torch.equal(a, out) and torch.equal(b, lse), i
