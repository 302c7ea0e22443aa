"""Rotary operators where they are easily wrong: infinities in the part of a
head that is not rotated, in the kernels for heads and strides that vectors do
not fit; plans of other lengths.

Elements past ``rotary_dim`` pass through (times the norm's factor and weight):
one of them that is infinite touches no other element of its row, except
through the norm's sum.  The comparisons are exact."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import rotary
from cacheslide_b200.rotary_rag import RotaryRagBatch

pytestmark = pytest.mark.gpu

INF = float("inf")
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
# tokens, dim, rotated, interleaved, dtype, odd start: what vectors do not fit
# (dims that are no power of two of vectors; starts that are no multiple of
# one) and, last, two that they do
ROWS = [(9, 80, 40, False, BF, 0), (9, 80, 40, True, HF, 0), (5, 96, 6, False, FP, 0),
        (9, 64, 32, False, BF, 1), (9, 128, 64, True, HF, 1), (5, 64, 32, True, FP, 1),
        (9, 128, 64, False, BF, 0), (9, 64, 32, True, HF, 0)]


def rows(device, tokens, heads, dim, dtype, odd, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    wide = torch.randn(tokens, heads * dim + odd, generator=g, device=device).to(dtype)
    return wide[:, odd:].unflatten(1, (heads, dim))


def args_of(device, tokens, dim, rot, inter):
    cos, sin = rotary.rotary_tables(64, rot, device=device)
    return dict(positions=torch.arange(3, 3 + tokens, device=device), cos=cos, sin=sin,
                interleaved=inter)


def places(dim, rot):
    """Elements past the rotated part: its first, one in the middle, the last."""
    return sorted({rot, rot + (dim - rot) // 2, dim - 1})


@pytest.mark.parametrize("tokens,dim,rot,inter,dtype,odd", ROWS)
def test_an_infinity_past_the_rotated_part_stays_where_it_is(cuda, tokens, dim, rot, inter, dtype,
                                                             odd):
    args = args_of(cuda, tokens, dim, rot, inter)
    q, k = rows(cuda, tokens, 3, dim, dtype, odd, 1), rows(cuda, tokens, 2, dim, dtype, odd, 2)
    want_q, want_k = (x.clone() for x in rotary.qk_norm_rope(q, k, **args))
    for n, e in enumerate(places(dim, rot)):
        for x, want in ((q, want_q), (k, want_k)):
            x[n + 1, 1, e] = want[n + 1, 1, e] = -INF if n % 2 else INF
    got_q, got_k = rotary.qk_norm_rope(q, k, **args)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    # with a norm the row's factor is zero: the infinity itself gives NaN, the rest zeros
    w = torch.ones(dim, dtype=dtype, device=cuda)
    got_q, _ = rotary.qk_norm_rope(q, k, q_weight=w, **args)
    for n, e in enumerate(places(dim, rot)):
        row = got_q[n + 1, 1]
        rest = torch.arange(dim, device=cuda) != e
        assert torch.isnan(row[e]) and not row[rest].any()


@pytest.mark.parametrize("tokens,dim,rot,inter,dtype,odd", ROWS)
def test_an_infinite_gradient_past_the_rotated_part(cuda, tokens, dim, rot, inter, dtype, odd):
    args = args_of(cuda, tokens, dim, rot, inter)
    q, k = rows(cuda, tokens, 3, dim, dtype, odd, 3), rows(cuda, tokens, 2, dim, dtype, odd, 4)
    w = rows(cuda, 1, 1, dim, dtype, 0, 5)[0, 0]

    def grads(gq, gk, weight):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, w)]
        out = rotary.qk_norm_rope(leaves[0], leaves[1], k_weight=leaves[2] if weight else None,
                                  **args)
        return torch.autograd.grad(out, leaves[:2 + weight], (gq, gk))

    gq, gk = torch.randn_like(q), torch.randn_like(k)
    want_q, want_k = (x.clone() for x in grads(gq, gk, False))
    _, _, want_w = grads(gq, gk, True)
    bad = places(dim, rot)
    for n, e in enumerate(bad):
        gq[n + 1, 1, e] = gk[n + 1, 1, e] = INF
        want_q[n + 1, 1, e] = want_k[n + 1, 1, e] = INF
    got_q, got_k = grads(gq, gk, False)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    # a weight's gradient is a sum over rows of its own element
    got_w = grads(gq, gk, True)[2]
    rest = torch.ones(dim, dtype=torch.bool, device=cuda)
    rest[bad] = False
    assert torch.equal(got_w[rest], want_w[rest])
    assert not torch.isfinite(got_w[~rest]).any()


@pytest.mark.parametrize("tokens,dim,rot,inter,dtype,odd", ROWS)
def test_append_of_an_infinity_past_the_rotated_part(cuda, tokens, dim, rot, inter, dtype, odd):
    args = args_of(cuda, tokens, dim, rot, inter)
    q, k = rows(cuda, tokens, 3, dim, dtype, odd, 6), rows(cuda, tokens, 2, dim, dtype, odd, 7)
    v = rows(cuda, tokens, 2, dim, dtype, odd, 8)
    slots = torch.randperm(32, device=cuda)[:tokens].contiguous()
    cache = torch.zeros(2, 2, 16, 2 * dim, dtype=dtype, device=cuda)
    want_q = rotary.append_rotated(cache, slots, k, v, query=q, **args).clone()
    want = cache.clone()
    for n, e in enumerate(places(dim, rot)):
        slot = int(slots[n + 1])
        q[n + 1, 1, e] = want_q[n + 1, 1, e] = INF
        k[n + 1, 1, e] = want[slot // 16, 1, slot % 16, e] = -INF
    got_q = rotary.append_rotated(cache, slots, k, v, query=q, **args)
    assert torch.equal(got_q, want_q) and torch.equal(cache, want)


def test_a_batch_refuses_a_plan_of_other_lengths_and_writes_nothing(cuda):
    rand = lambda *s: torch.randn(*s, device=cuda).to(BF)  # noqa: E731
    pool = torch.zeros(30, 2, 16, 256, dtype=BF, device=cuda)
    batch = RotaryRagBatch(pool, 8, 200, 2, 64)
    batch.write_prefix(rand(200, 2, 128), rand(200, 2, 128))
    args = rand(4, 8, 128), rand(4, 2, 128), rand(4, 2, 128)
    before, other = pool.clone(), batch.plan([1, 3])  # the same sums
    with pytest.raises(ValueError, match="plan"):
        batch.step(*args, [3, 1], other)
    assert torch.equal(pool, before) and batch.lengths == [0, 0]
    got = batch.step(*args, [3, 1], batch.plan([3, 1]))
    batch.lengths = [0, 0]
    assert torch.equal(batch.step(*args, [3, 1]), got)
    batch.check()


@pytest.mark.parametrize("dim,dtype", [(128, BF), (80, HF)])
def test_append_in_a_graph(cuda, dim, dtype):
    """The append as it is captured in a decode step, replayed with new tokens."""
    args = args_of(cuda, 9, dim, dim // 2, False)
    q, k = rows(cuda, 9, 4, dim, dtype, 0, 1), rows(cuda, 9, 2, dim, dtype, 0, 2)
    v, w = rows(cuda, 9, 2, dim, dtype, 0, 3), torch.ones(dim, dtype=dtype, device=cuda)
    slots = torch.arange(9, device=cuda)
    cache = torch.zeros(4, 2, 16, 2 * dim, dtype=dtype, device=cuda)
    call = lambda pool: rotary.append_rotated(  # noqa: E731
        pool, slots, k, v, query=q, q_weight=w, k_weight=w, **args)
    call(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(cache)
    for x in (q, k, v):
        x.copy_(x.roll(1, 0))
    slots.copy_(torch.randperm(64, device=cuda)[:9])
    cache.zero_()
    graph.replay()
    other = torch.zeros_like(cache)
    assert torch.equal(out, call(other)) and torch.equal(cache, other) and other.any()
