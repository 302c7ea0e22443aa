"""The rotary operators together: a retrieval batch that writes its prefix,
prefills questions of several lengths and decodes, against float64 attention
over the normed, rotated keys (``oracle.rotary``, dense softmax).

Tolerance: keys and queries are rounded once after the rotation (u each, u the
unit roundoff of the type), so a score is off by at most 2 u S (S = sum |q k|
scale) and every weight by a factor exp(2 * 2 u S) at most; weights and the
output are rounded once more (u)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cacheslide_b200.rotary_rag import RotaryRagBatch
from oracle import rotary as orot

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-20}


@pytest.mark.parametrize("dtype,hq,hk,d,rot,inter", [
    (torch.bfloat16, 8, 2, 128, 128, False),
    (torch.float16, 16, 4, 64, 32, True),
    (torch.float32, 4, 2, 32, 32, False),
])
def test_questions_and_decode(cuda, dtype, hq, hk, d, rot, inter):
    g = torch.Generator(device=cuda).manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)  # noqa: E731
    prefix, lens, block = 333, [17, 1, 40], 16
    pool = torch.full((40, hk, block, 2 * d), float("nan"), dtype=dtype, device=cuda)
    qw, kw = 1 + 0.2 * rand(d), 1 + 0.2 * rand(d)
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(1)).tolist()
    batch = RotaryRagBatch(pool, hq, prefix, 3, 48, rotary_dim=rot, q_weight=qw, k_weight=kw,
                           interleaved=inter, block_ids=ids)
    pk, pv = rand(prefix, hk, d), rand(prefix, hk, d)
    batch.write_prefix(pk, pv)
    f = lambda x: x.double().cpu().numpy()  # noqa: E731
    cos, sin = f(batch.cos), f(batch.sin)
    keys, values = [[f(pk)] for _ in lens], [[f(pv)] for _ in lens]
    have = [0] * 3
    for counts in (lens, [1, 1, 1], [3, 0, 2], [1, 1, 1]):
        total = sum(counts)
        q, k, v = rand(total, hq, d), rand(total, hk, d), rand(total, hk, d)
        out = f(batch.step(q, k, v, counts))
        at = 0
        for b, n in enumerate(counts):
            keys[b].append(f(k[at:at + n]))
            values[b].append(f(v[at:at + n]))
            if n:
                pos = np.arange(prefix + have[b] + n)
                rk = orot.norm_rope(np.concatenate(keys[b]), f(kw), cos[pos], sin[pos],
                                    interleaved=inter).repeat(hq // hk, 1)
                new = pos[-n:]
                rq = orot.norm_rope(f(q[at:at + n]), f(qw), cos[new], sin[new], interleaved=inter)
                vv = np.concatenate(values[b]).repeat(hq // hk, 1)
                z = np.einsum("nhd,khd->nhk", rq, rk) / math.sqrt(d)
                size = (np.einsum("nhd,khd->nhk", abs(rq), abs(rk)) / math.sqrt(d)).max(-1)
                z[np.broadcast_to((pos > new[:, None])[:, None], z.shape)] = -np.inf
                p = np.exp(z - z.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                want = np.einsum("nhk,khd->nhd", p, vv)
                u = U[dtype]
                rel = np.expm1(4 * u * size)[..., None] + u
                bound = u * abs(want) + rel * np.einsum("nhk,khd->nhd", p, abs(vv)) + 2.0**-14 * u
                assert (abs(out[at:at + n] - want) <= bound).all()
            have[b] += n
            at += n
    batch.check()
    assert batch.lengths == [22, 3, 44]
    with pytest.raises(ValueError):
        batch.plan([5, 1, 5])  # past the third request's blocks
    with pytest.raises(ValueError):
        RotaryRagBatch(pool, hq, prefix, 3, 400)
    with pytest.raises(ValueError):
        RotaryRagBatch(pool, hq, prefix, 3, 48, block_ids=ids[:20])


def test_one_plan_for_all_layers(cuda):
    """Layers of one step share the plan; a layer's result does not depend on
    the others'."""
    rand = lambda *s: torch.randn(*s, device=cuda).bfloat16()  # noqa: E731
    layers = []
    for _ in range(3):
        batch = RotaryRagBatch(torch.zeros(30, 2, 16, 256, dtype=torch.bfloat16, device=cuda), 8,
                               200, 4, 64)
        batch.write_prefix(rand(200, 2, 128), rand(200, 2, 128))
        layers.append((batch, rand(20, 8, 128), rand(20, 2, 128), rand(20, 2, 128)))
    plan = layers[0][0].plan([5] * 4)
    shared = [b.step(q, k, v, [5] * 4, plan) for b, q, k, v in layers]
    for (b, q, k, v), got in zip(layers, shared):
        b.lengths = [0] * 4  # the same step again, with a plan of its own
        assert torch.equal(b.step(q, k, v, [5] * 4), got)
        b.check()
