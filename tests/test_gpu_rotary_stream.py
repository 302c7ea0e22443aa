"""The gradient of the norm and rotation over many tokens, against float64: each
warp of the streamed kernel takes tens of tokens of one to five row groups, so
that its rings of rows and angles turn over many times (tolerances as in
``test_gpu_rotary``)."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import rotary
from test_gpu_rotary import check_grad, grads, inputs, rows_of

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
# tokens, q heads, kv heads, dim, rotated, interleaved, dtype; heads that leave
# the last row group of a token partly empty, one token short of an even share
CASES = [
    (20000, 8, 2, 64, 64, False, BF), (20000, 8, 2, 64, 32, True, HF),
    (9999, 20, 3, 64, 32, False, HF), (9999, 20, 3, 64, 64, True, BF),
    (7001, 33, 5, 128, 128, False, BF), (7001, 12, 4, 128, 64, True, BF),
    (7001, 6, 3, 256, 128, False, HF), (9999, 10, 3, 64, 64, False, FP),
    (5003, 9, 2, 128, 64, True, FP), (30011, 24, 9, 16, 16, False, BF),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,inter,dtype", CASES)
def test_gradient_of_many_tokens(cuda, tokens, hq, hk, dim, rot, inter, dtype):
    s = inputs(cuda, tokens, hq, hk, dim, rot, dtype, seed=11)
    g = torch.Generator(device=cuda).manual_seed(12)
    gq = torch.randn(tokens, hq, dim, generator=g, device=cuda).to(dtype)
    gk = torch.randn(tokens, hk, dim, generator=g, device=cuda).to(dtype)
    dq, dk, dqw, dkw = grads(s, gq, gk, interleaved=inter)
    cos, sin = rows_of(s)
    check_grad(dq, dqw, s["query"], s["q_weight"], gq, cos, sin, inter, dtype, dtype)
    check_grad(dk, dkw, s["key"], s["k_weight"], gk, cos, sin, inter, dtype, dtype)


@pytest.mark.parametrize("dim,rot,inter,dtype", [(64, 32, False, BF), (64, 64, True, HF),
                                                 (128, 64, False, FP), (80, 40, False, BF)])
def test_gradient_of_positions_outside_the_table(cuda, dim, rot, inter, dtype):
    """Their rows are NaN where they turn, no other row is touched, and the
    status says so (the last heads on the one-warp-a-row kernel)."""
    tokens = 9001
    s = inputs(cuda, tokens, 12, 3, dim, rot, dtype, seed=13, table=4096)
    s["q_weight"] = s["k_weight"] = None
    gq, gk = torch.randn_like(s["query"]), torch.randn_like(s["key"])
    want = grads(s, gq, gk, interleaved=inter)
    bad = torch.zeros(tokens, dtype=torch.bool, device=cuda)
    bad[[0, 1, 17, 2368, 4000, 4001, 8999, 9000]] = True
    s["positions"][bad] = torch.tensor([-1, 4096, 1 << 40, -7, 4096, 5000, -1, 4097], device=cuda)
    status = N.Status(cuda)
    leaves = [x.detach().requires_grad_(True) for x in (s["query"], s["key"])]
    out = rotary.qk_norm_rope(*leaves, s["positions"], s["cos"], s["sin"], interleaved=inter,
                              status=status)
    assert status.read() == N.ST_POS_RANGE
    status.word.zero_()
    got = torch.autograd.grad(out, leaves, (gq, gk))
    assert status.read() == N.ST_POS_RANGE
    for x, y in zip(got, want):
        assert torch.equal(x[~bad], y[~bad])
        assert torch.isnan(x[bad][..., :rot]).all()
        assert torch.equal(x[bad][..., rot:], y[bad][..., rot:])


def test_gradient_of_weights_in_many_types(cuda):
    s = inputs(cuda, 6007, 12, 3, 64, 64, BF, seed=14, wdtype=FP)
    gq, gk = torch.randn_like(s["query"]), torch.randn_like(s["key"])
    dq, dk, dqw, dkw = grads(s, gq, gk)
    cos, sin = rows_of(s)
    assert dqw.dtype is FP and dkw.dtype is FP
    check_grad(dq, dqw, s["query"], s["q_weight"], gq, cos, sin, False, BF, FP)
    check_grad(dk, dkw, s["key"], s["k_weight"], gk, cos, sin, False, BF, FP)
