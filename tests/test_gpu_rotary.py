"""Head norms with rotation, their gradient and the rotated append, against
float64 (``oracle.rotary``).

Tolerances.  The kernels compute in float32 and round once: an output is off
by at most u * |y| for the rounding (u = half the spacing of 1 + x: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and
by a few float32 units of the row's largest term for the arithmetic (a sum of
squares of up to 512 terms in 16 partial sums of 32 lanes, one reciprocal square root of two
units, four products, one sum: 32 units of 2^-24 bounds it).  The gradient has
two sums over the row: 64 units of its largest term.  dw adds one term a row:
units of 2^-24 of the sum of the terms' sizes, as many as the longest chain of
additions (rows a thread adds, then at most 64 for the joins)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import rotary
from cacheslide_b200.paged import NativePagedKV
from oracle import rotary as orot

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}  # subnormal halves
F32 = 2.0**-24


def f64(x):
    return None if x is None else x.detach().double().cpu().numpy()


def inputs(device, tokens, hq, hk, dim, rot, dtype, seed=0, table=None, wdtype=None):
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    table = table or max(4096, tokens)
    cos, sin = rotary.rotary_tables(table, max(rot, 2), device=device)
    cos, sin = cos[:, :rot // 2], sin[:, :rot // 2]
    wdtype = wdtype or dtype
    return dict(
        query=(1.5 * rand(tokens, hq, dim)).to(dtype), key=(1.5 * rand(tokens, hk, dim)).to(dtype),
        positions=torch.randint(0, table, (tokens,), generator=g, device=device), cos=cos, sin=sin,
        q_weight=(1 + 0.3 * rand(dim)).to(wdtype), k_weight=(1 + 0.3 * rand(dim)).to(wdtype))


def rows_of(s):
    p = s["positions"].cpu().numpy()
    return f64(s["cos"])[p], f64(s["sin"])[p]


def check_rows(got, x, w, cos, sin, interleaved, dtype, eps=1e-6):
    want = orot.norm_rope(f64(x), f64(w), cos, sin, eps, interleaved)
    size = np.abs(want).max(-1, keepdims=True) if want.size else want
    bound = U[dtype] * np.abs(want) + 32 * F32 * size + TINY[dtype]
    assert (np.abs(f64(got) - want) <= bound).all()


SHAPES = [  # tokens, q heads, kv heads, dim, rotated, interleaved, dtype
    (1, 32, 8, 128, 128, False, torch.bfloat16),
    (1, 1, 1, 2, 2, False, torch.float32),
    (7, 4, 2, 16, 16, False, torch.float32),
    (33, 64, 8, 64, 64, True, torch.float16),
    (257, 32, 8, 128, 64, False, torch.float16),
    (64, 5, 3, 80, 40, True, torch.bfloat16),
    (50, 6, 3, 96, 96, False, torch.bfloat16),
    (19, 3, 1, 100, 6, False, torch.float32),
    (40, 8, 2, 256, 256, True, torch.bfloat16),
    (21, 2, 2, 512, 512, False, torch.float32),
    (21, 2, 2, 512, 256, False, torch.float16),
    (12, 4, 4, 64, 0, False, torch.bfloat16),
    (1025, 8, 1, 128, 128, False, torch.float32),
    (300, 16, 4, 32, 32, True, torch.bfloat16),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,inter,dtype", SHAPES)
def test_forward(cuda, tokens, hq, hk, dim, rot, inter, dtype):
    s = inputs(cuda, tokens, hq, hk, dim, rot, dtype)
    q, k = rotary.qk_norm_rope(**s, interleaved=inter)
    cos, sin = rows_of(s)
    check_rows(q, s["query"], s["q_weight"], cos, sin, inter, dtype)
    check_rows(k, s["key"], s["k_weight"], cos, sin, inter, dtype)


@pytest.mark.parametrize("which", ["neither", "query", "key"])
def test_forward_with_some_norms(cuda, which):
    s = inputs(cuda, 77, 8, 2, 128, 128, torch.bfloat16)
    if which != "query":
        s["q_weight"] = None
    if which != "key":
        s["k_weight"] = None
    q, k = rotary.qk_norm_rope(**s)
    cos, sin = rows_of(s)
    check_rows(q, s["query"], s["q_weight"], cos, sin, False, torch.bfloat16)
    check_rows(k, s["key"], s["k_weight"], cos, sin, False, torch.bfloat16)


def test_zero_rows_huge_rows_and_infinities(cuda):
    s = inputs(cuda, 6, 4, 2, 64, 64, torch.float16)
    s["query"][1] = 0
    s["query"][2] = 60000.0  # its squares pass fp16, not float32
    s["query"][3, 1, 5] = float("inf")
    s["key"][4, 0, 0] = float("nan")
    q, k = rotary.qk_norm_rope(**s)
    cos, sin = rows_of(s)
    assert not q[1].any()
    clean = [0, 1, 2, 4, 5]
    check_rows(q[clean], s["query"][clean], s["q_weight"], cos[clean], sin[clean], False,
               torch.float16)
    assert torch.isnan(k[4, 0]).all() and torch.isfinite(k[4, 1]).all()
    assert torch.isfinite(q[3, 0]).all() and not torch.isfinite(q[3, 1]).all()


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float32)])
def test_strided_views_of_one_projection(cuda, dim, dtype):
    """q, k and v as slices of one projection output: other strides, an odd
    row pitch in elements, and a start that no vector load may use."""
    g = torch.Generator(device=cuda).manual_seed(1)
    s = inputs(cuda, 45, 4, 2, dim, dim, dtype)
    for pad, off in ((0, 0), (8, 8), (3, 1)):
        wide = torch.randn(45, 8 * dim + pad, generator=g, device=cuda).to(dtype)
        q = wide[:, off:off + 4 * dim].unflatten(1, (4, dim))
        k = wide[:, off + 4 * dim - (off and 1):][:, :2 * dim].unflatten(1, (2, dim))
        out = rotary.qk_norm_rope(**{**s, "query": q, "key": k})
        cos, sin = rows_of(s)
        check_rows(out[0], q, s["q_weight"], cos, sin, False, dtype)
        check_rows(out[1], k, s["k_weight"], cos, sin, False, dtype)
    t = torch.randn(4, 45, dim, generator=g, device=cuda).to(dtype).transpose(0, 1)  # head-major
    out = rotary.qk_norm_rope(**{**s, "query": t})
    check_rows(out[0], t, s["q_weight"], cos, sin, False, dtype)
    n = torch.randn(45, dim, 4, generator=g, device=cuda).to(dtype).transpose(1, 2)  # dim-strided
    out = rotary.qk_norm_rope(**{**s, "query": n})
    check_rows(out[0], n, s["q_weight"], cos, sin, False, dtype)


def test_no_tokens(cuda):
    s = inputs(cuda, 0, 4, 2, 64, 64, torch.bfloat16)
    s["query"].requires_grad_(True)
    s["q_weight"].requires_grad_(True)
    q, k = rotary.qk_norm_rope(**s)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    dq, dw = torch.autograd.grad(q.sum(), (s["query"], s["q_weight"]))
    assert dq.shape == (0, 4, 64) and not dw.any()


def test_positions_outside_the_table(cuda):
    s = inputs(cuda, 4, 2, 1, 32, 16, torch.float32)
    s["positions"][1], s["positions"][2] = -1, 4096
    status = N.Status(cuda)
    q, _ = rotary.qk_norm_rope(**s, status=status)
    assert status.read() == N.ST_POS_RANGE
    assert torch.isnan(q[1:3, :, :16]).all() and torch.isfinite(q[1:3, :, 16:]).all()
    assert torch.isfinite(q[[0, 3]]).all()


def test_weights_of_another_type(cuda):
    s = inputs(cuda, 31, 4, 2, 128, 128, torch.bfloat16, wdtype=torch.float32)
    q, _ = rotary.qk_norm_rope(**s)
    cos, sin = rows_of(s)
    check_rows(q, s["query"], s["q_weight"], cos, sin, False, torch.bfloat16)


def test_on_another_stream(cuda):
    s = inputs(cuda, 2000, 32, 8, 128, 128, torch.bfloat16)
    want = rotary.qk_norm_rope(**s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        query = s["query"] * 1  # written on this stream, read by the launch behind it
        got = rotary.qk_norm_rope(**{**s, "query": query})
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def grads(s, gq, gk, **kw):
    leaves = [s[n].detach().requires_grad_(True) if s[n] is not None else None
              for n in ("query", "key", "q_weight", "k_weight")]
    q, k = rotary.qk_norm_rope(leaves[0], leaves[1], s["positions"], s["cos"], s["sin"],
                               leaves[2], leaves[3], **kw)
    some = [x for x in leaves if x is not None]
    out = iter(torch.autograd.grad((q, k), some, (gq, gk)))
    return [next(out) if x is not None else None for x in leaves]


def check_grad(dx, dw, x, w, dy, cos, sin, inter, dtype, wdtype):
    want, wantw = orot.norm_rope_grad(f64(x), f64(w), f64(dy), cos, sin, 1e-6, inter)
    g = np.abs(orot.rotation(f64(dy), cos, -sin, inter))
    x64 = f64(x)
    if w is None:
        size = g.max(-1, keepdims=True) * np.ones_like(want)
    else:
        r = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-6)
        n, wg = np.abs(x64) * r, np.abs(f64(w)) * g
        size = r * (wg.max(-1, keepdims=True) + n * (wg * n).mean(-1, keepdims=True))
    # g itself is a difference of two products of the size of dy
    pair = 2 * np.abs(f64(dy)).max(-1, keepdims=True) * (1 if w is None else r)
    bound = U[dtype] * np.abs(want) + 64 * F32 * (size + pair) + TINY[dtype]
    assert (np.abs(f64(dx) - want) <= bound).all()
    if w is not None:
        rows = x.shape[0] * x.shape[1]
        terms = (np.abs(f64(dy)).max(-1, keepdims=True) * 2 * n).sum((0, 1))
        bound = U[wdtype] * np.abs(wantw) + (rows / 4736 + 64) * F32 * terms
        assert (np.abs(f64(dw) - wantw) <= bound).all()


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,inter,dtype", SHAPES)
def test_gradient(cuda, tokens, hq, hk, dim, rot, inter, dtype):
    s = inputs(cuda, tokens, hq, hk, dim, rot, dtype, seed=3)
    g = torch.Generator(device=cuda).manual_seed(9)
    gq = torch.randn(tokens, hq, dim, generator=g, device=cuda).to(dtype)
    gk = torch.randn(tokens, hk, dim, generator=g, device=cuda).to(dtype)
    dq, dk, dqw, dkw = grads(s, gq, gk, interleaved=inter)
    cos, sin = rows_of(s)
    check_grad(dq, dqw, s["query"], s["q_weight"], gq, cos, sin, inter, dtype, dtype)
    check_grad(dk, dkw, s["key"], s["k_weight"], gk, cos, sin, inter, dtype, dtype)


def test_gradient_without_norms_and_with_strided_inputs(cuda):
    s = inputs(cuda, 45, 4, 2, 64, 64, torch.float32)
    g = torch.Generator(device=cuda).manual_seed(2)
    s["query"] = torch.randn(45, 5 * 64 + 1, generator=g, device=cuda)[:, 1:257].unflatten(1, (4, 64))
    s["k_weight"] = None
    gq = torch.randn(4, 45, 64, generator=g, device=cuda).transpose(0, 1)
    gk = torch.randn(45, 2, 64, generator=g, device=cuda)
    dq, dk, dqw, dkw = grads(s, gq, gk)
    cos, sin = rows_of(s)
    assert dkw is None
    check_grad(dq, dqw, s["query"], s["q_weight"], gq, cos, sin, False, torch.float32,
               torch.float32)
    check_grad(dk, None, s["key"], None, gk, cos, sin, False, torch.float32, torch.float32)


def test_gradient_is_the_same_bit_for_bit(cuda):
    s = inputs(cuda, 3001, 8, 2, 128, 128, torch.bfloat16)
    gq, gk = torch.randn_like(s["query"]), torch.randn_like(s["key"])
    a, b = grads(s, gq, gk), grads(s, gq, gk)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_against_differences(cuda):
    """float32 forwards at x +- h v: truncation h^2 |f'''| / 6 and rounding
    2^-24 |y| sqrt(values) / h, each below 1e-3 of the directional derivative."""
    s = inputs(cuda, 40, 4, 2, 32, 32, torch.float32)
    g = torch.Generator(device=cuda).manual_seed(4)
    gq, gk = (torch.randn(x.shape, generator=g, device=cuda) for x in (s["query"], s["key"]))
    d = dict(zip(("query", "key", "q_weight", "k_weight"), grads(s, gq, gk)))

    def loss(at):
        q, k = rotary.qk_norm_rope(**at)
        return ((q.double() * gq).sum() + (k.double() * gk).sum()).item()

    h = 2.0**-7
    for name, grad in d.items():
        v = grad / grad.abs().max()  # along the gradient: no cancellation
        slope = (loss({**s, name: s[name] + h * v}) - loss({**s, name: s[name] - h * v})) / (2 * h)
        want = (grad.double() * v).sum().item()
        assert abs(slope - want) < 2e-3 * want, name


# ------------------------------------------------------------------- append
def pool(device, blocks, hk, bs, dim, dtype):
    return torch.full((blocks, hk, bs, 2 * dim), 7.0, dtype=dtype, device=device)


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,inter,dtype", SHAPES)
@pytest.mark.parametrize("block", [16, 5])
def test_append(cuda, tokens, hq, hk, dim, rot, inter, dtype, block):
    s = inputs(cuda, tokens, hq, hk, dim, rot, dtype, seed=7)
    value = torch.randn(tokens, hk, dim, device=cuda).to(dtype)
    blocks = tokens // block + 3
    cache = pool(cuda, blocks, hk, block, dim, dtype)
    slots = torch.randperm(blocks * block, device=cuda)[:tokens].contiguous()
    status = N.Status(cuda)
    args = dict(positions=s["positions"], cos=s["cos"], sin=s["sin"], interleaved=inter)
    q = rotary.append_rotated(cache, slots, s["key"], value, query=s["query"],
                              q_weight=s["q_weight"], k_weight=s["k_weight"], status=status,
                              **args)
    assert status.read() == 0
    # the dense operator's rows, and nothing else of the pool touched
    want_q, want_k = rotary.qk_norm_rope(s["query"], s["key"], q_weight=s["q_weight"],
                                         k_weight=s["k_weight"], **args)
    assert torch.equal(q, want_q)
    want = pool(cuda, blocks, hk, block, dim, dtype)
    want[slots // block, :, slots % block] = torch.cat((want_k, value), -1)
    assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_without_queries_or_norms_padded_and_in_place(cuda, dtype):
    s = inputs(cuda, 9, 4, 2, 64, 64, dtype)
    args = dict(positions=s["positions"], cos=s["cos"], sin=s["sin"])
    value = torch.randn(9, 2, 64, device=cuda).to(dtype)
    want_q, want_k = rotary.qk_norm_rope(s["query"], s["key"], **args)
    cache = pool(cuda, 2, 2, 16, 64, dtype)
    slots = torch.tensor([0, -1, 31, 5, 32, -2, 1 << 40, 6, 7], device=cuda)
    status = N.Status(cuda)
    assert rotary.append_rotated(cache, slots, s["key"], value, status=status, **args) is None
    assert status.read() == N.ST_SLOT_RANGE
    want = pool(cuda, 2, 2, 16, 64, dtype)
    for t in (0, 2, 3, 7, 8):
        slot = int(slots[t])
        want[slot // 16, :, slot % 16] = torch.cat((want_k, value), -1)[t]
    assert torch.equal(cache, want)
    # padding alone sets no bit; the queries may be rotated in place
    status = N.Status(cuda)
    query = s["query"].clone()
    out = rotary.append_rotated(cache, torch.full((9,), -1, device=cuda), s["key"], value,
                                query=query, out=query, status=status, **args)
    assert status.read() == 0 and out is query and torch.equal(query, want_q)
    assert torch.equal(cache, want)


def test_append_skips_positions_outside_the_table(cuda):
    s = inputs(cuda, 3, 2, 1, 32, 32, torch.float16)
    s["positions"][1] = 4096
    cache, status = pool(cuda, 1, 1, 16, 32, torch.float16), N.Status(cuda)
    rotary.append_rotated(cache, torch.tensor([0, 1, 2], device=cuda), s["key"], s["key"],
                          s["positions"], s["cos"], s["sin"], status=status)
    assert status.read() == N.ST_POS_RANGE
    assert (cache[0, 0, 1] == 7).all() and not (cache[0, 0, [0, 2]] == 7).all()


def test_append_to_strided_pools(cuda):
    """The pool as [block, offset, head, 2 * dim] memory, and as one whose
    innermost stride is 2."""
    s = inputs(cuda, 20, 4, 2, 64, 64, torch.bfloat16)
    value = torch.randn(20, 2, 64, device=cuda).bfloat16()
    slots = torch.randperm(48, device=cuda)[:20].contiguous()
    args = (slots, s["key"], value, s["positions"], s["cos"], s["sin"])
    want = pool(cuda, 3, 2, 16, 64, torch.bfloat16)
    rotary.append_rotated(want, *args)
    major = torch.full((3, 16, 2, 128), 7.0, dtype=torch.bfloat16, device=cuda).transpose(1, 2)
    rotary.append_rotated(major, *args)
    assert torch.equal(major, want)
    wide = torch.full((3, 2, 16, 256), 7.0, dtype=torch.bfloat16, device=cuda)
    rotary.append_rotated(wide[..., ::2], *args)
    assert torch.equal(wide[..., ::2], want) and (wide[..., 1::2] == 7).all()


def test_append_past_32_bit_offsets(cuda):
    blocks = 70_000  # 64 KB a block: 4.6 GB
    cache = torch.zeros(blocks, 8, 16, 256, dtype=torch.bfloat16, device=cuda)
    s = inputs(cuda, 5, 8, 8, 128, 128, torch.bfloat16)
    slots = torch.tensor([0, 17, 40_000 * 16 + 3, 69_999 * 16, 69_999 * 16 + 15], device=cuda)
    rotary.append_rotated(cache, slots, s["key"], s["query"], s["positions"], s["cos"], s["sin"])
    _, want = rotary.qk_norm_rope(s["query"], s["key"], s["positions"], s["cos"], s["sin"])
    got = cache[slots // 16, :, slots % 16]
    assert torch.equal(got, torch.cat((want, s["query"]), -1))
    assert int((cache != 0).any(-1).any(1).sum()) == 5


def test_append_to_an_arena_and_its_sidecar(cuda):
    cache = torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16, device=cuda)
    arena = NativePagedKV(cache, [0, 1], 20, 4)
    s = inputs(cuda, 3, 4, 2, 64, 64, torch.bfloat16)
    with pytest.raises(ValueError):
        rotary.append_rotated(arena, torch.zeros(3, dtype=torch.int64, device=cuda),
                              s["query"], s["query"], s["positions"], s["cos"], s["sin"])
    arena.write_prefill(*(torch.randn(20, 2, 64, device=cuda).bfloat16() for _ in range(2)))
    arena.promote_selected([3], *(torch.randn(1, 2, 64, device=cuda).bfloat16()
                                  for _ in range(2))).result()
    slots = torch.cat((arena.slot_table([3]), torch.tensor([20, 21], device=cuda)))
    assert int(slots[0]) >= 64
    rotary.append_rotated(arena, slots, s["key"], s["key"], s["positions"], s["cos"], s["sin"])
    _, want = rotary.qk_norm_rope(s["query"], s["key"], s["positions"], s["cos"], s["sin"])
    key, value = arena.gather([3])
    assert torch.equal(key[0], want[0]) and torch.equal(value[0], s["key"][0])
    assert torch.equal(cache[1, :, 4:6, :64].transpose(0, 1), want[1:])


def test_append_refuses(cuda):
    s = inputs(cuda, 3, 4, 2, 64, 64, torch.bfloat16)
    cache = pool(cuda, 2, 2, 16, 64, torch.bfloat16)
    slots = torch.arange(3, device=cuda)
    good = dict(kv=cache, slots=slots, key=s["key"], value=s["key"], positions=s["positions"],
                cos=s["cos"], sin=s["sin"], query=s["query"])
    for change in (dict(kv=cache.float()), dict(kv=cache[:, :1]), dict(kv=cache[..., :64]),
                   dict(slots=slots.int()), dict(slots=slots[:2]), dict(slots=slots.cpu()),
                   dict(value=s["key"].float()), dict(value=s["key"][:2]),
                   dict(query=s["query"][:2]), dict(out=torch.empty_like(s["key"])),
                   dict(query=None, out=s["query"]), dict(query=None, q_weight=s["q_weight"]),
                   dict(positions=s["positions"].cpu()), dict(cos=s["cos"].cpu())):
        with pytest.raises(ValueError):
            rotary.append_rotated(**{**good, **change})
