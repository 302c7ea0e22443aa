"""The restatement of the 4-bit pool: the codes' float32 difference, and the bounds
that the attention is held to (the stated roundings, done in float64, stay inside,
and mistakes do not)."""

from __future__ import annotations

import math

import pytest
import torch

from cacheslide_b200 import kv4
from oracle import kv4 as okv4

CASES = [(torch.bfloat16, 128, 64), (torch.float16, 128, 128), (torch.float16, 64, 32)]


def _case(dtype, dim, group, n, length=600, hq=8, hk=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    blocks = -(-length // 16)

    def rows():
        x = torch.randn(16 * blocks, hk, dim, generator=g)
        x[..., 3] *= 9
        return x.to(dtype)

    storage = torch.zeros(blocks, hk, 1, kv4.unit_bytes(dim, group), dtype=torch.uint8)
    okv4.write(storage, torch.arange(16 * blocks), rows(), rows(), group)
    q = (1.5 * torch.randn(n, hq, dim, generator=g)).to(dtype)
    return q, storage, torch.randperm(blocks, generator=g).int()


def _kernel(q, storage, table, length, group, scale, wide, *, shift=0, drop=None, parts=2):
    """The roundings of the kernel: its operands, and weights in fp16 below a
    maximum that is taken up 64 keys at a time when it grew by 2^8 (wide), or by
    2^14 after a rise of 2^6 (with the scales in it).  `shift`: the mask is off by so
    many keys; `drop`: a unit that is left out; `parts` 1: float16 operands of one
    part."""
    n, hq, d = q.shape
    at = torch.arange(length)
    slots = table[at // 16].long() * 16 + at % 16
    (kc, ks, kz), (vc, vs, vz) = okv4._parts(storage, slots, d, group, q.dtype)
    hk = kc.shape[1]
    kind = torch.bfloat16 if parts == 1 else q.dtype
    k, v = (okv4.operands(c, s, z, kind) if wide else z + s * c
            for c, s, z in ((kc, ks, kz), (vc, vs, vz)))
    z = torch.einsum("nhgd,khd->nhgk", q.double().view(n, hk, -1, d), k) * scale * math.log2(math.e)
    seen = at <= (length - n + shift + torch.arange(n))[:, None]
    if drop is not None:
        seen = seen & (at // 16 != drop)
    z = torch.where(seen[:, None, None], z, -math.inf)
    ref = torch.full(z.shape[:3], -math.inf, dtype=torch.float64)
    o, total = 0.0, 0.0
    for lo in range(0, length, 64):
        part = z[..., lo:lo + 64]
        size = torch.zeros(part.shape[-1], hk, dtype=torch.float64) if wide else \
            vs[lo:lo + 64].amax(-1).log2()
        top = (part + size.t()[None, :, None]).amax(-1)
        new = torch.where(top > ref + (8 if wide else 14), top, ref)
        down = torch.where(ref == new, 1.0, (ref - new).exp2()).nan_to_num(0.0)
        ref = new
        p = (part - torch.where(ref == -math.inf, 0.0, ref)[..., None] + (7 if wide else 6)).exp2()
        total = total * down + p.sum(-1)
        if wide:
            here = torch.einsum("nhgk,khd->nhgd", p.half().double(), v[lo:lo + 64])
        else:
            c, s, m = vc[lo:lo + 64] - 8, vs[lo:lo + 64], vz[lo:lo + 64] + 8 * vs[lo:lo + 64]
            w = (p.permute(0, 3, 1, 2)[..., None] * s[None, :, :, None]).half().double()
            here = (w * c[None, :, :, None]).sum(1) + torch.einsum("nhgk,khd->nhgd", p, m)
        o = o * down[..., None] + here
    some = total != 0
    out = torch.where(some[..., None], o / torch.where(some, total, 1.0)[..., None], 0.0)
    total = torch.where(some, total, 1.0)
    lse = torch.where(some, ref - (7 if wide else 6) + total.log2(), -math.inf)
    return out.reshape(n, hq, d).to(q.dtype), lse.reshape(n, hq) * math.log(2)


def _inside(got, lse, b, dtype):
    eps = torch.finfo(dtype).eps / 2
    bound = b.err + eps * (b.out.abs() + b.err) + torch.finfo(dtype).smallest_normal * eps
    square = (b.var + (okv4.ROUNDING * eps * b.out) ** 2).sum()
    return (((got.double() - b.out).abs() <= bound).all(),
            ((lse - b.lse).abs() <= b.lse_err)[b.lse != -math.inf].all(),
            math.sqrt(((got.double() - b.out) ** 2).sum() / square))


@pytest.mark.parametrize("dtype,dim,group", CASES)
@pytest.mark.parametrize("wide,n", [(True, 129), (False, 4)])
def test_the_stated_roundings_are_inside_and_mistakes_are_not(dtype, dim, group, wide, n):
    q, storage, table = _case(dtype, dim, group, n)
    args = q, storage, table, 600
    b = okv4.bounds(*args, n, group, dim ** -0.5, wide)
    run = [_inside(*_kernel(*args, group, dim ** -0.5, wide, **kw), b, dtype)
           for kw in ({}, dict(shift=1), dict(shift=-1), dict(drop=11),
                      *([dict(parts=1)] if wide and dtype == torch.float16 else []))]
    (o, l, ratio), mistakes = run[0], run[1:]
    # (a weight at its reference is a power of two, which no rounding changes: the
    # squares may be less)
    assert o and l and ratio < 1.1
    for o, l, ratio in mistakes[:3]:
        assert not o and not l
    for o, l, ratio in mistakes[3:]:
        assert ratio > 1.15


def test_codes_go_by_the_difference_in_float32():
    """2^-24 + 832 is 832 in float32, six and a half scales of 128."""
    x = torch.zeros(1, 32, dtype=torch.float16)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = -832.0, 1088.0, 2.0 ** -24, 1.0
    scale, low = okv4.params(x, 32)
    assert scale.item() == 128 and low.item() == -832
    assert okv4.codes(x, scale, low, 32)[0, :4].tolist() == [0, 15, 6, 7]


def test_codes_of_the_widest_groups():
    """Differences past float32's largest number, and far below its smallest scale."""
    big = torch.finfo(torch.bfloat16).max
    for unit in (big, 1e-37):
        x = (torch.linspace(-1, 1, 32) * unit).bfloat16()[None]
        scale, low = okv4.params(x, 32)
        got = okv4.codes(x, scale, low, 32)[0].double()
        exact = (x[0].double() - low.double()) / scale.double()
        assert ((got - exact).abs() <= 0.5 + (exact - 15).clamp(min=0)).all()


def test_a_scale_whose_last_value_would_round_to_infinity():
    """low + 15 scale exactly half a step past the largest number: the scale below."""
    x = torch.zeros(1, 32, dtype=torch.bfloat16)
    x[0, 0] = -6.911985578081563e37
    x[0, 1] = torch.finfo(torch.bfloat16).max
    scale, low = okv4.params(x, 32)
    assert torch.isfinite((low.double() + 15 * scale.double()).to(torch.bfloat16)).all()
