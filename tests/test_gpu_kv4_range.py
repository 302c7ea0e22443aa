"""Attention over the 4-bit pool with values of all sizes that its records can
hold: constants, the ends of the types, sizes far apart in one context."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4
from oracle import kv4 as okv4
from test_gpu_kv4 import FORMS, _check, _pool, _rows, _wide

pytestmark = pytest.mark.gpu


def _filled(cuda, seed, new, lengths, hq, hk, dim, group, dtype, values, keys=None):
    """A pool in order, `values` [slot, head, dim] (or a number for all), random
    keys (or `keys`), and queries."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // 16) for n in lengths]
    blocks, width = sum(per), max(per)
    table, at = torch.full((len(new), width), -3, dtype=torch.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    pool = _pool(cuda, blocks, hk, 16, dim, group, dtype)
    n = 16 * blocks
    k = _rows(seed, n, hk, dim, dtype) if keys is None else keys
    v = values if isinstance(values, torch.Tensor) else torch.full((n, hk, dim), values)
    kv4.append(pool, torch.arange(n, device=cuda), k.to(cuda), v.to(dtype).to(cuda))
    q = (0.5 * torch.randn(sum(new), hq, dim, generator=g)).to(dtype)
    return pool, table, q, torch.tensor([0, *new]).cumsum(0).int()


def _attend(cuda, pool, table, q, starts, lengths, scale=None):
    status = N.Status(cuda)
    got = kv4.attention(q.to(cuda), pool, table.to(cuda),
                        torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda),
                        scale=scale, return_lse=True, status=status)
    assert status.read() == 0
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_by_differences_that_float32_rounds(cuda, dtype):
    """Lowest values and elements far apart, at and beside the half ways."""
    x = torch.zeros(60, 1, 64)
    for i in range(60):
        low = -832.0 * 2 ** (i % 5) if i % 2 else -13.0 * 2 ** (i % 7)
        scale = -low * 2 / 13
        x[i, 0, 0], x[i, 0, 1] = low, low + 15 * scale
        x[i, 0, 2:34] = 2.0 ** -torch.arange(32) * (-1) ** (i // 3)
        x[i, 0, 34:48] = low + scale * (torch.arange(14) + 0.5)
    x = x.to(dtype)
    slots = torch.arange(60)
    pool = _pool(cuda, 4, 1, 16, 64, 64, dtype)
    want = pool.storage.cpu()
    okv4.write(want, slots, x, x.flip(0), 64)
    kv4.append(pool, slots.to(cuda), x.to(cuda), x.flip(0).to(cuda))
    assert torch.equal(pool.storage.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group", FORMS)
def test_records_of_any_bits(cuda, dtype, dim, group):
    """Numbers of all patterns: within a few powers of two, to the types' ends, and
    with infinities and NaN among them (a group of one is NaN, whichever)."""
    g = torch.Generator().manual_seed(dim + group)
    top = 0x7C00 if dtype == torch.float16 else 0x7F80
    first = torch.randint(0, top, (400, 1, 1), generator=g)
    size = 2 ** torch.randint(0, 15, (400, 1, 1), generator=g)
    bits = first + torch.randint(0, 1 << 15, (400, 2, dim), generator=g) % size
    bits = bits.clamp(max=top - 1) | torch.randint(0, 2, bits.shape, generator=g) << 15
    bits[:40] = torch.randint(0, 1 << 16, (40, 2, dim), generator=g)
    x = bits.to(torch.int32).to(torch.int16).view(dtype)
    slots = torch.arange(400)
    pool = _pool(cuda, 25, 2, 16, dim, group, dtype)
    want = pool.storage.cpu()
    okv4.write(want, slots, x, x.flip(0), group)
    kv4.append(pool, slots.to(cuda), x.to(cuda), x.flip(0).to(cuda))
    for a, b in zip(*(okv4.read(s, slots, dim, group, dtype) for s in (pool.storage.cpu(), want))):
        assert ((a == b) | a.isnan() & b.isnan()).all()


CONSTANTS = [(torch.float16, 60000.0), (torch.float16, -1000.0), (torch.float16, 6e-8),
             (torch.bfloat16, 1e7), (torch.bfloat16, 2.0 ** 22), (torch.bfloat16, -3e38),
             (torch.bfloat16, 1e-38), (torch.bfloat16, 1.0), (torch.float16, 0.0)]


@pytest.mark.parametrize("dtype,value", CONSTANTS)
@pytest.mark.parametrize("dim,group", [(128, 32), (64, 64)])
@pytest.mark.parametrize("new", [1, 3])
def test_constant_values_come_back(cuda, dtype, value, dim, group, new):
    """Every group of every value is one number, whose scale is 0: any weights
    give that number, to float32's rounding (256 additions a thread at most, 2^-16
    of it), which the output's rounding takes away."""
    lengths = [max(new, n) for n in (1, 17, 1024, 8192, 30000)]
    pool, table, q, starts = _filled(cuda, 3, [new] * 5, lengths, 8, 2, dim, group, dtype, value)
    got, lse = _attend(cuda, pool, table, q, starts, lengths)
    want = torch.tensor(value, dtype=dtype, device=cuda)
    assert torch.equal(got, want.expand_as(got)) and torch.isfinite(lse).all()


SPANS = [[0.0, 1e7], [0.0, 1e20], [1e7, 0.0], [1e-30, 1e20], [1e30, 1e-20, 1.0], [1e-35, 1e38],
         [1e38, 1e-35], [1e38, 1e-6, 0.0, 1e-30], [1.0, 1e-12], [1e-20], [1e35], [1e37, 1e34], [1e-31],
         [1e-34], [1e-33, 1.0]]


@pytest.mark.parametrize("sizes", SPANS)
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("few", [False, True])
def test_sizes_far_apart_in_one_context(cuda, sizes, new, few):
    """Runs of keys whose values differ by many powers of two, in either order:
    each keeps its weight in the softmax denominator."""
    dtype = torch.bfloat16
    lengths = [3 * 256, 97, 64] if few else [40, 640, 4096]
    lengths = [max(new, n) for n in lengths]
    n = 16 * sum(-(-a // 16) for a in lengths)
    size = torch.tensor(sizes, dtype=torch.float64)[torch.arange(n) // 32 % len(sizes)]
    v = (_rows(8, n, 2, 128, torch.float32).double().clamp(-2.5, 2.5) * size[:, None, None])
    pool, table, q, starts = _filled(cuda, 5, [new] * 3, lengths, 8, 2, 128, 64, dtype, v.float())
    got, lse = _attend(cuda, pool, table, q, starts, lengths)
    _check(got, lse, pool, table, q, starts, lengths, 128 ** -0.5, _wide([new] * 3, 4))


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("what", ["keys", "values"])
def test_groups_at_the_end_of_float16(cuda, dim, group, new, what):
    """-65504 .. 65504 and the like: whatever the operands are, they hold it."""
    dtype, lengths = torch.float16, [max(new, n) for n in (20, 300, 77)]
    n = 16 * sum(-(-a // 16) for a in lengths)
    x = _rows(6, n, 2, dim, torch.float32)
    ends = torch.tensor([65504.0, 62000.0, 61000.0, 65000.0])[torch.arange(n) % 4][:, None]
    at = torch.arange(n) % 3 > 0
    x[at, :, 5] = ends[at]
    x[at, :, 30] = -ends[at]
    x[at, :, 31] = 12345.0
    values = x if what == "values" else _rows(7, n, 2, dim, torch.float32)
    keys = x.half() if what == "keys" else None
    pool, table, q, starts = _filled(cuda, 5, [new] * 3, lengths, 8, 2, dim, group, dtype, values,
                                     keys)
    scale = 1e-5 if what == "keys" else dim ** -0.5
    got, lse = _attend(cuda, pool, table, q, starts, lengths, scale)
    assert torch.isfinite(got).all() and torch.isfinite(lse).all()
    _check(got, lse, pool, table, q, starts, lengths, scale, _wide([new] * 3, 4))


@pytest.mark.parametrize("value", [65504.0, -65504.0])
@pytest.mark.parametrize("length", [130, 4000])
@pytest.mark.parametrize("new", [1, 4, 60])
@pytest.mark.parametrize("spread", [False, True])
@pytest.mark.parametrize("odd", [False, True])
def test_means_of_the_largest_number_stay_in_float16(cuda, value, length, new, spread, odd):
    """A mean of numbers of a type is none that the type does not hold, however
    the weights are rounded: all keys but the first 64 are equal, so that their
    weights' roundings add up."""
    lengths = [length + 5 * b for b in range(6)]
    n = 16 * sum(-(-a // 16) for a in lengths)
    keys, at = _rows(9, n, 2, 128, torch.float16), 0
    for a in lengths:
        keys[at:at + 64] = keys[at]
        at += 16 * -(-a // 16)
        keys[at - 16 * -(-a // 16) + 64:at] = keys[at - 1]
    v = torch.full((n, 2, 128), value)
    if spread:  # a scale of 8728 whose top is 65512, which rounds to the largest number
        v[..., 1::2] = -65408.0 if value > 0 else 65408.0
    pool, table, q, starts = _filled(cuda, 5, [new] * 6, lengths, 8, 2, 128, 64, torch.float16, v,
                                     keys)
    rows = torch.empty(*q.shape[:2], 133, dtype=q.dtype, device=cuda)[..., 1:129]
    rows.copy_(q)
    got = kv4.attention(rows, pool, table.to(cuda),
                        torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda),
                        out=rows if odd else None)
    assert torch.isfinite(got).all()
    _, held = kv4.gather(pool, torch.zeros(1, dtype=torch.int64, device=cuda))
    # weights rounded to 2^-11 each act on 15 scales at most
    assert ((got.float() - held[0, 0].float()).abs() <= 2.0 ** -11 * 2 * 65504 + 32).all()


@pytest.mark.parametrize("up", [-100, -60, 60, 100, 112])
@pytest.mark.parametrize("new", [1, 4, 60])
def test_queries_and_keys_of_opposite_sizes(cuda, up, new):
    """Powers of two that the scores do not show."""
    lengths = [max(new, n) for n in (40, 640, 97)]
    n = 16 * sum(-(-a // 16) for a in lengths)
    values = _rows(4, n, 2, 128, torch.bfloat16)
    keys = _rows(5, n, 2, 128, torch.float32)
    outs = []
    for power in (0, up):
        pool, table, q, starts = _filled(cuda, 5, [new] * 3, lengths, 8, 2, 128, 64, torch.bfloat16,
                                         values, torch.ldexp(keys, torch.tensor(-power)).bfloat16())
        q = torch.ldexp(q.float(), torch.tensor(power)).bfloat16()
        got, lse = _attend(cuda, pool, table, q, starts, lengths)
        _check(got, lse, pool, table, q, starts, lengths, 128 ** -0.5, _wide([new] * 3, 4))
        outs.append(got)
    # (numbers below fp16's normal ones may lose bits, 2^-27 of the largest at least)
    assert (outs[0].float() - outs[1].float()).abs().max() <= 2.0 ** -7 * outs[0].abs().max()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 4, 60])
def test_a_query_that_is_not_finite_reaches_its_own_row(cuda, bad, dtype, new):
    lengths = [max(new, n) for n in (40, 640, 97)]
    pool, table, q, starts = _filled(cuda, 5, [new] * 3, lengths, 8, 2, 128, 64, dtype,
                                     _rows(4, 16 * 88, 2, 128, dtype)[:16 * sum(
                                         -(-a // 16) for a in lengths)])
    want, want_lse = _attend(cuda, pool, table, q, starts, lengths)
    # newest tokens, which see keys of either sign: a score of +inf or NaN among theirs
    at = [(new - 1, 3), (2 * new - 1, 7), (3 * new - 1, 0)]
    for token, head in at:
        q[token, head, 77] = bad
    got, lse = _attend(cuda, pool, table, q, starts, lengths)
    own = torch.zeros(q.shape[:2], dtype=torch.bool)
    for token, head in at:
        own[token, head] = True
    assert torch.isnan(got[own]).all() and not torch.isfinite(lse[own]).any()
    assert torch.equal(got[~own], want[~own]) and torch.equal(lse[~own], want_lse[~own])
