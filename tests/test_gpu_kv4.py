"""The 4-bit pool on the GPU against float64: records bit for bit, values and
attention within bounds that count roundings (oracle/kv4.py)."""

from __future__ import annotations

import math

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4
from oracle import kv4 as okv4

pytestmark = pytest.mark.gpu
FORMS = [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)]
TYPES = [torch.bfloat16, torch.float16]


def _rows(seed, n, heads, dim, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g) * scale
    x[..., 3] *= 9  # a loud channel
    return x.to(dtype)


def _pool(cuda, blocks, heads, block, dim, group, dtype, fill=0):
    pool = kv4.empty_pool(blocks, heads, block, dim, dtype, cuda, group)
    pool.storage.fill_(fill)
    return pool


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("n,heads,block", [(1, 1, 16), (37, 3, 48), (300, 8, 32)])
def test_records_bit_for_bit(cuda, dtype, dim, group, n, heads, block):
    k, v = _rows(n, n, heads, dim, dtype), _rows(n + 1, n, heads, dim, dtype, 0.01)
    blocks = -(-n // block) + 3
    slots = torch.randperm(blocks * block, generator=torch.Generator().manual_seed(7))[:n]
    pool = _pool(cuda, blocks, heads, block, dim, group, dtype, 0xA5)
    want = pool.storage.cpu()
    okv4.write(want, slots, k, v, group)
    status = N.Status(cuda)
    kv4.append(pool, slots.to(cuda), k.to(cuda), v.to(cuda), status=status)
    assert torch.equal(pool.storage.cpu(), want)  # the records, and nothing else
    gk, gv = kv4.gather(pool, slots.to(cuda), status=status)
    wk, _, wv, _ = okv4.read(want, slots, dim, group, dtype)
    # one rounding of the exact value (float32's own sum is rounded before: half
    # an ulp of it more)
    for got, exact in ((gk, wk), (gv, wv)):
        half = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10)
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((got.cpu().double() - exact).abs() <= half * exact.abs() + tiny / 2).all()
    assert status.read() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_constants_extremes_and_tiny_values(cuda, dtype):
    dim, group = 128, 32
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(14, 1, dim)
    steps = torch.arange(31) * 0.5  # halves of a scale of 1: ties at every odd one
    x[0, 0, :31] = steps
    x[0, 0, 31] = 15
    x[1, 0] = 3.25
    x[2, 0] = torch.linspace(-1, 1, dim) * big
    x[3, 0] = torch.linspace(0, 1, dim) * big
    x[4, 0] = torch.linspace(0, 1, dim) * tiny
    x[5, 0] = torch.linspace(-1, 1, dim) * tiny * 2.0 ** -6
    x[6, 0] = torch.linspace(-2, -1, dim)
    x[7, 0] = torch.where(torch.arange(dim) % 2 == 0, 1.0, 1.0 + torch.finfo(dtype).eps)
    x[8, 0] = -big
    x[9, 0, ::32] = big
    x[10, 0] = torch.linspace(0, 1, dim) ** 9
    x[11, 0] = -steps.repeat(5)[:dim] * 0.125
    x[12, 0] = torch.where(torch.arange(dim) % 3 == 0, -0.0, 0.0)
    x[13, 0] = torch.where(torch.arange(dim) % 3 == 0, -0.0, 1.0)
    x = x.to(dtype)
    slots = torch.arange(14)
    pool = _pool(cuda, 1, 1, 16, dim, group, dtype)
    want = pool.storage.cpu()
    okv4.write(want, slots, x, x.flip(0), group)
    kv4.append(pool, slots.to(cuda), x.to(cuda), x.flip(0).to(cuda))
    assert torch.equal(pool.storage.cpu(), want)
    k, _ = kv4.gather(pool, slots.to(cuda))
    assert torch.isfinite(k).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_not_finite_stands_for_nan(cuda, dtype, bad):
    k, v = _rows(1, 5, 2, 128, dtype), _rows(2, 5, 2, 128, dtype)
    k[2, 1, 40] = bad
    v[3, 0, 127] = bad
    pool = _pool(cuda, 1, 2, 16, 128, 32, dtype)
    slots = torch.arange(5, device=cuda)
    kv4.append(pool, slots, k.to(cuda), v.to(cuda))
    gk, gv = (x.cpu() for x in kv4.gather(pool, slots))
    nk, nv = torch.zeros_like(gk, dtype=torch.bool), torch.zeros_like(gv, dtype=torch.bool)
    nk[2, 1, 32:64] = True
    nv[3, 0, 96:] = True
    assert torch.equal(torch.isnan(gk), nk) and torch.equal(torch.isnan(gv), nv)


def test_padding_strides_and_slots_outside(cuda):
    dim, group, dtype = 64, 32, torch.bfloat16
    k = _rows(3, 6, 7, 2 * dim + 1, dtype)
    v = _rows(4, 7, 6, dim, dtype)
    kc, vc = k[:, 1:6, 1:dim + 1], v.transpose(0, 1)[:, :5]  # odd offset; heads and tokens swapped
    slots = torch.tensor([5, -1, 31, 32, -9, 0])
    pool = _pool(cuda, 2, 5, 16, dim, group, dtype, 0x11)
    want = pool.storage.cpu()
    okv4.write(want, slots, kc.contiguous(), vc.contiguous(), group)
    status = N.Status(cuda)
    ks, vs = k.to(cuda)[:, 1:6, 1:dim + 1], v.to(cuda).transpose(0, 1)[:, :5]
    kv4.append(pool, slots.to(cuda), ks, vs, status=status)
    assert status.read() == N.ST_SLOT_RANGE
    assert torch.equal(pool.storage.cpu(), want)
    status = N.Status(cuda)
    gk, gv = kv4.gather(pool, slots.to(cuda), status=status)
    assert status.read() == N.ST_SLOT_RANGE
    for x in (gk, gv):
        assert x[[1, 3, 4]].eq(0).all() and x[[0, 2, 5]].ne(0).any(-1).all()
    status = N.Status(cuda)
    only = torch.tensor([-1], device=cuda)
    kv4.append(pool, only, ks[:1], vs[:1], status=status)
    kv4.append(pool, only[:0], ks[:0], vs[:0], status=status)
    assert kv4.gather(pool, only[:0])[0].shape == (0, 5, dim)
    assert status.read() == 0 and torch.equal(pool.storage.cpu(), want)


# ------------------------------------------------------------------ attention
def _batch(cuda, seed, new, lengths, hq, hk, dim, group, block, dtype, spare=2, scale_k=1.0):
    """A pool of random records, tables over shuffled blocks and queries."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-max(a, 0) // block) for a in lengths]
    blocks = sum(per) + spare
    width = max(per + [1])
    perm = torch.randperm(blocks, generator=g).int()
    table, at = torch.full((len(new), width), -3, dtype=torch.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = perm[at:at + n]
        at += n
    n = blocks * block
    pool = _pool(cuda, blocks, hk, block, dim, group, dtype)
    kv4.append(pool, torch.arange(n, device=cuda), _rows(seed, n, hk, dim, dtype, scale_k).to(cuda),
               _rows(seed + 1, n, hk, dim, dtype).to(cuda))
    q = (1.5 * torch.randn(sum(new), hq, dim, generator=g)).to(dtype)
    starts = torch.tensor([0, *new]).cumsum(0).int()
    return pool, table, q, starts


def _wide(new, heads):
    """Whether the kernel for many query rows a KV head takes such a batch."""
    return len(new) > 0 and sum(new) * heads // len(new) > 32


def _check(got, lse, pool, table, q, starts, lengths, scale, wide, rows=None):
    storage = pool.storage.cpu()
    eps = torch.finfo(pool.dtype).eps / 2
    tiny = torch.finfo(pool.dtype).smallest_normal * eps
    got, lse = got.cpu().double(), lse.cpu().double()
    for b, length in enumerate(lengths):
        lo, hi = int(starts[b]), int(starts[b + 1])
        if hi == lo:
            continue
        o, l, err = okv4.attention(q[lo:hi], storage, table[b], length, hi - lo, pool.group, scale,
                                   wide)
        assert torch.equal(torch.isnan(got[lo:hi]), torch.isnan(o)), b
        bound = err + eps * (o.abs() + err) + tiny
        off = ((got[lo:hi] - o).abs() <= bound) | torch.isnan(o)
        assert off.all(), (b, ((got[lo:hi] - o).abs() / bound).nan_to_num().max())
        some = l != -math.inf
        assert torch.equal(lse[lo:hi] == -math.inf, ~some), b
        near = (lse[lo:hi] - l).abs() <= 2.0 ** (-9 if wide else -16) * (1 + l.abs())
        off = (lse[lo:hi] - l).abs().masked_fill(~some | torch.isnan(l), 0)
        assert (near | ~some | torch.isnan(l)).all(), (b, off.max(), off.argmax(), l.flatten()[off.argmax()])


def _run(cuda, new, lengths, hq, hk, dim, group, block, dtype, seed=0, scale=None, one=False,
         scale_k=1.0):
    pool, table, q, starts = _batch(cuda, seed, new, lengths, hq, hk, dim, group, block, dtype,
                                    scale_k=scale_k)
    status = N.Status(cuda)
    got, lse = kv4.attention(
        q.to(cuda), pool, table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
        None if one else starts.to(cuda), scale=scale, return_lse=True, status=status)
    assert status.read() == 0
    wide = _wide(new, hq // hk)
    _check(got, lse, pool, table, q, starts, lengths, dim ** -0.5 if scale is None else scale, wide)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("hq,hk", [(8, 2), (5, 5), (16, 1)])
def test_decode(cuda, dtype, dim, group, hq, hk):
    lengths = [1, 15, 16, 17, 63, 64, 65, 200, 511, 1300]
    _run(cuda, [1] * 10, lengths, hq, hk, dim, group, 32, dtype, one=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [2, 3, 4, 7, 9, 20])
def test_drafts(cuda, dtype, new):
    _run(cuda, [new] * 6, [new, new + 1, 30, 64, 129, 700], 8, 2, 128, 64, 16, dtype)


@pytest.mark.parametrize("dtype,dim,group", [(torch.bfloat16, 128, 64), (torch.float16, 64, 32),
                                             (torch.float16, 128, 128),
                                             (torch.bfloat16, 128, 32)])
def test_questions(cuda, dtype, dim, group):
    _run(cuda, [40, 150, 1, 64, 129], [40, 333, 90, 64, 600], 8, 2, dim, group, 48, dtype)


def test_long_contexts_are_cut_and_joined(cuda):
    _run(cuda, [1, 1, 1], [9000, 40, 23456], 8, 1, 128, 128, 16, torch.bfloat16, one=True)
    _run(cuda, [3, 2], [9000, 4001], 8, 2, 64, 64, 16, torch.float16)


def test_idle_requests_empty_rows_and_lengths_below_the_new_tokens(cuda):
    _run(cuda, [1, 0, 5, 0, 3, 2], [0, 50, 2, 0, 100, 1], 4, 2, 128, 64, 16, torch.bfloat16)
    _run(cuda, [70, 0, 50], [20, 50, 0], 4, 1, 128, 64, 16, torch.bfloat16)
    _run(cuda, [1, 1], [0, 0], 4, 2, 64, 32, 16, torch.float16, one=True)


def test_one_request_of_many_rows_among_decodes(cuda):
    _run(cuda, [1] * 30 + [90], [33] * 30 + [200], 8, 2, 128, 64, 16, torch.bfloat16)


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales(cuda, scale, new):
    _run(cuda, [new, new], [77, 300], 4, 2, 128, 64, 16, torch.bfloat16, scale=scale)


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("scale_k", [1e-6, 1e5])
def test_small_and_large_keys(cuda, scale_k, new):
    """Keys far outside fp16's range, with the scale that makes their scores ordinary."""
    _run(cuda, [new, new], [77, 300], 4, 2, 128, 64, 16, torch.bfloat16, scale=0.1 / scale_k,
         scale_k=scale_k)


@pytest.mark.parametrize("dtype,dim,group", [(torch.float16, 64, 32), (torch.bfloat16, 128, 128)])
@pytest.mark.parametrize("hq,hk,new", [(16, 4, [3, 150, 40, 66, 7, 149, 12, 64, 65, 90, 3, 128, 130]),
                                       (8, 8, [129, 300, 5, 260, 128, 511, 1, 257, 256, 140]),
                                       (8, 1, [5, 16, 30, 2, 17, 33, 9])])
def test_row_tiles_of_all_sizes_over_and_over(cuda, dtype, dim, group, hq, hk, new):
    """Blocks that go from tiles of one row half to tiles of two and back: the
    results are right, and the same in every call."""
    lengths = [n + 53 * (b * b % 29) for b, n in enumerate(new)]
    pool, table, q, starts = _batch(cuda, 4, new, lengths, hq, hk, dim, group, 16, dtype)
    args = (q.to(cuda), pool, table.to(cuda),
            torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda))
    status = N.Status(cuda)
    got, lse = kv4.attention(*args, return_lse=True, status=status)
    _check(got, lse, pool, table, q, starts, lengths, dim ** -0.5, _wide(new, hq // hk))
    busy = torch.empty(1 << 26, dtype=torch.uint8, device=cuda)
    for i in range(60):
        if i % 3 == 0:
            busy.fill_(i)  # another state of the caches, other times of arrival
        assert torch.equal(kv4.attention(*args, status=status), got), i
    assert status.read() == 0


def test_more_requests_than_threads(cuda):
    _run(cuda, [1] * 700, [1 + 37 * b % 120 for b in range(700)], 2, 1, 64, 32, 16,
         torch.bfloat16, one=True)


@pytest.mark.parametrize("new", [1, 3, 50])
def test_records_that_are_not_finite_reach_the_rows_that_see_them(cuda, new):
    lengths = [max(new, 3), 200]
    pool, table, q, starts = _batch(cuda, 5, [new, new], lengths, 4, 2, 128, 32, 16,
                                    torch.bfloat16)
    bad = _rows(9, 3, 2, 128, torch.bfloat16)
    bad[0, 1, 77] = math.inf  # a value seen by all of request 1's rows
    keys = bad.clone()
    keys[:] = 0.5
    keys[2, 0, 5] = math.nan  # a key that only the newest row sees
    at = torch.tensor([30, 3, lengths[1] - 1])
    slots = table[1][at // 16].long() * 16 + at % 16
    free = sorted(set(range(pool.num_blocks)) - set(table[table >= 0].tolist()))
    kv4.append(pool, slots.to(cuda), keys.to(cuda), bad.to(cuda))
    pool.storage[free] = 0xFF  # blocks of nobody: NaN pairs
    # and the places behind the requests' last tokens
    behind = torch.cat([table[b][(lengths[b] - 1) // 16].long() * 16
                        + torch.arange((lengths[b] - 1) % 16 + 1, 16) for b in (0, 1)])
    nan = torch.full((behind.numel(), 2, 128), math.nan, dtype=torch.bfloat16, device=cuda)
    kv4.append(pool, behind.to(cuda), nan, nan)
    status = N.Status(cuda)
    got, lse = kv4.attention(
        q.to(cuda), pool, table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
        starts.to(cuda), return_lse=True, status=status)
    assert status.read() == 0 and torch.isnan(got).any() and not torch.isnan(got).all()
    _check(got, lse, pool, table, q, starts, lengths, 128 ** -0.5, _wide([new, new], 2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 4, 40])
def test_whatever_lies_behind_the_last_token(cuda, dtype, new):
    """Blocks full of large numbers, infinities and NaN behind the lengths, and
    the same left in shared memory by a call before."""
    lengths = [max(new, n) for n in (1, 9, 16, 65, 130, 260)]
    pool, table, q, starts = _batch(cuda, 12, [new] * 6, lengths, 8, 2, 128, 64, 16, dtype)
    args = (table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda))
    want = kv4.attention(q.to(cuda), pool, *args)
    big = torch.finfo(dtype).max
    for value in (big, -big, math.nan, math.inf):
        rows = torch.full((pool.num_blocks * 16, 2, 128), value, dtype=dtype, device=cuda)
        rows[..., ::2] = 0
        other = kv4.empty_pool(pool.num_blocks, 2, 16, 128, dtype, cuda, 64)
        kv4.append(other, torch.arange(len(rows), device=cuda), rows, rows)
        kv4.attention(q.to(cuda), other, *args)
        for b, length in enumerate(lengths):
            at = torch.arange(length)
            slots = (table[b][at // 16].long() * 16 + at % 16).to(cuda)
            # exact copies of the records
            unit, r = slots // 16, slots % 16
            for base, size in ((0, 64), (1024, 64), (2048, 8), (2176, 8)):
                where = (base + r[:, None] * size + torch.arange(size, device=cuda))[:, None]
                where = where.expand(-1, 2, -1)
                src = pool.storage[unit][:, :, 0].gather(2, where)
                for h in (0, 1):
                    other.storage[unit[:, None], h, 0, where[:, h]] = src[:, h]
        assert torch.equal(kv4.attention(q.to(cuda), other, *args), want), value


@pytest.mark.parametrize("new", [1, 40])
def test_bad_tables_lengths_and_starts_are_reported(cuda, new):
    pool, table, q, starts = _batch(cuda, 6, [new] * 4, [100] * 4, 4, 2, 128, 64, 16,
                                    torch.bfloat16)
    lengths = torch.tensor([100] * 4, dtype=torch.int32)
    want = kv4.attention(q.to(cuda), pool, table.to(cuda), lengths.to(cuda), starts.to(cuda))

    def call(table=table, lengths=lengths, starts=starts):
        status = N.Status(cuda)
        out = torch.full_like(q, 7.0, device=cuda)
        kv4.attention(q.to(cuda), pool, table.to(cuda), lengths.to(cuda), starts.to(cuda),
                      out=out, status=status)
        return out, status.read()

    bad = table.clone()
    bad[2, 3] = pool.num_blocks
    bad[3, 1] = -1
    out, bits = call(table=bad)
    assert bits == N.ST_SLOT_RANGE
    assert torch.equal(out[:2 * new], want[:2 * new])
    # zero keys and values in their place
    zero = kv4.empty_pool(pool.num_blocks + 1, 2, 16, 128, torch.bfloat16, cuda, 64)
    zero.storage[:-1] = pool.storage
    bad[3, 1] = pool.num_blocks
    same = kv4.attention(q.to(cuda), zero, bad.to(cuda), lengths.to(cuda), starts.to(cuda))
    assert torch.equal(out, same)
    long = lengths.clone()
    long[1] = 10_000  # cut at the tables' width
    cut = lengths.clone()
    cut[1] = 16 * table.shape[1]
    out, bits = call(lengths=long, table=table.clamp(min=0))
    assert bits == N.ST_CAPACITY and torch.equal(out, call(lengths=cut, table=table.clamp(min=0))[0])
    fall = starts.clone()
    fall[2] = fall[1] - 1  # (request 2 then has rows of request 0 and 1 too)
    out, bits = call(starts=fall)
    assert bits == N.ST_CAPACITY and torch.equal(out[3 * new:], want[3 * new:])
    past = starts.clone()
    past[4] += 1
    out, bits = call(starts=past)
    assert bits == N.ST_CAPACITY
    assert torch.equal(out[:3 * new], want[:3 * new]) and out[3 * new:].eq(7).all()


@pytest.mark.parametrize("new", [1, 40])
def test_rows_of_no_request(cuda, new):
    pool, table, q, starts = _batch(cuda, 8, [new, 2, new], [90, 40, 70], 4, 2, 128, 64, 16,
                                    torch.bfloat16)
    lengths = torch.tensor([90, 40, 70], dtype=torch.int32, device=cuda)
    shifted = (starts + 5).to(cuda)
    rows = torch.zeros(5 + len(q) + 2, 4, 128, dtype=torch.bfloat16, device=cuda)
    rows[5:5 + len(q)] = q.to(cuda)
    want = kv4.attention(q.to(cuda), pool, table.to(cuda), lengths, starts.to(cuda))
    out = torch.full_like(rows, 3.0)
    kv4.attention(rows, pool, table.to(cuda), lengths, shifted, out=out)
    n = len(rows)
    assert torch.equal(out[5:5 + len(q)], want)
    assert out[:5].eq(3).all() and out[5 + len(q):].eq(3).all()
    new_out, lse = kv4.attention(rows, pool, table.to(cuda), lengths, shifted, return_lse=True)
    assert torch.equal(new_out[5:5 + len(q)], want)
    for lo, hi in ((0, 5), (5 + len(q), n)):
        assert new_out[lo:hi].eq(0).all() and lse[lo:hi].eq(-math.inf).all()


@pytest.mark.parametrize("new", [1, 30])
def test_strides_and_an_output_over_the_queries(cuda, new):
    pool, table, q, starts = _batch(cuda, 9, [new] * 3, [90, 400, 70], 8, 2, 128, 64, 16,
                                    torch.float16)
    lengths = torch.tensor([90, 400, 70], dtype=torch.int32, device=cuda)
    args = pool, table.to(cuda), lengths, starts.to(cuda)
    want = kv4.attention(q.to(cuda), *args)
    odd = torch.zeros(len(q), 9, 133, dtype=torch.float16, device=cuda)
    odd[:, 1:, 3:131] = q.to(cuda)
    out = torch.zeros(8, len(q), 131, dtype=torch.float16, device=cuda).transpose(0, 1)
    got = kv4.attention(odd[:, 1:, 3:131], *args, out=out[..., 1:129])
    assert torch.equal(got, want) and out[..., 0].eq(0).all() and out[..., 129:].eq(0).all()
    over = q.to(cuda)
    assert torch.equal(kv4.attention(over, *args, out=over), want) and torch.equal(over, want)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device=cuda)
    wide[:, 2:2 + table.shape[1]] = table.to(cuda)
    view = wide[:, 2:2 + table.shape[1]]
    assert torch.equal(kv4.attention(q.to(cuda), pool, view, *args[2:]), want)
    for _ in range(5):  # equal calls give equal bits
        assert torch.equal(kv4.attention(q.to(cuda), *args), want)


def test_streams_and_graphs(cuda):
    """Maps, append and attention of a decode loop in one graph on a side
    stream, against eager calls; two graphs share nothing."""
    from cacheslide_b200.tables import step_maps

    hq, hk, dim, block, steps = 8, 2, 128, 16, 20
    g = torch.Generator().manual_seed(3)
    k, v = ((torch.randn(steps, 3, hk, dim, generator=g)).bfloat16().to(cuda) for _ in "kv")
    q = torch.randn(steps, 3, hq, dim, generator=g).bfloat16().to(cuda)

    def fresh():
        pool = kv4.empty_pool(12, hk, block, dim, torch.bfloat16, cuda)
        return dict(pool=pool, lengths=torch.tensor([0, 15, 30], dtype=torch.int32, device=cuda),
                    table=torch.tensor([[0] * 4, [7, 0, 0, 0], [3, 4, 0, 0]], dtype=torch.int32,
                                       device=cuda),
                    free=torch.tensor([0, 1, 2, 5, 6, 8, 9, 10], dtype=torch.int32, device=cuda),
                    count=torch.tensor([8], dtype=torch.int32, device=cuda),
                    one=torch.ones(3, dtype=torch.int32, device=cuda),
                    at=torch.zeros(1, dtype=torch.int64, device=cuda),
                    out=torch.zeros(steps, 3, hq, dim, dtype=torch.bfloat16, device=cuda),
                    status=N.Status(cuda))

    def step(s):
        s["lengths"].add_(1)
        m = step_maps(s["lengths"], s["one"], s["table"], block, 12, tokens=3, free=s["free"],
                      free_count=s["count"], status=s["status"])
        s["count"].copy_(m.free_left)
        kv4.append(s["pool"], m.slots, k[s["at"]][0], v[s["at"]][0], status=s["status"])
        o = kv4.attention(q[s["at"]][0], s["pool"], s["table"], s["lengths"], status=s["status"])
        s["out"].index_copy_(0, s["at"], o[None])
        s["at"].add_(1)

    eager = fresh()
    for _ in range(steps):
        step(eager)
    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    runs = []
    with torch.cuda.stream(stream):
        for _ in range(2):
            s = fresh()
            keep = {n: t.clone() for n, t in s.items() if isinstance(t, torch.Tensor)}
            step(s)
            for n, t in keep.items():
                s[n].copy_(t)
            s["pool"].storage.zero_()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step(s)
            runs.append((s, graph))
        for _ in range(steps):
            for _, graph in runs:
                graph.replay()
    stream.synchronize()
    assert eager["status"].read() == 0
    for s, _ in runs:
        assert torch.equal(s["out"], eager["out"]) and s["status"].read() == 0
        assert torch.equal(s["pool"].storage, eager["pool"].storage)


@pytest.mark.parametrize("new", [1, 50])
def test_byte_offsets_past_32_bits(cuda, new):
    pool, table, q, starts = _batch(cuda, 13, [new] * 2, [400, 555], 4, 1, 128, 128, 16,
                                    torch.bfloat16)
    lengths = torch.tensor([400, 555], dtype=torch.int32, device=cuda)
    args = (lengths, starts.to(cuda))
    want = kv4.attention(q.to(cuda), pool, table.to(cuda), *args)
    blocks = (1 << 32) // pool.storage[0].numel() + 200_000  # 4.7 GB
    far = kv4.PagedKV4(torch.empty((blocks, *pool.storage.shape[1:]), dtype=torch.uint8,
                                   device=cuda), 128, torch.bfloat16, 128)
    shift = blocks - pool.num_blocks
    slots = torch.arange(pool.num_blocks * 16, device=cuda)
    k, v = kv4.gather(pool, slots)
    far.storage[shift:] = pool.storage
    for a, b in zip(kv4.gather(far, slots + 16 * shift), (k, v)):
        assert torch.equal(a, b)
    got = kv4.attention(q.to(cuda), far, (table + shift).to(cuda), *args)
    assert torch.equal(got, want)
    kv4.append(pool, slots, k, v)
    kv4.append(far, slots + 16 * shift, k, v)
    assert torch.equal(far.storage[shift:], pool.storage)


def test_calls_at_once_on_several_streams(cuda):
    """Few and many rows side by side over one pool: each call has its own
    workspace."""
    cases = []
    for seed, new in ((1, [1] * 9), (2, [70, 3, 200]), (3, [4] * 5), (4, [90] * 4)):
        lengths = [n + 300 * (b + 1) for b, n in enumerate(new)]
        pool, table, q, starts = _batch(cuda, seed, new, lengths, 8, 2, 128, 64, 16,
                                        torch.bfloat16)
        args = (q.to(cuda), pool, table.to(cuda),
                torch.tensor(lengths, dtype=torch.int32, device=cuda), starts.to(cuda))
        cases.append((args, kv4.attention(*args), torch.cuda.Stream(cuda)))
    torch.cuda.synchronize()
    out = []
    for i in range(10):
        for args, _, stream in cases:
            with torch.cuda.stream(stream):
                out.append(kv4.attention(*args))
    torch.cuda.synchronize()
    for i, got in enumerate(out):
        assert torch.equal(got, cases[i % 4][1]), i


def test_refusals(cuda):
    pool, table, q, starts = _batch(cuda, 1, [2, 2], [20, 30], 4, 2, 128, 64, 16, torch.bfloat16)
    table, q, starts = table.to(cuda), q.to(cuda), starts.to(cuda)
    lengths = torch.tensor([20, 30], dtype=torch.int32, device=cuda)
    kv4.attention(q, pool, table, lengths, starts)
    for bad in (dict(query=q.half()), dict(query=q[:, :3]), dict(query=q[..., :64]),
                dict(tables=table.long()), dict(tables=table[0]), dict(lengths=lengths.long()),
                dict(lengths=lengths[:1]), dict(starts=None), dict(starts=starts[:2]),
                dict(starts=starts.long()), dict(lengths=lengths.cpu()), dict(query=q.cpu()),
                dict(scale=math.inf), dict(scale=1e39), dict(out=q[:1]), dict(out=q.float()),
                dict(status=N.Status(torch.device("cpu"))), dict(pool=pool.storage)):
        args = dict(query=q, pool=pool, tables=table, lengths=lengths, starts=starts) | bad
        with pytest.raises(ValueError):
            kv4.attention(**args)
    slots = torch.arange(3, device=cuda)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=cuda)
    for bad in (dict(slots=slots.int()), dict(slots=slots[None]), dict(key=k.half()),
                dict(value=k[:2]), dict(key=k.cpu()), dict(slots=slots.cpu())):
        with pytest.raises(ValueError):
            kv4.append(**(dict(pool=pool, slots=slots, key=k, value=k) | bad))
    with pytest.raises(ValueError):
        kv4.gather(pool, slots.int())
    empty = kv4.attention(q[:0], pool, table[:0], lengths[:0])
    assert empty.shape == (0, 4, 128)
