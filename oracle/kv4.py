"""Float64 restatement of the 4-bit pool: records, attention, slot maps.

    low = min x,  scale = (max x - min x) / 15,  code = (x - low in float32) / scale,
    nearest
    value = low + scale code
    o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max)
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

UNIT = 16


def params(x: torch.Tensor, group: int):
    """Scale and lowest value of each group of 16-bit x, in its type."""
    y = x.float().unflatten(-1, (-1, group))
    low, high = y.amin(-1) + 0.0, y.amax(-1)  # (a zero without a sign)
    # the quotient in float32 (its exact range in float64), then 16 bits
    scale = ((high.double() - low.double()) / 15).abs().float().to(x.dtype)
    # half a step past the largest number, which rounds to infinity
    top = torch.finfo(x.dtype).max + {torch.float16: 16.0, torch.bfloat16: 2.0 ** 119}[x.dtype]
    over = low.double() + 15 * scale.double() >= top
    down = (scale.view(torch.int16) - 1).view(x.dtype)
    scale = torch.where(over, down, scale)
    bad = ~torch.isfinite(y).all(-1)
    nan = torch.full_like(scale, math.nan)
    return torch.where(bad, nan, scale), torch.where(bad, nan, low.to(x.dtype))


def codes(x: torch.Tensor, scale: torch.Tensor, low: torch.Tensor, group: int) -> torch.Tensor:
    # (a power of two keeps the difference below float32's largest number)
    up = torch.where(scale.float() < 2.0 ** -60, 2.0 ** 60, 2.0 ** -4)[..., None]
    y = x.float().unflatten(-1, (-1, group)) * up - low.float()[..., None] * up
    s = scale.double()[..., None] * up
    c = torch.where(s > 0, y.double() / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15)
    return c.flatten(-2).to(torch.uint8)


def values(c: torch.Tensor, scale: torch.Tensor, low: torch.Tensor, group: int) -> torch.Tensor:
    y = c.double().unflatten(-1, (-1, group))
    return (y * scale.double()[..., None] + low.double()[..., None]).flatten(-2)


def order(dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The nibble of a row's codes that holds element e, of keys and of values."""
    e, w = torch.arange(dim), dim // 32
    return ((e % 32 // 8 * w + e // 32) * 8 + e % 8, (e % 32 // 4 * w + e // 32) * 4 + e % 4)


def record(k, v, group):
    """Codes and pairs of one token's heads as rows of bytes: key codes, value
    codes, key pairs, value pairs (each [..., bytes])."""
    out = []
    for x, at in zip((k, v), order(k.shape[-1])):
        s, z = params(x, group)
        c = codes(x, s, z, group)
        n = torch.empty_like(c)
        n[..., at] = c
        out += [n[..., 0::2] | n[..., 1::2] << 4,
                torch.stack((s, z), -1).flatten(-2).contiguous().view(torch.uint8)]
    return out[0], out[2], out[1], out[3]


def write(storage, slots, k, v, group):
    """The records of the slots in `storage` [block, head, units, unit bytes]."""
    d = k.shape[-1]
    row, pair = d // 2, 4 * (d // group)
    bs = storage.shape[2] * UNIT
    parts = record(k, v, group)
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < storage.shape[0] * bs:
            continue
        unit = storage[slot // bs, :, slot % bs // UNIT]
        r, base = slot % UNIT, 0
        for x, size in zip(parts, (row, row, pair, pair)):
            unit[:, base + r * size: base + (r + 1) * size] = x[t]
            base += UNIT * size


def _parts(storage, slots, dim, group, dtype):
    """Of keys, then of values: codes, scales and lowest values of the elements,
    float64 [n, heads, dim]."""
    row, pair = dim // 2, 4 * (dim // group)
    bs = storage.shape[2] * UNIT
    unit = storage[slots // bs, :, slots % bs // UNIT]  # [n, heads, bytes]
    r = (slots % UNIT)[:, None, None]
    out, base = [], 0
    for size in (row, row, pair, pair):
        at = base + r * size + torch.arange(size)
        out.append(unit.gather(2, at.expand(-1, unit.shape[1], -1)))
        base += UNIT * size
    res = []
    for raw, pairs, at in ((out[0], out[2], order(dim)[0]), (out[1], out[3], order(dim)[1])):
        n = torch.stack((raw & 15, raw >> 4), -1).flatten(-2)[..., at]
        p = pairs.contiguous().view(dtype).unflatten(-1, (-1, 2)).double()
        res.append((n.double(), *(p[..., i].repeat_interleave(group, -1) for i in (0, 1))))
    return res


def read(storage, slots, dim, group, dtype):
    """float64 keys and values, and float64 scales of the values' elements."""
    (kc, ks, kz), (vc, vs, vz) = _parts(storage, slots, dim, group, dtype)
    return [kc * ks + kz, ks, vc * vs + vz, vs]


def half(x: torch.Tensor) -> torch.Tensor:
    """float64 x rounded to fp16's 11 bits, whatever its exponent."""
    m, e = torch.frexp(x)
    return torch.where(torch.isfinite(x), torch.ldexp((m * 2048).round(), e - 11), x)


def operands(c, s, z, dtype):
    """The values as the kernel for many rows has them: bfloat16 records rounded to
    fp16 (with a power of two, which changes no bit but below 2^-37 of the largest),
    float16 ones as two fp16 numbers, scale of 7 bits times the code's distance from
    the one nearest to zero, and the rest."""
    if dtype != torch.float16:
        return half(z + s * c)
    main = ((s.half().view(torch.int16).int() + 8) & 0xfff0).to(torch.int16)
    main = main.view(torch.float16).double()
    zero = torch.where(s != 0, -z / torch.where(s != 0, s, 1.0), 0.0).nan_to_num().round()
    d = c - zero.clamp(0, 15)
    return main * d + half(half(z + (c - d) * s) + (s - main) * d)


# A rounding to 11 bits is off by 2^-11 of the number at most, and by this much of
# that in the mean square: 1 / sqrt 3 of half a step, which is 1 / m of 2^-11 for a
# number m 2^e; the mean of 1 / m^2 over even logarithms is 3 / (8 ln 2).
ROUNDING = math.sqrt(1 / 3 * 3 / (8 * math.log(2)))


class Bounds(NamedTuple):
    """One request's attention in float64, and what a kernel may be off."""

    out: torch.Tensor      #: [n, hq, d]
    lse: torch.Tensor      #: [n, hq]
    err: torch.Tensor      #: the most, before the output is rounded
    lse_err: torch.Tensor  #: the most
    var: torch.Tensor      #: what squares are in the mean, before the output is rounded


def bounds(q, storage, table, length, n, group, scale, wide) -> Bounds:
    """The attention, and the roundings that a kernel's comments name.

    Scores: float32 sums of products of codes (15 s + |low| bounds what is added
    up), 2^-21 of what is added up; and the exponent's argument, whose terms are
    the score and the power of two that the values' size gives the weights.  Of the
    kernel for many rows, `operands`: the outputs of those numbers are worked out,
    so that only their own distance counts.
    Weights are rounded to fp16 (half a step, 2^-11): that acts on the codes'
    distance from their middle (8 s at most) or, of the kernel for many rows, on
    the value; weights below fp16's normal numbers by 2^-25 of 2^6 (2^7)."""
    hk, d = storage.shape[1], q.shape[-1]
    bs = storage.shape[2] * UNIT
    at = torch.arange(max(0, length))
    slots = table[at // bs].long() * bs + at % bs
    g = q.shape[1] // hk
    empty = torch.zeros(n, hk * g, d, dtype=torch.float64)
    if length <= 0:
        nothing = torch.full((n, hk * g), -math.inf, dtype=torch.float64)
        return Bounds(empty, nothing, empty, torch.zeros_like(nothing), empty)
    (kc, ks, kz), (vc, vs, vz) = _parts(storage, slots, d, group, q.dtype)
    k, v = kc * ks + kz, vc * vs + vz
    x = q.double().view(n, hk, g, d)
    seen = at <= (length - n + torch.arange(n))[:, None]
    shown = seen[:, :, None, None, None]
    seen = seen[:, None, None]

    def mix(weights, rows):  # a key that is not seen has no part, not even NaN
        rows = rows[None, :, :, None, :].expand(n, -1, -1, 1, -1)
        y = weights.permute(0, 3, 1, 2)[..., None] * rows
        return torch.where(shown, y, 0.0).sum(1)

    def soft(keys):
        z = torch.einsum("nhgd,khd->nhgk", x, keys) * scale
        z = torch.where(seen, z, -math.inf)
        top = z.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.where(seen, (z - top).exp(), 0.0)
        total = p.sum(-1, keepdim=True)
        some = total != 0  # (true of NaN)
        total = torch.where(some, total, 1.0)
        lse = torch.where(some, top + total.log(), -math.inf)[..., 0]
        return z, torch.where(some, p / total, 0.0), lse

    z, w, lse = soft(k)
    o = mix(w, v)
    size = torch.einsum("nhgd,khd->nhgk", x.abs(), k.abs() + 16 * ks) * abs(scale)
    # the power of two in the weights' exponents: of the values' sizes
    reach = torch.maximum(v.abs(), vs).nan_to_num(0, 0, 0).amax((1, 2))
    power = torch.where(reach > 0, reach, 2.0 ** -86).log2().abs().amax()
    dz = 2.0 ** -21 * (size + 1 + z.masked_fill(~seen, 0).abs() + power)
    dz = dz.nan_to_num(0, 0, 0)
    most, widest = w.nan_to_num().amax(-1)[..., None], v.nan_to_num(0, 0, 0).abs().amax()
    step = vs.nan_to_num(0, 0, 0).amax()
    err = 2 * mix(w * dz, v.abs())
    lse_err = (w * dz).sum(-1).nan_to_num()
    lse_err = lse_err + 2.0 ** -20 * (1 + lse.abs().nan_to_num(0, 0, 0) + power)
    if wide:
        k2, v2 = operands(kc, ks, kz, q.dtype), operands(vc, vs, vz, q.dtype)
        _, w2, lse2 = soft(k2)
        off = mix(w2, v2) - o
        err = err + off.abs() + 2.0 ** -11 * mix(w2, v2.abs())
        err = err + 2.0 ** -31 * length * most * widest + 2.0 ** -34 * widest
        lse_err = lse_err + (lse2 - lse).nan_to_num().abs()
        var = off ** 2 + (ROUNDING * 2.0 ** -11) ** 2 * mix(w2 ** 2, v2 ** 2)
    else:
        err = err + 2.0 ** -11 * mix(w, 8 * vs) + 2.0 ** -20 * step + \
            2.0 ** -28 * length * most * step
        var = (ROUNDING * 2.0 ** -11) ** 2 * mix(w ** 2, (vs * (vc - 8)) ** 2)
    shape = (n, hk * g, d)
    return Bounds(o.reshape(shape), lse.reshape(shape[:2]), err.reshape(shape),
                  lse_err.reshape(shape[:2]), var.reshape(shape))


def attention(q, storage, table, length, n, group, scale, wide):
    """One request: out [n, hq, d] and lse [n, hq] in float64, and how far a
    kernel may be from them before its output is rounded."""
    return bounds(q, storage, table, length, n, group, scale, wide)[:3]


def step_maps(lengths, new, tables, block, blocks, tokens, keys=0, offset=0, free=None,
              free_count=0):
    """Lists, token by token; the tables are changed in place.  None: refused."""
    tables = [list(t) for t in tables]
    width = len(tables[0]) if tables else 0
    if any(n < 0 or a < n or -(-a // block) > width for a, n in zip(lengths, new)) or \
            sum(new) > tokens or keys and sum(lengths) > keys:
        return None
    left = free_count
    if free is not None:
        for b, (a, n) in enumerate(zip(lengths, new)):
            for j in range(-(-(a - n) // block), -(-a // block)):
                if left == 0:
                    return None
                left -= 1
                tables[b][j] = free[left]

    def slot(b, p):
        at = tables[b][p // block]
        return at * block + p % block if 0 <= at < blocks else -1

    starts, key_starts, positions, slots, key_slots = [0], [0], [], [], []
    for b, (a, n) in enumerate(zip(lengths, new)):
        starts.append(starts[-1] + n)
        key_starts.append(key_starts[-1] + a)
        positions += [offset + p for p in range(a - n, a)]
        slots += [slot(b, p) for p in range(a - n, a)]
        if keys:
            key_slots += [slot(b, p) for p in range(a)]
    positions += [0] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    key_slots += [-1] * (keys - len(key_slots))
    return dict(tables=tables, starts=starts, key_starts=key_starts, positions=positions,
                slots=slots, key_slots=key_slots, left=left)
