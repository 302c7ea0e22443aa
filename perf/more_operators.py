"""Serving from a paged cache held in 4 bits: its operators and their cases.

* ``maps``: the slots and positions of a step's tokens, the blocks that they
  need taken from the free ones, and the slots of every request's keys, from
  the requests' lengths on the device (``tables.step_maps``);
* ``append``: keys and values rounded to 4 bits (a scale and a lowest value a
  group) into their slots of the pool, and read back as the values that the
  pool now stands for (``kv4.append``, ``kv4.gather``);
* ``attend``: attention over such a pool through block tables and lengths on
  the device -- decodes, drafted tokens, whole questions (``kv4.attention``).

``run`` computes either the plain form (elementary torch operations) or, with
``own`` set, the framework's operators; ``exact`` restates the definition in
64 bits.

The pool is bytes, [block, kv_head, block_size / 16, unit]: a unit holds 16
tokens of one head, their key codes (head_dim / 2 bytes a token), their value
codes, and the 16-bit pairs (scale, lowest value) of the keys' groups and of
the values', token by token.  A key's codes lie in words of 8: word 4-bit
code i of word t * (head_dim / 32) + w is element 32 w + 8 t + i; a value's in
half-words of 4: code i of half-word g * (head_dim / 32) + w is element
32 w + 4 g + i.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = 16  # tokens of a unit


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 32 chat sessions with histories up to 16K: one token
        # each, a block taken where it opens one
        dict(name="maps decode 32", op="maps", requests=32, new=1, new_max=1, length=256,
             length_max=16384, block=16, keys=False, order=1),
        # 64 retrieval questions of 64 tokens and the slots of all their own keys
        dict(name="maps questions 64", op="maps", requests=64, new=64, new_max=64, length=64,
             length_max=96, block=16, keys=True, order=2),
        # a large ragged batch, some requests idle, with every key's slot
        dict(name="maps ragged 500", op="maps", requests=500, new=0, new_max=7, length=8,
             length_max=8192, block=32, keys=True, order=3),
        # the tokens of a decode step of 32 chat sessions
        dict(name="append decode 32", op="append", tokens=32, kv_heads=8, dim=128, group=64,
             block=16, runs=1, dtype="bf16", order=4),
        # the turns those sessions append (256 to 1024 tokens each) in one call
        dict(name="append chat turns", op="append", tokens=20011, kv_heads=8, dim=128, group=32,
             block=16, runs=640, dtype="bf16", order=5),
        # one long document of 64K tokens moved to the 4-bit pool
        dict(name="append long document", op="append", tokens=65536, kv_heads=8, dim=128,
             group=128, block=32, runs=65536, dtype="fp16", order=6),
        # the smallest decode: 4 requests of about 512 tokens
        dict(name="attend decode 4", op="attend", requests=4, new=1, new_max=1, length=500,
             length_max=520, q_heads=8, kv_heads=2, dim=128, group=64, block=16, dtype="bf16",
             order=7),
        # 32 chat sessions decoding, histories up to 16K
        dict(name="attend decode 32", op="attend", requests=32, new=1, new_max=1, length=256,
             length_max=16384, q_heads=32, kv_heads=8, dim=128, group=64, block=16, dtype="bf16",
             order=8),
        # 8 decodes over 64K tokens each, 64 query heads on 8 KV heads
        dict(name="attend long 8", op="attend", requests=8, new=1, new_max=1, length=65000,
             length_max=65536, q_heads=64, kv_heads=8, dim=128, group=128, block=32,
             dtype="bf16", order=9),
        # the chat sessions again, four drafted tokens each to verify
        dict(name="attend drafts 32", op="attend", requests=32, new=4, new_max=4, length=256,
             length_max=16384, q_heads=32, kv_heads=8, dim=128, group=32, block=16, dtype="fp16",
             order=10),
        # 8 requests whose next 512-token chunk attends to 4096 tokens
        dict(name="attend chunks 8", op="attend", requests=8, new=512, new_max=512, length=4096,
             length_max=4096, q_heads=32, kv_heads=8, dim=128, group=64, block=16, dtype="bf16",
             order=11),
        # questions of odd lengths behind odd histories, small heads
        dict(name="attend odd questions", op="attend", requests=13, new=3, new_max=150,
             length=150, length_max=2999, q_heads=16, kv_heads=4, dim=64, group=32, block=48,
             dtype="fp16", order=12),
    ]


def _log(rng, low, high):
    """A whole number, its logarithm spread evenly over [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["maps", "append", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    dtype, block = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([16, 16, 32, 48, 64])
    order = rng.randrange(1000, 1 << 30)
    if op == "maps":
        requests = _log(rng, 1, 500)
        new = rng.choice([1, 1, 0, _log(rng, 1, 64)])
        longest = _log(rng, 16, 8192)
        return dict(op=op, requests=requests, new=new, new_max=max(1, new + rng.choice([0, 0, 7])),
                    length=rng.choice([1, 8, longest]), length_max=longest, block=block,
                    keys=rng.random() < 0.6, order=order)
    heads = rng.choice([(8, 2), (32, 8), (64, 8), (16, 4), (8, 8), (8, 1)])
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 65536 * 8 // max(8, heads[1])), kv_heads=heads[1],
                    dim=dim, group=group, block=block, runs=_log(rng, 1, 4096), dtype=dtype,
                    order=order)
    new = rng.choice([1, 1, 1, 2, 4, 7, _log(rng, 8, 512)])
    requests = _log(rng, 1, 64 if new < 8 else 16)
    most = min(65536, (8 * 65536 * 8) // (requests * heads[1]))
    if new >= 8:  # no more products than the listed chunks have
        cells = 8 * 512 * 4096 * 32 * 128
        most = min(most, 32768, max(2 * new, cells // (2 * requests * new * heads[0] * dim)))
    longest = _log(rng, new, max(new, most))
    return dict(op=op, requests=requests, new=new,
                new_max=new + (rng.randrange(0, new) if new > 1 else 0) // 2,
                length=rng.choice([1, max(1, longest // 2), longest]), length_max=longest,
                q_heads=heads[0], kv_heads=heads[1], dim=dim, group=group, block=block,
                dtype=dtype, order=order)


def _lens(case):
    """New tokens and lengths of each request: the case's own, whatever the seed."""
    r = random.Random(case["order"])
    n = [r.randint(case["new"], case["new_max"]) for _ in range(case["requests"])]
    low = min(case["length"], case["length_max"])
    s = [r.randint(low, case["length_max"]) for _ in range(case["requests"])]
    return n, [max(a, b) for a, b in zip(n, s)]


# --------------------------------------------------------------------- inputs
def _blocks(lengths, block, spare, g):
    """A table [requests, width] of shuffled blocks that holds the lengths,
    rows filled up with 0, and the number of blocks (`spare` in no row)."""
    dev = torch.device("cuda")
    per = torch.tensor([-(-n // block) for n in lengths], device=dev)
    width, total = max(1, -(-max(lengths) // block)), int(per.sum()) + spare
    perm = torch.randperm(total, generator=g, device=dev)
    j = torch.arange(width, device=dev)
    at = (torch.cumsum(per, 0) - per)[:, None] + j
    held = j < per[:, None]
    return torch.where(held, perm[at.clamp(max=total - 1)], 0).int(), total, perm


def _group_params(x, group):
    """Scale and lowest value of each group of x [..., dim] (16-bit), in 16 bits."""
    y = x.double().unflatten(-1, (-1, group))
    low, high = y.amin(-1), y.amax(-1)
    return ((high - low) / 15).to(x.dtype), low.to(x.dtype)


def _codes(x, scale, low, group):
    """4-bit codes of x as whole numbers (in 64 bits: a tie goes to the even one)."""
    y = x.double().unflatten(-1, (-1, group)) - low.double()[..., None]
    s = scale.double()[..., None]
    c = torch.where(s > 0, y / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15)
    return c.flatten(-2)


def _pack(k, v, kp, vp):
    """Bytes of units: codes [..., 16, dim] (uint8) and pairs [..., 16, groups, 2]."""
    w = k.shape[-1] // 32
    k = k.unflatten(-1, (w, 4, 4, 2)).transpose(-4, -3)   # t, w, byte, half
    v = v.unflatten(-1, (w, 8, 2, 2)).transpose(-4, -3)   # g, w, byte, half
    flat = [(c[..., 0] | c[..., 1] << 4).flatten(-4) for c in (k, v)]
    flat += [p.contiguous().view(torch.uint8).flatten(-3) for p in (kp, vp)]
    return torch.cat(flat, -1)


def _unpack(raw, dim, group, dtype):
    """Key and value codes (uint8, [..., 16, dim]) and pairs of units' bytes."""
    w, half = dim // 32, UNIT * dim // 2
    k = raw[..., :half].unflatten(-1, (UNIT, 4, w, 4))
    v = raw[..., half:2 * half].unflatten(-1, (UNIT, 8, w, 2))
    codes = [torch.stack((c & 15, c >> 4), -1).transpose(-4, -3).flatten(-4) for c in (k, v)]
    p = raw[..., 2 * half:].contiguous().view(dtype).unflatten(-1, (2, UNIT, dim // group, 2))
    return codes[0], codes[1], p[..., 0, :, :, :], p[..., 1, :, :, :]


def _unit_bytes(case):
    return UNIT * case["dim"] + 8 * UNIT * (case["dim"] // case["group"])


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s, op, block = {}, case["op"], case["block"]
    if op == "append":
        t, hk, d, dt = case["tokens"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
        # keys after their rotation: some channels are far larger than others
        loud = 1 + 3 * (torch.rand(hk, d, generator=g, device=dev) < 0.06)
        s["k"] = (torch.randn(t, hk, d, generator=g, device=dev) * loud).to(dt)
        s["v"] = torch.randn(t, hk, d, generator=g, device=dev).to(dt)
        n = min(case["runs"], t)
        blocks = -(-t // block) + -(-n // block) + 64
        # tokens fill shuffled blocks in order, in runs from different places
        perm = torch.randperm(blocks, generator=g, device=dev)
        place = torch.arange(blocks * block, device=dev)
        slots = perm[place // block] * block + place % block
        if n < t:
            starts = torch.randperm(blocks * block // n, generator=g, device=dev)[: -(-t // n)]
            slots = slots[(starts[:, None] * n + torch.arange(n, device=dev)).reshape(-1)]
        s["slots"] = slots[:t].contiguous()
        s["storage"] = torch.zeros(blocks, hk, block // UNIT, _unit_bytes(case),
                                   dtype=torch.uint8, device=dev)
        return s
    new, lengths = _lens(case)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    s["tokens"] = sum(new)
    if op == "maps":
        had = [-(-(a - n) // block) for a, n in zip(lengths, new)]
        need = sum(-(-a // block) - h for a, h in zip(lengths, had))
        full, total, perm = _blocks(lengths, block, 32, g)
        j = torch.arange(full.shape[1], device=dev)
        kept = j < torch.tensor(had, device=dev)[:, None]
        # what the requests do not hold yet is free, in another order
        taken = torch.zeros(total, dtype=torch.bool, device=dev)
        taken[full[kept].long()] = True
        free = perm[torch.randperm(total, generator=g, device=dev)]
        free = free[~taken[free]]
        s["tables"] = torch.where(kept, full, 0).int()
        s["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
        s["free"] = free.int()
        s["free_count"] = torch.tensor([free.numel()], dtype=torch.int32, device=dev)
        s["blocks"], s["need"] = total, need
        s["keys"] = sum(lengths) if case["keys"] else 0
        return s
    hq, hk, d, group = case["q_heads"], case["kv_heads"], case["dim"], case["group"]
    dt = DTYPES[case["dtype"]]
    s["q"] = (1.5 * torch.randn(s["tokens"], hq, d, generator=g, device=dev)).to(dt)
    s["tables"], blocks, _ = _blocks(lengths, block, 8, g)
    s["starts"] = torch.tensor([0, *new], device=dev).cumsum(0).int()
    units = block // UNIT
    s["storage"] = torch.empty(blocks, hk, units, _unit_bytes(case), dtype=torch.uint8, device=dev)
    loud = 1 + 3 * (torch.rand(hk, 1, 1, d, generator=g, device=dev) < 0.06)
    at = max(1, (1 << 25) // (hk * block * d))  # the pool is filled some blocks at a time
    for lo in range(0, blocks, at):
        n = min(at, blocks - lo)
        parts = []
        for wide in (loud, 1.0):
            x = (torch.randn(n, hk, units, UNIT, d, generator=g, device=dev) * wide).to(dt)
            scale, low = _group_params(x, group)
            parts.append((_codes(x, scale, low, group).byte(), torch.stack((scale, low), -1)))
        (kc, kp), (vc, vp) = parts
        s["storage"][lo:lo + n] = _pack(kc, vc, kp, vp)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "attend":  # the batch's lengths, as the plain form reads them
        new, lengths = _lens(case)
        s["longest"], s["most_new"] = max(lengths), max(new)
    if own and case["op"] != "maps":  # the handle of the pool that a server keeps
        from cacheslide_b200 import kv4

        s["pool"] = kv4.PagedKV4(s["storage"], case["dim"], DTYPES[case["dtype"]], case["group"])
    return s


# ------------------------------------------------------------------ plain form
def _plain_maps(s):
    case, dev = s["case"], s["lengths"].device
    block, table = case["block"], s["tables"].long()
    length, new = s["lengths"].long(), s["new"].long()
    had, want = (length - new + block - 1) // block, (length + block - 1) // block
    need = want - had
    first = need.cumsum(0) - need
    j = torch.arange(table.shape[1], device=dev)
    at = s["free_count"].long() - 1 - (first[:, None] + j - had[:, None])
    fresh = (j >= had[:, None]) & (j < want[:, None])
    table = torch.where(fresh, s["free"].long()[at.clamp(0, s["free"].numel() - 1)], table)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    starts, key_starts = torch.cat((zero, new.cumsum(0))), torch.cat((zero, length.cumsum(0)))

    def slots(request, position):
        return table[request, position // block] * block + position % block

    i = torch.arange(s["tokens"], device=dev)
    r = torch.searchsorted(starts[1:], i, right=True)
    positions = (length - new)[r] + i - starts[r]
    out = dict(tables=table.int(), starts=starts.int(), positions=positions,
               slots=slots(r, positions), free_left=(s["free_count"] - need.sum()).int())
    if case["keys"]:
        i = torch.arange(s["keys"], device=dev)
        r = torch.searchsorted(key_starts[1:], i, right=True)
        out["key_slots"] = slots(r, i - key_starts[r])
    return out


def _plain_append(s):
    case, group = s["case"], s["case"]["group"]
    out = {}
    for name in ("k", "v"):
        x = s[name]
        scale, low = _group_params(x, group)
        c = _codes(x, scale, low, group).float().unflatten(-1, (-1, group))
        out[name] = (c * scale.float()[..., None] + low.float()[..., None]).flatten(-2).to(x.dtype)
    return out


def _plain_attend(s):
    case, q, dev = s["case"], s["q"], s["q"].device
    hk, d, group, block = case["kv_heads"], case["dim"], case["group"], case["block"]
    r, gq = case["requests"], case["q_heads"] // case["kv_heads"]
    units = -(-s["longest"] // UNIT)
    raw = s["storage"][s["tables"].long()].transpose(1, 2)  # [r, hk, blocks, units, bytes]
    raw = raw.flatten(2, 3)[:, :, :units]
    kc, vc, kp, vp = _unpack(raw, d, group, q.dtype)
    k, v = ((c.float().unflatten(-1, (-1, group)) * p[..., :1].float() + p[..., 1:].float())
            .flatten(-2).flatten(2, 3) for c, p in ((kc, kp), (vc, vp)))  # [r, hk, keys, d]
    start, n = s["starts"][:-1].long(), s["most_new"]
    count = s["starts"][1:].long() - start
    i, j = torch.arange(n, device=dev), torch.arange(units * UNIT, device=dev)
    live = i < count[:, None]
    row = torch.where(live, start[:, None] + i, 0)
    seen = j <= (s["lengths"].long() - count)[:, None, None] + i[:, None]  # [r, n, keys]
    x = q[row].float().view(r, n, hk, gq, d).permute(0, 2, 1, 3, 4).reshape(r, hk, n * gq, d)
    z = torch.matmul(x * (1 / math.sqrt(d)), k.transpose(-1, -2)).view(r, hk, n, gq, -1)
    z.masked_fill_(~seen[:, None, :, None], float("-inf"))
    z = z.sub_(z.amax(-1, keepdim=True)).exp_()
    total = z.sum(-1, keepdim=True)
    o = torch.matmul(z.view(r, hk, n * gq, -1), v).view(r, hk, n, gq, d) / total
    return o.permute(0, 2, 1, 3, 4).reshape(r, n, hk * gq, d)[live].to(q.dtype)


# --------------------------------------------------------------- the framework
def _own_maps(s):
    from cacheslide_b200 import tables

    case = s["case"]
    m = tables.step_maps(s["lengths"], s["new"], s["tables"], case["block"], s["blocks"],
                         tokens=s["tokens"], keys=s["keys"], free=s["free"],
                         free_count=s["free_count"])
    out = dict(tables=s["tables"], starts=m.starts, positions=m.positions, slots=m.slots,
               free_left=m.free_left)
    if case["keys"]:
        out["key_slots"] = m.key_slots
    return out


def _own_append(s):
    from cacheslide_b200 import kv4

    kv4.append(s["pool"], s["slots"], s["k"], s["v"])
    k, v = kv4.gather(s["pool"], s["slots"])
    return dict(k=k, v=v)


def _own_attend(s):
    from cacheslide_b200 import kv4

    one = s["case"]["new_max"] == 1  # a decode step has one token a request
    return kv4.attention(s["q"], s["pool"], s["tables"], s["lengths"],
                         None if one else s["starts"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"maps": _own_maps, "append": _own_append, "attend": _own_attend}[op](state)
    return {"maps": _plain_maps, "append": _plain_append, "attend": _plain_attend}[op](state)


# ------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "append":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        record = values // 2 + 4 * (values // case["group"])
        # rows in, records out; records in, values out
        return dict(bytes=2 * (2 * values + record + 8 * case["tokens"]), flops=8 * values)
    new, lengths = _lens(case)
    b, block = case["requests"], case["block"]
    if case["op"] == "maps":
        want = [-(-a // block) for a in lengths]
        need = [w - -(-(a - n) // block) for w, a, n in zip(want, lengths, new)]
        read = sum(want) if case["keys"] else sum(
            -(-a // block) - (a - n) // block for a, n in zip(lengths, new) if n)
        return dict(bytes=8 * b + 4 * (read + 2 * sum(need)) + 4 * (b + 1) + 16 * sum(new)
                    + (8 * sum(lengths) if case["keys"] else 0),
                    flops=4 * (sum(new) + (sum(lengths) if case["keys"] else 0)))
    d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    cells = sum(n * (a - n) + n * (n + 1) // 2 for n, a in zip(new, lengths))
    return dict(bytes=sum(lengths) * hk * (d + 8 * (d // case["group"]))
                + 4 * sum(-(-a // block) for a in lengths) + 4 * sum(new) * hq * d,
                flops=4 * d * hq * cells)


# ----------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "maps":  # whole numbers: nothing is rounded
        return None
    s = _inputs(case, seed)
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):  # the nearest of a group's sixteen values
            t, hk, d = s[name].shape
            x = s[name].view(t, hk, d // case["group"], case["group"])
            low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            step = ((high.double() - low.double()) / 15).to(x.dtype).double()
            low = low.double()
            part = (x.double() - low) / step.clamp(min=5e-324)
            out[name] = (low + step * part.round().clamp(0, 15)).view(t, hk, d)
        return out
    new, lengths = _lens(case)
    d, hk, group, block = case["dim"], case["kv_heads"], case["group"], case["block"]
    gq, t, out = case["q_heads"] // hk, 0, []
    w, half = d // 32, UNIT * d // 2
    e = torch.arange(d, device=s["q"].device)
    # the byte of an element's code in a token's codes, and the half of that byte
    key_at = 4 * ((e % 32 // 8) * w + e // 32) + e % 8 // 2
    value_at = 2 * ((e % 32 // 4) * w + e // 32) + e % 4 // 2
    shift = (4 * (e % 2)).to(torch.uint8)
    for b, (n, m) in enumerate(zip(new, lengths)):
        at = torch.arange(m, device=e.device)
        unit = s["storage"][s["tables"][b, at // block].long(), :, at % block // UNIT]
        lane = (at % UNIT)[:, None]
        pairs = unit[..., 2 * half:].contiguous().view(s["q"].dtype).double()
        rows = []
        for place, base, first in ((key_at, 0, 0), (value_at, half, 2 * UNIT * (d // group))):
            where = base + lane * (d // 2) + place
            code = unit.gather(2, where[:, None].expand(m, hk, d)) >> shift & 15
            pair = first + 2 * (lane * (d // group) + e // group)
            pick = [pairs.gather(2, (pair + o)[:, None].expand(m, hk, d)) for o in (0, 1)]
            rows.append(torch.addcmul(pick[1], code.double(), pick[0]))
        q = s["q"][t:t + n].double().view(n, hk, gq, d)
        z = torch.einsum("nhgd,khd->nhgk", q, rows[0]) / math.sqrt(d)
        z.masked_fill_((at > (m - n + at.new_tensor(range(n)))[:, None])[:, None, None], -math.inf)
        o = torch.einsum("nhgk,khd->nhgd", torch.softmax(z, -1), rows[1])
        out.append(o.reshape(n, hk * gq, d))
        t += n
    return torch.cat(out)
