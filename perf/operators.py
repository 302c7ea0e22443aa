"""Rotary attention over the paged KV pool: three operators and their cases.

* ``norm_rope``: RMS norm of each query / key head and the position rotation
  in one pass (``rotary.qk_norm_rope``), forward alone or with its gradients;
* ``append``: keys and values appended to the paged pool, the keys rotated
  (and normed) on the way, the queries rotated in the same call
  (``rotary.append_rotated``);
* ``prefix``: attention of a batch whose requests share a long prefix in the
  pool, the prefix read once for all of them (``prefix.SharedPrefixAttention``).

``run`` computes either the plain form (elementary torch operations in 32
bits) or, with ``own`` set, the framework's operators; ``exact`` restates the
definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # the tiny decoder of the CPU smoke configuration (3 chunks of 32
        # tokens and a 16-token suffix, 4/2 heads of 16), one training step
        dict(name="norm_rope tiny train", op="norm_rope", tokens=112, q_heads=4, kv_heads=2,
             dim=16, rot=16, interleaved=False, train=True, dtype="fp32", order=1),
        # an odd-length prompt's projections at inference, half of each head rotated
        dict(name="norm_rope odd forward", op="norm_rope", tokens=1537, q_heads=64, kv_heads=8,
             dim=64, rot=32, interleaved=True, train=False, dtype="fp16", order=2),
        # one layer of a training step: a batch of 8 sequences of 4096 tokens
        dict(name="norm_rope batch train", op="norm_rope", tokens=32768, q_heads=32, kv_heads=8,
             dim=128, rot=128, interleaved=False, train=True, dtype="bf16", order=3),
        # a decode step of 32 chat sessions: one token each, scattered slots
        dict(name="append decode 32", op="append", tokens=32, q_heads=32, kv_heads=8, dim=128,
             rot=128, interleaved=False, norm=True, block=16, runs=1, dtype="bf16", order=4),
        # the turns those sessions append (256 to 1024 tokens each) in one call
        dict(name="append chat turns", op="append", tokens=20011, q_heads=32, kv_heads=8,
             dim=128, rot=128, interleaved=False, norm=True, block=16, runs=640, dtype="bf16",
             order=5),
        # one long document of 64K tokens written to the pool, without head norms
        dict(name="append long document", op="append", tokens=65536, q_heads=64, kv_heads=8,
             dim=128, rot=128, interleaved=True, norm=False, block=16, runs=65536, dtype="fp16",
             order=6),
        # the smallest decode: 4 requests on one 512-token prompt
        dict(name="prefix decode 4", op="prefix", requests=4, queries=1, queries_max=1,
             prefix=512, suffix=1, suffix_max=64, groups=1, q_heads=8, kv_heads=2, dim=128,
             block=16, scattered=False, dtype="bf16", order=7),
        # a retrieval batch: 64 questions on the same ten 512-token chunks, decoding
        dict(name="prefix decode 64", op="prefix", requests=64, queries=1, queries_max=1,
             prefix=5120, suffix=64, suffix_max=96, groups=1, q_heads=32, kv_heads=8, dim=128,
             block=16, scattered=False, dtype="bf16", order=8),
        # 32 chat sessions in two tenants (a 2K system prompt each), histories
        # up to 16K, four drafted tokens a session to verify; relocated slots
        dict(name="prefix drafts 32", op="prefix", requests=32, queries=4, queries_max=4,
             prefix=2048, suffix=256, suffix_max=16384, groups=2, q_heads=32, kv_heads=8,
             dim=128, block=16, scattered=True, dtype="fp16", order=9),
        # 8 decodes over one 64K document, 64 query heads on 8 KV heads
        dict(name="prefix long 8", op="prefix", requests=8, queries=1, queries_max=1,
             prefix=65536, suffix=1, suffix_max=64, groups=1, q_heads=64, kv_heads=8, dim=128,
             block=16, scattered=False, dtype="bf16", order=10),
        # the questions of that retrieval batch prefilled: 64 tokens each
        dict(name="prefix questions 64", op="prefix", requests=64, queries=64, queries_max=64,
             prefix=5120, suffix=64, suffix_max=64, groups=1, q_heads=32, kv_heads=8, dim=128,
             block=16, scattered=False, dtype="bf16", order=11),
        # questions of odd lengths behind an odd prefix, small heads
        dict(name="prefix odd questions", op="prefix", requests=13, queries=3, queries_max=150,
             prefix=2999, suffix=150, suffix_max=333, groups=1, q_heads=16, kv_heads=4, dim=64,
             block=32, scattered=False, dtype="fp16", order=12),
    ]


def _log(rng, low, high):
    """A whole number, its logarithm spread evenly over [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "prefix", "prefix"])
    heads = rng.choice([(8, 2), (32, 8), (64, 8), (16, 4), (8, 8), (32, 4)])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    order = rng.randrange(1000, 1 << 30)
    if op == "norm_rope":
        train = rng.random() < 0.5
        return dict(op=op, tokens=_log(rng, 1, 32768 * 32 * 128 // (heads[0] * dim)
                                       if heads[0] * dim > 4096 else 32768),
                    q_heads=heads[0], kv_heads=heads[1], dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.4,
                    train=train, dtype=rng.choice([dtype, dtype, "fp32"]) if dim == 64 else dtype,
                    order=order)
    if op == "append":
        tokens = _log(rng, 1, 32768)
        return dict(op=op, tokens=tokens, q_heads=heads[0], kv_heads=heads[1], dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.6, block=rng.choice([16, 16, 32]),
                    runs=_log(rng, 1, 4096), dtype=dtype, order=order)
    groups = rng.choice([1, 1, 1, 2, 3])
    requests = groups * _log(rng, 1, 24 if groups > 1 else 64)
    queries = rng.choice([1, 1, 1, 2, 5, _log(rng, 6, 64)])
    prefix = _log(rng, 1, 32768 if queries < 6 and requests <= 32 else 5120)
    suffix = _log(rng, 1, 512)
    return dict(op=op, requests=requests, queries=queries,
                queries_max=queries + (rng.randrange(0, queries) if queries > 1 else 0) // 2,
                prefix=prefix, suffix=suffix,
                suffix_max=suffix + _log(rng, 1, 4096 if requests <= 32 else 256), groups=groups,
                q_heads=heads[0], kv_heads=heads[1], dim=dim, block=rng.choice([16, 16, 32]),
                scattered=rng.random() < 0.3, dtype=dtype, order=order)


def _lens(case):
    """Query and suffix lengths of each request: the case's own, whatever the seed."""
    r = random.Random(case["order"])
    q = [r.randint(case["queries"], case["queries_max"]) for _ in range(case["requests"])]
    s = [r.randint(case["suffix"], case["suffix_max"]) for _ in range(case["requests"])]
    return q, [max(a, b) for a, b in zip(q, s)]


# --------------------------------------------------------------------- inputs
def _tables(positions, rot, device):
    """cos and sin of every position below `positions`, [positions, rot / 2]."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        x = torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)
        return x.mul_(scale).to(dt)

    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    s = {}
    if case["op"] in ("norm_rope", "append"):
        t = case["tokens"]
        s["cos"], s["sin"] = _tables(max(t, 4096), case["rot"], dev)
        s["positions"] = torch.arange(t, device=dev)
        if t <= 4096:  # a decode batch or a short prompt: anywhere in its context
            s["positions"] = torch.randint(0, 4096, (t,), generator=g, device=dev)
        s["q"] = rand(t, hq, d, scale=1.5)
        s["k"] = rand(t, hk, d, scale=1.5)
        s["qw"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dt)
        s["kw"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dt)
        if case["op"] == "norm_rope":
            if case["train"]:
                s["gq"], s["gk"] = rand(t, hq, d), rand(t, hk, d)
        else:
            s["v"] = rand(t, hk, d)
            bs = case["block"]
            blocks = -(-t // bs) * 2 if t < 4096 else -(-t // bs) + 64
            s["cache"] = torch.zeros(blocks, hk, bs, 2 * d, dtype=dt, device=dev)
            # tokens fill shuffled blocks in order; a decode step's tokens
            # (short runs) come from different places of the pool
            perm = torch.randperm(blocks, generator=g, device=dev)
            place = torch.arange(blocks * bs, device=dev)
            slots = perm[place // bs] * bs + place % bs
            if case["runs"] < t:
                n = case["runs"]
                starts = torch.randperm(blocks * bs // n, generator=g, device=dev)[: -(-t // n)]
                at = (starts[:, None] * n + torch.arange(n, device=dev)).reshape(-1)[:t]
                slots = slots[at]
            s["slots"] = slots[:t].contiguous()
        return s
    bs, groups, length = case["block"], case["groups"], case["prefix"]
    ql, sl = _lens(case)
    tokens, own_keys = sum(ql), sum(sl)
    # every group's prefix and every request's own keys fill blocks of their own
    pb = -(-length // bs)
    lens = torch.tensor(sl, device=dev)
    sb = (lens + bs - 1) // bs
    blocks = groups * pb + int(sb.sum()) + 8
    perm = torch.randperm(blocks, generator=g, device=dev)
    at = torch.arange(length, device=dev)
    s["prefix_slots"] = (perm[(torch.arange(groups, device=dev)[:, None] * pb + at // bs)] * bs
                         + at % bs).reshape(-1)
    first = groups * pb + torch.cumsum(sb, 0) - sb
    begin = torch.cumsum(lens, 0) - lens
    of = torch.repeat_interleave(torch.arange(len(sl), device=dev), lens)
    j = torch.arange(own_keys, device=dev) - begin[of]
    s["suffix_slots"] = perm[first[of] + j // bs] * bs + j % bs
    if case["scattered"]:  # one key in eight was relocated: any other slot of the pool
        n = s["suffix_slots"].numel()
        move = torch.rand(n, generator=g, device=dev) < 0.125
        idx = move.nonzero().flatten()
        mixed = idx[torch.randperm(idx.numel(), generator=g, device=dev)]
        s["suffix_slots"][idx] = s["suffix_slots"][mixed]
    s["cache"] = rand(blocks, hk, bs, 2 * d)
    s["q"] = rand(tokens, hq, d, scale=1.5)
    s["query_lens"], s["suffix_lens"] = ql, sl
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "prefix":  # the batch's lengths, as the plain form reads them
        s.update(_padded(s["query_lens"], s["suffix_lens"]))
    if own and case["op"] == "prefix":  # the batch's work plan, kept for all layers of a step
        from cacheslide_b200 import prefix

        per = case["requests"] // case["groups"]
        s["plan"] = prefix.SharedPrefixAttention(
            case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]],
            torch.device("cuda"), query_lens=s["query_lens"], suffix_lens=s["suffix_lens"],
            prefix_lens=[case["prefix"]] * case["groups"], group_sizes=[per] * case["groups"])
    return s


def _padded(ql, sl):
    dev = torch.device("cuda")
    q, k = torch.tensor(ql, device=dev), torch.tensor(sl, device=dev)
    i, j = torch.arange(max(ql), device=dev), torch.arange(max(sl), device=dev)
    q0, k0 = torch.cumsum(q, 0) - q, torch.cumsum(k, 0) - k
    return dict(
        row=torch.where(i < q[:, None], q0[:, None] + i, 0),
        live=i < q[:, None],
        col=torch.where(j < k[:, None], k0[:, None] + j, 0),
        seen=j[None, None, :] <= (k - q)[:, None, None] + i[None, :, None])


# ------------------------------------------------------------------ plain form
def _turn(x, cos, sin, interleaved):
    """x [tokens, heads, dim] with its first 2 * cos.shape[-1] values rotated."""
    rot = 2 * cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        out = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = head[..., : rot // 2], head[..., rot // 2:]
        out = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((out, rest), -1)


def _norm_turn(x, w, cos, sin, interleaved):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    return _turn(x, cos, sin, interleaved)


def _norm_turn_grad(x, w, dy, cos, sin, interleaved):
    """Gradients of the above: the rotation undone, then the norm's."""
    x, w = x.float(), w.float()
    g = _turn(dy.float(), cos, -sin, interleaved)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    gw = g * w
    return r * (gw - n * (gw * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))


def _plain_norm_rope(s):
    case, dt = s["case"], s["q"].dtype
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    how = cos, sin, case["interleaved"]
    out = dict(q=_norm_turn(s["q"], s["qw"], *how).to(dt),
               k=_norm_turn(s["k"], s["kw"], *how).to(dt))
    if case["train"]:
        dq, dqw = _norm_turn_grad(s["q"], s["qw"], s["gq"], *how)
        dk, dkw = _norm_turn_grad(s["k"], s["kw"], s["gk"], *how)
        out.update(dq=dq.to(dt), dk=dk.to(dt), dqw=dqw.to(dt), dkw=dkw.to(dt))
    return out


def _plain_append(s):
    case, dt, cache = s["case"], s["q"].dtype, s["cache"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    how = cos, sin, case["interleaved"]
    bs, d = cache.shape[2], case["dim"]
    k = _norm_turn(s["k"], s["kw"] if case["norm"] else None, *how)
    block, at = s["slots"] // bs, s["slots"] % bs
    cache[block, :, at, :d] = k.to(dt)
    cache[block, :, at, d:] = s["v"]
    return dict(q=_norm_turn(s["q"], s["qw"] if case["norm"] else None, *how).to(dt), cache=cache)


def _plain_prefix(s):
    case, q, cache = s["case"], s["q"], s["cache"]
    bs, d, hk = cache.shape[2], case["dim"], case["kv_heads"]
    gq, groups, scale = case["q_heads"] // hk, case["groups"], 1 / math.sqrt(case["dim"])
    row, col, live, seen = s["row"], s["col"], s["live"], s["seen"]
    b, n = row.shape
    qp = q[row].float().view(b, n, hk, gq, d).permute(0, 2, 1, 3, 4).contiguous()  # [b, hk, n, gq, d]
    qp = qp * scale
    own_slots = s["suffix_slots"][col]
    kv = cache[own_slots // bs, :, own_slots % bs].float().permute(0, 2, 1, 3)  # [b, hk, keys, 2d]
    mine = torch.matmul(qp.reshape(b, hk, n * gq, d), kv[..., :d].transpose(-1, -2))
    hide = ~seen[:, None, :, None, :].expand(b, 1, n, gq, seen.shape[-1])
    mine = mine.view(b, hk, n, gq, -1).masked_fill(hide, float("-inf"))
    pkv = cache[s["prefix_slots"] // bs, :, s["prefix_slots"] % bs].float()
    pkv = pkv.view(groups, -1, hk, 2 * d).transpose(1, 2)  # [groups, hk, prefix, 2d]
    per = b // groups
    qg = qp.view(groups, per, hk, n * gq, d).transpose(1, 2).reshape(groups, hk, -1, d)
    shared = torch.matmul(qg, pkv[..., :d].transpose(-1, -2))
    top = shared.amax(-1).view(groups, hk, per, n, gq).transpose(1, 2).reshape(b, hk, n, gq)
    top = torch.maximum(top, mine.amax(-1))[..., None]
    tg = top.view(groups, per, hk, n * gq, 1).transpose(1, 2).reshape(groups, hk, -1, 1)
    shared, mine = torch.exp(shared.sub_(tg)), torch.exp(mine - top)
    part = torch.matmul(shared, pkv[..., d:])
    back = lambda x: x.view(groups, hk, per, n, gq, -1).transpose(1, 2).reshape(b, hk, n, gq, -1)  # noqa: E731
    total = back(shared.sum(-1, keepdim=True)) + mine.sum(-1, keepdim=True)
    out = back(part) + torch.matmul(mine.view(b, hk, n * gq, -1), kv[..., d:]).view(b, hk, n, gq, d)
    out = (out / total).permute(0, 2, 1, 3, 4).reshape(b, n, hk * gq, d)
    return out[live].to(q.dtype)


# --------------------------------------------------------------- the framework
def _own_norm_rope(s):
    from cacheslide_b200 import rotary

    case = s["case"]
    leaves = [s[n].detach().requires_grad_(case["train"]) for n in ("q", "k", "qw", "kw")]
    q, k = rotary.qk_norm_rope(*leaves[:2], s["positions"], s["cos"], s["sin"], *leaves[2:],
                               eps=EPS, interleaved=case["interleaved"])
    if not case["train"]:
        return dict(q=q, k=k)
    dq, dk, dqw, dkw = torch.autograd.grad((q, k), leaves, (s["gq"], s["gk"]))
    return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk, dqw=dqw, dkw=dkw)


def _own_append(s):
    from cacheslide_b200 import rotary

    case = s["case"]
    w = (s["qw"], s["kw"]) if case["norm"] else (None, None)
    q = rotary.append_rotated(s["cache"], s["slots"], s["k"], s["v"], s["positions"], s["cos"],
                              s["sin"], query=s["q"], q_weight=w[0], k_weight=w[1], eps=EPS,
                              interleaved=case["interleaved"])
    return dict(q=q, cache=s["cache"])


def _own_prefix(s):
    return s["plan"](s["q"], s["cache"], s["prefix_slots"], s["suffix_slots"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm_rope": _own_norm_rope, "append": _own_append, "prefix": _own_prefix}[op](state)
    return {"norm_rope": _plain_norm_rope, "append": _plain_append, "prefix": _plain_prefix}[op](state)


# ------------------------------------------------------------------------ work
def work(case):
    hq, hk, d, es = case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "prefix":
        ql, sl = _lens(case)
        keys = case["groups"] * case["prefix"] + sum(sl)
        cells = sum(q * case["prefix"] + q * (n - q) + q * (q + 1) // 2 for q, n in zip(ql, sl))
        return dict(bytes=keys * (hk * 2 * d * es + 8) + 2 * sum(ql) * hq * d * es,
                    flops=4 * d * hq * cells)
    t = case["tokens"]
    rows = t * (hq + hk) * d
    table = t * (8 + 4 * case["rot"])
    if case["op"] == "append":
        values = rows + t * hk * d
        return dict(bytes=2 * values * es + table + 8 * t, flops=8 * rows)
    if case["train"]:  # read x and dy, write y and dx
        return dict(bytes=4 * rows * es + table, flops=24 * rows)
    return dict(bytes=2 * rows * es + table, flops=8 * rows)


# ----------------------------------------------------------------------- exact
def _exact_rotation(x, cos, sin, interleaved):
    """The rotation as a product with complex numbers of modulus one."""
    rot = 2 * cos.shape[-1]
    z = x[..., :rot]
    z = (torch.complex(z[..., 0::2], z[..., 1::2]) if interleaved
         else torch.complex(z[..., : rot // 2], z[..., rot // 2:]))
    z = z * torch.complex(cos, sin)[:, None]
    out = x.clone()
    if interleaved:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., : rot // 2], out[..., rot // 2: rot] = z.real, z.imag
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "prefix":
        cache, bs, d, hk = s["cache"].double(), case["block"], case["dim"], case["kv_heads"]
        gq, per = case["q_heads"] // hk, case["requests"] // case["groups"]
        out, t, k0 = [], 0, 0
        for b, (n, m) in enumerate(zip(s["query_lens"], s["suffix_lens"])):
            grp, length = b // per, case["prefix"]
            slots = torch.cat((s["prefix_slots"][grp * length:(grp + 1) * length],
                               s["suffix_slots"][k0:k0 + m]))
            kv = cache[slots // bs, :, slots % bs]  # [keys, hk, 2d]
            q = s["q"][t:t + n].double().view(n, hk, gq, d)
            z = torch.einsum("nhgd,khd->nhgk", q, kv[..., :d]) / math.sqrt(d)
            limit = length + m - n + torch.arange(n, device=q.device)
            z.masked_fill_((torch.arange(len(slots), device=q.device) > limit[:, None])[:, None, None],
                           -math.inf)
            o = torch.einsum("nhgk,khd->nhgd", torch.softmax(z, -1), kv[..., d:])
            out.append(o.reshape(n, hk * gq, d))
            t, k0 = t + n, k0 + m
        return torch.cat(out)
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    normed = case["op"] == "norm_rope" or case["norm"]

    def forward(x, w):
        if normed:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        return _exact_rotation(x, cos, sin, case["interleaved"])

    train = case["op"] == "norm_rope" and case["train"]
    q, k, qw, kw = (s[n].detach().double().requires_grad_(train) for n in ("q", "k", "qw", "kw"))
    yq, yk = forward(q, qw), forward(k, kw)
    if case["op"] == "append":
        cache, bs, d = s["cache"].double(), case["block"], case["dim"]
        cache[s["slots"] // bs, :, s["slots"] % bs] = torch.cat((yk, s["v"].double()), -1)
        return dict(q=yq, cache=cache)
    if not train:
        return dict(q=yq, k=yk)
    dq, dk, dqw, dkw = torch.autograd.grad((yq, yk), (q, k, qw, kw),
                                           (s["gq"].double(), s["gk"].double()))
    return dict(q=yq.detach(), k=yk.detach(), dq=dq, dk=dk, dqw=dqw, dkw=dkw)
