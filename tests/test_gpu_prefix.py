"""Attention behind shared prefixes against float64 (``oracle.prefix``).

Tolerances.  With u the unit roundoff of the type (2^-8 bf16, 2^-11 fp16,
2^-24 fp32), A = sum p|v| / sum p and S the largest sum |q k| scale of the row:
the output is rounded once (u |o|), 16-bit kernels round each p once (u A),
scores carry float32 products and sums of D terms ((D + 32) 2^-23 S, a relative
error of p as large), 2^x is within 2^-19, and sums over n keys in float32
chains of at most n / 4 (and 64 joins) are within (n / 4 + 64) 2^-23."""

from __future__ import annotations

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200.paged import NativePagedKV
from cacheslide_b200.prefix import SharedPrefixAttention
from oracle import prefix as oprefix

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def batch(device, hq, hk, d, dtype, queries, suffixes, prefixes, sizes=None, block=16, seed=0,
          scattered=0.0, spare=3, fill=float("nan")):
    """A pool whose unused places hold NaN, and the batch's slots in it."""
    g = torch.Generator(device=device).manual_seed(seed)
    runs = list(prefixes) + list(suffixes)
    need = [-(-n // block) for n in runs]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=g, device=device)
    slots, at = [], 0
    for n, nb in zip(runs, need):
        j = torch.arange(n, device=device)
        slots.append(perm[at + j // block] * block + j % block)
        at += nb
    pre = torch.cat(slots[:len(prefixes)] or [perm[:0]])
    suf = torch.cat(slots[len(prefixes):] or [perm[:0]])
    if scattered:
        both = torch.cat((pre, suf))
        idx = (torch.rand(both.numel(), generator=g, device=device) < scattered).nonzero().flatten()
        both[idx] = both[idx[torch.randperm(idx.numel(), generator=g, device=device)]]
        pre, suf = both[:pre.numel()].clone(), both[pre.numel():].clone()
    cache = torch.full((blocks, hk, block, 2 * d), fill, dtype=dtype, device=device)
    used = torch.cat((pre, suf))
    cache[used // block, :, used % block] = torch.randn(
        used.numel(), hk, 2 * d, generator=g, device=device).to(dtype)
    q = (1.5 * torch.randn(sum(queries), hq, d, generator=g, device=device)).to(dtype)
    lens = dict(query_lens=list(queries), suffix_lens=list(suffixes), prefix_lens=list(prefixes),
                group_sizes=sizes)
    return dict(query=q, cache=cache, prefix_slots=pre, suffix_slots=suf), lens


def plan_of(s, lens):
    return SharedPrefixAttention(s["query"].shape[1], s["cache"].shape[1], s["query"].shape[2],
                                 s["query"].dtype, s["query"].device, **lens)


def bounds(dtype, d, lens, want, lse, size, score):
    n = max(lens["prefix_lens"]) + max(lens["suffix_lens"])
    rel = 2.0**-19 + (d + 32) * 2.0**-23 * score + (n / 4 + 64) * 2.0**-23
    p_round = U[dtype] if dtype != FP else 0.0
    tiny = 2.0**-24 if dtype == HF else 0.0  # fp16: the output's and p's subnormals
    out = U[dtype] * want.abs() + (p_round + rel[..., None]) * size + tiny * (1 + size)
    return out, rel + lse.abs().nan_to_num(0, 0, 0) * 2.0**-23


def check(s, lens, got, lse_got, **kw):
    want, lse, size, score = oprefix.attention(s["query"], s["cache"], s["prefix_slots"],
                                               s["suffix_slots"], **lens, **kw)
    b_out, b_lse = bounds(s["query"].dtype, s["query"].shape[2], lens, want, lse, size, score)
    empty = lse == -float("inf")
    assert torch.equal(empty, lse_got == -float("inf"))
    assert not got[empty].any()
    off = (got.double() - want).abs()
    assert (off <= b_out).all(), float((off / b_out.clamp_min(1e-30)).max())
    off = (lse_got.double() - lse).abs()[~empty]
    assert (off <= b_lse[~empty]).all(), float(off.max())


def run(s, lens, **kw):
    return plan_of(s, lens)(s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"],
                            return_lse=True, **kw)


LAYOUTS = {
    "one token one key": ([1], [1], [0]),
    "one token, prefix of one": ([1], [0], [1]),
    "one token long": ([1], [37], [2999]),
    "decode": ([1] * 13, list(range(1, 14)), [515]),
    "decode many": ([1] * 70, [64 + 5 * (i % 9) for i in range(70)], [1280]),
    "drafts": ([4, 1, 3, 4, 2] * 3, [300, 1, 70, 1500, 2] * 3, [640]),
    "questions": ([50, 1, 130, 17, 0, 64], [50, 9, 130, 300, 12, 64], [400]),
    "no prefix": ([5, 1, 33], [5, 700, 129], [0]),
    "rows that see nothing": ([6, 3, 2], [2, 0, 5], [0]),
    "fewer own keys than queries": ([9, 4], [4, 0], [130]),
    "only the prefix": ([3, 40], [0, 0], [257]),
    "groups": ([1, 2, 5, 1, 1, 7], [3, 200, 5, 1, 90, 300], [130, 0, 700], [2, 1, 3]),
    "empty groups": ([1, 1, 1], [5, 6, 7], [100, 50, 0, 33], [1, 0, 2, 0]),
    "long question": ([700], [700], [300]),
    "wide batch": ([64] * 12, [64] * 12, [513]),
    "wide ragged": ([90, 64, 128, 3, 200, 77], [90, 100, 128, 3, 400, 77], [385]),
    "wide groups": ([100, 80, 128, 60], [100, 80, 200, 60], [129, 600], [1, 3]),
}
HEADS = [(32, 8, 128, BF), (8, 2, 64, HF), (16, 1, 128, HF), (3, 3, 64, BF)]


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("hq,hk,d,dtype", HEADS)
def test_layouts(cuda, name, hq, hk, d, dtype):
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    status = N.Status(cuda)
    got, lse = run(s, lens, status=status)
    assert status.read() == 0
    check(s, lens, got, lse)


@pytest.mark.parametrize("hq,hk,d,dtype", [
    (4, 2, 16, FP), (6, 3, 80, BF), (4, 1, 256, HF), (2, 2, 128, FP), (5, 5, 33, FP),
    (256, 1, 128, BF), (24, 2, 64, BF), (40, 8, 128, HF), (2, 1, 512, FP)])
@pytest.mark.parametrize("name", ["decode", "questions", "groups"])
def test_other_heads(cuda, hq, hk, d, dtype, name):
    s, lens = batch(cuda, hq, hk, d, dtype, *LAYOUTS[name])
    check(s, lens, *run(s, lens))


@pytest.mark.parametrize("block,scattered", [(16, 0.2), (16, 1.0), (5, 0.0), (32, 0.1), (64, 0.0),
                                             (1, 0.0), (128, 0.0)])
@pytest.mark.parametrize("name", ["drafts", "questions", "wide ragged"])
def test_block_sizes_and_relocated_slots(cuda, name, block, scattered):
    s, lens = batch(cuda, 32, 8, 128, BF, *LAYOUTS[name], block=block, scattered=scattered)
    check(s, lens, *run(s, lens))


@pytest.mark.parametrize("name", ["decode", "wide batch"])
def test_strides(cuda, name):
    s, lens = batch(cuda, 16, 4, 128, BF, *LAYOUTS[name])
    plan = plan_of(s, lens)
    want, lse = plan(s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"], return_lse=True)
    check(s, lens, want, lse)
    slots = s["prefix_slots"], s["suffix_slots"]
    # queries inside a projection's output, outputs inside a wider buffer
    tokens = s["query"].shape[0]
    wide = torch.zeros(tokens, 24 * 128 + 8, dtype=BF, device=cuda)
    q = wide[:, 8:8 + 16 * 128].unflatten(1, (16, 128)).copy_(s["query"])
    out = torch.zeros(tokens, 20, 136, dtype=BF, device=cuda)
    got = plan(q, s["cache"], *slots, out=out[:, 2:18, 4:132])
    assert got.data_ptr() == out[:, 2:18, 4:132].data_ptr()
    assert torch.equal(got, want)
    assert not out[:, :2].any() and not out[:, 18:].any() and not out[..., :4].any()
    # an odd start, one that no 16-byte load may use, and a strided head dim
    odd = torch.zeros(tokens, 16 * 128 + 1, dtype=BF, device=cuda)
    assert torch.equal(plan(odd[:, 1:].unflatten(1, (16, 128)).copy_(s["query"]), s["cache"],
                            *slots), want)
    assert torch.equal(plan(s["query"].transpose(1, 2).contiguous().transpose(1, 2), s["cache"],
                            *slots), want)
    # the pool in [block, offset, head] memory, inside a wider record, and dim-strided
    major = s["cache"].transpose(1, 2).contiguous().transpose(1, 2)
    check(s, lens, *plan(s["query"], major, *slots, return_lse=True))
    big = torch.zeros(*s["cache"].shape[:3], 264, dtype=BF, device=cuda)
    check(s, lens, *plan(s["query"], big[..., 8:].copy_(s["cache"]), *slots, return_lse=True))
    check(s, lens, *plan(s["query"], big[..., 1:257].copy_(s["cache"]), *slots, return_lse=True))
    two = torch.zeros(*s["cache"].shape[:3], 512, dtype=BF, device=cuda)
    check(s, lens, *plan(s["query"], two[..., ::2].copy_(s["cache"]), *slots, return_lse=True))


@pytest.mark.parametrize("name", ["decode", "wide batch"])
@pytest.mark.parametrize("scale", [1.0, 0.0, -0.1, 3.0])
def test_scale(cuda, name, scale):
    """1 and 3 make the softmax near one-hot, with scores of some hundreds."""
    s, lens = batch(cuda, 16, 4, 128, HF, *LAYOUTS[name])
    got, lse = run(s, lens, scale=scale)
    s64, lens64 = s, lens
    want, lse_w, size, score = oprefix.attention(
        s64["query"], s64["cache"], s64["prefix_slots"], s64["suffix_slots"], scale=scale, **lens64)
    score = oprefix.attention(s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"],
                              scale=abs(scale), **lens)[3]
    b_out, b_lse = bounds(HF, 128, lens, want, lse_w, size, score)
    assert ((got.double() - want).abs() <= b_out).all()
    assert ((lse.double() - lse_w).abs() <= b_lse).all()


@pytest.mark.parametrize("name", ["decode", "wide batch", "drafts"])
def test_growing_scores(cuda, name):
    """Scores that rise along the keys, each tile's maximum far above the last."""
    s, lens = batch(cuda, 16, 4, 128, BF, *LAYOUTS[name])
    s["query"][..., 0] = 8.0
    both = torch.cat((s["prefix_slots"], s["suffix_slots"]))
    ramp = torch.linspace(-30, 60, both.numel(), device=cuda).to(BF)
    s["cache"][both // 16, :, both % 16, 0] = ramp[:, None].expand(-1, 4)
    check(s, lens, *run(s, lens))
    s["cache"][both // 16, :, both % 16, 0] = -ramp[:, None].expand(-1, 4)
    check(s, lens, *run(s, lens))


@pytest.mark.parametrize("name", ["questions", "wide batch", "drafts"])
def test_values_no_row_may_see_yet(cuda, name):
    """An infinite or NaN key and value at a request's last own position: only
    its last query sees them."""
    s, lens = batch(cuda, 8, 2, 128, BF, *LAYOUTS[name])
    clean, lse = run(s, lens)
    check(s, lens, clean, lse)
    ends, t, k0 = [], 0, 0
    for n, m in zip(lens["query_lens"], lens["suffix_lens"]):
        if n and m:
            slot = int(s["suffix_slots"][k0 + m - 1])
            s["cache"][slot // 16, 0, slot % 16, 5] = float("nan")
            s["cache"][slot // 16, 0, slot % 16, 130] = float("inf")
            s["cache"][slot // 16, 1, slot % 16, 131] = float("nan")
            ends.append(t + n - 1)
        t, k0 = t + n, k0 + m
    got, lse_got = run(s, lens)
    last = torch.zeros(t, dtype=torch.bool, device=cuda)
    last[ends] = True
    tol = bounds(BF, 128, lens, *oprefix.attention(
        s["query"], s["cache"].nan_to_num(0, 0, 0), s["prefix_slots"], s["suffix_slots"], **lens))[0]
    assert ((got.double() - clean.double()).abs()[~last] <= 2 * tol[~last]).all()
    assert torch.isnan(got[last][:, :4]).all() and torch.isnan(lse_got[last][:, :4]).all()
    assert torch.isnan(got[last][:, 4:, 3]).all()
    assert torch.isfinite(got[last][:, 4:, 4:]).all()


@pytest.mark.parametrize("name", ["decode", "wide batch"])
def test_keys_of_minus_infinity(cuda, name):
    """Scores of -inf weigh nothing, first or later; +inf makes the row NaN."""
    s, lens = batch(cuda, 4, 1, 64, HF, *LAYOUTS[name])
    s["query"][..., 0] = 1.0
    first = s["prefix_slots"][:200]
    s["cache"][first // 16, 0, first % 16, 0] = -float("inf")
    got, lse = run(s, lens)
    short = {**s, "prefix_slots": s["prefix_slots"][200:].contiguous()}
    lens2 = {**lens, "prefix_lens": [lens["prefix_lens"][0] - 200]}
    check(short, lens2, got, lse)
    s["cache"][first // 16, 0, first % 16, 0] = float("inf")
    got, _ = run(s, lens)
    assert torch.isnan(got).all()


def test_slots_outside_the_pool(cuda):
    for layout in (LAYOUTS["decode"], LAYOUTS["wide batch"]):
        s, lens = batch(cuda, 8, 2, 128, BF, *layout)
        total = s["cache"].shape[0] * 16
        bad = {}
        for name, i, slot in (("prefix_slots", 7, -1), ("prefix_slots", 300, total),
                              ("suffix_slots", 3, 1 << 40)):
            bad.setdefault(name, s[name].clone())[i] = slot
        status = N.Status(cuda)
        got, lse = run({**s, **bad}, lens, status=status)
        assert status.read() == N.ST_SLOT_RANGE
        zeros = torch.cat((s["cache"], torch.zeros_like(s["cache"][:1])))
        want = {**s, "cache": zeros}
        for name, slots in bad.items():
            want[name] = slots.clone()
            want[name][(slots < 0) | (slots >= total)] = total  # a block of zeros
        check(want, lens, got, lse)


def test_arena_with_a_sidecar(cuda):
    cache = torch.zeros(40, 2, 16, 256, dtype=BF, device=cuda)
    arena = NativePagedKV(cache, list(range(20, 40)), 300, 64)
    rand = lambda n: torch.randn(n, 2, 128, device=cuda).to(BF)  # noqa: E731
    arena.write_prefill(rand(300), rand(300))
    moved = list(range(5, 250, 5))
    arena.promote_selected(moved, rand(len(moved)), rand(len(moved))).result()
    slots = arena.slot_table(range(300))
    assert int(slots.max()) >= 640
    lens = dict(query_lens=[1, 2], suffix_lens=[30, 20], prefix_lens=[250], group_sizes=None)
    s = dict(query=torch.randn(3, 8, 128, device=cuda).to(BF), cache=cache,
             prefix_slots=slots[:250].clone(), suffix_slots=slots[250:].clone())
    plan = plan_of(s, lens)
    got, lse = plan(s["query"], arena, s["prefix_slots"], s["suffix_slots"], return_lse=True)
    side = arena._side_key, arena._side_value
    check(s, lens, got, lse, side=side)
    wide = dict(query_lens=[100, 90], suffix_lens=[30, 20], prefix_lens=[250], group_sizes=None)
    s["query"] = torch.randn(190, 8, 128, device=cuda).to(BF)
    got, lse = plan_of(s, wide)(s["query"], arena, s["prefix_slots"], s["suffix_slots"],
                                return_lse=True)
    check(s, wide, got, lse, side=side)


@pytest.mark.parametrize("queries", [1, 120])
def test_past_32_bit_offsets(cuda, queries):
    """A pool of 4.6 GB whose last blocks are the ones read."""
    cache = torch.zeros(70_000, 8, 16, 256, dtype=BF, device=cuda)
    cache[69_000:].normal_()
    cache[0].normal_()
    g = torch.Generator(device=cuda).manual_seed(1)
    slots = torch.randperm(16_000, generator=g, device=cuda)[:900] + 69_000 * 16
    s = dict(query=torch.randn(2 * queries, 8, 128, device=cuda).to(BF), cache=cache,
             prefix_slots=torch.cat((torch.arange(16, device=cuda), slots[:500])),
             suffix_slots=slots[500:].contiguous())
    lens = dict(query_lens=[queries] * 2, suffix_lens=[200, 200], prefix_lens=[516],
                group_sizes=None)
    got, lse = run(s, lens)
    local = {**s, "cache": torch.cat((cache[:1], cache[69_000:]))}
    for name in ("prefix_slots", "suffix_slots"):
        local[name] = torch.where(s[name] >= 16, s[name] - 69_000 * 16 + 16, s[name])
    check(local, lens, got, lse)


@pytest.mark.parametrize("name", ["decode", "wide batch"])
def test_same_bits_again_and_on_another_stream(cuda, name):
    s, lens = batch(cuda, 32, 8, 128, BF, *LAYOUTS[name])
    plan = plan_of(s, lens)
    slots = s["prefix_slots"], s["suffix_slots"]
    want = plan(s["query"], s["cache"], *slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        query = s["query"] * 1
        got = plan(query, s["cache"], *slots)
        again = plan(query, s["cache"], *slots)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(again, want)


def test_plan_dropped_before_its_call_has_run(cuda):
    """The plan's memory is not handed out while a call on another stream
    than the plan's own still waits for its turn."""
    s, lens = batch(cuda, 8, 2, 128, BF, [40] * 5, [50] * 5, [300])
    plan = plan_of(s, lens)
    words, place = plan.words.numel(), plan.words.data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        plan(s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"])
    del plan
    assert torch.empty(words, dtype=torch.int32, device=cuda).data_ptr() != place
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()


def test_no_tokens(cuda):
    s, lens = batch(cuda, 8, 2, 128, BF, [0, 0], [5, 0], [20])
    got, lse = run(s, lens)
    assert got.shape == (0, 8, 128) and lse.shape == (0, 8)
    s, lens = batch(cuda, 8, 2, 128, BF, [], [], [20])
    assert run(s, lens)[0].shape == (0, 8, 128)


def test_refusals(cuda):
    s, lens = batch(cuda, 8, 2, 128, BF, [1, 2], [5, 6], [20])
    plan = plan_of(s, lens)
    good = dict(query=s["query"], kv=s["cache"], prefix_slots=s["prefix_slots"],
                suffix_slots=s["suffix_slots"])
    for change in (dict(query=s["query"][:2]), dict(query=s["query"].half()),
                   dict(query=s["query"].cpu()), dict(query=s["query"][:, :4]),
                   dict(prefix_slots=s["prefix_slots"][1:]),
                   dict(prefix_slots=s["prefix_slots"].int()),
                   dict(suffix_slots=s["suffix_slots"].cpu()),
                   dict(suffix_slots=torch.zeros(22, dtype=torch.int64, device=cuda)[::2]),
                   dict(kv=s["cache"].half()), dict(kv=s["cache"][:, :1]),
                   dict(kv=s["cache"][..., :128]), dict(kv=s["cache"].cpu()), dict(kv=None),
                   dict(scale=float("inf")), dict(out=s["query"][:2]),
                   dict(out=s["query"].float())):
        with pytest.raises(ValueError):
            plan(**{**good, **change})


def test_both_blocks_and_the_row_kernel_are_reached(cuda):
    """The plan picks 128-row blocks for decodes, 256-row blocks for prefills of
    questions and single rows where the tensor cores do not apply."""
    for name, variant in (("decode many", 1), ("wide batch", 2)):
        s, lens = batch(cuda, 32, 8, 128, BF, *LAYOUTS[name])
        assert plan_of(s, lens).info.variant == variant
    s, lens = batch(cuda, 4, 2, 80, BF, *LAYOUTS["decode"])
    assert plan_of(s, lens).info.variant == 0


@pytest.mark.parametrize("name,variant", [("decode many", 1), ("wide ragged", 2)])
def test_in_a_graph(cuda, name, variant):
    s, lens = batch(cuda, 32, 8, 128, BF, *LAYOUTS[name])
    plan = plan_of(s, lens)
    args = s["query"], s["cache"], s["prefix_slots"], s["suffix_slots"]
    want = plan(*args)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):  # each replayed launch beside the end of the one before
            plan(*args, out=out)
    s["query"].copy_(s["query"].roll(1, 0))
    graph.replay()
    assert torch.equal(out, plan(*args))
    assert not torch.equal(out, want)
