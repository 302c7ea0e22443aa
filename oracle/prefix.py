"""Attention behind shared prefixes in float64, request by request."""

from __future__ import annotations

import math

import torch


def attention(query, cache, prefix_slots, suffix_slots, *, query_lens, suffix_lens, prefix_lens,
              group_sizes=None, scale=None, side=None):
    """Returns (o, lse, size, score): the outputs [token, head, dim] and lse
    [token, head]; size = sum_j p_j |v_j| / sum_j p_j, what a relative error of
    the p_j scales with; score = max_j scale * sum_d |q_d k_jd|, what an error
    of the scores scales with.  ``side`` is the (K, V) sidecar of slots past
    the pool."""
    bs, d, hk = cache.shape[2], cache.shape[3] // 2, cache.shape[1]
    hq = query.shape[1]
    scale = d ** -0.5 if scale is None else scale
    records = cache.transpose(1, 2).reshape(-1, hk, 2 * d)
    if side is not None:
        records = torch.cat((records, torch.cat(side, -1)))
    sizes = [len(query_lens)] if group_sizes is None else group_sizes
    outs, t, k0, p0, b = [], 0, 0, 0, 0
    for length, members in zip(prefix_lens, sizes):
        for _ in range(members):
            n, m = query_lens[b], suffix_lens[b]
            kv = records[torch.cat((prefix_slots[p0:p0 + length], suffix_slots[k0:k0 + m]))]
            kv = kv.double().repeat_interleave(hq // hk, 1)  # [keys, hq, 2d]
            q = query[t:t + n].double()
            k, v = kv[..., :d], kv[..., d:]
            z = torch.einsum("nhd,khd->nhk", q, k) * scale
            # the whole prefix, and own keys up to the query's own position
            limit = length + (m - n + torch.arange(n, device=q.device)).clamp_min(-1)
            hidden = (torch.arange(length + m, device=q.device) > limit[:, None])[:, None]
            z = z.masked_fill(hidden, -math.inf)
            size = torch.einsum("nhd,khd->nhk", q.abs(), k.abs()) * scale
            size = size.masked_fill(hidden, 0.0)
            if length + m == 0:
                zero = q.new_zeros(n, hq)
                outs.append((q.new_zeros(n, hq, d), zero - math.inf, q.new_zeros(n, hq, d), zero))
            else:
                lse = torch.logsumexp(z, -1)
                p = torch.exp(z - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
                # a masked key adds nothing, whatever its value holds
                seen = (~hidden).expand_as(p)
                vp = torch.einsum("nhk,khd->nhd", p, v.nan_to_num(0, 0, 0)) if v.isfinite().all() \
                    else torch.stack([torch.stack([
                        (p[i, h, seen[i, h], None] * v[seen[i, h], h]).sum(0)
                        for h in range(hq)]) for i in range(n)]) if n else q.new_zeros(n, hq, d)
                outs.append((vp, lse, torch.einsum("nhk,khd->nhd", p, v.nan_to_num(0, 0, 0).abs()),
                             size.amax(-1) if n else q.new_zeros(n, hq)))
            t, k0, b = t + n, k0 + m, b + 1
        p0 += length
    return tuple(torch.cat(x) for x in zip(*outs))
