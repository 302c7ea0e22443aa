"""Rotary queries and keys over the paged pool.

A rotary model (or the rotary layers of a mixed one) serves from the same
paged pool as the contextual-position layers, with its keys rotated before
they are stored:

* ``rotary_tables``  -- float32 cosines and sines of every position;
* ``qk_norm_rope``   -- RMS norm of each query / key head and the rotation in
  one pass, differentiable in the queries, keys and both norm weights;
* ``append_rotated`` -- the serving form: the new tokens' keys (normed and
  rotated) and values go straight to their slots of the pool, and their
  queries come back normed and rotated, in one launch.

The reference has no rotary form (its layers count contextual positions,
position.py:295-307); slots, records and the sidecar are those of
``NativePagedKV`` (paged.py:205-240).  ``prefix.SharedPrefixAttention`` reads
what ``append_rotated`` writes.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _native as N
from .paged import NativePagedKV

MAX_HEAD_DIM = 512
_ROWS = torch.contiguous_format  # outputs are contiguous whatever the inputs' strides
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def rotary_tables(positions: int, rotary_dim: int, *, base: float = 10000.0,
                  device: torch.device | str = "cuda") -> tuple[Tensor, Tensor]:
    """cos and sin, float32 ``[positions, rotary_dim / 2]``, of the angles
    ``position * base^(-2 i / rotary_dim)`` (computed in float64)."""
    if type(positions) is not int or positions < 1:
        raise ValueError("positions must be a positive integer")
    if type(rotary_dim) is not int or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even integer")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] \
        * float(base) ** (-i / rotary_dim)
    return angle.cos().float(), angle.sin().float()


def _rows(name: str, x: Tensor) -> Tensor:
    if not isinstance(x, Tensor) or x.dim() != 3 or x.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32/float16/bfloat16 [token, head, dim]")
    return x if x.stride(2) == 1 else x.contiguous()


def _weight(w: Tensor, dim: int, device: int) -> int:
    if w.shape != (dim,) or w.dtype not in _TYPES or w.stride(0) != 1 and dim > 1:
        raise ValueError("norm weights must be contiguous floating [head dim]")
    if w.get_device() != device:
        raise ValueError("all tensors must be on the same CUDA device")
    return w.data_ptr()


def _params(query: Tensor | None, key: Tensor, positions: Tensor, cos: Tensor, sin: Tensor,
            q_weight: Tensor | None, k_weight: Tensor | None, eps: float, interleaved: bool,
            q_out: Tensor | None, k_out: Tensor | None,
            status: N.Status | None) -> N.RotaryParams:
    """The checks every entry point shares, and the C struct of the call."""
    tokens, k_heads, dim = key.shape
    dtype, device = key.dtype, key.get_device()
    if dim % 2 or not 2 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head dim must be even and at most {MAX_HEAD_DIM}")
    if (positions.shape != (tokens,) or positions.dtype is not torch.int64
            or tokens > 1 and positions.stride(0) != 1):
        raise ValueError("positions must be a contiguous int64 [token] vector")
    strides = cos.stride()
    if (len(strides) != 2 or cos.dtype is not torch.float32 or sin.dtype is not torch.float32
            or cos.shape != sin.shape or strides != sin.stride()
            or strides[1] != 1 and cos.shape[1] > 1):
        raise ValueError("cos and sin must be float32 [position, rotary_dim / 2]")
    rows, half = cos.shape
    if 2 * half > dim:
        raise ValueError("the rotated part is larger than the head")
    if not eps >= 0.0:
        raise ValueError("eps must be nonnegative")
    if (positions.get_device() != device or cos.get_device() != device
            or sin.get_device() != device):
        raise ValueError("all tensors must be on the same CUDA device")
    qw = kw = None
    weight_dtype = 0
    if q_weight is not None:
        qw = _weight(q_weight, dim, device)
        weight_dtype = N.DTYPES[q_weight.dtype]
    if k_weight is not None:
        kw = _weight(k_weight, dim, device)
        if q_weight is not None and k_weight.dtype is not q_weight.dtype:
            raise ValueError("norm weights must share a dtype")
        weight_dtype = N.DTYPES[k_weight.dtype]
    q = (None, 0, 0, 0)
    if query is not None:
        q_tokens, q_heads, q_dim = query.shape
        if q_tokens != tokens or q_dim != dim or query.dtype is not dtype:
            raise ValueError("query and key must share tokens, head dim and dtype")
        if query.get_device() != device:
            raise ValueError("all tensors must be on the same CUDA device")
        st = query.stride()
        q = (query.data_ptr(), st[0], st[1], q_heads)
    status_ptr = N.status_ptr(status, device)
    if device < 0:
        N.require_cuda(key)
    qo = ko = (None, 0, 0)
    if q_out is not None:
        st = q_out.stride()
        qo = (q_out.data_ptr(), st[0], st[1])
    if k_out is not None:
        st = k_out.stride()
        ko = (k_out.data_ptr(), st[0], st[1])
    st = key.stride()
    return N.RotaryParams(
        cos.data_ptr(), sin.data_ptr(), rows, strides[0], positions.data_ptr(), tokens, dim,
        2 * half, 1 if interleaved else 0, N.DTYPES[dtype], weight_dtype, eps, *q, qw, *qo,
        key.data_ptr(), st[0], st[1], k_heads, kw, *ko, status_ptr)


def _forward(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved, status):
    q_out = torch.empty_like(query, memory_format=_ROWS)
    k_out = torch.empty_like(key, memory_format=_ROWS)
    p = _params(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved, q_out,
                k_out, status)
    N.launch("cs_qk_norm_rope", key.device, p)
    return q_out, k_out


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved,
                status):
        ctx.save_for_backward(query, key, positions, cos, sin, q_weight, k_weight)
        ctx.how = eps, interleaved, status
        return _forward(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved,
                        status)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, q_dy, k_dy):
        query, key, positions, cos, sin, q_weight, k_weight = ctx.saved_tensors
        eps, interleaved, status = ctx.how
        q_dy, k_dy = q_dy.contiguous(), k_dy.contiguous()
        dq, dk = torch.empty_like(q_dy), torch.empty_like(k_dy)
        p = _params(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved, dq, dk,
                    status)
        dqw = None if q_weight is None else torch.empty_like(q_weight)
        dkw = None if k_weight is None else torch.empty_like(k_weight)
        workspace = torch.empty(N.load().cs_qk_norm_rope_grad_workspace(p), dtype=torch.uint8,
                                device=key.device)
        N.launch("cs_qk_norm_rope_grad", key.device, p, q_dy.data_ptr(), k_dy.data_ptr(),
                 N.ptr(dqw), N.ptr(dkw), workspace.data_ptr())
        return dq, dk, None, None, None, dqw, dkw, None, None, None


def qk_norm_rope(query: Tensor, key: Tensor, positions: Tensor, cos: Tensor, sin: Tensor,
                 q_weight: Tensor | None = None, k_weight: Tensor | None = None, *,
                 eps: float = 1e-6, interleaved: bool = False,
                 status: N.Status | None = None) -> tuple[Tensor, Tensor]:
    """RMS norm of each head (where its weight is given) and the position
    rotation of queries ``[token, q_head, dim]`` and keys ``[token, kv_head,
    dim]``, in float32 with one rounding to the input dtype.

    ``cos`` / ``sin`` come from ``rotary_tables``; twice their width is the
    rotated part of the head, the rest passes through.  ``interleaved`` pairs
    elements (2i, 2i + 1) instead of (i, i + rotary_dim / 2).  Gradients flow
    to query, key and the weights (cos and sin are constants); there is no
    forward-mode derivative, and a tensor that carries a tangent is refused.
    A position outside the tables makes the rotated elements of its rows NaN
    and sets ``ST_POS_RANGE`` in ``status`` (read it after the stream has
    drained)."""
    query, key = _rows("query", query), _rows("key", key)
    # (a level of dual numbers is rarely open, and this test of it is free)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None
            for t in (query, key, cos, sin, q_weight, k_weight)):
        raise ValueError("qk_norm_rope has no forward-mode derivative")
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (query, key, q_weight, k_weight)):
        return _NormRope.apply(query, key, positions, cos, sin, q_weight, k_weight, eps,
                               interleaved, status)
    return _forward(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved, status)


def pool_view(kv: Tensor | NativePagedKV | N.PagedKV) -> N.PagedKV:
    """The C-ABI view of a pool ``[blocks, kv_heads, block_size, 2 * dim]``, of
    an arena (with its sidecar), or a view made before."""
    if isinstance(kv, N.PagedKV):
        return kv
    if isinstance(kv, NativePagedKV):
        return kv.device_view()
    if not isinstance(kv, Tensor) or kv.device.type != "cuda":
        raise ValueError("kv must be a CUDA pool tensor or a NativePagedKV")
    return N.paged_view(kv)


def append_rotated(kv: Tensor | NativePagedKV | N.PagedKV, slots: Tensor, key: Tensor,
                   value: Tensor, positions: Tensor, cos: Tensor, sin: Tensor, *,
                   query: Tensor | None = None, q_weight: Tensor | None = None,
                   k_weight: Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                   out: Tensor | None = None, status: N.Status | None = None) -> Tensor | None:
    """Write new tokens to the paged pool: the record of ``slots[t]`` (int64)
    becomes the normed, rotated ``key[t]`` and ``value[t]``; with ``query``,
    its normed, rotated rows are returned (into ``out`` when given, which may
    be ``query`` itself and else overlaps no input).

    Norms, rotation and tables as in ``qk_norm_rope``.  Slot -1 marks padding
    and is not written; any other slot outside the pool (and sidecar), or a
    position outside the tables, is skipped and sets ``ST_SLOT_RANGE`` /
    ``ST_POS_RANGE`` in ``status`` (a query there has NaN in its rotated
    elements).  Distinct tokens need distinct slots: equal ones leave a mix of
    their rows.  The
    slot map's guards are the caller's: this writes where it is told, as a
    model runner's cache write does.  A serving operator: it has no derivative
    of either mode, and what it returns is a constant to autograd."""
    key, value = _rows("key", key), _rows("value", value)
    device = key.get_device()
    if value.shape != key.shape or value.dtype is not key.dtype or value.get_device() != device:
        raise ValueError("key and value must share shape, dtype and device")
    tokens = key.shape[0]
    if (slots.shape != (tokens,) or slots.dtype is not torch.int64
            or slots.get_device() != device or tokens > 1 and slots.stride(0) != 1):
        raise ValueError("slots must be a contiguous int64 [token] vector")
    view = pool_view(kv)
    N.require_pool_on(view, device)
    if query is not None:
        query = _rows("query", query)
        if out is None:
            out = torch.empty_like(query, memory_format=_ROWS)
        elif (out.shape != query.shape or out.dtype is not query.dtype
              or out.get_device() != device or out.stride(2) != 1):
            raise ValueError("out must match query, with a contiguous last dimension")
    elif out is not None or q_weight is not None:
        raise ValueError("out and q_weight need a query")
    p = _params(query, key, positions, cos, sin, q_weight, k_weight, eps, interleaved, out, None,
                status)
    if view.dtype != p.dtype or view.kv_heads != p.k_heads or view.head_dim != p.head_dim:
        raise ValueError("K/V must match the pool's dtype, KV heads and head dim")
    st = value.stride()
    N.launch("cs_kv_append_rotated", key.device, p, view, slots.data_ptr(), value.data_ptr(),
             st[0], st[1])
    return out
