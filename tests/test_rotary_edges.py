"""Rotary entry points without a GPU: what they refuse before any launch."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from cacheslide_b200 import _native as N
from cacheslide_b200 import rotary
from cacheslide_b200.prefix import SharedPrefixAttention


def _good():
    t = torch.zeros
    return dict(query=t(3, 4, 8), key=t(3, 2, 8), positions=t(3, dtype=torch.int64),
                cos=t(5, 4), sin=t(5, 4), q_weight=t(8), k_weight=t(8))


@pytest.mark.parametrize("name", ["query", "key", "q_weight", "k_weight", "cos", "sin"])
@pytest.mark.parametrize("grad", [True, False])
def test_norm_rope_refuses_forward_derivatives(name, grad):
    """A tangent would be lost in the launch: it raises, also without autograd."""
    good = _good()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(good[name], torch.ones_like(good[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            rotary.qk_norm_rope(**{**good, name: dual})
        # an ordinary call inside the level gets as far as the device check
        with pytest.raises(ValueError, match="CUDA"):
            rotary.qk_norm_rope(**good)


def _append_args():
    g = _good()
    return dict(slots=torch.zeros(3, dtype=torch.int64), key=g["key"], value=g["key"],
                positions=g["positions"], cos=g["cos"], sin=g["sin"])


def _view(device, **kw):
    """A pool's view as paged_view makes it, on a device that is only named."""
    kv = N.PagedKV(cache=16, num_blocks=1, kv_heads=2, block_size=16, head_dim=8,
                   dtype=N.CS_F32, **kw)
    kv.device = device
    return kv


def test_views_know_their_device():
    assert N.paged_view(torch.zeros(2, 2, 4, 16)).device == -1
    assert N.PagedKV().device is None  # a view made by hand: not known


def test_append_refuses_a_pool_on_another_device():
    with pytest.raises(ValueError, match="same CUDA device"):
        rotary.append_rotated(_view(1), **_append_args())
    for same in (_view(-1), _view(None)):  # as far as the device check of the tensors
        with pytest.raises(ValueError, match="CUDA tensors only"):
            rotary.append_rotated(same, **_append_args())


class _OnDevice:
    """What the checks read of a tensor, on a device that is only named."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self._device = torch.Size(shape), dtype, device
        self._strides = torch.empty(shape, dtype=dtype).stride()

    def get_device(self):
        return self._device

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def data_ptr(self):
        raise AssertionError("the call got past its checks")


class _Status:
    def __init__(self, device):
        self.word = _OnDevice((1,), torch.int32, device)
        self.ptr = 16


def _attention():
    plan = SharedPrefixAttention(4, 2, 8, torch.float32, "cpu", query_lens=[1, 2],
                                 suffix_lens=[1, 2], prefix_lens=[4])
    plan.device = torch.device("cuda", 0)
    on = lambda shape, dtype=torch.float32: _OnDevice(shape, dtype, 0)  # noqa: E731
    args = dict(query=on((3, 4, 8)), kv=_view(0), prefix_slots=on((4,), torch.int64),
                suffix_slots=on((3,), torch.int64), out=on((3, 4, 8)))
    return plan, args


def test_attention_refuses_a_pool_or_status_on_another_device():
    plan, args = _attention()
    with pytest.raises(AssertionError, match="past its checks"):
        plan(**args, status=_Status(0))
    with pytest.raises(ValueError, match="device"):
        plan(**{**args, "kv": _view(1)})
    with pytest.raises(ValueError, match="device"):
        plan(**args, status=_Status(1))


def test_norm_rope_and_append_refuse_a_status_on_another_device():
    with pytest.raises(ValueError, match="same CUDA device"):
        rotary.qk_norm_rope(**_good(), status=_Status(1))
    with pytest.raises(ValueError, match="same CUDA device"):
        rotary.append_rotated(_view(-1), **_append_args(), status=_Status(1))
