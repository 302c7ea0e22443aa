"""The rotary operators without a GPU: the oracle's gradient against
differences, and the refusals of the Python and C entry points."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import rotary
from oracle import rotary as orot


def _tables(positions, rot):
    inv = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    angle = np.asarray(positions)[:, None] * inv
    return np.cos(angle), np.sin(angle)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(16, 16), (12, 6), (8, 0)])
@pytest.mark.parametrize("normed", [True, False])
def test_oracle_gradient_equals_differences(dim, rot, interleaved, normed):
    g = np.random.default_rng(5)
    x, dy = g.standard_normal((3, 2, dim)), g.standard_normal((3, 2, dim))
    w = 1 + 0.3 * g.standard_normal(dim) if normed else None
    cos, sin = _tables([0, 7, 1000], rot)
    dx, dw = orot.norm_rope_grad(x, w, dy, cos, sin, 1e-3, interleaved)
    loss = lambda x, w: (orot.norm_rope(x, w, cos, sin, 1e-3, interleaved) * dy).sum()  # noqa: E731
    h = 1e-6  # truncation h^2 ~ 1e-12, rounding 1e-16 * |loss| / h ~ 1e-9
    for index in np.ndindex(x.shape):
        e = np.zeros_like(x)
        e[index] = h
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - dx[index]) < 1e-7
    if normed:
        for i in range(dim):
            e = np.zeros(dim)
            e[i] = h
            assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - dw[i]) < 1e-7


def test_tables_are_the_angles_of_the_formula():
    cos, sin = rotary.rotary_tables(50, 12, base=500.0, device="cpu")
    angle = np.arange(50)[:, None] * 500.0 ** (-np.arange(0, 12, 2) / 12)
    # float64 angles rounded once to float32: half a unit of values at most 1
    np.testing.assert_allclose(cos.numpy(), np.cos(angle), atol=2.0**-25 + 1e-12, rtol=0)
    np.testing.assert_allclose(sin.numpy(), np.sin(angle), atol=2.0**-25 + 1e-12, rtol=0)
    for bad in ((0, 4), (4, 3), (4, 0), (2.0, 4)):
        with pytest.raises(ValueError):
            rotary.rotary_tables(*bad, device="cpu")


def _good():
    t = torch.zeros
    return dict(query=t(3, 4, 8), key=t(3, 2, 8), positions=t(3, dtype=torch.int64),
                cos=t(5, 4), sin=t(5, 4), q_weight=t(8), k_weight=t(8))


@pytest.mark.parametrize("change", [
    dict(query=torch.zeros(2, 4, 8)),
    dict(query=torch.zeros(3, 4, 6)),
    dict(query=torch.zeros(3, 4, 8, dtype=torch.float16)),
    dict(key=torch.zeros(3, 8)),
    dict(key=torch.zeros(3, 2, 8, dtype=torch.float64)),
    dict(key=torch.zeros(3, 2, 7), query=torch.zeros(3, 4, 7)),
    dict(key=torch.zeros(3, 2, 514), query=torch.zeros(3, 4, 514)),
    dict(positions=torch.zeros(3, dtype=torch.int32)),
    dict(positions=torch.zeros(4, dtype=torch.int64)),
    dict(positions=torch.zeros(6, dtype=torch.int64)[::2]),
    dict(cos=torch.zeros(5, 4, dtype=torch.float64)),
    dict(cos=torch.zeros(5, 3)),
    dict(cos=torch.zeros(5, 6), sin=torch.zeros(5, 6)),
    dict(q_weight=torch.zeros(4)),
    dict(q_weight=torch.zeros(8, dtype=torch.float16)),
    dict(q_weight=torch.zeros(16)[::2]),
    dict(eps=-1.0),
    dict(eps=float("nan")),
    dict(),  # right but for the device
])
def test_norm_rope_refuses(change):
    with pytest.raises(ValueError):
        rotary.qk_norm_rope(**{**_good(), **change})


def test_append_refuses_cpu_pools_and_other_objects():
    g = _good()
    args = (torch.zeros(3, dtype=torch.int64), g["key"], g["key"], g["positions"], g["cos"],
            g["sin"])
    with pytest.raises(ValueError):
        rotary.append_rotated(torch.zeros(2, 2, 4, 16), *args)
    with pytest.raises(ValueError):
        rotary.append_rotated(None, *args)


def _c_params(**kw):
    p = N.RotaryParams(cos=16, sin=16, table_rows=4, table_stride=4, positions=16, tokens=2,
                       head_dim=8, rot=8, dtype=N.CS_F32, eps=1e-6, q=16, q_heads=1, q_out=16,
                       k=16, k_heads=1, k_out=16)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("change,want", [
    (dict(head_dim=7), N.CS_ERR_INVALID), (dict(head_dim=0), N.CS_ERR_INVALID),
    (dict(rot=10), N.CS_ERR_INVALID), (dict(rot=3), N.CS_ERR_INVALID),
    (dict(tokens=-1), N.CS_ERR_INVALID), (dict(eps=-1.0), N.CS_ERR_INVALID),
    (dict(positions=None), N.CS_ERR_INVALID), (dict(cos=None), N.CS_ERR_INVALID),
    (dict(q=None), N.CS_ERR_INVALID), (dict(k_out=None), N.CS_ERR_INVALID),
    (dict(q_weight=16, weight_dtype=N.CS_F64), N.CS_ERR_INVALID),
    (dict(head_dim=1024, rot=8), N.CS_ERR_UNSUPPORTED),
    (dict(dtype=N.CS_F64), N.CS_ERR_UNSUPPORTED),
])
def test_c_entry_refuses(change, want):
    lib = N.load()
    assert lib.cs_qk_norm_rope(ctypes.byref(_c_params(**change)), None) == want
    assert lib.cs_qk_norm_rope_grad(ctypes.byref(_c_params(**change)), 16, 16, 16, 16, 16,
                                    None) == want


def test_c_append_refuses():
    lib = N.load()
    kv = N.PagedKV(cache=16, num_blocks=1, kv_heads=2, block_size=16, head_dim=8,
                   dtype=N.CS_F32)
    ok = _c_params()
    assert lib.cs_kv_append_rotated(ctypes.byref(ok), ctypes.byref(kv), 16, 16, 8, 8,
                                    None) == N.CS_ERR_INVALID  # other KV heads
    kv.kv_heads = 1
    assert lib.cs_kv_append_rotated(ctypes.byref(ok), ctypes.byref(kv), None, 16, 8, 8,
                                    None) == N.CS_ERR_INVALID
    kv.dtype = N.CS_BF16
    assert lib.cs_kv_append_rotated(ctypes.byref(ok), ctypes.byref(kv), 16, 16, 8, 8,
                                    None) == N.CS_ERR_INVALID
    assert lib.cs_kv_append_rotated(ctypes.byref(ok), None, 16, 16, 8, 8,
                                    None) == N.CS_ERR_INVALID
    empty = _c_params(tokens=0)
    kv.dtype = N.CS_F32
    assert lib.cs_kv_append_rotated(ctypes.byref(empty), ctypes.byref(kv), None, None, 8, 8,
                                    None) == N.CS_OK
