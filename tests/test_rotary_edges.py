"""Rotary entry points without a GPU: what they refuse before any launch."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from cacheslide_b200 import rotary


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
