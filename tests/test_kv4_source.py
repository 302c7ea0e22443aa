"""What the 4-bit kernels' sources have to hold and no run can show."""

from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "cacheslide_b200" / "csrc"


def test_a_warpgroup_sets_its_registers_at_one_instruction():
    """Warps of a warpgroup that change their registers at different instructions
    (or under conditions that differ among them) are undefined, and the warps
    that wait for those registers may wait for ever."""
    calls = re.findall(r"regs_(?:up|down)<(Sh::\w+)>\(\)", (CSRC / "kv4_sm100.cu").read_text())
    assert sorted(calls) == ["Sh::kMakeRegs", "Sh::kRestRegs", "Sh::kSoftRegs"]
