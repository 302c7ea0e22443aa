"""The ctypes structures of the rotary and shared-prefix entries have the C
compiler's sizes and field offsets."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from cacheslide_b200 import _native as N

INCLUDE = Path(__file__).resolve().parents[1] / "include"
PAIRS = {"cs_rotary_params": N.RotaryParams, "cs_prefix_shape": N.PrefixShape,
         "cs_prefix_plan_info": N.PrefixPlanInfo, "cs_prefix_params": N.PrefixParams}


@pytest.mark.parametrize("name", PAIRS)
def test_structure_matches_the_c_compiler(name, tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [f[0] for f in PAIRS[name]._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "cacheslide_b200.h"\n'
                   "int main(void) {\n"
                   f'  printf("size %zu\\n", sizeof({name}));\n'
                   + "".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    cuda = "/usr/local/cuda/include"
    subprocess.run([cc, f"-I{INCLUDE}", f"-I{cuda}", str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in
               subprocess.run([str(exe)], check=True, capture_output=True,
                              text=True).stdout.splitlines())
    assert int(got.pop("size")) == ctypes.sizeof(PAIRS[name])
    for f in fields:
        assert int(got[f]) == getattr(PAIRS[name], f).offset, f
