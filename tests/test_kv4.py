"""The 4-bit pool and the slot maps without a GPU: structures, checks of
arguments, and the restatement's own properties."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cacheslide_b200 import _native as N
from cacheslide_b200 import kv4, tables
from oracle import kv4 as okv4

INCLUDE = Path(__file__).resolve().parents[1] / "include"
PAIRS = {"cs_step_maps_params": N.StepMapsParams, "cs_kv4_pool": N.KV4Pool,
         "cs_kv4_attn_params": N.KV4AttnParams}


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
    subprocess.run([cc, f"-I{INCLUDE}", str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in
               subprocess.run([str(exe)], check=True, capture_output=True,
                              text=True).stdout.splitlines())
    assert int(got.pop("size")) == ctypes.sizeof(PAIRS[name])
    for f in fields:
        assert int(got[f]) == getattr(PAIRS[name], f).offset, f


def _pool(dim=128, group=64, dtype=torch.bfloat16):
    return kv4.empty_pool(3, 2, 32, dim, dtype, "cpu", group)


def test_cpu_tensors_are_refused():
    pool = _pool()
    slots = torch.arange(4)
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    table, lengths = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kv4.append(pool, slots, k, k)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kv4.gather(pool, slots)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kv4.attention(torch.zeros(4, 4, 128, dtype=torch.bfloat16), pool, table, lengths)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        tables.step_maps(lengths, lengths, table, 16, 3, tokens=4)


@pytest.mark.parametrize("shape,dim,dtype,group", [
    ((3, 2, 2, 2304), 128, torch.float32, 64), ((3, 2, 2, 2304), 96, torch.float16, 32),
    ((3, 2, 2, 2304), 128, torch.float16, 16), ((3, 2, 2, 2304), 64, torch.float16, 128),
    ((3, 2, 2, 2303), 128, torch.float16, 64), ((3, 2, 2304), 128, torch.float16, 64),
    ((3, 0, 2, 2304), 128, torch.float16, 64)])
def test_pools_that_are_none(shape, dim, dtype, group):
    with pytest.raises(ValueError):
        kv4.PagedKV4(torch.zeros(shape, dtype=torch.uint8), dim, dtype, group)


def test_more_pools_that_are_none():
    x = torch.zeros(4, 2, 2, 2304, dtype=torch.uint8)
    kv4.PagedKV4(x, 128, torch.float16, 64)
    for bad in (x[::2], x.to(torch.int8), x.transpose(1, 2), None):
        with pytest.raises(ValueError):
            kv4.PagedKV4(bad, 128, torch.float16, 64)
    odd = torch.zeros(4 * 2304 + 1, dtype=torch.uint8)
    shift = 1 if odd.data_ptr() % 16 == 0 else 0
    with pytest.raises(ValueError, match="aligned"):
        kv4.PagedKV4(odd[shift:shift + 4 * 2304].view(4, 1, 1, 2304), 128, torch.float16, 64)
    for block in (0, 8, 24, 16.0):
        with pytest.raises(ValueError):
            kv4.empty_pool(3, 2, block, 128, torch.float16, "cpu")


def test_arguments_are_checked():
    pool = _pool()
    slots, k = torch.arange(4), torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    for bad in (dict(slots=slots.int()), dict(slots=slots.view(2, 2)), dict(key=k[:3]),
                dict(key=k.half()), dict(value=k[..., :64]), dict(pool=pool.storage),
                dict(slots=torch.arange(8)[::2])):
        with pytest.raises(ValueError) as e:
            kv4.append(**(dict(pool=pool, slots=slots, key=k, value=k) | bad))
        assert "CUDA tensors only" not in str(e.value)
    table, lengths = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    for bad in (dict(query=q[:, :3]), dict(query=q.half()), dict(query=q[0]),
                dict(tables=table.long()), dict(tables=table.t()), dict(tables=table[:1].expand(4, 2)),
                dict(lengths=lengths.long()), dict(lengths=lengths[:3]), dict(query=q[:3]),
                dict(starts=lengths), dict(scale=float("nan")), dict(scale=1e300),
                dict(out=q[:3]), dict(out=torch.zeros(4, 4, 256, dtype=q.dtype)[..., ::2])):
        with pytest.raises(ValueError) as e:
            kv4.attention(**(dict(query=q, pool=pool, tables=table, lengths=lengths) | bad))
        assert "CUDA tensors only" not in str(e.value)
    for bad in (dict(lengths=lengths[:3]), dict(new=lengths.long()), dict(tables=table.long()),
                dict(tables=table.t()), dict(block_size=0), dict(block_size=16.0),
                dict(num_blocks=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(keys=-1),
                dict(offset=-1), dict(free=lengths), dict(free_count=lengths[:1]),
                dict(free=lengths, free_count=lengths), dict(tables=table[:1].expand(4, 2))):
        with pytest.raises(ValueError) as e:
            tables.step_maps(**(dict(lengths=lengths, new=lengths, tables=table, block_size=16,
                                     num_blocks=3, tokens=4) | bad))
        assert "CUDA tensors only" not in str(e.value)


def test_entry_points_refuse_what_no_kernel_takes():
    lib = N.load()
    pool = N.KV4Pool(None, 0, 2, 16, 128, 64, N.CS_BF16)
    p = N.KV4AttnParams()
    p.pool, p.q_heads, p.scale = pool, 4, 1.0
    assert lib.cs_kv4_attn(p, None, None) == N.CS_OK  # no rows: nothing to do
    for change in (dict(q_heads=3), dict(q_heads=0), dict(tokens=-1), dict(requests=-1),
                   dict(tokens=1), dict(scale=float("inf")), dict(table_width=-1)):
        bad = N.KV4AttnParams.from_buffer_copy(p)
        for name, value in change.items():
            setattr(bad, name, value)
        assert lib.cs_kv4_attn(bad, None, None) == N.CS_ERR_INVALID, change
        assert lib.cs_kv4_attn_workspace(bad) == 0
    for name, value, rc in (("head_dim", 96, 3), ("group", 16, 3), ("block_size", 24, 3),
                            ("dtype", N.CS_F32, 3), ("kv_heads", 0, 1), ("num_blocks", -1, 1)):
        bad = N.KV4Pool.from_buffer_copy(pool)
        setattr(bad, name, value)
        for call in (lib.cs_kv4_append, lib.cs_kv4_gather):
            assert call(bad, None, 1, None, 0, 0, None, 0, 0, None, None) == rc, name
    assert lib.cs_kv4_append(pool, None, 1, None, 0, 0, None, 0, 0, None, None) == N.CS_ERR_INVALID
    assert lib.cs_kv4_append(pool, None, 0, None, 0, 0, None, 0, 0, None, None) == N.CS_OK
    m = N.StepMapsParams()
    assert lib.cs_step_maps(m, None) == N.CS_ERR_INVALID  # no block size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group", [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)])
def test_records_round_trip(dtype, dim, group):
    """Every element comes back within half a step (and the scale's rounding)."""
    g = torch.Generator().manual_seed(dim + group)
    k, v = (torch.randn(40, 3, dim, generator=g).to(dtype) for _ in "kv")
    storage = torch.zeros(4, 3, 1, kv4.unit_bytes(dim, group), dtype=torch.uint8)
    slots = torch.randperm(64, generator=g)[:40]
    okv4.write(storage, slots, k, v, group)
    rk, ks, rv, vs = okv4.read(storage, slots, dim, group, dtype)
    for x, y, s in ((k, rk, ks), (v, rv, vs)):
        # 15 steps of a scale rounded by half an ulp reach that much short
        assert ((x.double() - y).abs() <= s * (0.5 + 15 * torch.finfo(dtype).eps / 2)).all()
    for at in okv4.order(dim):
        assert sorted(at.tolist()) == list(range(dim))
