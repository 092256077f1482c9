"""Calls of the 4-bit cache's entry points that are refused before a kernel starts; every check but the last, for a CUDA
device, holds on any device."""
import pytest
import torch

from ridgefill_data_b200.ops import kv4

from test_kv4 import _args


@pytest.mark.parametrize("T", [3, 300])
@pytest.mark.parametrize("where", ["row0 on the device", "pos", "row0 on the host"])
def test_rope_tables_without_positions(T, where):
    """No position can be valid, and the kernels look entries up beside the rows whose position is not."""
    pool, src, table = _args(pages=20, T=T)
    table = torch.arange(20, dtype=torch.int32)
    none = torch.empty(0, 32).bfloat16()
    kw = dict(row0=0, q_heads=4, rot=64, tables=(none, none))
    if where == "row0 on the device":
        kw["row0"] = torch.zeros(1, dtype=torch.int32)
    elif where == "pos":
        kw["pos"] = torch.arange(T, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="RoPE tables|positions past"):
        kv4.append(src, pool, [table], **kw)
