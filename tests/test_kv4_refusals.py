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


@pytest.mark.parametrize("hq,gate_head", [(5, 2 ** 62), (3, 2 ** 63 - 8), (2, 2 ** 63 - 8), (5, 2 ** 61), (2, 520)])
def test_gate_columns_past_the_row(hq, gate_head):
    """The last head's gate would lie outside the row; (hq - 1) gate_head may pass 64 bits."""
    pool, _, table = _args(hkv=1, hq=hq)
    with pytest.raises(RuntimeError, match="gate rows"):
        kv4.attention(torch.zeros(1, hq, 128).bfloat16(), pool, [table], torch.zeros(1, dtype=torch.int32), 0.1,
                      gate=torch.zeros(1, 512).bfloat16(), gate_head=gate_head)


@pytest.mark.parametrize("hq", [2 ** 63 - 1, 2 ** 62, 65536, -1])
def test_query_heads_at_their_ends(hq):
    pool, src, table = _args(T=0)
    with pytest.raises(RuntimeError, match="up to 65535 heads"):
        kv4.append(src, pool, [table], 0, q_heads=hq)


def test_one_heads_gate_has_no_pitch():
    """With one query head nothing is taken gate_head columns further."""
    pool, _, table = _args(hkv=1, hq=1)
    with pytest.raises(RuntimeError, match="CUDA device"):
        kv4.attention(torch.zeros(1, 1, 128).bfloat16(), pool, [table], torch.zeros(1, dtype=torch.int32), 0.1,
                      gate=torch.zeros(1, 128).bfloat16(), gate_head=256)
