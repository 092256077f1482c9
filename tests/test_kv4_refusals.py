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


def _strided(shape, strides, offset=0, base=torch.zeros(1 << 14).bfloat16()):
    return base.as_strided(shape, strides, offset)


@pytest.mark.parametrize("strides", [(64, 128, 1), (128, 128, 1), (520, 64, 1), (128, 256, 1), (0, 128, 1)])
def test_query_rows_on_each_other(strides):
    pool, src, table = _args()
    with pytest.raises(RuntimeError, match="memory location|on each other"):
        kv4.append(src, pool, [table], 0, q_heads=4, q_out=_strided((3, 4, 128), strides))


@pytest.mark.parametrize("stride", [0, 64, 504])
def test_attention_rows_on_each_other(stride):
    pool, _, table = _args()
    with pytest.raises(RuntimeError, match="memory location|on each other"):
        kv4.attention(torch.zeros(2, 4, 128).bfloat16(), pool, [table, table], torch.zeros(2, dtype=torch.int32), 0.1,
                      out=_strided((2, 512), (stride, 1)))


@pytest.mark.parametrize("k,v", [((384, 0), (384, 0)), ((384, 0), (384, 384)), ((384, 128), (384, 0)), ((128, 0), (128, 4096)),
                                 ((1024, 1024), (1024, 0)), ((1024, 0), (1024, 376)), ((1024, 256), (1024, 1024))])
def test_read_rows_on_each_other(k, v):
    """(head pitch, first element) of k and v [2 heads, 3 rows, 128], in one buffer."""
    pool, _, table = _args()
    out = tuple(_strided((2, 3, 128), (pitch, 128, 1), at) for pitch, at in (k, v))
    with pytest.raises(RuntimeError, match="on each other"):
        kv4.read(pool, table, 3, 0, out=out)
    with pytest.raises(RuntimeError, match="on each other"):
        kv4.read(pool, table, 3, 0, out=(torch.zeros(2, 3, 128).bfloat16(),) * 2)


def test_interleaved_outputs_are_taken():
    """Views of one buffer that share no element."""
    pool, src, table = _args()
    for shape, strides in (((3, 4, 128), (128, 384, 1)), ((3, 4, 128), (1024, 128, 1)), ((3, 4, 128), (136, 416, 1))):
        with pytest.raises(RuntimeError, match="CUDA device"):
            kv4.append(src, pool, [table], 0, q_heads=4, q_out=_strided(shape, strides))
    for pitch, first, second in ((768, 0, 384), (768, 384, 0), (384, 0, 768), (1024, 0, 512)):
        out = tuple(_strided((2, 3, 128), (pitch, 128, 1), at) for at in (first, second))
        with pytest.raises(RuntimeError, match="CUDA device"):
            kv4.read(pool, table, 3, 0, out=out)
    one, two = pool[:1], torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):              # sequences inside heads
        kv4.read(one, [two, two], 3, torch.zeros(2, dtype=torch.int32),
                 out=tuple(_strided((2, 2, 3, 128), (384, 768, 128, 1), at) for at in (0, 1536)))
